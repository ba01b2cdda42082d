// The tiled attention kernels (paged_attn_mfma.h) of one type of heads, cache and form of scores.
#include "paged_attn_mfma.h"

int intent::launch_attn_bf16_fp8_sloped(const AttnArgs& a, int items, int rows, const AttnArgs* few, int few_items,
                             hipStream_t stream) {
  return attn::launch_any<true, kCacheFp8, kSloped>(a, items, rows, few, few_items, stream);
}
