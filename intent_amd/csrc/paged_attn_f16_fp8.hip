// The tiled attention kernels (paged_attn_mfma.h) of one type of heads and cache.
#include "paged_attn_mfma.h"

int intent::launch_attn_f16_fp8(const AttnArgs& a, int items, int rows, hipStream_t stream) {
  return attn::launch_any<false, true>(a, items, rows, stream);
}
