// The tiled attention kernels (paged_attn_mfma.h) of one type of heads, cache and form of scores.
#include "paged_attn_mfma.h"

int intent::launch_attn_bf16_capped(const AttnArgs& a, int items, int rows, const AttnArgs* few, int few_items,
                             hipStream_t stream) {
  return attn::launch_any<true, kCacheSame, kCapped>(a, items, rows, few, few_items, stream);
}

int intent::launch_join_bf16_prefix(const AttnJoin& j, int side, hipStream_t stream) {
  return attn::launch_join<true, true>(j, side, stream);
}
