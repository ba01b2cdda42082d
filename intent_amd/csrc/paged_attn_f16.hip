// The tiled attention kernels (paged_attn_mfma.h) of one type of heads and cache.
#include "paged_attn_mfma.h"

int intent::launch_attn_f16(const AttnArgs& a, int items, int rows, hipStream_t stream) {
  return attn::launch_any<false, false>(a, items, rows, stream);
}

int intent::launch_join_f16(const AttnJoin& j, int side, hipStream_t stream) {
  return attn::launch_join<false>(j, side, stream);
}
