// Attention of new tokens over a paged cache: what its kernels share.
//
// Sequence s owns the query rows q_offsets[s] .. q_offsets[s+1] and the first kv_lens[s] tokens of
// its pages (the new tokens among them, appended before the call). Its row i of n stands at position
// p = kv_len - n + i and sees the tokens t with
//   t < kv_len,   t <= p (causal),   t > p - window (window > 0).
//   out = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q.k_t - max),   0 where nothing is seen.
// Offsets, lengths and page ids come from device memory: they are clamped to the tensors' extents,
// so a wrong one gives a wrong row and no access outside them.
#pragma once

#include "common.h"
#include "internal.h"

namespace intent {

struct AttnArgs {
  const uint16_t* q;
  int64_t q_ld;
  const void *k_cache, *v_cache;
  int64_t k_page, v_page;  // elements from a page to the next
  const float *k_scales, *v_scales;
  int64_t ks_page, vs_page;
  const int32_t* page_table;
  int64_t table_ld;
  const int32_t *q_offsets, *kv_lens;
  uint16_t* out;
  int64_t out_ld;
  float scale_log2;  // scale * log2(e): the kernels work with exp2
  int T, S, HQ, HK, group, D, pages, page_shift, most_kv, causal, window;
};

// Query rows [start, start + count) and cached tokens of sequence s.
struct Sequence {
  int start, count, kv;
};

INTENT_DEVICE Sequence sequence_of(const AttnArgs& a, int s) {
  Sequence r;
  r.start = min(max(a.q_offsets[s], 0), a.T);
  r.count = max(min(a.q_offsets[s + 1], a.T) - r.start, 0);
  r.kv = min(max(a.kv_lens[s], 0), a.most_kv);
  return r;
}

// First and one past the last token that the row at position p sees.
INTENT_DEVICE int first_seen(const AttnArgs& a, int p) { return a.window > 0 && p >= a.window ? p - a.window + 1 : 0; }
INTENT_DEVICE int end_seen(const AttnArgs& a, int p, int kv) { return a.causal ? min(max(p + 1, 0), kv) : kv; }

// Page of token t (t < most_kv) of sequence s.
INTENT_DEVICE int page_of(const AttnArgs& a, int s, int t) {
  return (int)min((uint32_t)a.page_table[(int64_t)s * a.table_ld + (t >> a.page_shift)], (uint32_t)a.pages - 1u);
}

// Row of token t of a page and head in a cache with `row` elements for each token.
INTENT_DEVICE int64_t row_in_cache(const AttnArgs& a, int page, int64_t page_ld, int head, int t, int row) {
  return (int64_t)page * page_ld + (((int64_t)head << a.page_shift) + (t & ((1 << a.page_shift) - 1))) * row;
}

}  // namespace intent
