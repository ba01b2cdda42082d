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
  // the page strides again for the tiled kernels: in 16 bytes, and in scales
  uint32_t k_step, v_step, ks_step, vs_step;
  // work list of the tiled kernels (find_span)
  int min_rows, max_rows;  // sequences with more rows (new tokens times group) than min, up to max
  int target;              // workgroups for each cached head that tiles are split for; 0: none
  float* partial;          // [slot][HK][tile rows][D] unnormalised sums, then [slot][HK][tile rows][2]
  float* partial_stats;
};

// A launch of the tiled kernels: the arguments, workgroups for each cached head, of the kernel and of
// the join of its splits (0: none).
struct AttnLaunch {
  AttnArgs a;
  int items, joins, join_rows;
};

// The tiled kernels for one type and cache (paged_attn_*.hip): 16 * tiles rows over one workgroup's
// four waves, which split the tokens ("rows" kernel, tiles 1, 2 or 4), or 128 rows, 32 to a wave.
int launch_attn_f16(const AttnLaunch& l, int tiles, hipStream_t stream);
int launch_attn_bf16(const AttnLaunch& l, int tiles, hipStream_t stream);
int launch_attn_f16_fp8(const AttnLaunch& l, int tiles, hipStream_t stream);
int launch_attn_bf16_fp8(const AttnLaunch& l, int tiles, hipStream_t stream);

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

constexpr int kMostSplits = 256;

// A workgroup's share: rows row0 .. row0 + rows of a sequence (row = new token * group + head of the
// group) and the tokens begin .. end.
struct Span {
  int s, row0, rows, begin, end, splits, slot;
  Sequence q;
};

// Rows, row tiles and units of tokens of sequence s.
struct Extent {
  Sequence q;
  int tiles, units;
};

template <int ROWS, int UNIT>
INTENT_DEVICE Extent extent_of(const AttnArgs& a, int s) {
  Extent e{};
  if (s >= a.S) return e;
  e.q = sequence_of(a, s);
  const int64_t rows = (int64_t)e.q.count * a.group;
  if (rows <= a.min_rows || rows > a.max_rows) return e;
  e.tiles = (int)((rows + ROWS - 1) / ROWS);
  const int lo = first_seen(a, e.q.kv - e.q.count) & ~63;
  e.units = (e.q.kv - lo + UNIT - 1) / UNIT;
  return e;
}

INTENT_DEVICE int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Finds share `item` of one head's list: the sequences in order, each with its row tiles from the last
// (which sees most) to the first, each tile in `splits` parts of its tokens. The parts are sized so
// that all sequences together give about a.target of them: units / chunk of each, chunk = the units
// that a workgroup would get of an even share. With `joins`, the list of the tiles that are split.
// Every wave does it by itself: no plan is kept, so a captured call follows lengths that change.
template <int ROWS, int UNIT>
INTENT_DEVICE bool find_span(const AttnArgs& a, int item, bool joins, Span& r) {
  const int lane = threadIdx.x & 63;
  const Extent first = extent_of<ROWS, UNIT>(a, lane);
  int64_t chunk = INT32_MAX;
  if (a.target > 0) {
    int64_t all = (int64_t)first.tiles * first.units;
    for (int s0 = 64; s0 < a.S; s0 += 64) {
      const Extent e = extent_of<ROWS, UNIT>(a, s0 + lane);
      all += (int64_t)e.tiles * e.units;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off);
    chunk = (all + a.target - 1) / a.target;
    if (chunk < 1) chunk = 1;
  }
  int64_t base = 0;  // shares (low half) and slots of split tiles (high half) before sequence s0
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const Extent e = s0 == 0 ? first : extent_of<ROWS, UNIT>(a, s0 + lane);
    int splits = 1;
    if (e.units > chunk) {
      splits = (int)((e.units + chunk - 1) / chunk);
      if (splits > kMostSplits) splits = kMostSplits;
    }
    const int parts = e.tiles * splits;
    const int64_t mine = (int64_t)(splits > 1 ? parts : 0) << 32 | (uint32_t)(joins ? (splits > 1 ? e.tiles : 0) : parts);
    int64_t up = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t v = __shfl_up(up, off);
      if (lane >= off) up += v;
    }
    up += base;
    const uint64_t past = __ballot((int)(uint32_t)up > item);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int64_t before = up - mine;
      r.s = s0 + at;
      r.q.start = lane_value(e.q.start, at), r.q.count = lane_value(e.q.count, at), r.q.kv = lane_value(e.q.kv, at);
      r.splits = lane_value(splits, at);
      const int tiles = lane_value(e.tiles, at);
      const int local = item - lane_value((int)(uint32_t)before, at);
      r.slot = lane_value((int)(before >> 32), at) + (joins ? local * r.splits : local);
      const int turn = joins ? local : local / r.splits, split = joins ? 0 : local - turn * r.splits;
      r.row0 = (tiles - 1 - turn) * ROWS;
      r.rows = min(ROWS, r.q.count * a.group - r.row0);
      const int p0 = r.q.kv - r.q.count + r.row0 / a.group;
      const int p1 = r.q.kv - r.q.count + (r.row0 + r.rows - 1) / a.group;
      const int lo = first_seen(a, p0) & ~63, hi = end_seen(a, p1, r.q.kv);
      const int64_t units = hi > lo ? (hi - lo + UNIT - 1) / UNIT : 0;
      r.begin = lo + (int)(units * split / r.splits) * UNIT;
      r.end = min(hi, lo + (int)(units * (split + 1) / r.splits) * UNIT);
      return true;
    }
    base = __shfl(up, 63);
  }
  return false;
}

// Page of token t (t < most_kv) of sequence s.
INTENT_DEVICE int page_of(const AttnArgs& a, int s, int t) {
  return (int)min((uint32_t)a.page_table[(int64_t)s * a.table_ld + (t >> a.page_shift)], (uint32_t)a.pages - 1u);
}

// The table's entry of token t as it is, and the page that it names.
INTENT_DEVICE uint32_t table_entry(const AttnArgs& a, int s, int t) {
  return (uint32_t)a.page_table[(int64_t)s * a.table_ld + (t >> a.page_shift)];
}
INTENT_DEVICE uint32_t page_named(const AttnArgs& a, uint32_t entry) { return min(entry, (uint32_t)a.pages - 1u); }

// Row of token t of a page and head in a cache with `row` elements for each token.
INTENT_DEVICE int64_t row_in_cache(const AttnArgs& a, int page, int64_t page_ld, int head, int t, int row) {
  return (int64_t)page * page_ld + (((int64_t)head << a.page_shift) + (t & ((1 << a.page_shift) - 1))) * row;
}

}  // namespace intent
