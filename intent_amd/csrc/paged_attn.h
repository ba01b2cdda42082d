// Attention of new tokens over a paged cache: what its kernels share.
//
// Sequence s owns the query rows q_offsets[s] .. q_offsets[s+1] and the first kv_lens[s] tokens of
// its pages (the new tokens among them, appended before the call). Its row i of n stands at position
// p = kv_len - n + i and sees the tokens t with
//   t < kv_len,   t <= p (causal),   t > p - window (window > 0).
//   out = sum_t w_t v_t / sum_t w_t,   w_t = exp(x_t - max),   0 where nothing is seen,
//   x_t = scale q.k_t.
// Biased, each where it is asked for:
//   x_t = cap tanh(scale q.k_t / cap),   then less slope[head] |p - t|;
//   t <= p or t < prefix_len (causal): a prefix is seen by every row.
// Offsets, lengths and page ids come from device memory: they are clamped to the tensors' extents,
// so a wrong one gives a wrong row and no access outside them.
#pragma once

#include "common.h"
#include "internal.h"
#include "paged_cache.h"

namespace intent {

// Forms of scores that a kernel knows; all but the first know prefixes.
enum ScoreForms { kPlain = 0, kCapped = 1, kSloped = 2, kBoth = 3 };

constexpr const char* form_name(int forms) {
  return forms == kCapped ? ", capped" : forms == kSloped ? ", sloped" : forms == kBoth ? ", capped and sloped" : "";
}

struct AttnArgs {
  const uint16_t* q;
  int64_t q_ld;
  const void *k_cache, *v_cache;
  int64_t k_page, v_page;  // elements from a page to the next
  const float *k_scales, *v_scales;  // of 8 bits; of 4: the groups' pairs of f16
  int64_t ks_page, vs_page;          // scales (pairs) from a page to the next
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
  int slots;               // parts of split tiles of one head that the workspace holds
  float* partial;          // [slot][HK][tile rows][D] unnormalised sums, then [slot][HK][tile rows][2]
  float* partial_stats;
  // biased: null and zero where a form is not asked for
  const float* slopes;  // of a query head, times log2(e) where they are used
  const int32_t* prefix_lens;
  float cap_log2;  // cap * log2(e)
};

// The tiled kernels for one type, cache and form of scores (paged_attn_*.hip), by the rows of a tile: 16 to 64,
// whose tokens are spread over a workgroup's four waves, or 128 or 256, 32 to a wave. `items` workgroups for each
// cached head.
// `few`: the list of a mixture's short sequences (16 rows, heads of 64), in the same launch with tiles of 128 rows.
typedef int LaunchAttn(const AttnArgs& a, int items, int rows, const AttnArgs* few, int few_items, hipStream_t stream);
LaunchAttn launch_attn_f16, launch_attn_bf16, launch_attn_f16_fp8, launch_attn_bf16_fp8, launch_attn_f16_int4,
    launch_attn_bf16_int4, launch_attn_f16_capped, launch_attn_bf16_capped, launch_attn_f16_fp8_capped,
    launch_attn_bf16_fp8_capped, launch_attn_f16_int4_capped, launch_attn_bf16_int4_capped, launch_attn_f16_sloped,
    launch_attn_bf16_sloped, launch_attn_f16_fp8_sloped, launch_attn_bf16_fp8_sloped, launch_attn_f16_int4_sloped,
    launch_attn_bf16_int4_sloped, launch_attn_f16_both, launch_attn_bf16_both, launch_attn_f16_fp8_both,
    launch_attn_bf16_fp8_both, launch_attn_f16_int4_both, launch_attn_bf16_int4_both;

// One launch for the joins of the split tiles of up to two lists: the rows of each one's tiles, its units of
// tokens (their logarithm) and workgroups for each cached head (0: no list), and the second list's own
// arguments where they differ.
struct AttnJoin {
  int items[2], tile[2], unit_log[2];
  int min_rows, max_rows, target, slots;
  float *partial, *partial_stats;
  AttnArgs a;
};
// with `side` workgroups for the rows of a tile
typedef int LaunchJoin(const AttnJoin& j, int side, hipStream_t stream);
LaunchJoin launch_join_f16, launch_join_bf16, launch_join_f16_prefix, launch_join_bf16_prefix;

// Query rows [start, start + count), cached tokens and prefix of sequence s.
struct Sequence {
  int start, count, kv, front;
};

INTENT_DEVICE Sequence sequence_of(const AttnArgs& a, int s) {
  Sequence r;
  r.start = min(max(a.q_offsets[s], 0), a.T);
  r.count = max(min(a.q_offsets[s + 1], a.T) - r.start, 0);
  r.kv = min(max(a.kv_lens[s], 0), a.most_kv);
  r.front = 0;
  return r;
}

// The tokens of sequence s that every row sees (a window aside).
INTENT_DEVICE int prefix_of(const AttnArgs& a, int s) { return a.prefix_lens != nullptr ? max(a.prefix_lens[s], 0) : 0; }

// First and one past the last token that the row at position p sees.
INTENT_DEVICE int first_seen(const AttnArgs& a, int p) { return a.window > 0 && p >= a.window ? p - a.window + 1 : 0; }
INTENT_DEVICE int end_seen(const AttnArgs& a, int p, const Sequence& q) {
  return a.causal ? min(max(p + 1, q.front), q.kv) : q.kv;
}

// Parts of a tile. One sequence on one cached head would be cut further to fill the GPU, but its join goes through
// the parts of a row in one workgroup: 131000 tokens take 40 us in 256 parts and 111 in 1024; on two heads 47 and
// 68, on eight (fewer parts by themselves) 117 and 117.
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

INTENT_DEVICE Extent extent_of(const AttnArgs& a, int tile, int unit_log, int s) {
  Extent e;
  e.q = sequence_of(a, min(s, a.S - 1));
  const int rows = e.q.count * a.group;
  const bool listed = s < a.S && rows > a.min_rows && rows <= a.max_rows;
  const int lo = first_seen(a, e.q.kv - e.q.count) & ~63;
  e.tiles = listed ? (int)(((uint32_t)rows + (uint32_t)tile - 1u) / (uint32_t)tile) : 0;
  e.units = listed ? (e.q.kv - lo + (1 << unit_log) - 1) >> unit_log : 0;
  return e;
}

INTENT_DEVICE int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Sum over the wave, and sum of the lanes up to this one (DPP: shifts in rows of 16, then each row's
// last value to the rows behind it).
template <int CTRL, int ROWS>
INTENT_DEVICE int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
INTENT_DEVICE int wave_prefix(int v) {
  v = dpp_add<0x111, 0xf>(v);
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);
  return dpp_add<0x143, 0xc>(v);
}
INTENT_DEVICE float wave_total(float v) {
  const float in[1] = {v};
  float out[1];
  WaveReduce<1>::run(in, out);
  return out[0];
}

// Rows and tokens of share `local` of a sequence's (r.s, r.q and r.splits are set; with `joins`, of its
// tiles), whose parts begin at `slot`.
INTENT_DEVICE bool span_of(const AttnArgs& a, int tile, int unit_log, int tiles, int local, int slot, bool joins,
                           Span& r) {
  r.slot = slot + (joins ? local * r.splits : local);
  const int turn = joins ? local : (int)((uint32_t)local / (uint32_t)r.splits);
  const int split = joins ? 0 : local - turn * r.splits;
  // offsets that overlap may count up to anything: nothing outside the rows and the workspace then
  if (local < 0 || turn >= tiles || (r.splits > 1 && (r.slot < 0 || r.slot >= a.slots))) return false;
  if (joins && r.slot + r.splits > a.slots) return false;
  r.row0 = (tiles - 1 - turn) * tile;
  r.rows = min(tile, r.q.count * a.group - r.row0);
  const int before = r.q.kv - r.q.count;
  const int p0 = before + (int)((uint32_t)r.row0 / (uint32_t)a.group);
  const int p1 = before + (int)((uint32_t)(r.row0 + r.rows - 1) / (uint32_t)a.group);
  const int lo = first_seen(a, p0) & ~63, hi = end_seen(a, p1, r.q);
  const uint32_t units = hi > lo ? (uint32_t)(hi - lo + (1 << unit_log) - 1) >> unit_log : 0u;
  const uint32_t each = units / (uint32_t)r.splits, more = units - each * (uint32_t)r.splits;
  const uint32_t from = each * split + min((uint32_t)split, more);
  const uint32_t to = from + each + ((uint32_t)split < more ? 1u : 0u);
  r.begin = lo + ((int)from << unit_log);
  r.end = min(hi, lo + ((int)to << unit_log));
  return true;
}

// Finds share `item` of one head's list of tiles of `tile` rows, tokens in units of 1 << unit_log: the
// sequences in order, each with its row tiles from the last (which sees most) to the first, each tile in
// `splits` parts of its tokens. The parts are sized so that all sequences together give about a.target of
// them: units / chunk of each, to the nearest number, chunk = the units that a workgroup would get of an
// even share (rounded up, so never less than that: the workspace is sized by it), but for tiles of more
// than 64 rows no fewer than 8 units (a join costs as many). With `joins`, the list of the tiles that are
// split. Every wave does it by itself: no plan is kept, so a captured call follows lengths that change. The
// counts of one list fit 32 bits (the host bounds the grid).
//
// Lanes take a sequence each of 64, or of AT times 64 whose extents are all loaded before the first is
// used: 2048 sequences of 512 tokens take 1245 us with 64 at a time, 935 with 256; one sequence takes 7.1
// us with 64 and would wait for three useless loads with 256.
template <int AT, bool kBiased>
INTENT_DEVICE bool find_span_by(const AttnArgs& a, int tile, int unit_log, int item, bool joins, Span& r) {
  const int lane = threadIdx.x & 63;
  Extent e[AT];
#pragma unroll
  for (int i = 0; i < AT; ++i) e[i] = extent_of(a, tile, unit_log, i * 64 + lane);
  int chunk = INT32_MAX;
  if (a.target > 0) {
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < AT; ++i) all += (float)e[i].tiles * (float)e[i].units;
    for (int s0 = AT * 64; s0 < a.S; s0 += AT * 64) {
      Extent f[AT];
#pragma unroll
      for (int i = 0; i < AT; ++i) f[i] = extent_of(a, tile, unit_log, s0 + i * 64 + lane);
#pragma unroll
      for (int i = 0; i < AT; ++i) all += (float)f[i].tiles * (float)f[i].units;
    }
    chunk = (int)fminf(wave_total(all) * (1.0f + 0x1p-12f) / (float)a.target, 1.0e9f) + 1;
    if (tile > 64) chunk = max(chunk, 8);
  }
  int base = 0, slots = 0;  // shares, and slots of split tiles, before sequence s0
  for (int s0 = 0;;) {
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      const uint32_t near = ((uint32_t)e[i].units + (uint32_t)chunk / 2u) / (uint32_t)chunk;  // to the nearest
      const int splits = near > 1u ? min((int)near, kMostSplits) : 1;
      const int parts = e[i].tiles * splits, kept = splits > 1 ? parts : 0;
      const int mine = joins ? (splits > 1 ? e[i].tiles : 0) : parts;
      const int up = wave_prefix(mine) + base, kept_up = wave_prefix(kept) + slots;
      const uint64_t past = __ballot(up > item);
      if (past) {
        const int at = __builtin_ctzll(past);
        r.s = s0 + i * 64 + at;
        r.q.start = lane_value(e[i].q.start, at), r.q.count = lane_value(e[i].q.count, at);
        r.q.kv = lane_value(e[i].q.kv, at), r.q.front = kBiased ? prefix_of(a, r.s) : 0;
        r.splits = lane_value(splits, at);
        const int local = item - lane_value(up - mine, at), slot = lane_value(kept_up - kept, at);
        return span_of(a, tile, unit_log, lane_value(e[i].tiles, at), local, slot, joins, r);
      }
      base = lane_value(up, 63), slots = lane_value(kept_up, 63);
    }
    s0 += AT * 64;
    if (s0 >= a.S) return false;
#pragma unroll
    for (int i = 0; i < AT; ++i) e[i] = extent_of(a, tile, unit_log, s0 + i * 64 + lane);
  }
}
template <bool kBiased>
INTENT_DEVICE bool find_span(const AttnArgs& a, int tile, int unit_log, int item, bool joins, Span& r) {
  if (a.S <= 64) return find_span_by<1, kBiased>(a, tile, unit_log, item, joins, r);
  return find_span_by<4, kBiased>(a, tile, unit_log, item, joins, r);
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

// The score's form in base 2: x times log2(e) in and out. tanh(y) = 1 - 2 / (exp(2 y) + 1): 2^-23 of the cap
// off at most, the rounding of scores as large as it. exp2 may end at infinity or zero: tanh is 1 or -1 there.
INTENT_DEVICE float capped(float x, float cap_log2, float rate) {
  const float e = __builtin_amdgcn_exp2f(x * rate);
  return __builtin_fmaf(-2.0f * cap_log2, __builtin_amdgcn_rcpf(e + 1.0f), cap_log2);
}
// `rate` of capped(): 2 log2(e) / cap_log2.
INTENT_DEVICE float cap_rate(const AttnArgs& a) { return 2.88539008177792681472f / a.cap_log2; }

// Row of token t of a page and head in a cache with `row` elements for each token.
INTENT_DEVICE int64_t row_in_cache(const AttnArgs& a, int page, int64_t page_ld, int head, int t, int row) {
  return (int64_t)page * page_ld + (((int64_t)head << a.page_shift) + (t & ((1 << a.page_shift) - 1))) * row;
}

}  // namespace intent
