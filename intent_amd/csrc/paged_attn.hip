// Attention of new tokens over a paged cache (gfx950): the entry, and the kernel for any head size.
#include "paged_attn.h"

namespace {

using namespace intent;

constexpr int64_t kMostTokens = (int64_t)1 << 30;  // of a sequence: positions stay far inside 32 bits
constexpr int64_t kMostStride = UINT32_MAX;

template <bool kBf16>
INTENT_DEVICE float widen1(uint16_t v) {
  if constexpr (kBf16) return bit_cast<float>((uint32_t)v << 16);
  else return (float)bit_cast<f16>(v);
}

template <bool kBf16, bool kFp8>
INTENT_DEVICE void widen8(const void* p, float (&v)[8]) {
  if constexpr (kFp8) {
    const u32x2 raw = *(const u32x2*)p;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[j], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[j], true);
      v[4 * j] = lo[0], v[4 * j + 1] = lo[1], v[4 * j + 2] = hi[0], v[4 * j + 3] = hi[1];
    }
  } else {
    const u32x4 raw = load16(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = widen1<kBf16>((uint16_t)(raw[j] & 0xffffu));
      v[2 * j + 1] = widen1<kBf16>((uint16_t)(raw[j] >> 16));
    }
  }
}

template <bool kBf16, bool kFp8>
INTENT_DEVICE float widen_one(const void* cache, int64_t index) {
  if constexpr (kFp8) return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)cache)[index], 0);
  else return widen1<kBf16>(((const uint16_t*)cache)[index]);
}

INTENT_DEVICE float wave_max(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}
INTENT_DEVICE float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Any D that is a multiple of 8 up to 512: one wave for each query row. A lane takes one token of 64
// for the products with the keys, then D / 64 columns of the values, whose tokens the wave goes
// through one by one; tokens that the row does not see are not read.
template <bool kBf16, bool kFp8>
__global__ __launch_bounds__(256) void paged_attn_row_kernel(const AttnArgs a) {
  __shared__ float qs[4][512];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + wave;
  if (item >= (int64_t)a.T * a.HQ) return;
  const int row = (int)(item / a.HQ), head = (int)(item - (int64_t)row * a.HQ), kv_head = head / a.group;
  int s = -1;
  for (int s0 = 0; s0 < a.S && s < 0; s0 += 64) {
    bool owns = false;
    if (s0 + lane < a.S) {
      const Sequence q = sequence_of(a, s0 + lane);
      owns = row >= q.start && row < q.start + q.count;
    }
    const uint64_t found = __ballot(owns);
    if (found) s = s0 + __builtin_ctzll(found);
  }
  if (s < 0) return;  // a row of no sequence is left as it is
  const Sequence seq = sequence_of(a, s);
  const int p = seq.kv - seq.count + (row - seq.start);
  const int first = first_seen(a, p), end = end_seen(a, p, seq.kv);
  const uint16_t* q = a.q + (int64_t)row * a.q_ld + (int64_t)head * a.D;
  for (int d = lane; d < a.D; d += 64) qs[wave][d] = widen1<kBf16>(q[d]) * a.scale_log2;
  __builtin_amdgcn_wave_barrier();

  constexpr int kBytes = kFp8 ? 1 : 2;
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  float top = -INFINITY, total = 0.f;
  for (int t0 = first; t0 < end; t0 += 64) {
    const int t = t0 + lane;
    float score = -INFINITY, v_scale = 1.f;
    int page = 0;
    if (t < end) {
      page = page_of(a, s, t);
      const char* k = (const char*)a.k_cache + row_in_cache(a, page, a.k_page, kv_head, t, a.D) * kBytes;
      float sum = 0.f;
      for (int d = 0; d < a.D; d += 8) {
        float kv[8];
        widen8<kBf16, kFp8>(k + d * kBytes, kv);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(kv[j], qs[wave][d + j], sum);
      }
      if constexpr (kFp8) {
        sum *= a.k_scales[row_in_cache(a, page, a.ks_page, kv_head, t, 1)];
        v_scale = a.v_scales[row_in_cache(a, page, a.vs_page, kv_head, t, 1)];
      }
      score = sum;
    }
    const float m = fmaxf(top, wave_max(score));
    const float base = m == -INFINITY ? 0.f : m;
    const float keep = __builtin_amdgcn_exp2f(top - base);
    const float w = t < end ? __builtin_amdgcn_exp2f(score - base) : 0.f;
    total = total * keep + wave_sum(w);
    const float wv = w * v_scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= keep;
    const int n = min(end - t0, 64);
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl(wv, i);
      const int64_t v = row_in_cache(a, __shfl(page, i), a.v_page, kv_head, t0 + i, a.D);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (lane + 64 * j < a.D)
          acc[j] = __builtin_fmaf(wi, widen_one<kBf16, kFp8>(a.v_cache, v + lane + 64 * j), acc[j]);
    }
    top = m;
  }
  const float inv = end > first ? 1.0f / total : 0.f;
  uint16_t* out = a.out + (int64_t)row * a.out_ld + (int64_t)head * a.D;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (lane + 64 * j < a.D) {
      const float o = end > first ? acc[j] * inv : 0.f;
      if constexpr (kBf16) out[lane + 64 * j] = (uint16_t)(bf16x2_rne(o, o) & 0xffffu);
      else out[lane + 64 * j] = bit_cast<uint16_t>((f16)o);
    }
  }
}

template <bool kBf16, bool kFp8>
int launch_rows(const AttnArgs& a, hipStream_t stream) {
  const int64_t blocks = ((int64_t)a.T * a.HQ + 3) / 4;
  hipLaunchKernelGGL((paged_attn_row_kernel<kBf16, kFp8>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  static const KernelName name("paged_attn_row_kernel<%s%s>", kBf16 ? "bf16" : "f16", kFp8 ? ", fp8 cache" : "");
  return launch_status(name.text);
}

// ---- which kernel, and into how many parts --------------------------------------------

struct Part {
  int rows;  // of a tile
  int min_rows, max_rows;
  int unit_log() const { return rows <= 64 ? 7 : 6; }  // of the tokens that a share is a multiple of
  // Workgroups that the tiles are split for: what the 256 CUs hold at one time (by the kernels' registers),
  // and twice that where a CU holds three, which evens out sequences of different lengths and costs
  // little (four sequences of 60000 to 131000 tokens: 300 us at 512, 235 at 768, 239 at 1536; 64 of 300
  // to 8191 126, 128 and 119 us). One workgroup to a CU loses by a second round (16 sequences of five
  // drafted tokens: 28 us at 256, 34 at 512).
  int fill(int64_t D) const {
    if (rows > 64) return rows == 256 || D > 128 ? 256 : 512;
    return D > 128 ? 256 : rows * D <= 2048 ? 1536 : rows * D <= 4096 ? 512 : 256;
  }
};

struct Plan {
  Part part[2];
  int parts;
};

bool tiled(int64_t D) { return D == 64 || D == 96 || D == 128 || D == 256; }

// The host knows the extents only. Sequences of one new token each, and one sequence, are all alike, and as many
// new tokens as equal chunks make are taken to be: the kernel that spreads the tokens over the waves takes up to
// 64 rows of them in the tile that holds one, the other kernel more. Heads of 256 leave it registers for 16
// rows: up to 32 rows still do better in two of those tiles than in half of a tile of 128 (24 rows of 16
// sequences over 5000 tokens: 51 and 57 us, in 8 bits 32 and 48; 40 rows 125 and 59), and so do fewer than 512
// rows in all (400 of one head over 4000: 26 and 37; 312 of 13 sequences 129 and 47). Any other batch may mix
// decoding sequences with chunks: beyond 2048 rows in all, each sequence goes by its own rows to one of the two;
// fewer rows do not repay the launches (12 sequences of 1 to 24 tokens, 460 rows: 19 us in one, 32 in two).
// Short sequences are those of up to 16 rows, or up to 32 where more than 16 heads share a cached one, so that
// decoding stays among them (15 decoding sequences and a chunk of 403, groups of 24: 87 us, 92 with up to 16
// rows; it loses with 63 of them, 120 and 112, and in groups of 32, 83 and 67).
//
// That the sequences divide the tokens is a guess at equal chunks, and a mixture (or a padded batch) may meet
// it by chance. Both sides, one list and two, 32 heads on 8 of 128 over 1500 to 6000 cached tokens and over 50
// to 400: 63 decoding and a chunk of 961 296 and 276 us, 73 and 63; 7 and a chunk of 2041 193 and 187, 70 and
// 76; heads of 256, 31 and a chunk of 609: 182 and 148, 43 and 56. Equal ones pay for a launch that finds
// nothing: 4 chunks of 512 202 and 205, 44 and 47; 128 of five drafted tokens 387 and 398, 38 and 49 (64 of
// them in groups of 8 150 and 123, 20 and 23: their 40 rows then run in tiles of 128).
//
// More than 64 rows: with fewer than 22 tiles of 128 the other kernel's 64 rows, whose waves share the tokens,
// still fill more of the GPU (397 rows of two heads over 594 tokens: 17 us, 29 in tiles of 128; 758 x 4 of one
// head over 917 21 and 21; 512 x 4 of eight over 512 22 and 20). Tiles of 256 halve what is loaded for a row
// but need one and a half rounds of them to even out (4096 x 4 rows of eight heads over 4096: 157 us, 163 in
// tiles of 128; 2048 x 4 over 2048: 71 and 59).
Plan plan_of(int64_t T, int64_t S, int64_t HK, int64_t group, int64_t D) {
  const int64_t mean = (T * group + S - 1) / S;
  const int most = D > 128 ? 32 : 64, few = D > 128 || group <= 16 ? 16 : 32;
  const int64_t all = T * group * HK;
  const int tile = D > 128 ? (all < 4 * 128 ? 16 : 128) : all < 22 * 128 ? 64 : all < 384 * 256 ? 128 : 256;
  Plan p{};
  if (T > S && T % S != 0 && T * group > 2048) {
    p.parts = 2;
    p.part[0] = {tile, few, INT32_MAX};
    p.part[1] = {few, 0, few};
  } else {
    p.parts = 1;
    const int few_rows = D > 128 ? 16 : (int)((mean + 15) / 16) * 16;
    p.part[0] = {mean <= 16 ? 16 : mean <= most ? few_rows : tile, 0, INT32_MAX};
  }
  return p;
}

// Tiles of one head: every sequence's last one may be partly filled, and sequences of at most a tile have one.
int64_t tiles_bound(const Part& p, int64_t T, int64_t S, int64_t group) {
  const int64_t some = S < T ? S : T;
  return p.max_rows <= p.rows ? some : T * group / p.rows + some;
}

// Shares of one head that its tiles are split for. Sequences of a tile each that take half the GPU and more
// as they are: with heads of 256, whose tiles have a CU to themselves, lengths that differ leave a second
// round of a few long shares, so twice as many (111 sequences of 2600 to 7500 tokens on two heads: 612 us
// with 256 shares, 401 with 512; 128 of them 570 and 434; all of 5000 332 and 360). More tiles to a sequence
// even out by themselves.
int64_t target_of(const Part& p, int64_t T, int64_t S, int64_t group, int64_t HK, int64_t D) {
  const int64_t fill = p.fill(D);
  const bool uneven = D > 128 && p.rows == 128 && T * group <= S * p.rows && S * HK * 2 > fill;
  return (fill * (uneven ? 2 : 1) + HK - 1) / HK;
}

// Parts of all split tiles of one head: fewer than twice the target (a tile of one and a half shares and
// more is cut to the nearest number of them), and at most every tile's most.
int64_t slots_bound(const Part& p, int64_t T, int64_t S, int64_t group, int64_t HK, int64_t D, int64_t most_kv) {
  const int64_t target = target_of(p, T, S, group, HK, D);
  int64_t splits = (most_kv + (1 << p.unit_log()) - 1) >> p.unit_log();
  if (splits > kMostSplits) splits = kMostSplits;
  if (splits < 2) return 0;
  const int64_t all = tiles_bound(p, T, S, group) * splits;
  return all < 2 * target ? all : 2 * target;
}

size_t part_bytes(const Part& p, int64_t T, int64_t S, int64_t group, int64_t HK, int64_t D, int64_t most_kv) {
  return (size_t)(slots_bound(p, T, S, group, HK, D, most_kv) * HK * p.rows * (D + 2) * 4);
}

int launch_tiled(AttnArgs a, bool bf16, bool fp8, float* workspace, size_t bytes, hipStream_t stream) {
  const Plan plan = plan_of(a.T, a.S, a.HK, a.group, a.D);
  size_t need = 0;
  for (int i = 0; i < plan.parts; ++i) need += part_bytes(plan.part[i], a.T, a.S, a.group, a.HK, a.D, a.most_kv);
  AttnJoin join{};
  int lists = 0;
  for (int i = 0; i < plan.parts; ++i) {
    const Part& p = plan.part[i];
    const int64_t slots = slots_bound(p, a.T, a.S, a.group, a.HK, a.D, a.most_kv);
    // one sequence's tiles all attend the same tokens: enough of them even out by themselves
    const bool many = a.S == 1 && (int64_t)a.T * a.group / p.rows * a.HK >= 2 * p.fill(a.D);
    const bool split = slots > 0 && workspace != nullptr && bytes >= need && !many;
    a.min_rows = p.min_rows, a.max_rows = p.max_rows;
    a.target = split ? (int)target_of(p, a.T, a.S, a.group, a.HK, a.D) : 0;
    a.slots = split ? (int)slots : 0;
    a.partial = workspace;
    a.partial_stats = split ? workspace + slots * a.HK * p.rows * a.D : nullptr;
    const int64_t tiles = tiles_bound(p, a.T, a.S, a.group);
    // workgroups of 256 or 512 lanes: the grid's work items stay below 2^32
    INTENT_REQUIRE((tiles + a.target) * a.HK < ((int64_t)1 << 23), INTENT_ERR_UNSUPPORTED,
                   "%lld tiles of %d heads exceed the %lld workgroups that a launch covers", (long long)tiles, a.HK,
                   (long long)((int64_t)1 << 23));
    const int items = (int)(tiles + a.target);
    const auto go = fp8 ? (bf16 ? launch_attn_bf16_fp8 : launch_attn_f16_fp8) : (bf16 ? launch_attn_bf16 : launch_attn_f16);
    const int status = go(a, items, p.rows, stream);
    if (status != INTENT_OK) return status;
    if (!split) continue;
    // a tile is split from one and a half shares on
    const int64_t most = a.target * 2 / 3 + 1;
    if (lists == 0) {
      join.a = a;
    } else {
      join.min_rows = a.min_rows, join.max_rows = a.max_rows, join.target = a.target, join.slots = a.slots;
      join.partial = a.partial, join.partial_stats = a.partial_stats;
    }
    join.tile[lists] = p.rows, join.unit_log[lists] = p.unit_log();
    join.items[lists++] = (int)(tiles < most ? tiles : most);
    workspace += part_bytes(p, a.T, a.S, a.group, a.HK, a.D, a.most_kv) / 4;
  }
  if (lists == 0) return INTENT_OK;
  // workgroups for the rows of a split tile: one for each of a mean sequence, up to 1024 in all
  const int64_t mean = ((int64_t)a.T * a.group + a.S - 1) / a.S;
  const int64_t room = 1024 / ((int64_t)(join.items[0] + join.items[1]) * a.HK), rows = plan.part[0].rows;
  const int64_t side = mean < rows ? mean : rows;
  const int sides = (int)(room < 1 ? 1 : room < side ? room : side);
  return bf16 ? launch_join_bf16(join, sides, stream) : launch_join_f16(join, sides, stream);
}

}  // namespace

extern "C" size_t intent_paged_attention_workspace_size(int64_t T, int64_t HQ, int64_t HK, int64_t D, int64_t S,
                                                        int64_t table_width, int64_t page_size) {
  if (T <= 0 || HQ <= 0 || HK <= 0 || S <= 0 || HQ % HK || table_width <= 0 || page_size <= 0 || !tiled(D) ||
      table_width > kMostTokens / page_size || HQ > 65536 || T * HQ >= ((int64_t)1 << 25))
    return 0;
  const Plan plan = plan_of(T, S, HK, HQ / HK, D);
  size_t need = 0;
  for (int i = 0; i < plan.parts; ++i)
    need += part_bytes(plan.part[i], T, S, HQ / HK, HK, D, table_width * page_size);
  return need;
}

extern "C" int intent_paged_attention(const void* q, int64_t T, int64_t HQ, int64_t q_ld, int is_bf16,
                                      int cache_is_fp8, const void* k_cache, int64_t k_page_ld, const void* v_cache,
                                      int64_t v_page_ld, const float* k_scales, int64_t k_scales_ld,
                                      const float* v_scales, int64_t v_scales_ld, int64_t pages, int64_t HK,
                                      int64_t page_size, int64_t D, const int32_t* page_table, int64_t S,
                                      int64_t table_width, int64_t table_ld, const int32_t* q_offsets,
                                      const int32_t* kv_lens, float scale, int causal, int64_t window, void* out,
                                      int64_t out_ld, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  INTENT_REQUIRE(T >= 0 && HQ >= 0 && HK >= 0 && D >= 0 && S >= 0 && pages >= 0 && page_size >= 0 && table_width >= 0 &&
                     window >= 0 && T <= INT32_MAX && HQ <= 65536 && HK <= 65536 && S < INT32_MAX &&
                     pages <= INT32_MAX && page_size <= INT32_MAX,
                 INTENT_ERR_INVALID_ARGUMENT, "bad extents (T=%lld HQ=%lld HK=%lld D=%lld S=%lld pages=%lld of %lld)",
                 (long long)T, (long long)HQ, (long long)HK, (long long)D, (long long)S, (long long)pages,
                 (long long)page_size);
  if (T == 0 || HQ == 0 || D == 0 || S == 0) return INTENT_OK;
  const float scale_log2 = scale * 1.44269504088896340736f;
  INTENT_REQUIRE(__builtin_isfinite(scale_log2), INTENT_ERR_INVALID_ARGUMENT, "scale * log2(e) must be finite, got %g",
                 (double)scale_log2);
  INTENT_REQUIRE(HK > 0 && HQ % HK == 0, INTENT_ERR_INVALID_ARGUMENT,
                 "HQ=%lld query heads must be a multiple of the HK=%lld heads of the cache", (long long)HQ,
                 (long long)HK);
  INTENT_REQUIRE(D % 8 == 0 && D <= 512, INTENT_ERR_UNSUPPORTED, "D must be a multiple of 8 up to 512, got %lld",
                 (long long)D);
  const bool any = pages > 0 && page_size > 0 && table_width > 0;
  INTENT_REQUIRE(!any || (page_size & (page_size - 1)) == 0, INTENT_ERR_UNSUPPORTED,
                 "the page size must be a power of two, got %lld", (long long)page_size);
  INTENT_REQUIRE(!any || table_width <= kMostTokens / page_size, INTENT_ERR_UNSUPPORTED,
                 "a table of %lld pages of %lld tokens exceeds 2^30 tokens", (long long)table_width,
                 (long long)page_size);
  INTENT_REQUIRE(!any || HK <= UINT32_MAX / page_size, INTENT_ERR_UNSUPPORTED, "pages of %lld tokens of %lld heads",
                 (long long)page_size, (long long)HK);
  // at most a wave for each row of a head: the grid's work items stay below 2^32
  INTENT_REQUIRE(T * HQ < ((int64_t)1 << 25), INTENT_ERR_UNSUPPORTED,
                 "T * HQ = %lld rows exceed the %lld a launch covers", (long long)(T * HQ),
                 (long long)((int64_t)1 << 25));
  INTENT_REQUIRE(q && out && q_offsets && kv_lens && (!any || (k_cache && v_cache && page_table)) &&
                     (!any || !cache_is_fp8 || (k_scales && v_scales)),
                 INTENT_ERR_INVALID_ARGUMENT, "null pointer argument");
  INTENT_REQUIRE(T == 1 || (q_ld >= HQ * D && out_ld >= HQ * D), INTENT_ERR_INVALID_ARGUMENT,
                 "token stride smaller than the heads");
  INTENT_REQUIRE(intent::aligned16(q) && intent::aligned16(out) && (T == 1 || (q_ld % 8 == 0 && out_ld % 8 == 0)),
                 INTENT_ERR_ALIGNMENT, "q and out must be 16-byte aligned with token strides %% 8 == 0");
  if (any) {
    const int64_t step = cache_is_fp8 ? 16 : 8;
    INTENT_REQUIRE(S == 1 || table_ld >= table_width, INTENT_ERR_INVALID_ARGUMENT, "table stride smaller than the row");
    INTENT_REQUIRE(pages == 1 || (k_page_ld >= HK * page_size * D && v_page_ld >= HK * page_size * D &&
                                  (!cache_is_fp8 || (k_scales_ld >= HK * page_size && v_scales_ld >= HK * page_size))),
                   INTENT_ERR_INVALID_ARGUMENT, "page stride smaller than the page");
    INTENT_REQUIRE(intent::aligned16(k_cache) && intent::aligned16(v_cache) &&
                       (pages == 1 || (k_page_ld % step == 0 && v_page_ld % step == 0)) &&
                       (!cache_is_fp8 || (intent::aligned4(k_scales) && intent::aligned4(v_scales))),
                   INTENT_ERR_ALIGNMENT, "the cache must be 16-byte aligned with page strides of whole 16 bytes");
  }
  INTENT_REQUIRE(!any || pages == 1 || (k_page_ld <= kMostStride && v_page_ld <= kMostStride &&
                                        k_scales_ld <= kMostStride && v_scales_ld <= kMostStride),
                 INTENT_ERR_UNSUPPORTED, "page stride past 2^32 elements");
  AttnArgs a{};
  a.q = (const uint16_t*)q, a.q_ld = q_ld;
  a.k_cache = k_cache, a.v_cache = v_cache, a.k_page = k_page_ld, a.v_page = v_page_ld;
  a.k_scales = k_scales, a.v_scales = v_scales, a.ks_page = k_scales_ld, a.vs_page = v_scales_ld;
  const int64_t units = cache_is_fp8 ? 16 : 8;
  a.k_step = (uint32_t)(k_page_ld / units), a.v_step = (uint32_t)(v_page_ld / units);
  a.ks_step = (uint32_t)k_scales_ld, a.vs_step = (uint32_t)v_scales_ld;
  a.page_table = page_table, a.table_ld = table_ld;
  a.q_offsets = q_offsets, a.kv_lens = kv_lens;
  a.out = (uint16_t*)out, a.out_ld = out_ld;
  a.scale_log2 = scale_log2;
  a.T = (int)T, a.S = (int)S, a.HQ = (int)HQ, a.HK = (int)HK, a.group = (int)(HQ / HK), a.D = (int)D;
  a.pages = any ? (int)pages : 0, a.page_shift = any ? __builtin_ctzll((unsigned long long)page_size) : 0;
  a.most_kv = any ? (int)(table_width * page_size) : 0;
  a.causal = causal != 0, a.window = (int)(window < INT32_MAX ? window : INT32_MAX);
  hipStream_t st = (hipStream_t)stream;
  if (tiled(D)) {
    const bool aligned = workspace != nullptr && intent::aligned16(workspace);
    return launch_tiled(a, is_bf16 != 0, cache_is_fp8 != 0, aligned ? (float*)workspace : nullptr, workspace_bytes, st);
  }
  if (cache_is_fp8) return is_bf16 ? launch_rows<true, true>(a, st) : launch_rows<false, true>(a, st);
  return is_bf16 ? launch_rows<true, false>(a, st) : launch_rows<false, false>(a, st);
}
