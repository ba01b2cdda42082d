// The tiled attention kernels (see paged_attn.h for the operator). Included by one source file for each
// type of heads and cache.
//
// Both compute the transposed products, S^T = K Q^T and O^T = V^T P^T. An MFMA leaves four consecutive
// rows of a column in a lane, so S^T puts the scores of one query row in one lane column: its softmax
// needs no exchange but a maximum over two or four lane groups, and the weights are already where the
// second product reads its right operand (its sum over tokens may go in any order: k index (g, j) of
// lane group g is the token that the first product left there). The left operand V^T is read from
// row-major values in LDS by the transposing read (ds_read_b64_tr_b16: of 16 lanes' 8 bytes, four rows
// of 16 columns, each lane gets one column).
//
// Running softmax in base 2: weights w = exp2(t - M) with t the score times scale log2(e). M follows
// the maximum only when that has risen by 8, so weights reach 2^8 at most and the sums are rescaled
// rarely. With an 8-bit cache the value's scale is part of the weight that is rounded: M follows the
// maximum of t + log2(scale), w = exp2(t - M) * scale, and only the sum of weights takes exp2(t - M) by
// itself. The codes are exact in 16 bits.
//
// 4 bits are widened to f16, for heads of bf16 too (its packed operations have no counterpart for bf16): lowest +
// scale code in one rounding, 2^-12 of it off at most where the code itself stands for a thirtieth of the group's
// range. Scores are then 2^-12 sum |q k| off, weights by as much (f16 heads: 5e-4 of the output against 2e-4 with
// f32 rows; bf16's own rounding is 17e-4); to leave the scale out of the product would keep the codes exact, but
// takes an accumulator and a weight for every group. Queries of bf16 are brought into f16's range row by row
// (query_f16); weights are f16's.
//
// The product with the values takes the weights rounded to the heads' type, half a step of it each, like
// the values beside them; the sums of weights are those before the rounding. bf16 has the exponents of
// f32. f16 ends at 2^-24, and a long flat tail behind one token that outweighs it may lie below: there all
// weights are 2^kLift higher (2^15 at most), so each is off by half a step or by 2^-32 of the highest, and
// numerators, sums and parts alike carry the factor, which their quotient drops.
//
// A weight of zero does not keep an infinity or NaN out of a product. Values of tokens that no row of a
// tile sees (pages behind a sequence's end hold anything) are set to zero; where rows of a tile see
// different tokens (the last of a chunk, the first of a window), values and scales that are not finite
// go into the product as zeros, and once the loop is over they are added to the rows that see them, which
// makes those infinite or NaN.
#pragma once

#include "paged_attn.h"

namespace intent {
namespace attn {

using ::load16;

constexpr float kRise = 8.0f;
template <bool kBf16>
constexpr float kLift = kBf16 ? 0.f : 7.f;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A cached token's row or scale: global addresses, so that the loads count on vmcnt alone.
typedef const __attribute__((address_space(1))) char* global_bytes;
INTENT_DEVICE global_bytes as_global(const void* p) { return (global_bytes)p; }
// Bytes of a token's head in the cache, and scales (or pairs of f16) beside it.
template <int kCache, int D>
constexpr int cached_bytes() {
  return kCache == kCacheInt4 ? D / 2 : kCache == kCacheFp8 ? D : D * 2;
}
template <int kCache, int D>
constexpr int cached_params() {
  return kCache == kCacheInt4 ? D / kGroup4 : 1;
}
// Rows (of kRowBytes) of a head from token t on, t and the page uniform or not.
template <int kRowBytes>
INTENT_DEVICE global_bytes cached_rows(const AttnArgs& a, const void* base, uint32_t page, uint32_t step, int head,
                                       int t) {
  const uint32_t row = ((uint32_t)head << a.page_shift) + ((uint32_t)t & ((1u << a.page_shift) - 1u));
  return as_global(base) + ((uint64_t)page * step + (uint64_t)row * (kRowBytes / 16)) * 16;
}
// Their scales or pairs, kParams of them to a token.
template <int kParams>
INTENT_DEVICE global_bytes cached_scales(const AttnArgs& a, const float* base, uint32_t page, uint32_t step, int head,
                                         int t) {
  const uint32_t row = ((uint32_t)head << a.page_shift) + ((uint32_t)t & ((1u << a.page_shift) - 1u));
  return as_global(base) + ((uint64_t)page * step + (uint64_t)row * kParams) * 4;
}
INTENT_DEVICE float load_float(global_bytes p) { return *(const __attribute__((address_space(1))) float*)p; }
INTENT_DEVICE u32x4 load16(global_bytes p) { return *(const __attribute__((address_space(1))) u32x4*)p; }
INTENT_DEVICE uint32_t load4(global_bytes p) { return *(const __attribute__((address_space(1))) uint32_t*)p; }
INTENT_DEVICE u32x2 load8(global_bytes p) { return *(const __attribute__((address_space(1))) u32x2*)p; }

template <bool kBf16>
INTENT_DEVICE f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bit_cast<bf16x8>(a), bit_cast<bf16x8>(b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(bit_cast<f16x8>(a), bit_cast<f16x8>(b), c, 0, 0, 0);
}
template <bool kBf16>
INTENT_DEVICE f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bit_cast<bf16x8>(a), bit_cast<bf16x8>(b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<f16x8>(a), bit_cast<f16x8>(b), c, 0, 0, 0);
}

// Keeps the compiler from turning a rarely taken uniform branch into selects on the common path.
INTENT_DEVICE void rarely() { asm volatile(""); }

template <bool kBf16>
INTENT_DEVICE uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) return bf16x2_rne(lo, hi);
  else return bit_cast<uint32_t>(__builtin_convertvector(f32x2{lo, hi}, f16x2));
}

// Eight E4M3FN codes as eight 16-bit floats (exact).
template <bool kBf16>
INTENT_DEVICE u32x4 widen_codes(uint32_t lo, uint32_t hi) {
  u32x4 r;
  if constexpr (kBf16) {
    r[0] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    r[1] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    r[2] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    r[3] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    r[0] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    r[1] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    r[2] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    r[3] = bit_cast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
  }
  return r;
}

// 16 bytes of cached values with zeros for infinities and NaN, which are noted in `found`. (All exponent
// bits of a 16-bit float set: one more in the exponent's last place carries into the sign's place, which
// the mask has cleared. E4M3FN: all bits but the sign's, and there are no infinities.)
template <bool kBf16, bool kFp8>
INTENT_DEVICE u32x4 only_finite(u32x4 v, bool& found) {
  constexpr uint32_t kExponent = kFp8 ? 0x7f7f7f7fu : kBf16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t kStep = kFp8 ? 0x01010101u : kBf16 ? 0x00800080u : 0x04000400u;
  constexpr uint32_t kSigns = kFp8 ? 0x80808080u : 0x80008000u;
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t out = ((v[e] & kExponent) + kStep) & kSigns;
    any |= out;
    v[e] &= ~((out >> (kFp8 ? 7 : 15)) * (kFp8 ? 0xffu : 0xffffu));
  }
  found = found || any != 0;
  return v;
}

// Element d of token t of a page and head in the values, as it goes into the product (8 bits: times its scale).
template <bool kBf16, int kCache, int D>
INTENT_DEVICE float cached_value(const AttnArgs& a, int page, int head, int t, int d) {
  constexpr int kRow = cached_bytes<kCache, D>(), kParams = cached_params<kCache, D>();
  const char* row = (const char*)cached_rows<kRow>(a, a.v_cache, page, a.v_step, head, t);
  const char* params = (const char*)cached_scales<kParams>(a, a.v_scales, page, a.vs_step, head, t);
  if constexpr (kCache == kCacheInt4) {
    const f16x2 pair = bit_cast<f16x2>(((const uint32_t*)params)[d / kGroup4]);
    const uint32_t code = ((const uint32_t*)row)[d / 8] >> code_bit(d) & 15u;
    return (float)__builtin_elementwise_fma((f16)(int)code, pair[0], pair[1]);
  } else if constexpr (kCache == kCacheFp8) {
    return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)row)[d], 0) * *(const float*)params;
  } else if constexpr (kBf16) {
    return bit_cast<float>((uint32_t)((const uint16_t*)row)[d] << 16);
  } else {
    return (float)((const f16*)row)[d];
  }
}
INTENT_DEVICE u32x2 read_transposed(const char* lds) {
  return bit_cast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)(__attribute__((address_space(3))) char*)lds));
}

// Rows of LDS tiles are a power of two of bytes (RB); the 16-byte chunk c of token t is kept at
// c ^ swizzle(t). LDS has 64 banks of 4 bytes, so that 16 lanes of a 16-byte access and 32 of an 8-byte
// one have to lie apart in 256 bytes: one chunk of 16 consecutive tokens (16 bytes each), and what a
// transposing read takes of 4 tokens (64 bytes each, the kernel of many rows) or of 8 (32 bytes each, the
// other). Rows of 128 bytes alternate between the halves of the banks by themselves.
template <int RB, bool kTileKernel>
INTENT_DEVICE int swizzle(int t) {
  if constexpr (kTileKernel) return RB == 128 ? (t >> 1 & 1) << 2 | (t >> 2 & 3) : (t & 3) << 2 | (t >> 2 & 3);
  else return RB == 128 ? (t >> 1 & 3) << 1 | (t >> 3 & 1) : (t & 7) << 1 | (t >> 3 & 1);
}

template <int D>
constexpr int row_bytes() {
  return D <= 64 ? 128 : D <= 128 ? 256 : 512;
}

// Orders a wave's LDS writes before its reads of other lanes' (the LDS itself takes them in order).
INTENT_DEVICE void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// log2|scale|, bounded so that sums of exp2(t - M), 2^(100 + kRise) at most, stay finite beside tokens of zeros.
template <bool kBf16>
INTENT_DEVICE float scale_exponent(float v) {
  return fmaxf(__builtin_amdgcn_logf(fabsf(v)), kLift<kBf16> - 100.0f);
}

// Where one query row of a tile (column r of S^T) stands: its position and the tokens lo <= t < hi that it sees.
struct RowView {
  int lo, hi, p;
};
INTENT_DEVICE RowView row_view(const AttnArgs& a, const Span& w, int r) {
  const int p = w.q.kv - w.q.count + (int)((uint32_t)(w.row0 + min(r, w.rows - 1)) / (uint32_t)a.group);
  return {first_seen(a, p), end_seen(a, p, w.q), p};
}

INTENT_DEVICE const uint16_t* q_row(const AttnArgs& a, const Span& w, int head, int r) {
  const int row = w.row0 + min(r, w.rows - 1), token = (int)((uint32_t)row / (uint32_t)a.group);
  return a.q + (int64_t)(w.q.start + token) * a.q_ld + (int64_t)(head * a.group + row - token * a.group) * a.D;
}
INTENT_DEVICE uint16_t* out_row(const AttnArgs& a, const Span& w, int head, int r) {
  const int row = w.row0 + r, token = (int)((uint32_t)row / (uint32_t)a.group);
  return a.out + (int64_t)(w.q.start + token) * a.out_ld + (int64_t)(head * a.group + row - token * a.group) * a.D;
}

// Queries with the sign of the scale, so that the kernels scale by its size and may take maxima first.
INTENT_DEVICE u32x4 signed_query(const AttnArgs& a, u32x4 v) {
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  return u32x4{v[0] ^ flip, v[1] ^ flip, v[2] ^ flip, v[3] ^ flip};
}

// The slope of a query row's head in base 2.
INTENT_DEVICE float slope_of(const AttnArgs& a, const Span& w, int head, int r) {
  if (a.slopes == nullptr) return 0.f;
  const int row = w.row0 + min(r, w.rows - 1);
  return a.slopes[head * a.group + (int)((uint32_t)row % (uint32_t)a.group)] * 1.44269504088896340736f;
}

// Queries of bf16 for products in f16 (a cache of 4 bits): a row is taken times a power of two that brings its
// largest element to 2^14 .. 2^15, so that elements down to 2^-28 of that are exact and smaller ones are 2^-39 of
// it off at most. `high`: the row's largest element's bits without its sign. An infinity or NaN stays one.
INTENT_DEVICE int query_exponent(uint32_t high) { return min(268 - (int)(high >> 7), 253); }  // biased
INTENT_DEVICE u32x4 query_f16(u32x4 v, int exponent) {
  const float by = bit_cast<float>((uint32_t)exponent << 23);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    v[e] = pack2<false>(bit_cast<float>(v[e] << 16) * by, bit_cast<float>(v[e] & 0xffff0000u) * by);
  return v;
}
INTENT_DEVICE uint32_t magnitude(u32x4 v) {
  uint32_t high = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) high = max(high, max(v[e] & 0x7fffu, v[e] >> 16 & 0x7fffu));
  return high;
}

// The size of the scale; instead of zero the smallest f32, which moves no finite score by more than 2^-20 and
// leaves a masked one at -inf.
INTENT_DEVICE float scale_of(const AttnArgs& a) { return fmaxf(fabsf(a.scale_log2), 0x1p-149f); }

// The scale of a row that query_f16 took times 2^(exponent - 127); nor is this ever zero.
INTENT_DEVICE float scale_behind(float scale, int exponent) {
  return fmaxf(scale * bit_cast<float>((uint32_t)(254 - exponent) << 23), 0x1p-149f);
}

INTENT_DEVICE float max_across16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return fmaxf(bit_cast<float>(r[0]), bit_cast<float>(r[1]));
}
INTENT_DEVICE float max_across32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return fmaxf(bit_cast<float>(r[0]), bit_cast<float>(r[1]));
}
INTENT_DEVICE float sum_across16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return bit_cast<float>(r[0]) + bit_cast<float>(r[1]);
}
INTENT_DEVICE float sum_across32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(v), bit_cast<uint32_t>(v), false, false);
  return bit_cast<float>(r[0]) + bit_cast<float>(r[1]);
}

// Eight codes of 4 bits as eight f16: 1024 + code and 1024 + 16 code come out of one bitwise operation each, less
// their 1024 (exact), times the scale plus the lowest value (one rounding). The constants that an operation takes
// two of are kept in vector registers.
struct Codes4 {
  uint32_t magic;
  f16x2 minus;
  INTENT_DEVICE Codes4() {
    magic = 0x64006400u;
    uint32_t m = 0xd400d400u;  // -64
    asm("" : "+v"(magic), "+v"(m));
    minus = bit_cast<f16x2>(m);
  }
  INTENT_DEVICE u32x4 widen(uint32_t word, uint32_t pair) const {
    const f16x2 h = bit_cast<f16x2>(pair), s = splat2(h[0]), m = splat2(h[1]);
    const uint32_t rest = word >> 8;
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t from = e < 2 ? word : rest;
      f16x2 code;
      if (e % 2 == 0) code = bit_cast<f16x2>(bfi(0x000f000fu, from, magic)) - splat2((f16)1024.f);
      else code = __builtin_elementwise_fma(bit_cast<f16x2>(bfi(0x00f000f0u, from, magic)), splat2((f16)0.0625f), minus);
      r[e] = bit_cast<uint32_t>(__builtin_elementwise_fma(code, s, m));
    }
    return r;
  }
};

// The forms of a row's scores, each in kernels of its own (kForms; a prefix alone runs among the sloped ones):
//   capped: cap tanh(x / cap) = cap - 2 cap r, r = 1 / (exp(2 x / cap) + 1): a product, an exponential, a sum and a
//           reciprocal. The softmax does not see the cap that is added to all of them, so a score becomes -r, and 2 cap
//           log2(e) brings it to base 2 in the exponent's own multiplication;
//   sloped: scores get their distance, slope |p - t|, in base 2: with all tokens at or before the row it is linear in
//           t, one operation, and the scale's product adds it.
// Written as branches of one kernel they cost the tiles of a prompt 10 to 20% by spilled registers.
template <int kCache, int kForms, int N, int kElements>
struct Scores {
  static constexpr bool kFp8 = kCache == kCacheFp8, kCap = (kForms & kCapped) != 0, kSlope = (kForms & kSloped) != 0;
  // whether they are in base 2 before the softmax takes its maximum
  static constexpr bool kScaled = kFp8 || kSlope;
  float in, out;  // capped: what a score is multiplied by before and behind the reciprocal
  float slope;
  int position;  // less the lane's first token: distances are exact below 2^24 tokens, wherever they lie

  INTENT_DEVICE void begin(const AttnArgs& a, float scale, float slope_log2, int p) {
    in = kCap ? fminf(kFp8 ? cap_rate(a) : scale * cap_rate(a), 0x1.fffffep127f) : scale;  // 0 times it stays 0
    out = kCap ? 2.0f * a.cap_log2 : scale;
    slope = slope_log2, position = p;
  }
  // s: element (u, r) of token t + token(u, r), of which `last` is the greatest; the rows stand at `top` and behind.
  // k_mul: scales of the keys, with the scores' own.
  template <typename S, typename Token, typename KMul>
  INTENT_DEVICE void apply(S (&s)[N], int t, int last, int top, Token token, KMul k_mul) const {
    if constexpr (kFp8 && !(kSlope && !kCap)) {
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int r = 0; r < kElements; ++r) s[u][r] *= k_mul(u, r);
    }
    if constexpr (kCap) {
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int r = 0; r < kElements; ++r) {
          s[u][r] = -__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[u][r] * in) + 1.0f);
          if constexpr (kFp8 && !kSlope) s[u][r] *= out;
        }
    }
    if constexpr (kSlope) {
      const float ahead = (float)(t - position);
      auto add = [&](int u, int r, float bias) {
        s[u][r] = __builtin_fmaf(s[u][r], kFp8 && !kCap ? k_mul(u, r) : out, bias);
      };
      if (t + last <= top) {
        const float first = slope * ahead;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int r = 0; r < kElements; ++r) add(u, r, __builtin_fmaf(slope, (float)token(u, r), first));
      } else {
        rarely();
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int r = 0; r < kElements; ++r) add(u, r, -slope * fabsf(ahead + (float)token(u, r)));
      }
    }
  }
};

// ---- few rows: 16 * MT of them, the tokens over the waves -----------------------------------------

// A wave takes 32 tokens of each 128: keys straight into the first product's left operand (a lane holds 8
// or 16 of a token's D), values through its own LDS rows; no barrier until the four waves' results are
// joined. Keys and values of its next 32 tokens are under way during the softmax and the second product.
//
// Bound by the reads of the cache: with 16 rows of heads of 128 three workgroups to a CU keep 12 waves of
// 16 KB (8 KB of 8-bit) under way. Four sequences of 60000 to 131000 tokens, 32 heads sharing 8 (1.42 GB):
// 242 us, 5.9 TB/s, where a large copy moves 5.1; 64 of 300 to 8191 tokens in 8 bits (645 MB): 124 us, 5.2
// TB/s, the lengths being uneven. One sequence of 4096 tokens (17 MB) is a chain of latencies, 7 us and 4
// for the join. The same in 4 bits: four (442 MB) 85 to 90 us, 5.0 TB/s, 64 (391 MB) 80 to 84 us, 4.8 TB/s, one 5.8 us.
// There 32 tokens are 300 vector instructions of a wave, two thirds of them to widen the codes, and the vector unit is
// busy for 56% of the time; four workgroups to a CU or three, and loads by 64-bit addresses or by buffers, make no
// difference to the long ones.
//
// Waves to a SIMD are what the registers hold. Rows of 4 bits leave more of them, slopes take some back (48 rows, 64
// sequences of 300 to 8191 tokens on eight heads: of 64 148 us with two waves, 110 with three; of 128 246 with one,
// 182 with two; 16 rows of 256, on four heads: 170 with one, 109 with two).
constexpr int rows_waves(int cache, int forms, int D, int mt) {
  if (cache == kCacheInt4) {
    const int spare = (forms & kSloped) != 0;
    if (D > 128) return 2;
    if (mt == 1) return 4;
    if (mt * D <= 192) return mt * D <= 128 ? 3 : 3 - spare;
    return mt * D > 384 ? 1 : D == 96 && mt == 4 ? 2 - spare : 2;
  }
  return D > 128 ? 1 : mt * D <= 128 ? 3 : mt * D <= 256 ? 2 : 1;
}

// Its LDS: the waves' values, then the joining buffer in their place.
template <bool kFp8, int D>
struct RowsShared {
  static constexpr int OB = D + 4;  // floats of a row in the joining buffer
  static constexpr int kValues = 4 * 32 * row_bytes<D>(), kJoin = 4 * 16 * OB * 4;
  __attribute__((aligned(16))) char lds[kValues > kJoin ? kValues : kJoin];
  __attribute__((aligned(16))) float scales[kFp8 ? 4 : 1][3][32];
  float stats[4][16][2];
};

template <bool kBf16, int kCache, int kForms, int D, int MT>
INTENT_DEVICE void attend_rows(const AttnArgs& a, int block, RowsShared<kCache == kCacheFp8, D>& shared) {
  constexpr bool kFp8 = kCache == kCacheFp8, kInt4 = kCache == kCacheInt4;
  constexpr bool kMath = kBf16 && !kInt4;              // products in bf16
  constexpr bool kBiased = kForms != kPlain;
  using Form = Scores<kCache, kForms, 2, 4>;
  constexpr bool kScaled = kFp8 || Form::kScaled;      // scores are scaled before the softmax
  constexpr int KS = D / 32, DT = D / 16, RB = row_bytes<D>();
  // elements of a lane's load of a token's row: 16 bytes of them if the row's quarter holds as many
  constexpr int ELEMS = kInt4 ? (D % 128 == 0 ? 32 : D % 64 == 0 ? 16 : 8) : kFp8 && D % 64 == 0 ? 16 : 8;
  constexpr int LOADS = D / 4 / ELEMS, CHUNKS = ELEMS / 8;  // loads, and 16 bytes of 16-bit elements of one
  constexpr int kRow = cached_bytes<kCache, D>(), kParams = cached_params<kCache, D>();
  constexpr int kLoad = kRow / 4 / LOADS;              // bytes of a load
  constexpr int OB = RowsShared<kFp8, D>::OB;
  auto& lds = shared.lds;
  auto& scales = shared.scales;
  auto& stats = shared.stats;

  const int head = block % a.HK;
  Span w;
  if (!find_span<kBiased>(a, 16 * MT, 7, block / a.HK, false, w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, g = lane >> 4;

  // element index of load i of lane group g in a token's row
  auto at = [&](int i) { return i * 4 * ELEMS + g * ELEMS; };
  u32x4 q[MT][KS];
  RowView view[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    view[m] = row_view(a, w, m * 16 + col);
    const uint16_t* row = q_row(a, w, head, m * 16 + col);
#pragma unroll
    for (int i = 0; i < KS; ++i)
      q[m][i] = signed_query(a, load16(row + at(i / CHUNKS) + i % CHUNKS * 8));
  }
  // the tokens that some row sees, and those that all rows see
  const RowView top = row_view(a, w, 0), bottom = row_view(a, w, w.rows - 1);
  const int some_lo = top.lo, some_hi = bottom.hi, all_lo = bottom.lo, all_hi = top.hi;
  const float scale = scale_of(a);
  float row_scale[MT];
  Form forms[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    row_scale[m] = scale;
    if constexpr (kBf16 && kInt4) {
      uint32_t high = 0;
#pragma unroll
      for (int i = 0; i < KS; ++i) high = max(high, magnitude(q[m][i]));
      // as floats: integers below 2^15 are exact
      const int exponent = query_exponent((uint32_t)max_across32(max_across16((float)high)));
#pragma unroll
      for (int i = 0; i < KS; ++i) q[m][i] = query_f16(q[m][i], exponent);
      row_scale[m] = scale_behind(scale, exponent);
    }
    if constexpr (kBiased) {
      forms[m].begin(a, row_scale[m], Form::kSlope ? slope_of(a, w, head, m * 16 + col) : 0.f, view[m].p - g * 4);
      row_scale[m] = forms[m].out;
    }
  }

  f32x4 o[MT][DT];
  float ref[MT], total[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    ref[m] = -INFINITY, total[m] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  char* mine = lds + wave * 32 * RB;
  const Codes4 codes4;
  const int write_at = col * RB, swz = swizzle<RB, false>(col);
  // transposing reads: tokens 4 g .. 4 g + 3 of each 16, columns 16 d ..
  const int read_row = g * 4 + (col >> 2);
  const int read_at =
      wave * 32 * RB + read_row * RB + (((col >> 1 & 1) ^ swizzle<RB, false>(read_row)) << 4) + (col & 1) * 8;

  u32x4 kr[2][LOADS], vr[2][LOADS];
  uint32_t kg[2][LOADS], vg[2][LOADS];  // pairs of the codes' groups
  float ks[2], vs[2];
  // Pages of 16 tokens and more: each 16 tokens lie in one. The table's entries of this wave's next 32
  // times 32 tokens are kept one in each lane (a vector load every 32 times: scalar loads would make
  // every wait for LDS a wait for them) and clamped where they are used. Smaller pages: each lane looks
  // up its token's.
  const bool paged = a.page_shift >= 4;
  const uint32_t lane_at = col * kRow + g * kLoad;
  auto clamped = [&](int t) { return min(max(t, some_lo), max(some_hi - 1, 0)); };
  uint32_t entries = 0, next_entries = 0;
  auto batch = [&](int t) { return table_entry(a, w.s, clamped(t + (lane >> 1) * 128 + (lane & 1) * 16)); };
  auto issue = [&](int u, global_bytes k, global_bytes v, global_bytes kp, global_bytes vp) {
    auto codes = [](global_bytes from) {
      if constexpr (kLoad == 16) return load16(from);
      if constexpr (kLoad == 4) return u32x4{load4(from), 0u, 0u, 0u};
      const u32x2 two = load8(from);
      return u32x4{two[0], two[1], 0u, 0u};
    };
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      kr[u][i] = codes(k + i * 4 * kLoad);
      vr[u][i] = codes(v + i * 4 * kLoad);
      if constexpr (kInt4) kg[u][i] = load4(kp + at(i) / kGroup4 * 4), vg[u][i] = load4(vp + at(i) / kGroup4 * 4);
    }
    if constexpr (kFp8) ks[u] = load_float(kp), vs[u] = load_float(vp);
  };
  // 4 bits, in one page: buffer loads, whose base is scalar and whose lane offsets stay in two registers (with
  // addresses of 64 bits for each of the eight loads four waves to a SIMD spill them).
  const uint32_t pair_at = col * (4 * kParams) + g * ELEMS / kGroup4 * 4;
  auto issue4 = [&](u32x4(&codes)[LOADS], uint32_t(&pairs)[LOADS], global_bytes rows, global_bytes params) {
    const auto from = make_rsrc((const void*)rows), beside = make_rsrc((const void*)params);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if constexpr (kLoad == 16) {
        codes[i] = __builtin_amdgcn_raw_buffer_load_b128(from, lane_at, i * 4 * kLoad, 0);
      } else if constexpr (kLoad == 8) {
        const u32x2 two = __builtin_amdgcn_raw_buffer_load_b64(from, lane_at, i * 4 * kLoad, 0);
        codes[i] = u32x4{two[0], two[1], 0u, 0u};
      } else {
        codes[i] = u32x4{(uint32_t)__builtin_amdgcn_raw_buffer_load_b32(from, lane_at, i * 4 * kLoad, 0), 0u, 0u, 0u};
      }
      pairs[i] = __builtin_amdgcn_raw_buffer_load_b32(beside, pair_at, i * (ELEMS / 2), 0);
    }
  };
  int place = 0;  // of the entries of the tokens to load next
  // Tokens that no row sees are loaded too (a page that is there, whatever it holds): their scores are
  // masked, their values set to zero when they are stored.
  auto load_rows = [&](int t) {
    if (paged) {
      if (place == 64) entries = next_entries, next_entries = batch(t + 32 * 128), place = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t page = page_named(a, (uint32_t)lane_value((int)entries, place + u));
        const int t16 = t + 16 * u;
        if constexpr (kInt4) {
          issue4(kr[u], kg[u], cached_rows<kRow>(a, a.k_cache, page, a.k_step, head, t16),
                 cached_scales<kParams>(a, a.k_scales, page, a.ks_step, head, t16));
          issue4(vr[u], vg[u], cached_rows<kRow>(a, a.v_cache, page, a.v_step, head, t16),
                 cached_scales<kParams>(a, a.v_scales, page, a.vs_step, head, t16));
          continue;
        }
        issue(u, cached_rows<kRow>(a, a.k_cache, page, a.k_step, head, t16) + lane_at,
              cached_rows<kRow>(a, a.v_cache, page, a.v_step, head, t16) + lane_at,
              cached_scales<kParams>(a, a.k_scales, page, a.ks_step, head, t16) + col * (4 * kParams),
              cached_scales<kParams>(a, a.v_scales, page, a.vs_step, head, t16) + col * (4 * kParams));
      }
      place += 2;
    } else {
      rarely();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int tk = t + 16 * u + col;
        const uint32_t page = page_named(a, table_entry(a, w.s, clamped(tk)));
        issue(u, cached_rows<kRow>(a, a.k_cache, page, a.k_step, head, tk) + g * kLoad,
              cached_rows<kRow>(a, a.v_cache, page, a.v_step, head, tk) + g * kLoad,
              cached_scales<kParams>(a, a.k_scales, page, a.ks_step, head, tk),
              cached_scales<kParams>(a, a.v_scales, page, a.vs_step, head, tk));
        if constexpr (kInt4) __builtin_amdgcn_sched_barrier(0);  // the addresses of one of them at a time
      }
    }
  };

  // whether rows of this tile see different ones of the tokens t ..
  auto apart = [&](int t) { return (some_lo != all_lo || some_hi != all_hi) && (t < all_lo || t + 32 > all_hi); };
  bool found = false;
  int t = w.begin + wave * 32;
  if (t < w.end) {
    if (paged) entries = batch(t), next_entries = batch(t + 32 * 128);
    load_rows(t);
  }
  for (; t < w.end; t += 128) {
    // values and scales of these tokens to LDS, the scores' operands from the registers
    const bool masked = t < all_lo || t + 32 > all_hi;
    if (t < some_lo || t + 32 > some_hi) {
      rarely();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int tk = t + 16 * u + col;
        if (tk < some_lo || tk >= some_hi) {
          vs[u] = 0.f;
#pragma unroll
          for (int i = 0; i < LOADS; ++i) vr[u][i] = u32x4{0u, 0u, 0u, 0u}, vg[u][i] = 0u;
        }
      }
    }
    if (!kInt4 && apart(t)) {
      rarely();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) vr[u][i] = only_finite<kBf16, kFp8>(vr[u][i], found);
      if constexpr (kFp8) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool good = fabsf(vs[u]) < INFINITY;
          found = found || !good;
          vs[u] = good ? vs[u] : 0.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        char* row = mine + u * 16 * RB + write_at;
        const int chunk = at(i) / 8;
        if constexpr (kInt4) {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c)
            *(u32x4*)(row + (((chunk + c) ^ swz) << 4)) = codes4.widen(vr[u][i][c], vg[u][i]);
        } else if constexpr (kFp8) {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c)
            *(u32x4*)(row + (((chunk + c) ^ swz) << 4)) = widen_codes<kBf16>(vr[u][i][2 * c], vr[u][i][2 * c + 1]);
        } else {
          *(u32x4*)(row + ((chunk ^ swz) << 4)) = vr[u][i];
        }
      }
      if constexpr (kFp8) {
        if (g == 0) {
          scales[wave][0][u * 16 + col] = ks[u] * scale;
          scales[wave][1][u * 16 + col] = vs[u];
          scales[wave][2][u * 16 + col] = scale_exponent<kMath>(vs[u]);
        }
      }
    }
    if (kInt4 && apart(t)) {  // what is not finite taken out again, by the lane that wrote it
      rarely();
#pragma unroll 1
      for (int i = 0; i < 2 * LOADS * CHUNKS; ++i) {
        const int chunk = at(i % (LOADS * CHUNKS) / CHUNKS) / 8 + i % CHUNKS;
        u32x4* to = (u32x4*)(mine + i / (LOADS * CHUNKS) * 16 * RB + write_at + ((chunk ^ swz) << 4));
        *to = only_finite<false, false>(*to, found);
      }
    }
    wave_lds_order();
    f32x4 s[MT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m) s[m][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        u32x4 k;
        const int l = i / CHUNKS, c = i % CHUNKS;
        if constexpr (kInt4) k = codes4.widen(kr[u][l][c], kg[u][l]);
        else if constexpr (kFp8) k = widen_codes<kBf16>(kr[u][l][2 * c], kr[u][l][2 * c + 1]);
        else k = kr[u][i];
#pragma unroll
        for (int m = 0; m < MT; ++m) s[m][u] = mfma16<kMath>(k, q[m][i], s[m][u]);
      }
    }
    const int now = t;
    if (now + 128 < w.end) load_rows(now + 128);
    u32x4 p[MT];
    f32x4 k_mul[2], v_mul[2], v_exp[2];
    if constexpr (kFp8) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        k_mul[u] = *(const f32x4*)&scales[wave][0][u * 16 + g * 4];
        v_mul[u] = *(const f32x4*)&scales[wave][1][u * 16 + g * 4];
        v_exp[u] = *(const f32x4*)&scales[wave][2][u * 16 + g * 4];
        if constexpr (!kBiased) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[m][u][r] *= k_mul[u][r];
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (kBiased) {
        // the branch, always taken, keeps the forms apart from the products: without it 16 rows of heads of 256 over
        // 32 caches of 2000 to 8000 tokens take 187 us, with it 174
        if (!Form::kCap || a.cap_log2 != 0.f)
          forms[m].apply(s[m], now, 31, top.p, [](int u, int r) { return 16 * u + r; },
                       [&](int u, int r) { return k_mul[u][r]; });
      }
      // the highest score, times the value's scale; s is a score or, scaled already, its t
      float high = -INFINITY;
      if (masked) {
        rarely();
        const int lo = view[m].lo - now - g * 4, hi = view[m].hi - now - g * 4;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool seen = 16 * u + r >= lo && 16 * u + r < hi;
            s[m][u][r] = seen ? s[m][u][r] : -INFINITY;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) high = fmaxf(high, kFp8 ? s[m][u][r] + v_exp[u][r] : s[m][u][r]);
      high = max_across32(max_across16(high));
      if constexpr (!kScaled) high *= row_scale[m];
      if (__any(high > ref[m] + kRise)) {
        const float next = fmaxf(ref[m], high);
        const float keep = __builtin_amdgcn_exp2f(ref[m] - (next == -INFINITY ? 0.f : next));
        ref[m] = next;
        total[m] *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[m][d] *= keep;
      }
      const float base = (ref[m] == -INFINITY ? 0.f : ref[m]) - kLift<kMath>;
      float wt[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(kScaled ? s[m][u][r] - base
                                                         : __builtin_fmaf(s[m][u][r], row_scale[m], -base));
          total[m] += e;
          wt[u][r] = kFp8 ? e * v_mul[u][r] : e;
        }
      }
      p[m] = u32x4{pack2<kMath>(wt[0][0], wt[0][1]), pack2<kMath>(wt[0][2], wt[0][3]), pack2<kMath>(wt[1][0], wt[1][1]),
                   pack2<kMath>(wt[1][2], wt[1][3])};
    }
    // V^T: tokens 4 g .. of the first 16, then of the second
    auto value = [&](int d) {
      const char* from = lds + (read_at ^ (d * 32));
      const u32x2 lo = read_transposed(from), hi = read_transposed(from + 16 * RB);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const u32x4 v = value(d);
#pragma unroll
      for (int m = 0; m < MT; ++m) o[m][d] = mfma16<kMath>(v, p[m], o[m][d]);
    }
    wave_lds_order();
  }
  if (__any(found)) {  // values left out of the products above
    for (t = w.begin + wave * 32; t < w.end; t += 128) {
      for (int tk = max(t, some_lo); apart(t) && tk < min(t + 32, some_hi); ++tk) {
        const int page = page_of(a, w.s, tk);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = cached_value<kBf16, kCache, D>(a, page, head, tk, d * 16 + g * 4 + r);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              if (tk >= view[m].lo && tk < view[m].hi && !(fabsf(v) < INFINITY)) o[m][d][r] += v;
          }
        }
      }
    }
  }

  // join the four waves, 16 rows at a time
  float* rows = (float*)lds;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m * 16 >= w.rows) break;
    __syncthreads();
    const float sum = sum_across32(sum_across16(total[m]));
    if (g == 0) stats[wave][col][0] = ref[m], stats[wave][col][1] = sum;
#pragma unroll
    for (int d = 0; d < DT; ++d) *(f32x4*)&rows[(wave * 16 + col) * OB + d * 16 + g * 4] = o[m][d];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
      const int r = i / (D / 4), d = i % (D / 4) * 4, row = m * 16 + r;
      if (row >= w.rows) break;
      float high = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) high = fmaxf(high, stats[k][r][0]);
      const float base = high == -INFINITY ? 0.f : high;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
      float all = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float keep = __builtin_amdgcn_exp2f(stats[k][r][0] - base);
        all += keep * stats[k][r][1];
        acc += keep * *(const f32x4*)&rows[(k * 16 + r) * OB + d];
      }
      if (w.splits == 1) {
        const RowView rv = row_view(a, w, row);
        const float inv = rv.hi > rv.lo ? 1.0f / all : 0.f;
        *(u32x2*)(out_row(a, w, head, row) + d) =
            u32x2{pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv)};
      } else {
        const int64_t to = ((int64_t)w.slot * a.HK + head) * (16 * MT) + row;
        *(f32x4*)(a.partial + to * D + d) = acc;
        if (d == 0) *(f32x2*)(a.partial_stats + to * 2) = f32x2{high, all};
      }
    }
  }
}

template <bool kBf16, int kCache, int kForms, int D, int MT>
__global__ __launch_bounds__(256, rows_waves(kCache, kForms, D, MT)) void attn_rows_kernel(const AttnArgs a) {
  __shared__ RowsShared<kCache == kCacheFp8, D> shared;
  attend_rows<kBf16, kCache, kForms, D, MT>(a, (int)blockIdx.x, shared);
}

// ---- many rows: 128 or 256, 32 to a wave, all of them over the same tokens ----------------------------

// 64 tokens of keys and values in LDS at a time, in two buffers: the next ones are loaded into
// registers while these are worked on and stored to the other buffer behind them, so one barrier for
// each 64 tokens.
//
// The matrix unit and the softmax have about the same to do for 32 rows and 64 tokens of heads of 128: 32
// MFMAs of 32 cycles, and 180 vector instructions, of which 32 exponentials at a quarter of the rate. So the
// next tokens' products with the queries are issued between the exponentials of these, which needs the
// scores of both: heads of 64, whose products are half as long, do better with three waves to a SIMD and
// without (1925 tokens in 24 sequences over a window of 1000: 24 us against 29). Prefill of 4096 tokens,
// 32 heads sharing 8 (137 GFLOP): 152 to 161 us, 850 to 900 TFLOP/s, where the library's product of
// 8192^3 reaches 1200; 3696 tokens in two chunks over 10000 to 18000 in 8 bits 1115 to 1170 us, 780 to 820
// TFLOP/s. What is left: with the loads of the cache taken away it takes 140 us, with the vector work
// 117, with the products 111; each wave's own chain, not one unit, sets the time. 64 rows to a wave read LDS
// half as often, but one wave to a SIMD and 1500 copies between the two halves of its registers take 215 us.
//
// Capped scores (4096 tokens of which the first 1000 are a prefix, 141 GFLOP): 208 to 237 us; an exponential and a
// reciprocal more for each score cost what they take to issue, 43 cycles, also if they stand between the products.
// 4 bits (1834 + 1862 tokens over 9000 to 16000 others, 911 GFLOP): 1010 to 1050 us, 870 to 900 TFLOP/s. The codes are
// widened on their way to LDS, 16 bytes of a token to a lane (heads of 64: 8), between a load's arrival and the barrier:
// keys by four of eight waves and values by the other four, 3% less than both by the first four. Their stores meet four
// to a bank; to turn them apart costs more registers and selects than it gains (1220 against 1195 us).
template <bool kFp8, int D>
struct TileShared {
  __attribute__((aligned(16))) char lds[2][2][64 * row_bytes<D>()];
  __attribute__((aligned(16))) float scales[kFp8 ? 2 : 1][3][64];
  int left_out;  // values that are not finite were left out of a product
};

template <bool kBf16, int kCache, int kForms, int D, int WAVES>
INTENT_DEVICE void attend_tile(const AttnArgs& a, int block, TileShared<kCache == kCacheFp8, D>& shared) {
  constexpr bool kFp8 = kCache == kCacheFp8, kInt4 = kCache == kCacheInt4;
  constexpr bool kMath = kBf16 && !kInt4;             // products in bf16
  constexpr bool kBiased = kForms != kPlain;
  using Form = Scores<kCache, kForms, 2, 16>;
  constexpr bool kScaled = kFp8 || Form::kScaled;     // scores are scaled before the softmax
  constexpr int KS = D / 16, DT = D / 32, RB = row_bytes<D>();
  constexpr int kRow = cached_bytes<kCache, D>(), kParams = cached_params<kCache, D>();
  constexpr int kLoad = kInt4 && D == 64 ? 8 : 16;    // bytes of a lane's load: rows of 32 bytes take four lanes too
  constexpr int CHUNKS = kRow / kLoad, WORDS = kLoad / 4;  // loads of a token's row
  // lanes that take one (a power of two)
  constexpr int SPREAD = kInt4 ? RB / kLoad / 4 : kFp8 ? RB / 32 : RB / 16;
  constexpr int EACH = 64 / SPREAD;                   // tokens that a wave loads at once
  constexpr int STEP = EACH * WAVES;                  // and the workgroup
  constexpr int LOADS = STEP >= 64 ? 1 : 64 / STEP, ROWS = 32 * WAVES;
  // Whether the scores of the next 64 tokens are computed during the softmax of these.
  constexpr bool kAhead = D > 64;
  auto& lds = shared.lds;
  auto& scales = shared.scales;
  int& left_out = shared.left_out;

  const int head = block % a.HK;
  Span w;
  if (!find_span<kBiased>(a, ROWS, 6, block / a.HK, false, w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, h = lane >> 5;
  const int r0 = wave * 32;

  u32x4 q[KS];
  const RowView view = row_view(a, w, r0 + col);
  {
    const uint16_t* row = q_row(a, w, head, r0 + col);
#pragma unroll
    for (int i = 0; i < KS; ++i) q[i] = signed_query(a, load16(row + i * 16 + h * 8));
  }
  const RowView first = row_view(a, w, 0), last = row_view(a, w, w.rows - 1);
  const int some_lo = first.lo, some_hi = last.hi, all_lo = last.lo, all_hi = first.hi;
  const RowView top = row_view(a, w, r0), bottom = row_view(a, w, r0 + 31);  // of this wave
  const bool idle = r0 >= w.rows;
  const float scale = scale_of(a);
  float row_scale = scale;
  Form forms;
  if constexpr (kBf16 && kInt4) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < KS; ++i) most = max(most, magnitude(q[i]));
    const int exponent = query_exponent((uint32_t)max_across32((float)most));  // as floats: exact
#pragma unroll
    for (int i = 0; i < KS; ++i) q[i] = query_f16(q[i], exponent);
    row_scale = scale_behind(scale, exponent);
  }
  if constexpr (kBiased) {
    forms.begin(a, row_scale, Form::kSlope ? slope_of(a, w, head, r0 + col) : 0.f, view.p - h * 4);
    row_scale = forms.out;
  }

  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float ref = -INFINITY, total = 0.f;

  // 4 bits and eight waves: 64 tokens' rows are one load of four waves, so half of them take the keys and half the
  // values (each widens half as much before the barrier).
  constexpr bool kHalves = kInt4 && STEP >= 128;
  const bool takes_keys = !kHalves || wave < WAVES / 2, takes_values = !kHalves || wave >= WAVES / 2;
  const Codes4 codes4;
  const int wave_token = wave * EACH & 63;  // where there are more waves than tokens, those behind idle
  const int load_token = wave_token + lane / SPREAD, load_chunk = lane % SPREAD;
  const bool loads = load_chunk < CHUNKS && (kHalves || wave * EACH < 64);
  u32x4 kr[LOADS], other[LOADS];
  uint32_t kg[LOADS], other_pairs[LOADS];  // pairs of the codes' groups
  u32x4(&vr)[LOADS] = kHalves ? kr : other;
  uint32_t(&vg)[LOADS] = kHalves ? kg : other_pairs;
  float ks = 0.f, vs = 0.f;
  // Pages of EACH tokens and more (16 at most): each load's tokens lie in one, whose id is a scalar.
  const bool paged = (1 << a.page_shift) >= EACH;
  const int chunk = load_chunk < CHUNKS ? load_chunk : 0;
  const int group = chunk * (kLoad / 4) * 8 / kGroup4;
  const uint32_t lane_at = (lane / SPREAD) * kRow + chunk * kLoad, pair_at = (lane / SPREAD) * (4 * kParams) + group * 4;
  // The table's entries of the next `span` times 64 tokens, one in each lane, in two batches (as above).
  const bool one_page = a.page_shift >= 6;  // the 64 tokens in one page
  constexpr int kLoadsLog = LOADS == 1 ? 0 : LOADS == 2 ? 1 : LOADS == 4 ? 2 : 3;
  const int pieces_log = one_page ? 0 : kLoadsLog, span_log = 6 - pieces_log, span = 1 << span_log;
  auto clamped = [&](int t) __attribute__((always_inline)) { return min(max(t, some_lo), max(some_hi - 1, 0)); };
  auto batch = [&](int t) __attribute__((always_inline)) {
    const int piece = lane & ((1 << pieces_log) - 1);
    return table_entry(a, w.s, clamped(t + (lane >> pieces_log) * 64 + piece * STEP + wave_token));
  };
  uint32_t entries[2] = {0, 0};
  // of the i-th load of the tokens n * 64 behind w.begin
  auto entry = [&](int n, int i) __attribute__((always_inline)) {
    return (uint32_t)lane_value((int)(n >> span_log & 1 ? entries[1] : entries[0]),
                                ((n & (span - 1)) << pieces_log) + (one_page ? 0 : i));
  };
  // Tokens that no row sees are loaded too (a page that is there, whatever it holds): their scores are
  // masked, their values set to zero when they are stored.
  auto load = [&](u32x4(&fetched)[LOADS], uint32_t(&pairs)[LOADS], const void* cache, uint32_t step,
                  const float* params, uint32_t pair_step, int t) __attribute__((always_inline)) {
    auto codes = [](global_bytes at) {
      if constexpr (kLoad == 16) return load16(at);
      const u32x2 two = load8(at);
      return u32x4{two[0], two[1], 0u, 0u};
    };
    const int n = (t - w.begin) >> 6;
    if (one_page) {
      const uint32_t page = page_named(a, entry(n, 0));
      const global_bytes from = cached_rows<kRow>(a, cache, page, step, head, t + wave_token);
      const global_bytes beside = cached_scales<kParams>(a, params, page, pair_step, head, t + wave_token);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        fetched[i] = codes(from + i * (STEP * kRow) + lane_at);
        if constexpr (kInt4) pairs[i] = load4(beside + i * (STEP * 4 * kParams) + pair_at);
      }
    } else if (paged) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t page = page_named(a, entry(n, i));
        const int tk = t + i * STEP + wave_token;
        fetched[i] = codes(cached_rows<kRow>(a, cache, page, step, head, tk) + lane_at);
        if constexpr (kInt4) pairs[i] = load4(cached_scales<kParams>(a, params, page, pair_step, head, tk) + pair_at);
      }
    } else {
      rarely();
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int tk = t + i * STEP + load_token;
        const uint32_t page = page_named(a, table_entry(a, w.s, clamped(tk)));
        fetched[i] = codes(cached_rows<kRow>(a, cache, page, step, head, tk) + chunk * kLoad);
        if constexpr (kInt4) pairs[i] = load4(cached_scales<kParams>(a, params, page, pair_step, head, tk) + group * 4);
      }
    }
  };
  auto load_share = [&](int keys, int values) __attribute__((always_inline)) {
    load(kr, kg, takes_keys ? a.k_cache : a.v_cache, takes_keys ? a.k_step : a.v_step,
         takes_keys ? a.k_scales : a.v_scales, takes_keys ? a.ks_step : a.vs_step, takes_keys ? keys : values);
  };
  auto load_keys = [&](int t) __attribute__((always_inline)) {
    load(kr, kg, a.k_cache, a.k_step, a.k_scales, a.ks_step, t);
  };
  auto load_values = [&](int t) __attribute__((always_inline)) {
    load(vr, vg, a.v_cache, a.v_step, a.v_scales, a.vs_step, t);
    if constexpr (kFp8) {
      if (wave == 0) {
        const int tk = t + lane;
        const uint32_t page = page_named(a, table_entry(a, w.s, clamped(tk)));
        ks = load_float(cached_scales<1>(a, a.k_scales, page, a.ks_step, head, tk));
        vs = load_float(cached_scales<1>(a, a.v_scales, page, a.vs_step, head, tk));
      }
    }
  };
  auto store = [&](char* to, const u32x4(&from)[LOADS], const uint32_t(&pairs)[LOADS]) __attribute__((always_inline)) {
    if (!loads) return;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int tk = load_token + i * STEP, swz = swizzle<RB, true>(tk);
      char* row = to + tk * RB;
      if constexpr (kInt4) {
#pragma unroll
        for (int c = 0; c < WORDS; ++c)
          *(u32x4*)(row + ((load_chunk * WORDS + c ^ swz) << 4)) = codes4.widen(from[i][c], pairs[i]);
      } else if constexpr (kFp8) {
        *(u32x4*)(row + ((load_chunk * 2 ^ swz) << 4)) = widen_codes<kBf16>(from[i][0], from[i][1]);
        *(u32x4*)(row + (((load_chunk * 2 + 1) ^ swz) << 4)) = widen_codes<kBf16>(from[i][2], from[i][3]);
      } else {
        *(u32x4*)(row + ((load_chunk ^ swz) << 4)) = from[i];
      }
    }
  };
  // whether rows of this tile see different ones of the tokens t ..
  auto apart = [&](int t) __attribute__((always_inline)) {
    return (some_lo != all_lo || some_hi != all_hi) && (t < all_lo || t + 64 > all_hi);
  };
  auto store_values = [&](int buffer, int t) __attribute__((always_inline)) {
    if (t < some_lo || t + 64 > some_hi) {
      rarely();
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int tk = t + i * STEP + load_token;
        if (tk < some_lo || tk >= some_hi) vr[i] = u32x4{0u, 0u, 0u, 0u}, vg[i] = 0u;
      }
      if (t + lane < some_lo || t + lane >= some_hi) vs = 0.f;
    }
    if (!kInt4 && apart(t)) {
      rarely();
      bool found = false;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) vr[i] = only_finite<kBf16, kFp8>(vr[i], found);
      if constexpr (kFp8) {
        const bool good = fabsf(vs) < INFINITY;
        found = found || !good;
        vs = good ? vs : 0.f;
      }
      if (found) left_out = 1;
    }
    store(lds[buffer][1], vr, vg);
    if (kInt4 && apart(t) && loads) {  // what is not finite taken out again, by the lane that wrote it
      rarely();
      bool found = false;
#pragma unroll 1
      for (int i = 0; i < LOADS * WORDS; ++i) {
        const int tk = load_token + i / WORDS * STEP;
        u32x4* to = (u32x4*)(lds[buffer][1] + tk * RB + ((load_chunk * WORDS + i % WORDS ^ swizzle<RB, true>(tk)) << 4));
        *to = only_finite<false, false>(*to, found);
      }
      if (found) left_out = 1;
    }
    if constexpr (kFp8) {
      if (wave == 0) {
        scales[buffer][0][lane] = ks * scale;
        scales[buffer][1][lane] = vs;
        scales[buffer][2][lane] = scale_exponent<kMath>(vs);
      }
    }
  };

  const int k_at = col * RB + ((h ^ swizzle<RB, true>(col)) << 4);
  const int i16 = lane & 15, read_row = h * 4 + (i16 >> 2);
  const int v_chunk = (lane >> 4 & 1) * 2 + (i16 >> 1 & 1);
  const int v_at = read_row * RB + ((v_chunk ^ swizzle<RB, true>(read_row)) << 4) + (i16 & 1) * 8;

  auto scores = [&](int buffer, f32x16(&s)[2]) __attribute__((always_inline)) {
    const char* keys = lds[buffer][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = mfma32<kMath>(*(const u32x4*)(keys + u * 32 * RB + (k_at ^ (i * 32))), q[i], s[u]);
  };

  // kAhead: of tokens t, values (and scales) in buffer j, their scores in registers; of t + 64, keys in
  // buffer j ^ 1; values of t + 64 and keys of t + 128 under way. Else keys and values of t in buffer j,
  // those of t + 64 under way.
  if (threadIdx.x == 0) left_out = 0;
  __syncthreads();
  f32x16 s[2];
  if (w.begin < w.end) {
    if (paged) entries[0] = batch(w.begin), entries[1] = batch(w.begin + span * 64);
    if constexpr (kHalves) {
      load_share(w.begin, w.begin);
    } else {
      load_keys(w.begin);
      load_values(w.begin);
    }
    if constexpr (kAhead) {
      u32x4 second[LOADS];
      uint32_t second_pairs[LOADS];
      load(second, second_pairs, a.k_cache, a.k_step, a.k_scales, a.ks_step, w.begin + 64);
      if (takes_keys) store(lds[0][0], kr, kg);
      if (takes_values) store_values(0, w.begin);
      if (takes_keys) store(lds[1][0], second, second_pairs);
    } else {
      if (takes_keys) store(lds[0][0], kr, kg);
      if (takes_values) store_values(0, w.begin);
    }
  }
  __syncthreads();
  if constexpr (kAhead) {
    if (w.begin < w.end) scores(0, s);
    __syncthreads();  // the first keys are read: their buffer may be written
  }
  int j = 0;
  for (int t = w.begin; t < w.end; t += 64, j ^= 1) {
    const bool more = t + 64 < w.end;
    if (more) {
      if constexpr (kHalves) {
        load_share(t + (kAhead ? 128 : 64), t + 64);
      } else {
        load_values(t + 64);
        load_keys(t + (kAhead ? 128 : 64));
      }
      const int n = (t + 64 - w.begin) >> 6;
      if (paged && (n & (span - 1)) == span - 1) {  // past a batch: the one behind the other takes its place
        rarely();
        const uint32_t later = batch(t + 64 + (span + 1) * 64);
        if (n >> span_log & 1) entries[1] = later;
        else entries[0] = later;
      }
    }
    if (!idle) {
      if constexpr (!kAhead) scores(j, s);
      const char* values = lds[j][1];
      const bool masked = t < bottom.lo || t + 64 > top.hi;
      float high = -INFINITY;
      if constexpr (kFp8 && !kBiased) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 k_mul = *(const f32x4*)&scales[j][0][u * 32 + i * 8 + h * 4];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[u][i * 4 + r] *= k_mul[r];
          }
      }
      if constexpr (kBiased)
        forms.apply(s, t, 63, top.p, [](int u, int r) { return u * 32 + (r >> 2) * 8 + (r & 3); },
                    [&](int u, int r) { return scales[j][0][u * 32 + (r >> 2) * 8 + h * 4 + (r & 3)]; });
      if (masked) {
        rarely();
        const int lo = view.lo - t - h * 4, hi = view.hi - t - h * 4;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int tk = u * 32 + (r >> 2) * 8 + (r & 3);
            s[u][r] = tk >= lo && tk < hi ? s[u][r] : -INFINITY;
          }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 v_exp;
          if constexpr (kFp8) v_exp = *(const f32x4*)&scales[j][2][u * 32 + i * 8 + h * 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) high = fmaxf(high, kFp8 ? s[u][i * 4 + r] + v_exp[r] : s[u][i * 4 + r]);
        }
      if constexpr (!kScaled) high *= row_scale;
      high = max_across32(high);
      if (__any(high > ref + kRise)) {
        rarely();
        const float next = fmaxf(ref, high);
        const float keep = __builtin_amdgcn_exp2f(ref - (next == -INFINITY ? 0.f : next));
        ref = next;
        total *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= keep;
      }
      const float base = (ref == -INFINITY ? 0.f : ref) - kLift<kMath>;
      // Sixteen steps, each with the weights of two tokens, its part of the next tokens' products with the
      // queries (kAhead; of what lies in that buffer behind the last tokens, too: not used then) and, four
      // steps behind, of the products with these values, so that the matrix unit works through all of them.
      constexpr int S_ALL = 2 * KS, V_ALL = 4 * DT, K_AHEAD = 4, V_AHEAD = 2;
      f32x16 after[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) after[u][r] = 0.f;
      const char* keys = lds[j ^ 1][0];
      auto key = [&](int n) __attribute__((always_inline)) {
        return *(const u32x4*)(keys + (n & 1) * 32 * RB + (k_at ^ ((n >> 1) * 32)));
      };
      auto value = [&](int n) __attribute__((always_inline)) {
        const int m = n / DT, d = n % DT;
        // tokens 8 further: their swizzle differs in one bit
        const u32x2 lo = read_transposed(values + (v_at ^ (d * 64)) + m * 16 * RB);
        const u32x2 hi = read_transposed(values + (v_at ^ (d * 64) ^ 32) + (m * 16 + 8) * RB);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      };
      u32x4 p[4], kf[S_ALL], vf[V_ALL];
      if constexpr (kAhead) {
#pragma unroll
        for (int n = 0; n < K_AHEAD; ++n) kf[n] = key(n);
      }
      auto products = [&](int from, int to) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < V_ALL; ++n) {
          if (n < from || n >= to) continue;
          if (n + V_AHEAD < V_ALL) vf[n + V_AHEAD] = value(n + V_AHEAD);
          o[n % DT] = mfma32<kMath>(vf[n], p[n / DT], o[n % DT]);
        }
      };
      float sums[2] = {0.f, 0.f};
      f32x4 v_mul;
      auto step = [&](int i) __attribute__((always_inline)) {
        if constexpr (kAhead) {
#pragma unroll
          for (int n = i * S_ALL / 16; n < (i + 1) * S_ALL / 16; ++n) {
            if (n + K_AHEAD < S_ALL) kf[n + K_AHEAD] = key(n + K_AHEAD);
            after[n & 1] = mfma32<kMath>(kf[n], q[n >> 1], after[n & 1]);
          }
        }
        if (i == 3) {
#pragma unroll
          for (int n = 0; n < V_AHEAD; ++n) vf[n] = value(n);
        }
        if (i >= 4) products((i - 4) * DT / 4, (i - 3) * DT / 4);
        if constexpr (kFp8)
          if (i % 2 == 0) v_mul = *(const f32x4*)&scales[j][1][(i / 2 / 4) * 32 + (i / 2 % 4) * 8 + h * 4];
        float wt[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = s[i / 8][i % 8 * 2 + e];
          const float y = __builtin_amdgcn_exp2f(kScaled ? x - base : __builtin_fmaf(x, row_scale, -base));
          sums[e] += y;
          wt[e] = kFp8 ? y * v_mul[i % 2 * 2 + e] : y;
        }
        p[i / 4][i % 4] = pack2<kMath>(wt[0], wt[1]);
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int i = 0; i < 16; ++i) step(i);
      products(3 * DT, V_ALL);
      total += sums[0] + sums[1];
      if constexpr (kAhead) s[0] = after[0], s[1] = after[1];
    }
    if (more) {
      if (takes_values) store_values(j ^ 1, t + 64);
      if (takes_keys) store(lds[kAhead ? j : j ^ 1][0], kr, kg);
    }
    __syncthreads();
  }

  if (left_out != 0) {
    for (int t = w.begin; t < w.end; t += 64) {
      for (int tk = max(t, some_lo); apart(t) && tk < min(t + 64, some_hi); ++tk) {
        const int page = page_of(a, w.s, tk);
        const bool seen = tk >= view.lo && tk < view.hi;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float v = cached_value<kBf16, kCache, D>(a, page, head, tk, d * 32 + (r >> 2) * 8 + h * 4 + (r & 3));
            if (seen && !(fabsf(v) < INFINITY)) o[d][r] += v;
          }
        }
      }
    }
  }
  const int r = r0 + col;
  if (r >= w.rows) return;
  const float all = sum_across32(total);
  if (w.splits == 1) {
    const float inv = view.hi > view.lo ? 1.0f / all : 0.f;
    uint16_t* to = out_row(a, w, head, r);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(u32x2*)(to + d * 32 + i * 8 + h * 4) = u32x2{pack2<kBf16>(o[d][i * 4] * inv, o[d][i * 4 + 1] * inv),
                                                       pack2<kBf16>(o[d][i * 4 + 2] * inv, o[d][i * 4 + 3] * inv)};
  } else {
    const int64_t to = ((int64_t)w.slot * a.HK + head) * ROWS + r;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f32x4*)(a.partial + to * D + d * 32 + i * 8 + h * 4) =
            f32x4{o[d][i * 4], o[d][i * 4 + 1], o[d][i * 4 + 2], o[d][i * 4 + 3]};
    if (h == 0) *(f32x2*)(a.partial_stats + to * 2) = f32x2{ref, all};
  }
}

template <bool kBf16, int kCache, int kForms, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D == 64 ? 3 : D <= 128 ? 2 : 1) void attn_tile_kernel(const AttnArgs a) {
  __shared__ TileShared<kCache == kCacheFp8, D> shared;
  attend_tile<kBf16, kCache, kForms, D, WAVES>(a, (int)blockIdx.x, shared);
}

// Both lists of a mixture of heads of 64 in one launch, whose registers and LDS let three workgroups of either share a
// CU: tiles of 128 rows in the first `tiles` workgroups, sequences of up to 16 rows in the others. The two take the same
// LDS: side by side they are 53764 bytes with 8 bits, of which a CU holds two (six chunks of 300 to 700 tokens over 500
// to 3000, 16 heads on 8: 90 us, 74 so; 127 decoding sequences and a chunk of 600, 32 heads on 8: 122 and 100).
template <bool kBf16, int kCache, int kForms>
__global__ __launch_bounds__(256, 3) void attn_mixed_kernel(const AttnArgs a, const AttnArgs b, int tiles) {
  __shared__ union {
    TileShared<kCache == kCacheFp8, 64> tile;
    RowsShared<kCache == kCacheFp8, 64> rows;
  } shared;
  if ((int)blockIdx.x < tiles) attend_tile<kBf16, kCache, kForms, 64, 4>(a, (int)blockIdx.x, shared.tile);
  else attend_rows<kBf16, kCache, kForms, 64, 1>(b, (int)blockIdx.x - tiles, shared.rows);
}

// ---- the join of split tiles ---------------------------------------------------------------------

// out = sum_j w_j O_j / sum_j w_j l_j, w_j = exp2(M_j - max M), over the parts of a tile in a fixed order.
// Up to 16 parts, a row is D / 4 lanes of four columns, and a wave takes as many rows as it holds. More
// parts are dealt to the four waves of a workgroup (D / 64 columns a lane), whose sums are added in
// order; each works out the weights of 64 parts at a time, one in each lane, while its first parts are on
// their way. What the first list needs to be found comes before the struct, where the kernel has it in
// registers when it starts. A launch and a chain of four latencies: 4.2 to 4.8 us for one tile of 32 parts;
// one launch for the tiles of a mixture's two lists 7.2 us, where two took 11.4.
template <bool kBf16, bool kBiased, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(int items, int tile, int unit_log, const AttnJoin j) {
  constexpr int E = (D + 63) / 64, AHEAD = 8, FEW = 16;
  constexpr int LANES = D == 96 ? 32 : D / 4, TOGETHER = 64 / LANES;  // lanes of a row, rows of a wave
  typedef float part __attribute__((ext_vector_type(E)));
  __shared__ part sums[4][64];
  AttnArgs a = j.a;
  const int head = blockIdx.x % a.HK;
  int item = blockIdx.x / a.HK;
  if (item >= items) {
    item -= items, tile = j.tile[1], unit_log = j.unit_log[1];
    a.min_rows = j.min_rows, a.max_rows = j.max_rows, a.target = j.target, a.slots = j.slots;
    a.partial = j.partial, a.partial_stats = j.partial_stats;
  }
  Span w;
  if (!find_span<kBiased>(a, tile, unit_log, item, true, w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w.splits <= FEW) {
    const int c = lane % LANES * 4 < D ? lane % LANES * 4 : 0;
    for (int first = (blockIdx.y * 4 + wave) * TOGETHER; first < w.rows; first += gridDim.y * 4 * TOGETHER) {
      const int r = first + lane / LANES, row = min(r, w.rows - 1);
      auto at = [&](int j) { return ((int64_t)(w.slot + j) * a.HK + head) * tile + row; };
      f32x2 st[FEW];
      float high = -INFINITY;
#pragma unroll
      for (int j = 0; j < FEW; ++j) {
        st[j] = f32x2{-INFINITY, 0.f};
        if (j < w.splits) st[j] = *(const f32x2*)(a.partial_stats + at(j) * 2);
      }
#pragma unroll
      for (int j = 0; j < FEW; ++j) high = fmaxf(high, st[j][0]);
      const float base = high == -INFINITY ? 0.f : high;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
      float total = 0.f;
#pragma unroll
      for (int j0 = 0; j0 < FEW; j0 += 4) {
        if (j0 < w.splits) {
          f32x4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = *(const f32x4*)(a.partial + at(min(j0 + j, w.splits - 1)) * D + c);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float keep = __builtin_amdgcn_exp2f(st[j0 + j][0] - base);
            total += keep * st[j0 + j][1];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(keep, j0 + j < w.splits ? v[j][e] : 0.f, acc[e]);
          }
        }
      }
      const RowView rv = row_view(a, w, row);
      const float inv = rv.hi > rv.lo ? 1.0f / total : 0.f;
      if (r < w.rows && lane % LANES * 4 < D)
        *(u32x2*)(out_row(a, w, head, row) + c) =
            u32x2{pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv)};
    }
    return;
  }
  const bool mine = lane * E < D;
  const int d0 = mine ? lane * E : 0;
  for (int r = blockIdx.y; r < w.rows; r += gridDim.y) {
    auto at = [&](int j) { return ((int64_t)(w.slot + j) * a.HK + head) * tile + r; };
    auto load = [&](int j) { return *(const part*)(a.partial + at(min(j, w.splits - 1)) * D + d0); };
    part ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = load(wave + i * 4);
    f32x2 st = f32x2{-INFINITY, 0.f};
    if (lane < w.splits) st = *(const f32x2*)(a.partial_stats + at(lane) * 2);
    float high = st[0];
    for (int j = lane + 64; j < w.splits; j += 64) high = fmaxf(high, a.partial_stats[at(j) * 2]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) high = fmaxf(high, __shfl_xor(high, off));
    const float base = high == -INFINITY ? 0.f : high;
    part acc{};
    float total = 0.f;
    for (int j0 = 0; j0 < w.splits; j0 += 64) {
      if (j0 > 0) {
        st = f32x2{-INFINITY, 0.f};
        if (j0 + lane < w.splits) st = *(const f32x2*)(a.partial_stats + at(j0 + lane) * 2);
      }
      const float keep = __builtin_amdgcn_exp2f(st[0] - base);
      float all = keep * st[1];
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off);
      total += all;
      const int n = min(w.splits - j0, 64);
      auto add = [&](part v, int i) {
        const float k = bit_cast<float>(__builtin_amdgcn_readlane(bit_cast<int>(keep), i));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(k, v[e], acc[e]);
      };
      int i = wave;
      if (j0 == 0) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (wave + k * 4 < n) add(ahead[k], wave + k * 4);
        i += AHEAD * 4;
      }
      for (; i < n; i += 4) add(load(j0 + i), i);
    }
    __syncthreads();
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || !mine) continue;
    acc = sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
    const RowView rv = row_view(a, w, r);
    const float inv = rv.hi > rv.lo ? 1.0f / total : 0.f;
    uint16_t* to = out_row(a, w, head, r) + d0;
    if constexpr (E == 1) *to = (uint16_t)(pack2<kBf16>(acc[0] * inv, 0.f) & 0xffffu);
    else if constexpr (E == 2) *(uint32_t*)to = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
    else *(u32x2*)to = u32x2{pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv)};
  }
}

// ROWS up to 64: rows of the first kernel; 128 or 256: of the second's four or eight waves.
template <bool kBf16, int kCache, int kForms, int D, int ROWS>
int launch(const AttnArgs& a, int items, hipStream_t stream) {
  const unsigned groups = (unsigned)items * (unsigned)a.HK;
  constexpr bool kFew = ROWS <= 64;
  if constexpr (kFew)
    hipLaunchKernelGGL((attn_rows_kernel<kBf16, kCache, kForms, D, ROWS / 16>), dim3(groups), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attn_tile_kernel<kBf16, kCache, kForms, D, ROWS / 32>), dim3(groups), dim3(ROWS * 2), 0, stream,
                       a);
  static const KernelName name("attn_%s_kernel<%s%s%s, D %d, %d rows>", kFew ? "rows" : "tile", kBf16 ? "bf16" : "f16",
                               cache_name(kCache), form_name(kForms), D, ROWS);
  return launch_status(name.text);
}

template <bool kBf16, int kCache, int kForms, int D>
int launch_d(const AttnArgs& a, int items, int rows, hipStream_t stream) {
  if (rows == 16) return launch<kBf16, kCache, kForms, D, 16>(a, items, stream);
  if constexpr (D <= 128) {
    if (rows == 32) return launch<kBf16, kCache, kForms, D, 32>(a, items, stream);
    if (rows == 48) return launch<kBf16, kCache, kForms, D, 48>(a, items, stream);
    if (rows == 64) return launch<kBf16, kCache, kForms, D, 64>(a, items, stream);
    if (rows == 256) return launch<kBf16, kCache, kForms, D, 256>(a, items, stream);
  }
  return launch<kBf16, kCache, kForms, D, 128>(a, items, stream);
}

template <bool kBf16, int kCache, int kForms = kPlain>
int launch_any(const AttnArgs& a, int items, int rows, const AttnArgs* few, int few_items, hipStream_t stream) {
  if (few != nullptr) {
    const int tiles = items * a.HK;
    hipLaunchKernelGGL((attn_mixed_kernel<kBf16, kCache, kForms>), dim3((unsigned)tiles + (unsigned)few_items * a.HK),
                       dim3(256), 0, stream, a, *few, tiles);
    static const KernelName name("attn_mixed_kernel<%s%s%s>", kBf16 ? "bf16" : "f16", cache_name(kCache),
                                 form_name(kForms));
    return launch_status(name.text);
  }
  switch (a.D) {
    case 64: return launch_d<kBf16, kCache, kForms, 64>(a, items, rows, stream);
    case 96: return launch_d<kBf16, kCache, kForms, 96>(a, items, rows, stream);
    case 128: return launch_d<kBf16, kCache, kForms, 128>(a, items, rows, stream);
    case 256: return launch_d<kBf16, kCache, kForms, 256>(a, items, rows, stream);
    default: return fail(INTENT_ERR_UNSUPPORTED, "no tiled attention kernel for heads of %d", a.D);
  }
}

template <bool kBf16, bool kBiased, int D>
int launch_join_d(const AttnJoin& j, int side, hipStream_t stream) {
  const unsigned groups = (unsigned)(j.items[0] + j.items[1]) * (unsigned)j.a.HK;
  hipLaunchKernelGGL((attn_join_kernel<kBf16, kBiased, D>), dim3(groups, side), dim3(256), 0, stream, j.items[0],
                     j.tile[0], j.unit_log[0], j);
  static const KernelName name("attn_join_kernel<%s%s, D %d> of splits", kBf16 ? "bf16" : "f16",
                               kBiased ? ", biased" : "", D);
  return launch_status(name.text);
}

template <bool kBf16, bool kBiased = false>
int launch_join(const AttnJoin& j, int side, hipStream_t stream) {
  switch (j.a.D) {
    case 64: return launch_join_d<kBf16, kBiased, 64>(j, side, stream);
    case 96: return launch_join_d<kBf16, kBiased, 96>(j, side, stream);
    case 128: return launch_join_d<kBf16, kBiased, 128>(j, side, stream);
    case 256: return launch_join_d<kBf16, kBiased, 256>(j, side, stream);
    default: return fail(INTENT_ERR_UNSUPPORTED, "no tiled attention kernel for heads of %d", j.a.D);
  }
}

}  // namespace attn
}  // namespace intent
