// What runs between the projection of queries, keys and values and the attention:
// norms of queries and keys for each head, the position rotation, and the append to a
// paged cache, in one pass over the projection's rows (gfx950).
//
//   norm:    y = x * rsqrt(mean(x^2) + eps) * w over the D elements of a head
//   rotate:  the first R elements as pairs (a, b): (i, i + R/2), or (2i, 2i + 1) interleaved:
//            a' = a cos - b sin, b' = b cos + a sin, cos and sin of the token's position
//   cache:   the row as it is (f16 / bf16), or E4M3FN codes with a scale for each token and head,
//            s = max(absmax, 1e-12) / 448, code = e4m3fn(clamp(y / s, +-448)): the groupwise FP8
//            quantizer's rule with one group for each head
//
// All of it in f32; each result is rounded once, when it is stored (y is not rounded between
// the norm, the rotation and the encoding). Values are neither normed nor rotated.
//
// A head is a row of D / 8 chunks of 16 bytes; LPR lanes (D / 8 rounded up to a power of two)
// hold one chunk each, so a row's sums stay inside a DPP row or a half-wave and a rotation
// partner is a lane of the same group. A group takes RPG heads of one token, which share its
// cosines and sines and whose loads are all issued before the first is used.
//
// Bound by memory for many tokens: 8192 of 32 + 8 heads of 128 (172 MB) take 36.7 us, 4.7 TB/s, with values
// into an f16 cache (206 MB) 40.1 us, 5.1 TB/s, the rate of a large copy; 64 tokens 4 us, a chain of
// latencies (position, table row, store).
#include "common.h"
#include "internal.h"

namespace {

struct PrepArgs {
  const uint16_t *q, *k, *v;
  int64_t q_ld, k_ld, v_ld;
  const uint16_t *q_weight, *k_weight;  // null: no norm
  const float* cos_sin;
  int64_t cos_sin_ld;
  const int32_t *positions, *slots;
  uint16_t* q_out;
  int64_t q_out_ld;
  uint16_t* k_out;
  int64_t k_out_ld;
  void *k_cache, *v_cache;
  int64_t k_page, v_page;  // elements from a page to the next
  float *k_scales, *v_scales;
  int64_t ks_page, vs_page;
  int64_t items;
  float eps;
  int HQ, HK, D, R, P, heads, items_per_token, interleaved, page_shift, slot_count;
};

enum Mode { kKeysOut = 0, kCacheSame = 1, kCacheFp8 = 2 };

// The larger of two floats without a sign, by their bits: NaN is the largest.
INTENT_DEVICE float magnitude_max(float a, float b) {
  return bit_cast<float>(max(bit_cast<uint32_t>(a), bit_cast<uint32_t>(b)));
}

// Sum or maximum over the LPR lanes of a group.
template <int LPR, bool kMax>
INTENT_DEVICE float group_reduce(float v) {
  auto join = [](float a, float b) { return kMax ? magnitude_max(a, b) : a + b; };
  v = join(v, dpp_f32<0xB1>(v));             // quad_perm [1,0,3,2]
  v = join(v, dpp_f32<0x4E>(v));             // quad_perm [2,3,0,1]
  v = join(v, dpp_f32<0x141>(v));            // mirrored in halves of a row: 8 lanes
  if constexpr (LPR >= 16) v = join(v, dpp_f32<0x140>(v));  // mirrored row: 16 lanes
  if constexpr (LPR >= 32) v = join(v, __shfl_xor(v, 16));
  if constexpr (LPR >= 64) v = join(v, __shfl_xor(v, 32));
  return v;
}

template <bool kBf16>
INTENT_DEVICE void widen(u32x4 raw, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kBf16) {
      v[2 * j] = bit_cast<float>(raw[j] << 16);
      v[2 * j + 1] = bit_cast<float>(raw[j] & 0xffff0000u);
    } else {
      const f16x2 h = bit_cast<f16x2>(raw[j]);
      v[2 * j] = (float)h[0];
      v[2 * j + 1] = (float)h[1];
    }
  }
}

template <bool kBf16>
INTENT_DEVICE u32x4 narrow(const float (&v)[8]) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kBf16) r[j] = bf16x2_rne(v[2 * j], v[2 * j + 1]);
    else r[j] = bit_cast<uint32_t>(__builtin_convertvector(f32x2{v[2 * j], v[2 * j + 1]}, f16x2));
  }
  return r;
}

// The row of a token and head in a paged cache [page][HK][page size], or -1 for a slot outside it.
INTENT_DEVICE int64_t cache_row(const PrepArgs& a, int slot, int head, int64_t page_ld, int row_size) {
  const int page = slot >> a.page_shift, place = slot & ((1 << a.page_shift) - 1);
  return (int64_t)page * page_ld + (((int64_t)head << a.page_shift) + place) * row_size;
}

template <bool kBf16, int MODE, int LPR, int RPG>
__global__ __launch_bounds__(256) void attn_prep_kernel(const PrepArgs a) {
  const int c = threadIdx.x % LPR;  // this lane's chunk of 8 elements
  const int64_t item = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (item >= a.items) return;
  const int64_t token = item / a.items_per_token;
  const int h0 = (int)(item - token * a.items_per_token) * RPG;
  const bool mine = c * 8 < a.D;

  u32x4 raw[RPG];
#pragma unroll
  for (int i = 0; i < RPG; ++i) {
    const int h = h0 + i;
    const uint16_t* row = h < a.HQ ? a.q + token * a.q_ld + (int64_t)h * a.D
                          : h < a.HQ + a.HK ? a.k + token * a.k_ld + (int64_t)(h - a.HQ) * a.D
                                            : a.v + token * a.v_ld + (int64_t)(h - a.HQ - a.HK) * a.D;
    raw[i] = mine && h < a.heads ? load16(row + c * 8) : u32x4{0u, 0u, 0u, 0u};
  }
  const int half = a.R >> 4;                    // chunks of one half of the rotated elements
  const bool turned = c < 2 * half;             // this chunk is rotated
  float cosv[8], sinv[8];
  int partner = c;
  bool second = false;
  if (a.R > 0 && h0 < a.HQ + a.HK) {
    const int p = min(max(a.positions[token], 0), a.P - 1);
    const float* row = a.cos_sin + (int64_t)p * a.cos_sin_ld;
    if (turned && a.interleaved) {
      *(f32x4*)cosv = *(const f32x4*)(row + c * 4);
      *(f32x4*)sinv = *(const f32x4*)(row + a.R / 2 + c * 4);
    } else if (turned) {
      second = c >= half;
      const int pair = second ? c - half : c;
      partner = second ? c - half : c + half;
      *(f32x4*)cosv = *(const f32x4*)(row + pair * 8);
      *(f32x4*)(cosv + 4) = *(const f32x4*)(row + pair * 8 + 4);
      *(f32x4*)sinv = *(const f32x4*)(row + a.R / 2 + pair * 8);
      *(f32x4*)(sinv + 4) = *(const f32x4*)(row + a.R / 2 + pair * 8 + 4);
    }
  }
  int slot = -1;
  if constexpr (MODE != kKeysOut) {
    if (h0 + RPG > a.HQ) {
      slot = a.slots[token];
      if (slot >= a.slot_count) slot = -1;
    }
  }

#pragma unroll
  for (int i = 0; i < RPG; ++i) {
    const int h = h0 + i;
    if (h >= a.heads) break;
    const bool is_q = h < a.HQ, is_v = h >= a.HQ + a.HK;
    float x[8];
    widen<kBf16>(raw[i], x);
    const uint16_t* weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    if (weight != nullptr) {
      float w[8];
      widen<kBf16>(mine ? load16(weight + c * 8) : u32x4{0u, 0u, 0u, 0u}, w);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
      const float r = rsqrtf(group_reduce<LPR, false>(sum) / (float)a.D + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j];
    }
    if (a.R > 0 && !is_v) {
      if (a.interleaved) {
        if (turned) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float even = x[2 * j] * cosv[j] - x[2 * j + 1] * sinv[j];
            x[2 * j + 1] = x[2 * j + 1] * cosv[j] + x[2 * j] * sinv[j];
            x[2 * j] = even;
          }
        }
      } else {
        float other[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) other[j] = __shfl(x[j], partner, LPR);
        if (turned) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float t = other[j] * sinv[j];
            x[j] = second ? x[j] * cosv[j] + t : x[j] * cosv[j] - t;
          }
        }
      }
    }
    if (is_q) {
      if (mine) store16(a.q_out + token * a.q_out_ld + (int64_t)h * a.D + c * 8, narrow<kBf16>(x));
      continue;
    }
    const int head = is_v ? h - a.HQ - a.HK : h - a.HQ;
    if constexpr (MODE == kKeysOut) {
      if (mine) store16(a.k_out + token * a.k_out_ld + (int64_t)head * a.D + c * 8, narrow<kBf16>(x));
    } else {
      const int64_t page_ld = is_v ? a.v_page : a.k_page;
      if constexpr (MODE == kCacheSame) {
        uint16_t* cache = (uint16_t*)(is_v ? a.v_cache : a.k_cache);
        if (mine && slot >= 0) store16(cache + cache_row(a, slot, head, page_ld, a.D) + c * 8, narrow<kBf16>(x));
      } else {
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = magnitude_max(amax, fabsf(x[j]));
        // a head that holds an infinity or NaN reads as NaN throughout: its scale is infinite or NaN, and
        // the clamp lets NaN pass
        const float scale = __fdiv_rn(magnitude_max(group_reduce<LPR, true>(amax), 1.0e-12f), 448.0f);
        uint32_t code[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float t[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            t[e] = __fdiv_rn(x[4 * j + e], scale);
            t[e] = t[e] < -448.0f ? -448.0f : t[e] > 448.0f ? 448.0f : t[e];
          }
          int word = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
          code[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], word, true);
        }
        if (slot >= 0) {
          uint8_t* cache = (uint8_t*)(is_v ? a.v_cache : a.k_cache);
          if (mine) *(u32x2*)(cache + cache_row(a, slot, head, page_ld, a.D) + c * 8) = u32x2{code[0], code[1]};
          if (c == 0) (is_v ? a.v_scales : a.k_scales)[cache_row(a, slot, head, is_v ? a.vs_page : a.ks_page, 1)] = scale;
        }
      }
    }
  }
}

template <bool kBf16, int MODE, int LPR, int RPG>
int launch(PrepArgs a, int64_t T, hipStream_t stream) {
  a.items_per_token = (a.heads + RPG - 1) / RPG;
  a.items = T * a.items_per_token;
  const int64_t blocks = (a.items + 256 / LPR - 1) / (256 / LPR);
  hipLaunchKernelGGL((attn_prep_kernel<kBf16, MODE, LPR, RPG>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  static const intent::KernelName name("attn_prep_kernel<%s%s, %d lanes, %d heads>", kBf16 ? "bf16" : "f16",
                                       MODE == kCacheFp8 ? ", fp8 cache" : MODE == kCacheSame ? ", cache" : "", LPR, RPG);
  return intent::launch_status(name.text);
}

// Two heads to a group once one each is more lanes than twice what the GPU holds (2^19): they share the
// table's row (8192 tokens of 32 + 8 heads of 128: 39.4 us with one, 36.7 with two, 36.5 with four; with
// values into an f16 cache 42.9, 40.1, 42.6). Fewer tokens are a matter of latency (64 tokens into an
// 8-bit cache: 4.0, 4.9 and 6.9 us).
template <bool kBf16, int MODE, int LPR>
int launch_heads(const PrepArgs& a, int64_t T, hipStream_t stream) {
  return T * a.heads * LPR >= (int64_t)1 << 20 ? launch<kBf16, MODE, LPR, 2>(a, T, stream)
                                               : launch<kBf16, MODE, LPR, 1>(a, T, stream);
}

template <bool kBf16, int MODE>
int launch_lanes(const PrepArgs& a, int64_t T, hipStream_t stream) {
  const int chunks = a.D / 8;
  if (chunks <= 8) return launch_heads<kBf16, MODE, 8>(a, T, stream);
  if (chunks <= 16) return launch_heads<kBf16, MODE, 16>(a, T, stream);
  if (chunks <= 32) return launch_heads<kBf16, MODE, 32>(a, T, stream);
  return launch_heads<kBf16, MODE, 64>(a, T, stream);
}

// The checks that both entries share; fills the arguments they share.
int check_heads(PrepArgs& a, const void* q, int64_t T, int64_t HQ, int64_t q_ld, const void* k, int64_t HK, int64_t k_ld,
                int64_t D, const void* q_weight, const void* k_weight, float eps, const float* cos_sin, int64_t P,
                int64_t R, int64_t cos_sin_ld, int interleaved, const int32_t* positions, void* q_out, int64_t q_out_ld) {
  INTENT_REQUIRE(T >= 0 && HQ >= 0 && HK >= 0 && D >= 0 && R >= 0 && P >= 0 && T <= INT32_MAX && HQ <= 65536 &&
                     HK <= 65536 && P <= INT32_MAX,
                 INTENT_ERR_INVALID_ARGUMENT, "bad extents (T=%lld HQ=%lld HK=%lld D=%lld R=%lld P=%lld)", (long long)T,
                 (long long)HQ, (long long)HK, (long long)D, (long long)R, (long long)P);
  INTENT_REQUIRE(R <= D && R % 2 == 0, INTENT_ERR_INVALID_ARGUMENT, "R=%lld rotated elements of heads of %lld",
                 (long long)R, (long long)D);
  INTENT_REQUIRE(D % 8 == 0 && D <= 512 && R % 16 == 0, INTENT_ERR_UNSUPPORTED,
                 "D=%lld must be a multiple of 8 up to 512 and R=%lld a multiple of 16", (long long)D, (long long)R);
  // a lane group of at most 64 for each head: the grid's work items stay below 2^32
  INTENT_REQUIRE(T * (HQ + 2 * HK) < ((int64_t)1 << 25), INTENT_ERR_UNSUPPORTED,
                 "T * (HQ + 2 HK) = %lld heads exceed the %lld a launch covers", (long long)(T * (HQ + 2 * HK)),
                 (long long)((int64_t)1 << 25));
  if (T == 0 || D == 0) return INTENT_OK;
  INTENT_REQUIRE((HQ == 0 || (q && q_out)) && (HK == 0 || k), INTENT_ERR_INVALID_ARGUMENT, "null pointer argument");
  INTENT_REQUIRE((HQ == 0 || ((T == 1 || (q_ld >= HQ * D && q_out_ld >= HQ * D)))) && (HK == 0 || T == 1 || k_ld >= HK * D),
                 INTENT_ERR_INVALID_ARGUMENT, "token stride smaller than the heads");
  INTENT_REQUIRE(intent::aligned16(q) && intent::aligned16(k) && intent::aligned16(q_out) &&
                     intent::aligned16(q_weight) && intent::aligned16(k_weight) &&
                     (T == 1 || ((HQ == 0 || (q_ld % 8 == 0 && q_out_ld % 8 == 0)) && (HK == 0 || k_ld % 8 == 0))),
                 INTENT_ERR_ALIGNMENT, "heads and weights must be 16-byte aligned with token strides %% 8 == 0");
  if (R > 0 && HQ + HK > 0) {
    INTENT_REQUIRE(cos_sin && positions, INTENT_ERR_INVALID_ARGUMENT, "null pointer argument");
    INTENT_REQUIRE(P > 0, INTENT_ERR_INVALID_ARGUMENT, "a rotation needs a table of at least one position");
    INTENT_REQUIRE(P == 1 || cos_sin_ld >= R, INTENT_ERR_INVALID_ARGUMENT, "table stride smaller than the row");
    INTENT_REQUIRE(intent::aligned16(cos_sin) && (P == 1 || cos_sin_ld % 4 == 0), INTENT_ERR_ALIGNMENT,
                   "cos_sin must be 16-byte aligned with a stride %% 4 == 0");
  }
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k;
  a.q_ld = q_ld, a.k_ld = k_ld;
  a.q_weight = (const uint16_t*)q_weight, a.k_weight = (const uint16_t*)k_weight;
  a.cos_sin = cos_sin, a.cos_sin_ld = cos_sin_ld, a.positions = positions;
  a.q_out = (uint16_t*)q_out, a.q_out_ld = q_out_ld;
  a.eps = eps;
  a.HQ = (int)HQ, a.HK = (int)HK, a.D = (int)D, a.R = (int)R, a.P = (int)P, a.interleaved = interleaved != 0;
  return INTENT_OK;
}

}  // namespace

extern "C" int intent_qk_norm_rope(const void* q, int64_t T, int64_t HQ, int64_t q_ld, const void* k, int64_t HK,
                                   int64_t k_ld, int64_t D, const void* q_weight, const void* k_weight, float eps,
                                   const float* cos_sin, int64_t P, int64_t R, int64_t cos_sin_ld, int interleaved,
                                   const int32_t* positions, int is_bf16, void* q_out, int64_t q_out_ld, void* k_out,
                                   int64_t k_out_ld, void* stream) {
  intent::clear_error();
  PrepArgs a{};
  if (const int status = check_heads(a, q, T, HQ, q_ld, k, HK, k_ld, D, q_weight, k_weight, eps, cos_sin, P, R,
                                     cos_sin_ld, interleaved, positions, q_out, q_out_ld))
    return status;
  if (T == 0 || D == 0 || HQ + HK == 0) return INTENT_OK;
  if (HK > 0) {
    INTENT_REQUIRE(k_out, INTENT_ERR_INVALID_ARGUMENT, "null pointer argument");
    INTENT_REQUIRE(T == 1 || k_out_ld >= HK * D, INTENT_ERR_INVALID_ARGUMENT, "token stride smaller than the heads");
    INTENT_REQUIRE(intent::aligned16(k_out) && (T == 1 || k_out_ld % 8 == 0), INTENT_ERR_ALIGNMENT,
                   "k_out must be 16-byte aligned with a token stride %% 8 == 0");
  }
  a.k_out = (uint16_t*)k_out, a.k_out_ld = k_out_ld;
  a.heads = a.HQ + a.HK;
  return is_bf16 ? launch_lanes<true, kKeysOut>(a, T, (hipStream_t)stream)
                 : launch_lanes<false, kKeysOut>(a, T, (hipStream_t)stream);
}

extern "C" int intent_paged_kv_append(const void* q, int64_t T, int64_t HQ, int64_t q_ld, const void* k, int64_t HK,
                                      int64_t k_ld, const void* v, int64_t v_ld, int64_t D, const void* q_weight,
                                      const void* k_weight, float eps, const float* cos_sin, int64_t P, int64_t R,
                                      int64_t cos_sin_ld, int interleaved, const int32_t* positions,
                                      const int32_t* slots, int is_bf16, int cache_is_fp8, void* k_cache,
                                      int64_t k_page_ld, void* v_cache, int64_t v_page_ld, float* k_scales,
                                      int64_t k_scales_ld, float* v_scales, int64_t v_scales_ld, int64_t pages,
                                      int64_t page_size, void* q_out, int64_t q_out_ld, void* stream) {
  intent::clear_error();
  PrepArgs a{};
  if (const int status = check_heads(a, q, T, HQ, q_ld, k, HK, k_ld, D, q_weight, k_weight, eps, cos_sin, P, R,
                                     cos_sin_ld, interleaved, positions, q_out, q_out_ld))
    return status;
  INTENT_REQUIRE(pages >= 0 && page_size >= 0 && pages <= INT32_MAX && page_size <= INT32_MAX &&
                     pages * page_size <= INT32_MAX,
                 INTENT_ERR_INVALID_ARGUMENT, "bad cache extents (%lld pages of %lld)", (long long)pages,
                 (long long)page_size);
  if (T == 0 || D == 0 || HQ + HK == 0) return INTENT_OK;
  if (HK > 0) {
    INTENT_REQUIRE(page_size > 0 && (page_size & (page_size - 1)) == 0, INTENT_ERR_UNSUPPORTED,
                   "the page size must be a power of two, got %lld", (long long)page_size);
    INTENT_REQUIRE(v && slots, INTENT_ERR_INVALID_ARGUMENT, "null pointer argument");
    INTENT_REQUIRE(T == 1 || v_ld >= HK * D, INTENT_ERR_INVALID_ARGUMENT, "token stride smaller than the heads");
    INTENT_REQUIRE(intent::aligned16(v) && (T == 1 || v_ld % 8 == 0), INTENT_ERR_ALIGNMENT,
                   "v must be 16-byte aligned with a token stride %% 8 == 0");
    if (pages > 0) {
      INTENT_REQUIRE(k_cache && v_cache && (!cache_is_fp8 || (k_scales && v_scales)), INTENT_ERR_INVALID_ARGUMENT,
                     "null pointer argument");
      INTENT_REQUIRE(pages == 1 || (k_page_ld >= HK * page_size * D && v_page_ld >= HK * page_size * D &&
                                    (!cache_is_fp8 || (k_scales_ld >= HK * page_size && v_scales_ld >= HK * page_size))),
                     INTENT_ERR_INVALID_ARGUMENT, "page stride smaller than the page");
      const int64_t step = cache_is_fp8 ? 16 : 8;
      INTENT_REQUIRE(intent::aligned16(k_cache) && intent::aligned16(v_cache) &&
                         (pages == 1 || (k_page_ld % step == 0 && v_page_ld % step == 0)) &&
                         (!cache_is_fp8 || (intent::aligned4(k_scales) && intent::aligned4(v_scales))),
                     INTENT_ERR_ALIGNMENT, "the cache must be 16-byte aligned with page strides of whole 16 bytes");
    }
  }
  a.v = (const uint16_t*)v, a.v_ld = v_ld, a.slots = slots;
  a.k_cache = k_cache, a.v_cache = v_cache, a.k_page = k_page_ld, a.v_page = v_page_ld;
  a.k_scales = k_scales, a.v_scales = v_scales, a.ks_page = k_scales_ld, a.vs_page = v_scales_ld;
  a.page_shift = page_size > 0 ? __builtin_ctzll((unsigned long long)page_size) : 0;
  a.slot_count = (int)(pages * page_size);
  a.heads = a.HQ + 2 * a.HK;
  hipStream_t st = (hipStream_t)stream;
  if (cache_is_fp8)
    return is_bf16 ? launch_lanes<true, kCacheFp8>(a, T, st) : launch_lanes<false, kCacheFp8>(a, T, st);
  return is_bf16 ? launch_lanes<true, kCacheSame>(a, T, st) : launch_lanes<false, kCacheSame>(a, T, st);
}
