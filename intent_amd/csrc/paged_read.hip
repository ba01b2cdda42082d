// Tokens of a paged cache as rows again: k[t] and v[t] are the keys and values at slot slots[t], widened to the
// heads' type; a slot outside the cache (padding) gives zeros (gfx950).
//
// A head is a row of D / 8 chunks of eight elements, one to each of LPR lanes (D / 8 rounded up to a power of two).
#include "paged_cache.h"

namespace {

using namespace intent;

struct ReadArgs {
  const void *k_cache, *v_cache;
  int64_t k_page, v_page;  // elements from a page to the next
  const void *k_params, *v_params;
  int64_t ks_page, vs_page;  // scales or pairs from a page to the next
  const int32_t* slots;
  uint16_t *k_out, *v_out;
  int64_t k_out_ld, v_out_ld;
  int64_t items;
  int HK, D, page_shift, slot_count, items_per_token;
};

template <bool kBf16, int FORMAT, int LPR, int RPG>
__global__ __launch_bounds__(256) void paged_read_kernel(const ReadArgs a) {
  const int c = threadIdx.x % LPR;
  const int64_t item = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (item >= a.items || c * 8 >= a.D) return;
  const int64_t token = item / a.items_per_token;
  const int first = (int)(item - token * a.items_per_token) * RPG, parts = 2 * a.HK;
  const int slot = a.slots[token];
  const bool inside = slot >= 0 && slot < a.slot_count;
  const int64_t page = slot >> a.page_shift;
  const int place = slot & ((1 << a.page_shift) - 1);
  const int groups = (a.D + kGroup4 - 1) / kGroup4;
  u32x4 raw[RPG];
  uint32_t param[RPG];
  if (inside) {
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      const int part = min(first + i, parts - 1);
      const bool is_v = part >= a.HK;
      const int64_t row = ((int64_t)(is_v ? part - a.HK : part) << a.page_shift) + place;
      const char* cache = (const char*)(is_v ? a.v_cache : a.k_cache);
      const int64_t at = page * (is_v ? a.v_page : a.k_page), beside = page * (is_v ? a.vs_page : a.ks_page);
      const uint32_t* params = (const uint32_t*)(is_v ? a.v_params : a.k_params);
      if constexpr (FORMAT == kCacheSame) {
        raw[i] = load16(cache + (at + row * a.D + c * 8) * 2);
      } else if constexpr (FORMAT == kCacheFp8) {
        const u32x2 two = *(const u32x2*)(cache + at + row * a.D + c * 8);
        raw[i] = u32x4{two[0], two[1], 0u, 0u};
        param[i] = params[beside + row];
      } else {
        raw[i] = u32x4{*(const uint32_t*)(cache + at + row * (a.D / 2) + c * 4), 0u, 0u, 0u};
        param[i] = params[beside + row * groups + c / 4];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RPG; ++i) {
    const int part = first + i;
    if (part >= parts) break;
    const bool is_v = part >= a.HK;
    uint16_t* to = (is_v ? a.v_out + token * a.v_out_ld : a.k_out + token * a.k_out_ld) +
                   (int64_t)(is_v ? part - a.HK : part) * a.D + c * 8;
    u32x4 out = u32x4{0u, 0u, 0u, 0u};
    if (inside && FORMAT == kCacheSame) out = raw[i];
    if constexpr (FORMAT != kCacheSame) {
      if (inside) {
        float v[8];
        if constexpr (FORMAT == kCacheFp8) {
          const float scale = bit_cast<float>(param[i]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[i][j], false);
            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[i][j], true);
            v[4 * j] = lo[0] * scale, v[4 * j + 1] = lo[1] * scale;
            v[4 * j + 2] = hi[0] * scale, v[4 * j + 3] = hi[1] * scale;
          }
        } else {
          widen4(raw[i][0], param[i], v);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kBf16) out[j] = bf16x2_rne(v[2 * j], v[2 * j + 1]);
          else out[j] = bit_cast<uint32_t>(__builtin_convertvector(f32x2{v[2 * j], v[2 * j + 1]}, f16x2));
        }
      }
    }
    store16(to, out);
  }
}

template <bool kBf16, int FORMAT, int LPR, int RPG>
int launch(ReadArgs a, int64_t T, hipStream_t stream) {
  a.items_per_token = (2 * a.HK + RPG - 1) / RPG;
  a.items = T * a.items_per_token;
  const int64_t blocks = (a.items + 256 / LPR - 1) / (256 / LPR);
  hipLaunchKernelGGL((paged_read_kernel<kBf16, FORMAT, LPR, RPG>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  static const KernelName name("paged_read_kernel<%s%s, %d lanes, %d heads>", kBf16 ? "bf16" : "f16", cache_name(FORMAT),
                               LPR, RPG);
  return launch_status(name.text);
}

// Four heads to a group once one each is more lanes than twice what the GPU holds: they share the slot, and their loads
// are all issued before the first is used (50001 tokens of 8 heads of 128 in 8 bits: 75 us with one, 57, 54 and 53 with
// two, four and eight; 4096 in 4 bits 8.3, 7.0, 6.9 and 7.6).
constexpr int kMany = 4;
template <bool kBf16, int FORMAT, int LPR>
int launch_heads(const ReadArgs& a, int64_t T, hipStream_t stream) {
  return T * 2 * a.HK * LPR >= (int64_t)1 << 20 ? launch<kBf16, FORMAT, LPR, kMany>(a, T, stream)
                                                : launch<kBf16, FORMAT, LPR, 1>(a, T, stream);
}

template <bool kBf16, int FORMAT>
int launch_lanes(const ReadArgs& a, int64_t T, hipStream_t stream) {
  const int chunks = a.D / 8;
  if (chunks <= 8) return launch_heads<kBf16, FORMAT, 8>(a, T, stream);
  if (chunks <= 16) return launch_heads<kBf16, FORMAT, 16>(a, T, stream);
  if (chunks <= 32) return launch_heads<kBf16, FORMAT, 32>(a, T, stream);
  return launch_heads<kBf16, FORMAT, 64>(a, T, stream);
}

}  // namespace

extern "C" int intent_paged_kv_read(int cache_format, const void* k_cache, int64_t k_page_ld, const void* v_cache,
                                    int64_t v_page_ld, const void* k_params, int64_t k_params_ld, const void* v_params,
                                    int64_t v_params_ld, int64_t pages, int64_t HK, int64_t page_size, int64_t D,
                                    const int32_t* slots, int64_t T, int is_bf16, void* k_out, int64_t k_out_ld,
                                    void* v_out, int64_t v_out_ld, void* stream) {
  clear_error();
  INTENT_REQUIRE(cache_format >= INTENT_CACHE_SAME && cache_format <= INTENT_CACHE_INT4, INTENT_ERR_INVALID_ARGUMENT,
                 "no cache has format %d", cache_format);
  INTENT_REQUIRE(T >= 0 && HK >= 0 && D >= 0 && pages >= 0 && page_size >= 0 && T <= INT32_MAX && HK <= 65536 &&
                     pages <= INT32_MAX && page_size <= INT32_MAX && pages * page_size <= INT32_MAX,
                 INTENT_ERR_INVALID_ARGUMENT, "bad extents (T=%lld HK=%lld D=%lld, %lld pages of %lld)", (long long)T,
                 (long long)HK, (long long)D, (long long)pages, (long long)page_size);
  INTENT_REQUIRE(D % 8 == 0 && D <= 512, INTENT_ERR_UNSUPPORTED, "D must be a multiple of 8 up to 512, got %lld",
                 (long long)D);
  // a lane group of at most 64 for each head: the grid's work items stay below 2^32
  INTENT_REQUIRE(T * HK < ((int64_t)1 << 24), INTENT_ERR_UNSUPPORTED,
                 "T * HK = %lld heads exceed the %lld a launch covers", (long long)(T * HK), (long long)((int64_t)1 << 24));
  if (T == 0 || D == 0 || HK == 0) return INTENT_OK;
  const bool any = pages > 0 && page_size > 0;
  INTENT_REQUIRE(!any || (page_size & (page_size - 1)) == 0, INTENT_ERR_UNSUPPORTED,
                 "the page size must be a power of two, got %lld", (long long)page_size);
  INTENT_REQUIRE(slots && k_out && v_out, INTENT_ERR_INVALID_ARGUMENT, "null pointer argument");
  INTENT_REQUIRE(T == 1 || (k_out_ld >= HK * D && v_out_ld >= HK * D), INTENT_ERR_INVALID_ARGUMENT,
                 "token stride smaller than the heads");
  INTENT_REQUIRE(aligned16(k_out) && aligned16(v_out) && (T == 1 || (k_out_ld % 8 == 0 && v_out_ld % 8 == 0)),
                 INTENT_ERR_ALIGNMENT, "k_out and v_out must be 16-byte aligned with token strides %% 8 == 0");
  const Cache cache{cache_format, k_cache, k_page_ld, v_cache, v_page_ld, k_params, k_params_ld, v_params, v_params_ld,
                    pages, HK, page_size};
  if (any)
    if (const int status = check_cache(cache, D)) return status;
  const RowSizes sizes = row_sizes(cache_format, D);
  ReadArgs a{};
  a.k_cache = k_cache, a.v_cache = v_cache, a.k_page = k_page_ld, a.v_page = v_page_ld;
  a.k_params = k_params, a.v_params = v_params;
  a.ks_page = k_params_ld / sizes.each, a.vs_page = v_params_ld / sizes.each;
  a.slots = slots;
  a.k_out = (uint16_t*)k_out, a.v_out = (uint16_t*)v_out, a.k_out_ld = k_out_ld, a.v_out_ld = v_out_ld;
  a.HK = (int)HK, a.D = (int)D;
  a.page_shift = any ? __builtin_ctzll((unsigned long long)page_size) : 0;
  a.slot_count = any ? (int)(pages * page_size) : 0;
  hipStream_t st = (hipStream_t)stream;
  switch (cache_format) {
    case kCacheInt4: return is_bf16 ? launch_lanes<true, kCacheInt4>(a, T, st) : launch_lanes<false, kCacheInt4>(a, T, st);
    case kCacheFp8: return is_bf16 ? launch_lanes<true, kCacheFp8>(a, T, st) : launch_lanes<false, kCacheFp8>(a, T, st);
    // the heads' type as it is: one kernel for both
    default: return launch_lanes<false, kCacheSame>(a, T, st);
  }
}
