// Calls kept as a row of 64-bit slots, one for each argument before the stream in the entry's order
// (pointers and integers as they are, a float by its bits in the low half): what a caller that repeats a
// call hands over again, in one argument.
#include <string.h>

#include <type_traits>
#include <utility>

#include "internal.h"

namespace {

template <typename T>
T slot_value(int64_t slot) {
  if constexpr (std::is_pointer<T>::value) {
    return reinterpret_cast<T>(slot);
  } else if constexpr (std::is_same<T, float>::value) {
    const uint32_t bits = (uint32_t)slot;
    float v;
    memcpy(&v, &bits, sizeof(v));
    return v;
  } else {
    return (T)slot;
  }
}

template <auto Entry, typename... A, size_t... I>
int call_with(int (*)(A...), const int64_t* slots, void* stream, std::index_sequence<I...>) {
  (void)stream;
  // the last parameter is the stream
  return Entry((I + 1 == sizeof...(A) ? slot_value<A>((int64_t)(intptr_t)stream) : slot_value<A>(slots[I]))...);
}

template <auto Entry, typename... A>
int call_slots(int (*entry)(A...), const int64_t* slots, int64_t count, void* stream) {
  INTENT_REQUIRE(slots != nullptr && count + 1 == (int64_t)sizeof...(A), INTENT_ERR_INVALID_ARGUMENT,
                 "the entry takes %lld slots, got %lld", (long long)(sizeof...(A) - 1), (long long)count);
  return call_with<Entry>(entry, slots, stream, std::make_index_sequence<sizeof...(A)>{});
}

}  // namespace

extern "C" int intent_amd_replay(int record, const int64_t* slots, int64_t count, void* stream) {
  switch (record) {
    case INTENT_RECORD_QK_NORM_ROPE: return call_slots<intent_qk_norm_rope>(intent_qk_norm_rope, slots, count, stream);
    case INTENT_RECORD_PAGED_KV_APPEND:
      return call_slots<intent_paged_kv_append>(intent_paged_kv_append, slots, count, stream);
    case INTENT_RECORD_PAGED_ATTENTION:
      return call_slots<intent_paged_attention>(intent_paged_attention, slots, count, stream);
    default: return intent::fail(INTENT_ERR_INVALID_ARGUMENT, "no entry has record number %d", record);
  }
}
