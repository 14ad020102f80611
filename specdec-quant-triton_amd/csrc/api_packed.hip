// One entry point for calls whose arguments come as 64-bit words (specq_call_packed): foreign-function
// bindings pay for every argument they convert -- ctypes some 3 us for the 33 of specq_rotary, 0.8 us for one
// packed buffer -- which is as much as a small launch takes.
#include <type_traits>
#include <utility>

#include "api_common.hpp"

namespace specq {
namespace {

// Whether a word holds an argument of type T.
template <typename T>
bool fits(int64_t w) {
  if constexpr (std::is_integral_v<T>) return static_cast<int64_t>(static_cast<T>(w)) == w;
  else return true;
}

template <typename T>
T from_word(int64_t w) {
  if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(w));
  } else if constexpr (std::is_floating_point_v<T>) {
    double d;
    memcpy(&d, &w, sizeof(d));
    return static_cast<T>(d);
  } else {
    return static_cast<T>(w);
  }
}

template <typename... A, size_t... I>
int apply(int (*fn)(A...), const int64_t* w, std::index_sequence<I...>) {
  SPECQ_REQUIRE((fits<A>(w[I]) && ...), SPECQ_EINVAL, "call_packed: an integer argument is out of its type's range");
  return fn(from_word<A>(w[I])...);
}

template <typename... A>
int call(int (*fn)(A...), const int64_t* w, int n) {
  SPECQ_REQUIRE(n == (int)sizeof...(A), SPECQ_EINVAL, "call_packed: %d arguments given, %d taken", n, (int)sizeof...(A));
  return apply(fn, w, std::index_sequence_for<A...>{});
}

}  // namespace
}  // namespace specq

extern "C" int specq_call_packed(const char* name, const int64_t* words, int n) {
  specq::clear_error();
  SPECQ_REQUIRE(name && words, SPECQ_EINVAL, "call_packed: null pointer");
#define SPECQ_PACKED(fn) \
  if (strcmp(name, #fn) == 0) return specq::call(fn, words, n)
  SPECQ_PACKED(specq_paged_attn_block);
  SPECQ_PACKED(specq_kv_append_block);
  SPECQ_PACKED(specq_rotary);
  SPECQ_PACKED(specq_kv_pages_reserve);
  SPECQ_PACKED(specq_kv_pages_free);
  SPECQ_PACKED(specq_kv_pages_fork);
  SPECQ_PACKED(specq_kv_pages_compact);
  SPECQ_PACKED(specq_kv_pages_copy);
#undef SPECQ_PACKED
  specq::set_error("call_packed: no entry point %s", name);
  return SPECQ_EINVAL;
}
