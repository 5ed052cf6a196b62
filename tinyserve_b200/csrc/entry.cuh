// Entry points whose arguments come as one run of 64-bit fields (integers and pointers; floats as doubles): with twenty or thirty of them, a
// foreign-function call that converts each takes longer than the launch behind it (32 arguments: 4.4 us of the host one by one, 0.9 packed).
#pragma once

#include <cstring>
#include <type_traits>
#include <utility>

#include "common.cuh"

template <typename T> inline T ts_field(const char* at) {
  if constexpr (std::is_floating_point<T>::value) {
    double v;
    std::memcpy(&v, at, 8);
    return static_cast<T>(v);
  } else {
    long long v;
    std::memcpy(&v, at, 8);
    return (T)v;
  }
}
template <typename... A, size_t... I>
inline int ts_unpacked(int (*fn)(A...), const char* fields, std::index_sequence<I...>) { return fn(ts_field<A>(fields + 8 * I)...); }
template <typename... A>
inline int ts_call(const char* name, int (*fn)(A...), const void* fields, int n) {
  TS_REQUIRE(n == (int)sizeof...(A), "%s takes %d fields, got %d", name, (int)sizeof...(A), n);
  return ts_unpacked(fn, static_cast<const char*>(fields), std::index_sequence_for<A...>{});
}
// the entry point ts_<name>(fields, how many) of a function <name> of this file
#define TS_ENTRY(name) \
  TS_EXPORT int ts_##name(const void* fields, int n) { return ts_call("ts_" #name, name, fields, n); }
