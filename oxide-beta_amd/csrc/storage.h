// storage.h -- element types of the sequence operators (internal to the library): values are kept
// as float32 or bfloat16, all arithmetic is float32, a stored bfloat16 is rounded once, to nearest
// even.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "common.h"

namespace oxh {
namespace storage {

typedef __bf16 bf16;

inline bool valid(int dtype) { return dtype == OXH_F32 || dtype == OXH_BF16; }
inline uint64_t bytes_of(int dtype) { return dtype == OXH_BF16 ? 2 : 4; }

template <typename T>
__device__ __forceinline__ float widen(T v) {
  return static_cast<float>(v);
}

// N consecutive values moved as one access (N * sizeof(T) bytes, up to 16).  The address need only
// be a multiple of a value's bytes: the device's vector accesses may lie anywhere.
template <typename T, int N>
struct Pack {
  typedef T vector __attribute__((ext_vector_type(N)));
  typedef vector type __attribute__((aligned(sizeof(T))));
};
template <typename T>
struct Pack<T, 1> {
  typedef T type;
};

template <typename T, int N>
__device__ __forceinline__ typename Pack<T, N>::type raw(const T *p) {
  return *reinterpret_cast<const typename Pack<T, N>::type *>(p);
}
template <typename T, int N>
__device__ __forceinline__ void widen_all(const typename Pack<T, N>::type &x, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = widen(x);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = widen(x[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void load(const T *p, float (&v)[N]) {
  widen_all<T, N>(raw<T, N>(p), v);
}

// The places of a row that N consecutive ones from `at` (< columns) stand for, columns >= N.
// Ragged rows, whose columns are no multiple of N, end in an access that begins early enough to
// stay within the row: its first `skip` values are the access's before it.
struct Places {
  uint32_t start, skip;
};
template <int N, bool Ragged>
__device__ __forceinline__ Places places_at(uint32_t at, uint32_t columns) {
  if constexpr (!Ragged) return {at, 0};
  const uint32_t start = min(at, columns - N);
  return {start, at - start};
}
// Skipped values are zero.
template <typename T, int N, bool Ragged>
__device__ __forceinline__ void load_places(const T *row, Places at, float (&v)[N]) {
  load<T, N>(row + at.start, v);
  if constexpr (Ragged) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = i < at.skip ? 0.0f : v[i];
  }
}

// Once: past the caches.
template <typename T, int N, bool Once = false>
__device__ __forceinline__ void store(T *p, const float (&v)[N]) {
  typename Pack<T, N>::type x;
  if constexpr (N == 1) {
    x = static_cast<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = static_cast<T>(v[i]);
  }
  if constexpr (Once)
    __builtin_nontemporal_store(x, reinterpret_cast<typename Pack<T, N>::type *>(p));
  else
    *reinterpret_cast<typename Pack<T, N>::type *>(p) = x;
}

// Skipped values are not stored.
template <typename T, int N, bool Ragged, bool Once = false>
__device__ __forceinline__ void store_places(T *row, Places at, const float (&v)[N]) {
  if (!Ragged || at.skip == 0) {
    store<T, N, Once>(row + at.start, v);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
      if (i >= at.skip) row[at.start + i] = static_cast<T>(v[i]);
  }
}

}  // namespace storage
}  // namespace oxh
