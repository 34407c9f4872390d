// Pieces of rows at any alignment, shared by the kernels that walk rows packet
// by packet: up to kVec elements from an element-aligned address. And the host's
// checks of which tensors share memory.
#pragma once

#include <initializer_list>

#include "common.h"

namespace dragon_hip {

// The first n (1 .. kVec) elements at p, the others as `fill`. Whole packets are
// one access; plain loads, so that a later pass finds them in the cache.
template <typename T>
__device__ __forceinline__ void load_span(const T* p, int n, typename IO<T>::Acc fill,
                                          typename IO<T>::Acc (&v)[IO<T>::kVec]) {
  if (n >= IO<T>::kVec) {
    IO<T>::unpack(load_packet_unaligned(p), v);
  } else {
#pragma unroll
    for (int e = 0; e < IO<T>::kVec; ++e) v[e] = e < n ? IO<T>::load1(p + e) : fill;
  }
}

// How many of `vec` elements are there where `left` remain.
__device__ __forceinline__ int span_of(int64_t left, int vec) {
  return left < vec ? static_cast<int>(left) : vec;
}
__device__ __forceinline__ int64_t ceil_div_device(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T>
__device__ __forceinline__ void store_span(T* p, int n, const typename IO<T>::Acc (&v)[IO<T>::kVec]) {
  if (n >= IO<T>::kVec) {
    store_packet_unaligned(p, IO<T>::pack(v));
  } else {
#pragma unroll
    for (int e = 0; e < IO<T>::kVec; ++e) {
      if (e < n) IO<T>::store1(p + e, v[e]);
    }
  }
}

// A tensor's memory, as the host's checks of arguments see it; a null pointer is no tensor.
struct Span {
  const void* p;
  uint64_t bytes;
};
// Bytes of a tensor of these extents (none negative), or more than any memory holds.
inline uint64_t bytes_of(uint64_t element, int64_t a, int64_t b = 1, int64_t c = 1) {
  uint64_t n = element;
  for (const int64_t extent : {a, b, c}) {
    if (__builtin_mul_overflow(n, static_cast<uint64_t>(extent), &n)) return UINT64_MAX;
  }
  return n;
}
inline bool overlap(const Span& a, const Span& b) {
  if (!a.p || !b.p || a.bytes == 0 || b.bytes == 0) return false;
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.p), q = reinterpret_cast<uintptr_t>(b.p);
  return p <= q ? q - p < a.bytes : p - q < b.bytes;
}
// Whether an output shares memory with none of the others.
inline bool apart(const Span& out, std::initializer_list<Span> others) {
  for (const Span& other : others) {
    if (overlap(out, other)) return false;
  }
  return true;
}
// Whether an output is the very buffer of each of these inputs of its size, or shares nothing with it.
inline bool on_or_apart(const Span& out, std::initializer_list<Span> inputs) {
  for (const Span& in : inputs) {
    if (out.p != in.p && overlap(out, in)) return false;
  }
  return true;
}

} // namespace dragon_hip
