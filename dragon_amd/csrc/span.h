// Pieces of rows at any alignment, shared by the kernels that walk rows packet
// by packet: up to kVec elements from an element-aligned address. And the host's
// check that an output does not lie across a tensor.
#pragma once

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

// Whether two tensors of so many bytes share memory; a null pointer is no tensor.
inline bool overlaps(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return p && q && p < q + b_bytes && q < p + a_bytes;
}
// Whether an output shares memory with an input of its size without being the very buffer of it.
inline bool across(const void* out, const void* in, uint64_t bytes) {
  return out != in && overlaps(out, bytes, in, bytes);
}

} // namespace dragon_hip
