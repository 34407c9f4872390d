// RMSNorm with the residual's addition, its 8-bit form and its gradient, for gfx950.
//
//   s = x + residual,  rsig = (mean(s^2) + eps)^(-1/2),  y = s * rsig * gamma,  h = s
//   z = dy * gamma,  dx = dh + rsig * (z - h * rsig^2 * mean(z * h)),  dgamma = sum dy * h * rsig
//
// The gradient follows from d rsig / d s_j = -rsig^3 s_j / C. All three are bound by HBM: x and
// residual in, h and y out; h, dy and dh in, dx out.
#include <climits>

#include "row_loop.h"
#include "row_tile.h"
#include "span.h"

namespace dragon_hip {
namespace {

constexpr float kFp8Max = 448.f;      // largest e4m3 value
constexpr float kAmaxFloor = 1e-30f;  // keeps the scale of a group of zeros a normal number

// Four values as e4m3 codes, in order from the lowest byte. Round to nearest even. The callers'
// values are y * (448 / max|y|), at most 448 (1 + 2^-23), which rounds to 448.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}

// The codes of the first n of kVec values at an address of any alignment.
typedef uint32_t u32_unaligned __attribute__((may_alias, aligned(1)));
typedef u32x2 u32x2_unaligned __attribute__((may_alias, aligned(1)));
template <int kVec>
__device__ __forceinline__ void store_codes(uint8_t* p, int n, const float (&v)[kVec]) {
  static_assert(kVec == 4 || kVec == 8, "a packet of 32- or 16-bit elements");
  const uint32_t lo = e4m3x4(v[0], v[1], v[2], v[3]);
  uint32_t hi = 0;
  if constexpr (kVec == 8) hi = e4m3x4(v[4], v[5], v[6], v[7]);
  if (n >= kVec) {
    if constexpr (kVec == 8) {
      const u32x2 w = {lo, hi};
      *reinterpret_cast<u32x2_unaligned*>(p) = w;
    } else {
      *reinterpret_cast<u32_unaligned*>(p) = lo;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (e < n) p[e] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
  }
}

// Largest value over `lanes` neighbouring lanes (a power of two, aligned).
__device__ __forceinline__ float cluster_max(float v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) v = MaxOp()(v, __shfl_xor(v, o, kWaveSize));
  return v;
}

// s = x (+ residual) of a packet.
template <typename T>
__device__ __forceinline__ void load_sum(const T* x, const T* residual, int n,
                                         typename IO<T>::Acc (&v)[IO<T>::kVec]) {
  using A = typename IO<T>::Acc;
  load_span<T>(x, n, A(0), v);
  if (residual) {
    A r[IO<T>::kVec];
    load_span<T>(residual, n, A(0), r);
#pragma unroll
    for (int e = 0; e < IO<T>::kVec; ++e) v[e] += r[e];
  }
}

// Any width and alignment: a workgroup walks a row two times (three with a scale per row), the
// later walks out of the L2. h and y are written by the last walk, by the thread that read the
// same elements, so either may lie on x or residual (no pointer is __restrict__).
template <typename T, bool kQuant>
__global__ __launch_bounds__(kLoopThreads) void rms_norm_rows_looped(
    const int64_t N, const int64_t C, const typename IO<T>::Acc eps, const T* x, const T* residual,
    const typename IO<T>::Acc* gamma, T* h, typename IO<T>::Acc* rsig, T* y, const int group,
    const int64_t groups, uint8_t* q, float* scale) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  __shared__ A slots[2][kLoopWaves];
  const int64_t npackets = ceil_div_device(C, kVec);
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* xr = x + row * C;
    const T* rr = residual ? residual + row * C : nullptr;
    A sum = A(0);
    for (int64_t p = threadIdx.x; p < npackets; p += kLoopThreads) {
      const int64_t col = p * kVec;
      A v[kVec];
      load_sum<T>(xr + col, rr ? rr + col : nullptr, span_of(C - col, kVec), v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += v[e] * v[e];
    }
    sum = block_allreduce<kLoopWaves>(sum, SumOp(), slots[0]);
    const A rs = acc_rsqrt_exact(sum / A(C) + eps);
    if (threadIdx.x == 0 && rsig) rsig[row] = rs;
    A row_scale = A(0);
    if constexpr (kQuant) {
      if (group == 0) {
        A top = A(0);
        for (int64_t p = threadIdx.x; p < npackets; p += kLoopThreads) {
          const int64_t col = p * kVec;
          const int n = span_of(C - col, kVec);
          A v[kVec], g[kVec];
          load_sum<T>(xr + col, rr ? rr + col : nullptr, n, v);
          load_params_ragged<kVec>(gamma + col, n, g);
#pragma unroll
          for (int e = 0; e < kVec; ++e) top = MaxOp()(top, fabsf(v[e] * rs * g[e]));
        }
        top = block_allreduce<kLoopWaves>(top, MaxOp(), slots[1]);
        row_scale = MaxOp()(top, kAmaxFloor);
        if (threadIdx.x == 0) scale[row] = row_scale / kFp8Max;
      }
    }
    // every lane takes part in every step: the scales of groups are found across lanes
    for (int64_t first = 0; first < npackets; first += kLoopThreads) {
      const int64_t p = first + threadIdx.x;
      const bool on = p < npackets;
      const int64_t col = p * kVec;
      const int n = on ? span_of(C - col, kVec) : 0;
      A v[kVec], g[kVec];
      if (on) {
        load_sum<T>(xr + col, rr ? rr + col : nullptr, n, v);
        load_params_ragged<kVec>(gamma + col, n, g);
        if (h) store_span<T>(h + row * C + col, n, v);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = on ? v[e] * rs * g[e] : A(0);
      if constexpr (kQuant) {
        float top = row_scale;
        if (group > 0) {
          top = 0.f;
#pragma unroll
          for (int e = 0; e < kVec; ++e) top = MaxOp()(top, fabsf(v[e]));
          top = MaxOp()(cluster_max(top, group / kVec), kAmaxFloor);
          if (on && col % group == 0) scale[row * groups + col / group] = top / kFp8Max;
        }
        const float inv = kFp8Max / top;
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] *= inv;
        if (on) store_codes<kVec>(q + row * C + col, n, v);
      } else {
        if (on) store_span<T>(y + row * C + col, n, v);
      }
    }
    __syncthreads();  // slots are reused by the next row
  }
}

template <typename T>
int launch_rms_norm(int64_t N, int64_t C, float eps, const void* x, const void* residual,
                    const void* gamma, void* h, void* rsig, void* y, hipStream_t stream) {
  using A = typename IO<T>::Acc;
  hipLaunchKernelGGL((rms_norm_rows_looped<T, false>), dim3(loop_grid(N)), dim3(kLoopThreads), 0,
                     stream, N, C, A(eps), static_cast<const T*>(x), static_cast<const T*>(residual),
                     static_cast<const A*>(gamma), static_cast<T*>(h), static_cast<A*>(rsig),
                     static_cast<T*>(y), 0, static_cast<int64_t>(0), static_cast<uint8_t*>(nullptr),
                     static_cast<float*>(nullptr));
  return status_of_launch();
}

template <typename T>
int launch_rms_norm_quant(int64_t N, int64_t C, int64_t group, float eps, const void* x,
                          const void* residual, const void* gamma, void* h, void* rsig, void* q,
                          void* scale, hipStream_t stream) {
  hipLaunchKernelGGL((rms_norm_rows_looped<T, true>), dim3(loop_grid(N)), dim3(kLoopThreads), 0,
                     stream, N, C, eps, static_cast<const T*>(x), static_cast<const T*>(residual),
                     static_cast<const float*>(gamma), static_cast<T*>(h), static_cast<float*>(rsig),
                     static_cast<T*>(nullptr), static_cast<int>(group),
                     group ? ceil_div(C, group) : static_cast<int64_t>(1), static_cast<uint8_t*>(q),
                     static_cast<float*>(scale));
  return status_of_launch();
}

// ------------------------------------------------------------------ gradient

// mean(z * h) * rsig^2 of each row, for the column kernel below.
template <typename T>
__global__ __launch_bounds__(kLoopThreads) void rms_norm_grad_dots(
    const int64_t N, const int64_t C, const T* __restrict__ h,
    const typename IO<T>::Acc* __restrict__ rsig, const typename IO<T>::Acc* __restrict__ gamma,
    const T* __restrict__ dy, typename IO<T>::Acc* __restrict__ coef) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  __shared__ A slots[kLoopWaves];
  const int64_t npackets = ceil_div_device(C, kVec);
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    A sum = A(0);
    for (int64_t p = threadIdx.x; p < npackets; p += kLoopThreads) {
      const int64_t col = p * kVec;
      const int n = span_of(C - col, kVec);
      A a[kVec], b[kVec], g[kVec];
      load_span<T>(h + row * C + col, n, A(0), a);
      load_span<T>(dy + row * C + col, n, A(0), b);
      load_params_ragged<kVec>(gamma + col, n, g);
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += b[e] * g[e] * a[e];
    }
    sum = block_allreduce<kLoopWaves>(sum, SumOp(), slots);
    if (threadIdx.x == 0) {
      const A rs = rsig[row];
      coef[row] = sum / A(C) * rs * rs;
    }
    __syncthreads();
  }
}

// dx, and per chunk of rows the column sums of dy * h * rsig: a thread owns one packet of
// columns and walks its chunk's rows. dx may lie on dy or dh: each element is read and then
// written by one thread.
constexpr int kColThreads = 256;
template <typename T>
__global__ __launch_bounds__(kColThreads) void rms_norm_grad_cols(
    const int64_t N, const int64_t C, const int64_t rows_per_chunk, const T* h,
    const typename IO<T>::Acc* rsig, const typename IO<T>::Acc* gamma, const T* dy, const T* dh,
    const typename IO<T>::Acc* coef, typename IO<T>::Acc* partial, T* dx) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * kColThreads + threadIdx.x) * kVec;
  if (col >= C) return;
  const int n = span_of(C - col, kVec);
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * rows_per_chunk;
  const int64_t end = begin + rows_per_chunk < N ? begin + rows_per_chunk : N;
  A g[kVec], acc[kVec];
  load_params_ragged<kVec>(gamma + col, n, g);
#pragma unroll
  for (int e = 0; e < kVec; ++e) acc[e] = A(0);
  for (int64_t row = begin; row < end; ++row) {
    const int64_t at = row * C + col;
    const A rs = rsig[row], c = coef[row];
    A a[kVec], b[kVec], d[kVec];
    load_span<T>(h + at, n, A(0), a);
    load_span<T>(dy + at, n, A(0), b);
    if (dh) {
      load_span<T>(dh + at, n, A(0), d);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) d[e] = A(0);
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      acc[e] += b[e] * a[e] * rs;
      d[e] += rs * (b[e] * g[e] - a[e] * c);
    }
    store_span<T>(dx + at, n, d);
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    if (e < n) partial[blockIdx.y * C + col + e] = acc[e];
  }
}

// dgamma = the chunks' sums, added in order.
template <typename A>
__global__ __launch_bounds__(kColThreads) void rms_norm_grad_join(const int64_t C, const int64_t chunks,
                                                                  const A* __restrict__ partial,
                                                                  A* __restrict__ dgamma) {
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kColThreads + threadIdx.x;
  if (col >= C) return;
  A sum = A(0);
  for (int64_t p = 0; p < chunks; ++p) sum += partial[p * C + col];
  dgamma[col] = sum;
}

struct GradCols {
  int64_t chunks, rows_per_chunk;
};
inline GradCols plan_grad_cols(int64_t N, int64_t C, int vec) {
  GradCols p;
  const int64_t tiles = ceil_div(C, static_cast<int64_t>(vec) * kColThreads);
  int64_t chunks = ceil_div(static_cast<int64_t>(num_cus()) * 4, tiles);
  if (chunks > N) chunks = N;
  p.rows_per_chunk = ceil_div(N, chunks > 0 ? chunks : 1);
  p.chunks = p.rows_per_chunk > 0 ? ceil_div(N, p.rows_per_chunk) : 0;
  return p;
}

template <typename T>
size_t grad_scratch_bytes(int64_t N, int64_t C) {
  using A = typename IO<T>::Acc;
  const GradCols p = plan_grad_cols(N, C, IO<T>::kVec);
  return static_cast<size_t>(N + p.chunks * C) * sizeof(A);
}

template <typename T>
int launch_rms_norm_grad(int64_t N, int64_t C, const void* h, const void* rsig, const void* gamma,
                         const void* dy, const void* dh, void* dgamma, void* dx, void* scratch,
                         size_t scratch_bytes, hipStream_t stream) {
  using A = typename IO<T>::Acc;
  if (N > 0 && (!scratch || scratch_bytes < grad_scratch_bytes<T>(N, C))) return DRAGON_HIP_ESCRATCH;
  const GradCols p = plan_grad_cols(N, C, IO<T>::kVec);
  A* coef = static_cast<A*>(scratch);
  A* partial = coef + N;
  if (N > 0) {
    hipLaunchKernelGGL((rms_norm_grad_dots<T>), dim3(loop_grid(N)), dim3(kLoopThreads), 0, stream, N, C,
                       static_cast<const T*>(h), static_cast<const A*>(rsig),
                       static_cast<const A*>(gamma), static_cast<const T*>(dy), coef);
    const dim3 grid(static_cast<unsigned>(ceil_div(C, static_cast<int64_t>(IO<T>::kVec) * kColThreads)),
                    static_cast<unsigned>(p.chunks));
    hipLaunchKernelGGL((rms_norm_grad_cols<T>), grid, dim3(kColThreads), 0, stream, N, C,
                       p.rows_per_chunk, static_cast<const T*>(h), static_cast<const A*>(rsig),
                       static_cast<const A*>(gamma), static_cast<const T*>(dy),
                       static_cast<const T*>(dh), coef, partial, static_cast<T*>(dx));
  }
  hipLaunchKernelGGL((rms_norm_grad_join<A>), dim3(static_cast<unsigned>(ceil_div(C, kColThreads))),
                     dim3(kColThreads), 0, stream, C, p.chunks, partial, static_cast<A*>(dgamma));
  return status_of_launch();
}

inline bool sizes_ok(int64_t N, int64_t C) { return N >= 0 && C > 0 && N <= INT_MAX && C <= INT_MAX; }

} // namespace
} // namespace dragon_hip

extern "C" {

using namespace dragon_hip;

int dragon_hip_rms_norm(int dtype, int64_t N, int64_t C, float eps, const void* x,
                        const void* residual, const void* gamma, void* h, void* rsig, void* y,
                        void* stream) {
  if (!sizes_ok(N, C)) return DRAGON_HIP_EINVAL;
  if (N == 0) return DRAGON_HIP_OK;
  if (!x || !gamma || !y || y == h) return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_DTYPE(dtype, launch_rms_norm, N, C, eps, x, residual, gamma, h, rsig, y, s);
}

int dragon_hip_rms_norm_quant(int dtype, int64_t N, int64_t C, int64_t group, float eps,
                              const void* x, const void* residual, const void* gamma, void* h,
                              void* rsig, void* q, void* scale, void* stream) {
  if (dtype != DRAGON_HIP_F16 && dtype != DRAGON_HIP_BF16 && dtype != DRAGON_HIP_F32)
    return DRAGON_HIP_EDTYPE;
  if (!sizes_ok(N, C)) return DRAGON_HIP_EINVAL;
  if (group != 0 && group != 32 && group != 64 && group != 128 && group != 256) return DRAGON_HIP_EINVAL;
  if (N == 0) return DRAGON_HIP_OK;
  if (!x || !gamma || !q || !scale) return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DRAGON_HIP_F16:
      return launch_rms_norm_quant<f16_t>(N, C, group, eps, x, residual, gamma, h, rsig, q, scale, s);
    case DRAGON_HIP_BF16:
      return launch_rms_norm_quant<bf16_t>(N, C, group, eps, x, residual, gamma, h, rsig, q, scale, s);
    default:
      return launch_rms_norm_quant<float>(N, C, group, eps, x, residual, gamma, h, rsig, q, scale, s);
  }
}

size_t dragon_hip_rms_norm_grad_scratch_bytes(int dtype, int64_t N, int64_t C) {
  if (!sizes_ok(N, C) || N == 0) return 0;
  switch (dtype) {
    case DRAGON_HIP_F16: return grad_scratch_bytes<f16_t>(N, C);
    case DRAGON_HIP_BF16: return grad_scratch_bytes<bf16_t>(N, C);
    case DRAGON_HIP_F32: return grad_scratch_bytes<float>(N, C);
    case DRAGON_HIP_F64: return grad_scratch_bytes<double>(N, C);
    default: return 0;
  }
}

int dragon_hip_rms_norm_grad(int dtype, int64_t N, int64_t C, const void* h, const void* rsig,
                             const void* gamma, const void* dy, const void* dh, void* dgamma,
                             void* dx, void* scratch, size_t scratch_bytes, void* stream) {
  if (!sizes_ok(N, C)) return DRAGON_HIP_EINVAL;
  if (!dgamma || (N > 0 && (!h || !rsig || !gamma || !dy || !dx || dx == h))) return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_DTYPE(dtype, launch_rms_norm_grad, N, C, h, rsig, gamma, dy, dh, dgamma, dx,
                            scratch, scratch_bytes, s);
}

} // extern "C"
