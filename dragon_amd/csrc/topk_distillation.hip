// Distillation of a student's logits from a teacher's top logits, forward and backward, for gfx950.
//
//   p_k = softmax over the listed entries of teacher / t,  lse = log sum_v exp(x_v / t)
//   loss of a row = t^2 sum_k p_k (log p_k - x[index_k] / t + lse)
//   dx_v = dl * t * (exp(x_v / t - lse) - sum_{k: index_k = v} p_k) / divisor
//
// The forward reads the logits once (running maximum and sum), the backward reads them once and
// writes the gradient once: both are bound by HBM; the teacher's K entries per row are a few
// hundred bytes against the row's tens or hundreds of KB.
#include <climits>

#include "row_loop.h"
#include "row_tile.h"
#include "span.h"

namespace dragon_hip {
namespace {

constexpr int kMaxK = 1024;

// A running maximum and the sum of exponentials relative to it. An empty pair, and one of
// nothing but -inf, is (-inf, 0); a NaN or +inf among the values makes the sum NaN.
template <typename A>
struct ExpSum {
  A m, s;
};
template <typename A>
__device__ __forceinline__ A finite_base(A m) {
  return m == acc_neg_inf<A>() ? A(0) : m;
}
template <typename A>
__device__ __forceinline__ ExpSum<A> join(const ExpSum<A>& a, const ExpSum<A>& b) {
  const A m = MaxOp()(a.m, b.m);
  const A base = finite_base(m);
  return {m, a.s * acc_exp(a.m - base) + b.s * acc_exp(b.m - base)};
}
// The pair of the whole workgroup, for every thread.
template <int kWaves, typename A>
__device__ __forceinline__ ExpSum<A> block_join(ExpSum<A> v, A (&slots)[2][kWaves]) {
  const A m = block_allreduce<kWaves>(v.m, MaxOp(), slots[0]);
  const A s = block_allreduce<kWaves>(v.s * acc_exp(v.m - finite_base(m)), SumOp(), slots[1]);
  return {m, s};
}

// Whether an entry is listed: its class is in the row and its teacher logit is not -inf.
template <typename A, typename IndexT>
__device__ __forceinline__ bool entry_listed(IndexT index, A logit, int64_t C) {
  return index >= 0 && static_cast<int64_t>(index) < C && logit != acc_neg_inf<A>();
}

// Forward of a row by one workgroup: two reads of K entries and one of the row.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kLoopThreads) void distill_forward_rows(
    const int64_t N, const int64_t C, const int K, const typename IO<T>::Acc inv_t,
    const typename IO<T>::Acc t2, const T* __restrict__ x, const IndexT* __restrict__ index,
    const typename IO<T>::Acc* __restrict__ teacher, typename IO<T>::Acc* __restrict__ stats,
    typename IO<T>::Acc* __restrict__ loss) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  __shared__ A slots[4][2][kLoopWaves];
  const int64_t npackets = ceil_div_device(C, kVec);
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    // the teacher: entry k belongs to thread k
    const bool has = static_cast<int>(threadIdx.x) < K;
    const IndexT cls = has ? index[row * K + threadIdx.x] : IndexT(-1);
    const A logit = has ? teacher[row * K + threadIdx.x] : acc_neg_inf<A>();
    const bool listed = entry_listed(cls, logit, C);
    if (!__syncthreads_or(listed)) {
      if (threadIdx.x == 0) {
        stats[row] = -acc_neg_inf<A>();
        loss[row] = A(0);
      }
      continue;
    }
    const A z = listed ? logit * inv_t : acc_neg_inf<A>();
    const ExpSum<A> tz = block_join<kLoopWaves, A>({z, listed ? A(1) : A(0)}, slots[0]);
    // the student
    ExpSum<A> run = {acc_neg_inf<A>(), A(0)};
    for (int64_t p = threadIdx.x; p < npackets; p += kLoopThreads) {
      const int64_t col = p * kVec;
      A v[kVec];
      load_span<T>(x + row * C + col, span_of(C - col, kVec), acc_neg_inf<A>(), v);
      A top = run.m;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        v[e] *= inv_t;
        top = MaxOp()(top, v[e]);
      }
      const A base = finite_base(top);
      A s = run.s * acc_exp(run.m - base);
#pragma unroll
      for (int e = 0; e < kVec; ++e) s += acc_exp(v[e] - base);
      run = {top, s};
    }
    run = block_join<kLoopWaves, A>(run, slots[1]);
    // a row of nothing but -inf has no distribution
    const A lse = run.m == acc_neg_inf<A>() ? A(__builtin_nanf("")) : run.m + acc_log(run.s);
    A part = A(0);
    if (listed) {
      const A log_p = z - tz.m - acc_log(tz.s);
      const A p = acc_exp(log_p);
      const A xk = IO<T>::load1(x + row * C + static_cast<int64_t>(cls)) * inv_t;
      if (p != A(0)) part = p * (log_p - xk + lse);
    }
    part = block_allreduce<kLoopWaves>(part, SumOp(), slots[2][0]);
    if (threadIdx.x == 0) {
      stats[row] = lse;
      loss[row] = part * t2;
    }
    __syncthreads();
  }
}

// The reduction of the rows' losses, and the divisor behind the rows' statistics. One workgroup,
// rows in a fixed order.
template <typename A>
__global__ __launch_bounds__(kLoopThreads) void distill_reduce(const int64_t N, const float normalizer,
                                                               const A* __restrict__ rows,
                                                               A* __restrict__ stats, A* __restrict__ loss) {
  __shared__ A slots[2][kLoopWaves];
  A sum = A(0), count = A(0);
  for (int64_t i = threadIdx.x; i < N; i += kLoopThreads) {
    sum += rows[i];
    count += stats[i] != -acc_neg_inf<A>() ? A(1) : A(0);
  }
  sum = block_allreduce<kLoopWaves>(sum, SumOp(), slots[0]);
  count = block_allreduce<kLoopWaves>(count, SumOp(), slots[1]);
  if (threadIdx.x == 0) {
    const A divisor = normalizer < 0.f ? count : A(normalizer);
    stats[N] = divisor;
    loss[0] = sum / (divisor > A(1) ? divisor : A(1));
  }
}
template <typename A>
__global__ void distill_no_reduction(const int64_t N, A* __restrict__ stats) {
  stats[N] = A(1);
}

template <typename T, typename IndexT>
int launch_forward(int64_t N, int64_t C, int64_t K, float temperature, float normalizer, const void* x,
                   const void* index, const void* teacher, void* stats, void* loss, void* scratch,
                   hipStream_t stream) {
  using A = typename IO<T>::Acc;
  const bool reduce = normalizer != 0.f;
  A* rows = static_cast<A*>(reduce ? scratch : loss);
  if (N > 0) {
    hipLaunchKernelGGL((distill_forward_rows<T, IndexT>), dim3(loop_grid(N)), dim3(kLoopThreads), 0,
                       stream, N, C, static_cast<int>(K), A(1) / A(temperature),
                       A(temperature) * A(temperature), static_cast<const T*>(x),
                       static_cast<const IndexT*>(index), static_cast<const A*>(teacher),
                       static_cast<A*>(stats), rows);
  }
  if (reduce) {
    hipLaunchKernelGGL((distill_reduce<A>), dim3(1), dim3(kLoopThreads), 0, stream, N, normalizer, rows,
                       static_cast<A*>(stats), static_cast<A*>(loss));
  } else {
    hipLaunchKernelGGL((distill_no_reduction<A>), dim3(1), dim3(1), 0, stream, N, static_cast<A*>(stats));
  }
  return status_of_launch();
}

// ------------------------------------------------------------------ gradient

// A workgroup writes the gradient of a row: first the softmax everywhere, then, behind a
// barrier, the listed classes again with the teacher's share taken off. The logits of the
// listed classes are read before the first store, so that dx may lie on x.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kLoopThreads) void distill_backward_rows(
    const int64_t N, const int64_t C, const int K, const typename IO<T>::Acc inv_t,
    const typename IO<T>::Acc temperature, const bool per_row, const T* x, const IndexT* index,
    const typename IO<T>::Acc* teacher, const typename IO<T>::Acc* stats,
    const typename IO<T>::Acc* dl, T* dx) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  __shared__ A slots[2][kLoopWaves];
  __shared__ int64_t classes[kMaxK];
  __shared__ A shares[kMaxK];
  const int64_t npackets = ceil_div_device(C, kVec);
  const A divisor = stats[N];
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const A lse = stats[row];
    T* out = dx + row * C;
    if (lse == -acc_neg_inf<A>()) {  // ignored
      A zero[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) zero[e] = A(0);
      for (int64_t p = threadIdx.x; p < npackets; p += kLoopThreads) {
        store_span<T>(out + p * kVec, span_of(C - p * kVec, kVec), zero);
      }
      continue;
    }
    const A w = dl[per_row ? row : 0] * temperature / (divisor > A(0.5) ? divisor : A(0.5));
    const bool has = static_cast<int>(threadIdx.x) < K;
    const IndexT cls = has ? index[row * K + threadIdx.x] : IndexT(-1);
    const A logit = has ? teacher[row * K + threadIdx.x] : acc_neg_inf<A>();
    const bool listed = entry_listed(cls, logit, C);
    const A z = listed ? logit * inv_t : acc_neg_inf<A>();
    const ExpSum<A> tz = block_join<kLoopWaves, A>({z, listed ? A(1) : A(0)}, slots);
    const A xk = listed ? IO<T>::load1(x + row * C + static_cast<int64_t>(cls)) : A(0);
    if (has) {
      classes[threadIdx.x] = listed ? static_cast<int64_t>(cls) : -1;
      shares[threadIdx.x] = listed ? acc_exp(z - tz.m) / tz.s : A(0);
    }
    __syncthreads();
    for (int64_t p = threadIdx.x; p < npackets; p += kLoopThreads) {
      const int64_t col = p * kVec;
      const int n = span_of(C - col, kVec);
      A v[kVec];
      load_span<T>(x + row * C + col, n, A(0), v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = w * acc_exp(v[e] * inv_t - lse);
      store_span<T>(out + col, n, v);
    }
    __syncthreads();  // the second store of a listed class comes behind the first
    if (listed) {
      A share = A(0);
      for (int k = 0; k < K; ++k) share += classes[k] == static_cast<int64_t>(cls) ? shares[k] : A(0);
      IO<T>::store1(out + cls, w * (acc_exp(xk * inv_t - lse) - share));
    }
    __syncthreads();
  }
}

template <typename T, typename IndexT>
int launch_backward(int64_t N, int64_t C, int64_t K, float temperature, float normalizer, const void* x,
                    const void* index, const void* teacher, const void* stats, const void* dl, void* dx,
                    hipStream_t stream) {
  using A = typename IO<T>::Acc;
  hipLaunchKernelGGL((distill_backward_rows<T, IndexT>), dim3(loop_grid(N)), dim3(kLoopThreads), 0,
                     stream, N, C, static_cast<int>(K), A(1) / A(temperature), A(temperature),
                     normalizer == 0.f, static_cast<const T*>(x), static_cast<const IndexT*>(index),
                     static_cast<const A*>(teacher), static_cast<const A*>(stats),
                     static_cast<const A*>(dl), static_cast<T*>(dx));
  return status_of_launch();
}

inline bool index_dtype_ok(int t) { return t == DRAGON_HIP_I32 || t == DRAGON_HIP_I64; }
inline bool dtype_ok(int d) { return d >= DRAGON_HIP_F16 && d <= DRAGON_HIP_F64; }
inline bool sizes_ok(int64_t N, int64_t C, int64_t K, float temperature, float normalizer) {
  // a temperature or a normalizer that is NaN fails every comparison
  return N >= 0 && N < INT_MAX && C > 0 && C <= INT_MAX && K > 0 && K <= kMaxK && temperature > 0.f &&
      temperature <= 3.4e38f && normalizer == normalizer;
}

// Calls FN<T, IndexT>(args...).
#define DRAGON_HIP_DISPATCH_INDEXED(dtype, index_dtype, FN, ...)                    \
  switch (dtype) {                                                                  \
    case DRAGON_HIP_F16:                                                            \
      return index_dtype == DRAGON_HIP_I32 ? FN<f16_t, int32_t>(__VA_ARGS__)        \
                                           : FN<f16_t, int64_t>(__VA_ARGS__);       \
    case DRAGON_HIP_BF16:                                                           \
      return index_dtype == DRAGON_HIP_I32 ? FN<bf16_t, int32_t>(__VA_ARGS__)       \
                                           : FN<bf16_t, int64_t>(__VA_ARGS__);      \
    case DRAGON_HIP_F32:                                                            \
      return index_dtype == DRAGON_HIP_I32 ? FN<float, int32_t>(__VA_ARGS__)        \
                                           : FN<float, int64_t>(__VA_ARGS__);       \
    default:                                                                        \
      return index_dtype == DRAGON_HIP_I32 ? FN<double, int32_t>(__VA_ARGS__)       \
                                           : FN<double, int64_t>(__VA_ARGS__);      \
  }

} // namespace
} // namespace dragon_hip

extern "C" {

using namespace dragon_hip;

size_t dragon_hip_topk_distillation_loss_scratch_bytes(int dtype, int64_t N, int64_t C) {
  if (!dtype_ok(dtype) || N < 0 || N >= INT_MAX || C <= 0 || C > INT_MAX) return 0;
  const size_t acc = dtype == DRAGON_HIP_F64 ? 8 : 4;
  return static_cast<size_t>(N) * acc;  // a loss per row
}

int dragon_hip_topk_distillation_loss_forward(int dtype, int index_dtype, int64_t N, int64_t C,
                                              int64_t K, float temperature, float normalizer,
                                              const void* x, const void* index,
                                              const void* teacher, void* stats, void* loss,
                                              void* scratch, size_t scratch_bytes, void* stream) {
  if (!dtype_ok(dtype) || !index_dtype_ok(index_dtype)) return DRAGON_HIP_EDTYPE;
  if (!sizes_ok(N, C, K, temperature, normalizer)) return DRAGON_HIP_EINVAL;
  if (!stats || (N > 0 && (!x || !index || !teacher)) || (!loss && (N > 0 || normalizer != 0.f)))
    return DRAGON_HIP_EINVAL;
  const size_t need = dragon_hip_topk_distillation_loss_scratch_bytes(dtype, N, C);
  if (need > 0 && (!scratch || scratch_bytes < need)) return DRAGON_HIP_ESCRATCH;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_INDEXED(dtype, index_dtype, launch_forward, N, C, K, temperature, normalizer, x,
                              index, teacher, stats, loss, scratch, s);
}

int dragon_hip_topk_distillation_loss_backward(int dtype, int index_dtype, int64_t N, int64_t C,
                                               int64_t K, float temperature, float normalizer,
                                               const void* x, const void* index,
                                               const void* teacher, const void* stats,
                                               const void* dl, void* dx, void* stream) {
  if (!dtype_ok(dtype) || !index_dtype_ok(index_dtype)) return DRAGON_HIP_EDTYPE;
  if (!sizes_ok(N, C, K, temperature, normalizer)) return DRAGON_HIP_EINVAL;
  if (N == 0) return DRAGON_HIP_OK;
  if (!x || !index || !teacher || !stats || !dl || !dx) return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_INDEXED(dtype, index_dtype, launch_backward, N, C, K, temperature, normalizer, x,
                              index, teacher, stats, dl, dx, s);
}

} // extern "C"
