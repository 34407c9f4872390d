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

// How exponentials of logits at a temperature are taken. `scale` turns a logit into the domain
// that running maxima m are held in; term(x) is exp of the logit x relative to m, shrink(d) the
// factor that a maximum which grows by -d leaves to a sum.
//   16-bit logits: the base-2 domain, one fused multiply-add and the hardware's exp2 per element.
//   The roundings of scale and m move a term by parts in 10^6, a thousandth of a logit's own.
//   32-bit logits: the natural domain, so that the argument of the largest terms, near 0, is
//   exact to its last bits; then exp2. 64-bit logits: the library's exp.
template <typename T>
struct ExpMath {
  using A = typename IO<T>::Acc;
  static constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
  static constexpr bool kBase2 = sizeof(T) == 2;
  static __device__ __forceinline__ A scale(A inv_t) {
    if constexpr (kBase2) return inv_t * kLog2e;
    return inv_t;
  }
  static __device__ __forceinline__ A shrink(A d) {
    if constexpr (kBase2) return __builtin_amdgcn_exp2f(d);
    else if constexpr (sizeof(A) == 4) return __builtin_amdgcn_exp2f(d * kLog2e);
    else return acc_exp(d);
  }
  static __device__ __forceinline__ A term(A x, A scale, A m) { return shrink(fma(x, scale, -m)); }
  // log of a sum relative to m, and a natural logarithm in the domain of m
  static __device__ __forceinline__ A log_of(A m, A s) {
    if constexpr (kBase2) return (m + __builtin_amdgcn_logf(s)) * kLn2;
    return m + acc_log(s);
  }
  static __device__ __forceinline__ A from_log(A l) {
    if constexpr (kBase2) return l * kLog2e;
    return l;
  }
};

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

// The kVec logits of kPackets packets joined to a thread's pair: one maximum and one rescaling
// for all of them.
template <typename T, int kPackets>
__device__ __forceinline__ void take_packets(const typename IO<T>::Acc (&v)[kPackets][IO<T>::kVec],
                                             const typename IO<T>::Acc scale,
                                             ExpSum<typename IO<T>::Acc>& run) {
  using A = typename IO<T>::Acc;
  A top = v[0][0];
#pragma unroll
  for (int k = 0; k < kPackets; ++k)
#pragma unroll
    for (int e = 0; e < IO<T>::kVec; ++e) top = MaxOp()(top, v[k][e]);
  const A m = MaxOp()(run.m, top * scale);
  const A base = finite_base(m);
  A s = run.s * ExpMath<T>::shrink(run.m - base);
#pragma unroll
  for (int k = 0; k < kPackets; ++k)
#pragma unroll
    for (int e = 0; e < IO<T>::kVec; ++e) s += ExpMath<T>::term(v[k][e], scale, base);
  run = {m, s};
}
template <typename T>
__device__ __forceinline__ void take_one(const typename IO<T>::Acc v, const typename IO<T>::Acc scale,
                                         ExpSum<typename IO<T>::Acc>& run) {
  using A = typename IO<T>::Acc;
  const A m = MaxOp()(run.m, v * scale);
  const A base = finite_base(m);
  run = {m, run.s * ExpMath<T>::shrink(run.m - base) + ExpMath<T>::term(v, scale, base)};
}

// All-reduce over the kTPR threads of a row's group: a wavefront, or a workgroup of several (one
// barrier; `slots` is used once).
template <int kTPR, typename A, typename Op>
__device__ __forceinline__ A group_reduce(A v, Op op, A* slots) {
  if constexpr (kTPR == kWaveSize) return wave_allreduce(v, op);
  else return block_allreduce<kTPR / kWaveSize>(v, op, slots);
}
template <typename T, int kTPR>
__device__ __forceinline__ ExpSum<typename IO<T>::Acc> group_join(
    const ExpSum<typename IO<T>::Acc> v, typename IO<T>::Acc (*slots)[kTPR / kWaveSize]) {
  using A = typename IO<T>::Acc;
  const A m = group_reduce<kTPR>(v.m, MaxOp(), slots[0]);
  return {m, group_reduce<kTPR>(v.s * ExpMath<T>::shrink(v.m - finite_base(m)), SumOp(), slots[1])};
}
template <int kTPR>
__device__ __forceinline__ bool group_any(bool v) {
  if constexpr (kTPR == kWaveSize) return __any(v);
  else return __syncthreads_or(v);
}

// Whether an entry is listed: its class is in the row and its teacher logit is not -inf.
template <typename A, typename IndexT>
__device__ __forceinline__ bool entry_listed(IndexT index, A logit, int64_t C) {
  return index >= 0 && static_cast<int64_t>(index) < C && logit != acc_neg_inf<A>();
}

// A row cut at the 16-byte boundaries of its memory: `head` elements, `packets` whole aligned
// packets, `tail` elements. Head and tail are shorter than a packet.
template <typename T>
struct RowCut {
  int head, tail;
  int64_t packets;
  __device__ __forceinline__ RowCut(const T* row, int64_t C) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15u);
    head = off ? static_cast<int>((16 - off) / sizeof(T)) : 0;
    if (head > C) head = static_cast<int>(C);
    packets = (C - head) / IO<T>::kVec;
    tail = static_cast<int>(C - head - packets * IO<T>::kVec);
  }
};

// The teacher's side and the loss of a row, from the pair of its logits, by the kTPR threads of
// its group.
template <typename T, typename IndexT, int kTPR>
__device__ __forceinline__ void finish_row(const int64_t row, const int64_t C, const int K,
                                           const typename IO<T>::Acc inv_t,
                                           const typename IO<T>::Acc t2, const T* x, const IndexT* index,
                                           const typename IO<T>::Acc* teacher,
                                           const ExpSum<typename IO<T>::Acc> run,
                                           typename IO<T>::Acc* stats, typename IO<T>::Acc* loss,
                                           typename IO<T>::Acc (*slots)[kTPR / kWaveSize]) {
  using A = typename IO<T>::Acc;
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  A m = acc_neg_inf<A>();  // the maximum passes over NaN; the sum keeps it
  for (int k = lane; k < K; k += kTPR) {
    const A logit = teacher[row * K + k];
    if (entry_listed(index[row * K + k], logit, C)) m = MaxOp()(m, logit * inv_t);
  }
  m = group_reduce<kTPR>(m, MaxOp(), slots[0]);
  A total = A(0);
  for (int k = lane; k < K; k += kTPR) {
    const A logit = teacher[row * K + k];
    if (entry_listed(index[row * K + k], logit, C)) total += acc_exp(logit * inv_t - m);
  }
  total = group_reduce<kTPR>(total, SumOp(), slots[1]);
  const A log_total = acc_log(total);
  // a row of nothing but -inf has no distribution
  const A lse = run.m == acc_neg_inf<A>() ? A(__builtin_nanf("")) : ExpMath<T>::log_of(run.m, run.s);
  A part = A(0);
  for (int k = lane; k < K; k += kTPR) {
    const A logit = teacher[row * K + k];
    const IndexT cls = index[row * K + k];
    if (entry_listed(cls, logit, C)) {
      const A log_p = logit * inv_t - m - log_total;
      const A p = acc_exp(log_p);
      const A xk = IO<T>::load1(x + row * C + static_cast<int64_t>(cls)) * inv_t;
      if (p != A(0)) part += p * (log_p - xk + lse);
    }
  }
  part = group_reduce<kTPR>(part, SumOp(), slots[2]);
  if (lane == 0) {
    stats[row] = lse;
    loss[row] = part * t2;
  }
}

// A group of kTPR threads (a wavefront, four of them to a workgroup, or a workgroup) reads segment
// blockIdx.y of a row. Where a row is one segment, it finishes the row; otherwise it leaves its
// pair. Rows that list nothing are not read.
constexpr int kSegmentThreads = 256;
template <typename T, typename IndexT, int kTPR, bool kWhole>
__global__ __launch_bounds__(kSegmentThreads) void distill_forward_segments(
    const int64_t N, const int64_t C, const int K, const int64_t segment_packets,
    const typename IO<T>::Acc inv_t, const typename IO<T>::Acc t2, const T* __restrict__ x,
    const IndexT* __restrict__ index, const typename IO<T>::Acc* __restrict__ teacher,
    typename IO<T>::Acc* __restrict__ stats, typename IO<T>::Acc* __restrict__ loss,
    ExpSum<typename IO<T>::Acc>* __restrict__ pairs) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  constexpr int kUnroll = 4;
  __shared__ A slots[5][kTPR / kWaveSize];
  constexpr int kRows = kSegmentThreads / kTPR;
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  const A scale = ExpMath<T>::scale(inv_t);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTPR; row < N;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    bool listed = false;
    for (int k = lane; k < K; k += kTPR)
      listed |= entry_listed(index[row * K + k], teacher[row * K + k], C);
    if (!group_any<kTPR>(listed)) {
      if (lane == 0 && blockIdx.y == 0) {
        stats[row] = -acc_neg_inf<A>();
        loss[row] = A(0);
      }
      continue;
    }
    const T* xr = x + row * C;
    const RowCut<T> cut(xr, C);
    const T* body = xr + cut.head;
    ExpSum<A> run = {acc_neg_inf<A>(), A(0)};
    int64_t p = static_cast<int64_t>(blockIdx.y) * segment_packets;
    const int64_t end = p + segment_packets < cut.packets ? p + segment_packets : cut.packets;
    if (blockIdx.y == 0) {
      if (lane < cut.head) take_one<T>(IO<T>::load1(xr + lane), scale, run);
      if (lane < cut.tail) take_one<T>(IO<T>::load1(body + cut.packets * kVec + lane), scale, run);
    }
    for (; p + kUnroll * kTPR <= end; p += kUnroll * kTPR) {
      u32x4 raw[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) raw[k] = load_packet(body + (p + k * kTPR + lane) * kVec);
      A v[kUnroll][kVec];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) IO<T>::unpack(raw[k], v[k]);
      take_packets<T, kUnroll>(v, scale, run);
    }
    for (p += lane; p < end; p += kTPR) {
      A v[1][kVec];
      load_unpack<T>(body + p * kVec, v[0]);
      take_packets<T, 1>(v, scale, run);
    }
    run = group_join<T, kTPR>(run, slots);
    if constexpr (kWhole) {
      finish_row<T, IndexT, kTPR>(row, C, K, inv_t, t2, x, index, teacher, run, stats, loss, slots + 2);
    } else if (lane == 0) {
      pairs[row * gridDim.y + blockIdx.y] = run;
    }
    if constexpr (kTPR > kWaveSize) __syncthreads();  // slots are reused by the next row
  }
}

// Joins the pairs of a row's segments and finishes the row: a wavefront per row.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kSegmentThreads) void distill_forward_join(
    const int64_t N, const int64_t C, const int K, const int segments, const typename IO<T>::Acc inv_t,
    const typename IO<T>::Acc t2, const T* __restrict__ x, const IndexT* __restrict__ index,
    const typename IO<T>::Acc* __restrict__ teacher, typename IO<T>::Acc* __restrict__ stats,
    typename IO<T>::Acc* __restrict__ loss, const ExpSum<typename IO<T>::Acc>* __restrict__ pairs) {
  using A = typename IO<T>::Acc;
  constexpr int kRows = kSegmentThreads / kWaveSize;
  const int lane = static_cast<int>(threadIdx.x) % kWaveSize;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kWaveSize; row < N;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    bool listed = false;
    for (int k = lane; k < K; k += kWaveSize)
      listed |= entry_listed(index[row * K + k], teacher[row * K + k], C);
    if (!__any(listed)) continue;  // written by the row's first segment
    ExpSum<A> run = {acc_neg_inf<A>(), A(0)};
    for (int i = lane; i < segments; i += kWaveSize) {
      const ExpSum<A> other = pairs[row * segments + i];
      const A m = MaxOp()(run.m, other.m);
      const A base = finite_base(m);
      run = {m, run.s * ExpMath<T>::shrink(run.m - base) + other.s * ExpMath<T>::shrink(other.m - base)};
    }
    run = group_join<T, kWaveSize>(run, static_cast<A(*)[1]>(nullptr));
    finish_row<T, IndexT, kWaveSize>(row, C, K, inv_t, t2, x, index, teacher, run, stats, loss,
                                     static_cast<A(*)[1]>(nullptr));
  }
}

// How a row is cut into segments. A wavefront takes rows of up to 512 packets whole. Longer rows are
// read by workgroups, 4096 packets (16 per thread) at most at a time, and 1024 at least where
// there are too few rows to give every compute unit eight workgroups.
struct SegmentPlan {
  bool wave_rows;
  int64_t segments, packets;  // per row, per segment
};
inline SegmentPlan plan_segments(int64_t N, int64_t C, int vec) {
  const int64_t packets = ceil_div(C, vec);
  if (packets <= 512) return {true, 1, packets};
  const int64_t fewest = ceil_div(packets, 4096), most = ceil_div(packets, 1024);
  int64_t segments = ceil_div(static_cast<int64_t>(num_cus()) * 8, N > 0 ? N : 1);
  segments = segments < fewest ? fewest : (segments > most ? most : segments);
  if (segments > 32768) segments = 32768;  // a launch's second extent holds 65535
  const int64_t each = ceil_div(packets, segments);
  return {false, ceil_div(packets, each), each};
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
  const SegmentPlan plan = plan_segments(N, C, IO<T>::kVec);
  ExpSum<A>* pairs = static_cast<ExpSum<A>*>(scratch);
  A* rows = reduce ? static_cast<A*>(scratch) + 2 * N * plan.segments : static_cast<A*>(loss);
  const T* xp = static_cast<const T*>(x);
  const IndexT* ip = static_cast<const IndexT*>(index);
  const A* tp = static_cast<const A*>(teacher);
  A* sp = static_cast<A*>(stats);
  const A inv_t = A(1) / A(temperature), t2 = A(temperature) * A(temperature);
  const int k = static_cast<int>(K);
  if (N > 0) {
    const dim3 block(kSegmentThreads), waves(row_grid(N, kSegmentThreads / kWaveSize));
    const dim3 grid(row_grid(N, 1), static_cast<unsigned>(plan.segments));
    if (plan.wave_rows) {
      hipLaunchKernelGGL((distill_forward_segments<T, IndexT, kWaveSize, true>), waves, block, 0, stream, N,
                         C, k, plan.packets, inv_t, t2, xp, ip, tp, sp, rows, pairs);
    } else if (plan.segments == 1) {
      hipLaunchKernelGGL((distill_forward_segments<T, IndexT, kSegmentThreads, true>), grid, block, 0,
                         stream, N, C, k, plan.packets, inv_t, t2, xp, ip, tp, sp, rows, pairs);
    } else {
      hipLaunchKernelGGL((distill_forward_segments<T, IndexT, kSegmentThreads, false>), grid, block, 0,
                         stream, N, C, k, plan.packets, inv_t, t2, xp, ip, tp, sp, rows, pairs);
      hipLaunchKernelGGL((distill_forward_join<T, IndexT>), waves, block, 0, stream, N, C, k,
                         static_cast<int>(plan.segments), inv_t, t2, xp, ip, tp, sp, rows, pairs);
    }
  }
  if (reduce) {
    hipLaunchKernelGGL((distill_reduce<A>), dim3(1), dim3(kLoopThreads), 0, stream, N, normalizer, rows,
                       sp, static_cast<A*>(loss));
  } else {
    hipLaunchKernelGGL((distill_no_reduction<A>), dim3(1), dim3(1), 0, stream, N, sp);
  }
  return status_of_launch();
}

// ------------------------------------------------------------------ gradient

// A workgroup writes the gradient of a segment of a row: the softmax everywhere, then, behind a
// barrier, the listed classes of the segment again with the teacher's share taken off. The logits
// of those are read before the first store, so that dx may lie on x.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kSegmentThreads) void distill_backward_segments(
    const int64_t N, const int64_t C, const int K, const int64_t segment_packets,
    const typename IO<T>::Acc inv_t, const typename IO<T>::Acc temperature, const bool per_row, const T* x,
    const IndexT* index, const typename IO<T>::Acc* teacher, const typename IO<T>::Acc* stats,
    const typename IO<T>::Acc* dl, T* dx) {
  using A = typename IO<T>::Acc;
  using Math = ExpMath<T>;
  constexpr int kVec = IO<T>::kVec, kThreads = kSegmentThreads, kWaves = kThreads / kWaveSize;
  constexpr int kUnroll = 4, kMine = kMaxK / kThreads;  // entries of a thread
  __shared__ A slots[2][kWaves];
  __shared__ int classes[kMaxK];
  __shared__ A shares[kMaxK];
  const int lane = threadIdx.x;
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const A lse = stats[row];
    T* out = dx + row * C;
    const T* in = x + row * C;
    const RowCut<T> cut(out, C);  // stores are aligned; loads are where x and dx lie alike
    const bool first = blockIdx.y == 0;
    int64_t p = static_cast<int64_t>(blockIdx.y) * segment_packets;
    const int64_t end = p + segment_packets < cut.packets ? p + segment_packets : cut.packets;
    if (lse == -acc_neg_inf<A>()) {  // ignored
      A zero[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) zero[e] = A(0);
      if (first && lane < cut.head) IO<T>::store1(out + lane, A(0));
      if (first && lane < cut.tail) IO<T>::store1(out + cut.head + cut.packets * kVec + lane, A(0));
      for (p += lane; p < end; p += kThreads) pack_store<T>(out + cut.head + p * kVec, zero);
      continue;
    }
    const A divisor = stats[N];
    const A w = dl[per_row ? row : 0] * temperature / (divisor > A(0.5) ? divisor : A(0.5));
    const A scale = Math::scale(inv_t), base = Math::from_log(lse);
    // the teacher's shares; entry k belongs to thread k % kThreads
    A z[kMine], m = acc_neg_inf<A>();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int k = i * kThreads + lane;
      z[i] = acc_neg_inf<A>();
      if (k < K) {
        const IndexT cls = index[row * K + k];
        const A logit = teacher[row * K + k];
        const bool listed = entry_listed(cls, logit, C);
        classes[k] = listed ? static_cast<int>(cls) : -1;
        if (listed) {
          z[i] = logit * inv_t;
          m = MaxOp()(m, z[i]);
        }
      }
    }
    m = block_allreduce<kWaves>(m, MaxOp(), slots[0]);
    A total = A(0);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      z[i] = z[i] == acc_neg_inf<A>() ? A(0) : acc_exp(z[i] - m);
      total += z[i];
    }
    total = block_allreduce<kWaves>(total, SumOp(), slots[1]);
    // the listed classes of this segment; the row's head and tail are the first segment's
    A kept[kMine];
    bool here[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int k = i * kThreads + lane;
      here[i] = false;
      kept[i] = A(0);
      if (k < K) {
        shares[k] = z[i] / total;
        const int64_t cls = classes[k];
        const bool edge = cls < cut.head || cls >= cut.head + cut.packets * kVec;
        here[i] = cls >= 0 && (edge ? first : cls >= cut.head + p * kVec && cls < cut.head + end * kVec);
        if (here[i]) kept[i] = IO<T>::load1(in + cls);
      }
    }
    __syncthreads();
    if (first) {
      if (lane < cut.head) IO<T>::store1(out + lane, w * Math::term(IO<T>::load1(in + lane), scale, base));
      const int64_t at = cut.head + cut.packets * kVec + lane;
      if (lane < cut.tail) IO<T>::store1(out + at, w * Math::term(IO<T>::load1(in + at), scale, base));
    }
    const T* src = in + cut.head;
    T* dst = out + cut.head;
    for (; p + kUnroll * kThreads <= end; p += kUnroll * kThreads) {
      u32x4 raw[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        raw[k] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4_unaligned*>(src + (p + k * kThreads + lane) * kVec));
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        A v[kVec];
        IO<T>::unpack(raw[k], v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = w * Math::term(v[e], scale, base);
        pack_store<T>(dst + (p + k * kThreads + lane) * kVec, v);
      }
    }
    for (p += lane; p < end; p += kThreads) {
      A v[kVec];
      IO<T>::unpack(load_packet_unaligned(src + p * kVec), v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = w * Math::term(v[e], scale, base);
      pack_store<T>(dst + p * kVec, v);
    }
    __syncthreads();  // the second store of a listed class comes behind the first
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if (!here[i]) continue;
      const int cls = classes[i * kThreads + lane];
      A share = A(0);
      for (int k = 0; k < K; ++k) share += classes[k] == cls ? shares[k] : A(0);
      IO<T>::store1(out + cls, w * (Math::term(kept[i], scale, base) - share));
    }
    __syncthreads();  // classes and shares are reused by the next row
  }
}

template <typename T, typename IndexT>
int launch_backward(int64_t N, int64_t C, int64_t K, float temperature, float normalizer, const void* x,
                    const void* index, const void* teacher, const void* stats, const void* dl, void* dx,
                    hipStream_t stream) {
  using A = typename IO<T>::Acc;
  const SegmentPlan plan = plan_segments(N, C, IO<T>::kVec);
  hipLaunchKernelGGL((distill_backward_segments<T, IndexT>),
                     dim3(row_grid(N, 1), static_cast<unsigned>(plan.segments)),
                     dim3(kSegmentThreads), 0, stream, N, C, static_cast<int>(K), plan.packets,
                     A(1) / A(temperature), A(temperature), normalizer == 0.f, static_cast<const T*>(x),
                     static_cast<const IndexT*>(index), static_cast<const A*>(teacher),
                     static_cast<const A*>(stats), static_cast<const A*>(dl), static_cast<T*>(dx));
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
  const int vec = dtype == DRAGON_HIP_F64 ? 2 : (dtype == DRAGON_HIP_F32 ? 4 : 8);
  // a pair per segment, then a loss per row
  return static_cast<size_t>(N) * (2 * plan_segments(N, C, vec).segments + 1) * acc;
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
