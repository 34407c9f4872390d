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
#include <limits>

#include "row_loop.h"
#include "row_tile.h"
#include "span.h"

namespace dragon_hip {
namespace {

constexpr int kMaxK = 1024;  // entries that a workgroup holds

// How exponentials of logits at a temperature are taken. `scale` turns a logit into the domain
// that running maxima m are held in; term(x) is exp of the logit x relative to m, shrink(d) the
// factor that a maximum which grows by -d leaves to a sum.
//   16-bit logits: the base-2 domain, one fused multiply-add and the hardware's exp2 per element.
//   The rounding of scale moves a term by 2^-24 of its logit's distance from the maximum, that of m all
//   terms alike, by 2^-24 |m| log 2 (8e-5 at most, below kFar); the loss adds distances from the rounded m,
//   in which that cancels.
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
  // log of a sum s relative to m; its two parts, and how far a logit lies below m, apart: the loss
  // adds these, which are smaller than the logarithm itself and lose less in rounding. Halves, so
  // that the type's lowest value has a distance in the base-2 domain too.
  static __device__ __forceinline__ A log_of(A m, A s) {
    if constexpr (kBase2) return fma(m, kLn2, acc_log(s));
    return m + acc_log(s);
  }
  static __device__ __forceinline__ A below(A x, A scale, A m) {
    if constexpr (kBase2) return fma(-x, scale * 0.5f, m * 0.5f) * (2.f * kLn2);
    return fma(-x, scale, m);
  }
  // a natural logarithm in the domain of m
  static __device__ __forceinline__ A from_log(A l) {
    if constexpr (kBase2) return l * kLog2e;
    return l;
  }
};

// A running maximum, never below -kFar, and the sum of exponentials relative to it. An empty pair is
// (-kFar, 0); a NaN or +inf among the values makes the sum NaN.
//
// term() multiplies without rounding and subtracts a maximum that was rounded: the term of the
// maximum itself is exp of that rounding, a part in 10^4 at 2048 and anything from 0 to infinity at
// the lowest value of a type, which masks are made of. The floor keeps masked stretches of a row
// (threads, segments) at sums of 0. Rows whose maximum is not inside (-kFar, kFar) are masked all
// over, or are logits of unusual size: they are read again by far_sum, which subtracts first. In the domain of
// m: 16-bit logits are held in base 2, where kFar is 1420 in x / t. The gradient, which has no maximum, goes by the
// log-sum, and by half of kFar.
constexpr int kFar = 2048;
template <typename A>
struct ExpSum {
  A m, s;
  static __device__ __forceinline__ ExpSum none() { return {A(-kFar), A(0)}; }
  __device__ __forceinline__ bool far() const { return !(m > A(-kFar) && m < A(kFar)); }
};

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
  A s = run.s * ExpMath<T>::shrink(run.m - m);
#pragma unroll
  for (int k = 0; k < kPackets; ++k)
#pragma unroll
    for (int e = 0; e < IO<T>::kVec; ++e) s += ExpMath<T>::term(v[k][e], scale, m);
  run = {m, s};
}
template <typename T>
__device__ __forceinline__ void take_one(const typename IO<T>::Acc v, const typename IO<T>::Acc scale,
                                         ExpSum<typename IO<T>::Acc>& run) {
  using A = typename IO<T>::Acc;
  const A m = MaxOp()(run.m, v * scale);
  run = {m, run.s * ExpMath<T>::shrink(run.m - m) + ExpMath<T>::term(v, scale, m)};
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
  return {m, group_reduce<kTPR>(v.s * ExpMath<T>::shrink(v.m - m), SumOp(), slots[1])};
}
template <int kTPR>
__device__ __forceinline__ bool group_any(bool v) {
  if constexpr (kTPR == kWaveSize) return __any(v);
  else return __syncthreads_or(v);
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

// A row by itself: its largest logit (not scaled), and the sum of exp((x - that) / t). By the kTPR
// threads of a group, which read it twice. A row of nothing but -inf, as one with NaN or +inf,
// has a NaN sum.
template <typename T, int kTPR>
__device__ __forceinline__ ExpSum<typename IO<T>::Acc> far_sum(
    const T* row, int64_t C, typename IO<T>::Acc inv_t, typename IO<T>::Acc (*slots)[kTPR / kWaveSize]) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  A m = acc_neg_inf<A>(), s = A(0);
#pragma unroll 1
  for (int64_t col = static_cast<int64_t>(lane) * kVec; col < C; col += kTPR * kVec) {
    A v[kVec];
    load_span<T>(row + col, span_of(C - col, kVec), acc_neg_inf<A>(), v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) m = MaxOp()(m, v[e]);
  }
  m = group_reduce<kTPR>(m, MaxOp(), slots[0]);
#pragma unroll 1
  for (int64_t col = static_cast<int64_t>(lane) * kVec; col < C; col += kTPR * kVec) {
    const int n = span_of(C - col, kVec);
    A v[kVec];
    load_span<T>(row + col, n, A(0), v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) s += e < n ? acc_exp((v[e] - m) * inv_t) : A(0);
  }
  return {m, group_reduce<kTPR>(s, SumOp(), slots[1])};
}

// The teacher's entries of a row in the registers of its group, one or four to a thread (four
// where K asks for them: they cost a kernel's occupancy): entry k belongs to thread k % kTPR, in
// slot k / kTPR. Everything is requested at once.
constexpr int kWaveK = 4 * kWaveSize;  // entries that a wavefront holds
template <typename T, typename IndexT, int kTPR, int kSlotsT>
struct Entries {
  using A = typename IO<T>::Acc;
  static constexpr int kSlots = kSlotsT;
  int cls[kSlots];  // -1: not listed
  A z[kSlots];      // teacher's logit, -inf where it is not listed
  __device__ __forceinline__ void load(int64_t row, int64_t C, int K, const IndexT* index, const A* teacher) {
    const int lane = static_cast<int>(threadIdx.x) % kTPR;
    IndexT c[kSlots];
    A l[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      c[i] = IndexT(-1);
      l[i] = acc_neg_inf<A>();
      if (i * kTPR + lane < K) {
        c[i] = index[row * K + i * kTPR + lane];
        l[i] = teacher[row * K + i * kTPR + lane];
      }
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const bool listed = c[i] >= 0 && static_cast<int64_t>(c[i]) < C && l[i] != acc_neg_inf<A>();
      cls[i] = listed ? static_cast<int>(c[i]) : -1;
      z[i] = listed ? l[i] : acc_neg_inf<A>();
    }
  }
  __device__ __forceinline__ bool any() const {
    bool on = false;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) on |= cls[i] >= 0;
    return group_any<kTPR>(on);
  }
  // How far entry i lies below the maximum m, at the temperature. The difference comes first: a quotient of
  // its own would be rounded relative to the logit, not to the difference that decides the share (parts in 10^3
  // of it at 30000), and the type's lowest value has none at t < 1.
  __device__ __forceinline__ A offset(int i, A m, A inv_t) const { return (z[i] - m) * inv_t; }
  // Their maximum (which passes over NaN) and the sum of their exponentials (which keeps it).
  __device__ __forceinline__ ExpSum<A> sum(A inv_t, A (*slots)[kTPR / kWaveSize]) const {
    A m = acc_neg_inf<A>();
#pragma unroll
    for (int i = 0; i < kSlots; ++i) m = MaxOp()(m, z[i]);
    m = group_reduce<kTPR>(m, MaxOp(), slots[0]);
    A total = A(0);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) total += cls[i] >= 0 ? acc_exp(offset(i, m, inv_t)) : A(0);
    return {m, group_reduce<kTPR>(total, SumOp(), slots[1])};
  }
};

// The loss of a row from the pair of its logits, by the kTPR threads of its group: every thread has
// it, one writes the row's log-sum.
template <typename T, typename IndexT, int kTPR, int kSlots>
__device__ __forceinline__ typename IO<T>::Acc finish_row(const int64_t row, const int64_t C,
                                           const typename IO<T>::Acc inv_t,
                                           const typename IO<T>::Acc t2, const T* x,
                                           const Entries<T, IndexT, kTPR, kSlots>& entries,
                                           const ExpSum<typename IO<T>::Acc> run,
                                           typename IO<T>::Acc* stats,
                                           typename IO<T>::Acc (*slots)[kTPR / kWaveSize]) {
  using A = typename IO<T>::Acc;
  A xk[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    xk[i] = entries.cls[i] >= 0 ? IO<T>::load1(x + row * C + entries.cls[i]) : A(0);
  const ExpSum<A> t = entries.sum(inv_t, slots);
  const A log_total = acc_log(t.s);
  const A scale = ExpMath<T>::scale(inv_t);
  A log_s = acc_log(run.s), lse = ExpMath<T>::log_of(run.m, run.s);
  const bool far = run.far();
  A largest = A(0);
  if (far) {
    const ExpSum<A> own = far_sum<T, kTPR>(x + row * C, C, inv_t, slots + 3);
    largest = own.m;
    log_s = acc_log(own.s);
    lse = largest * inv_t + log_s;
    // finite, though x / t may not be: +inf stands for an ignored row
    const A most = std::numeric_limits<A>::max();
    lse = lse > most ? most : (lse < -most ? -most : lse);
  }
  A part = A(0);
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    if (entries.cls[i] < 0) continue;
    const A log_p = entries.offset(i, t.m, inv_t) - log_total;
    const A p = acc_exp(log_p);
    const A below = far ? (largest - xk[i]) * inv_t : ExpMath<T>::below(xk[i], scale, run.m);
    if (p != A(0)) part += p * (log_p + (below + log_s));
  }
  part = group_reduce<kTPR>(part, SumOp(), slots[2]);
  if (threadIdx.x % kTPR == 0) stats[row] = lse;
  return part * t2;
}

// The divisor of a reduction.
template <typename A>
__device__ __forceinline__ A divisor_of(const float normalizer, const A count) {
  return normalizer < 0.f ? count : A(normalizer);
}

// The reduction where one workgroup has all rows, one to a wavefront of kRowWaves: the last launch
// does it by itself.
constexpr int kRowWaves = 16;
template <typename A>
__device__ __forceinline__ void reduce_waves(const int64_t N, const float normalizer, const A row_loss,
                                             const A row_count, A* stats, A* loss) {
  __shared__ A rows[2][kRowWaves];
  if (threadIdx.x % kWaveSize == 0) {
    rows[0][threadIdx.x / kWaveSize] = row_loss;
    rows[1][threadIdx.x / kWaveSize] = row_count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    A sum = A(0), count = A(0);
#pragma unroll
    for (int i = 0; i < kRowWaves; ++i) sum += rows[0][i], count += rows[1][i];
    const A divisor = divisor_of(normalizer, count);
    stats[N] = divisor;
    loss[0] = sum / (divisor > A(1) ? divisor : A(1));
  }
}

// A group of kTPR threads (a wavefront, four of them to a workgroup, or a workgroup) reads a segment
// of a row, the segments of a row by neighbouring groups. Where a row is one segment, it finishes
// the row; otherwise it leaves its pair. Rows that list nothing are not read. kReduce: the only
// workgroup, of rows by wavefronts, reduces them too.
constexpr int kSegmentThreads = 256;
constexpr int row_threads(bool reduce) { return reduce ? kRowWaves * kWaveSize : kSegmentThreads; }
template <typename T, typename IndexT, int kTPR, int kSlots, bool kWhole, bool kReduce = false>
__global__ __launch_bounds__(row_threads(kReduce)) void distill_forward_segments(
    const int64_t N, const int64_t C, const int K, const uint32_t segments, const int64_t segment_packets,
    const typename IO<T>::Acc inv_t, const typename IO<T>::Acc t2, const T* __restrict__ x,
    const IndexT* __restrict__ index, const typename IO<T>::Acc* __restrict__ teacher,
    typename IO<T>::Acc* __restrict__ stats, typename IO<T>::Acc* __restrict__ loss,
    ExpSum<typename IO<T>::Acc>* __restrict__ pairs, const float normalizer) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  // the divisor of single losses
  if (!kReduce && normalizer == 0.f && blockIdx.x == 0 && threadIdx.x == 0) stats[N] = A(1);
  constexpr int kUnroll = 4, kTake = 2;  // packets requested at once, and joined at once
  __shared__ A slots[7][kTPR / kWaveSize];
  constexpr int kRows = row_threads(kReduce) / kTPR;
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  A row_loss = A(0), row_count = A(0);
  const A scale = ExpMath<T>::scale(inv_t);
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTPR; item < N * segments;
       item += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t row = kWhole ? item : item / segments;
    const uint32_t segment = kWhole ? 0 : static_cast<uint32_t>(item - row * segments);
    Entries<T, IndexT, kTPR, kSlots> entries;
    entries.load(row, C, K, index, teacher);
    if (!entries.any()) {
      if (lane == 0 && segment == 0) {
        stats[row] = -acc_neg_inf<A>();
        if constexpr (!kReduce) loss[row] = A(0);
      }
      continue;
    }
    const T* xr = x + row * C;
    const RowCut<T> cut(xr, C);
    const T* body = xr + cut.head;
    ExpSum<A> run = ExpSum<A>::none();
    int64_t p = segment * segment_packets;
    const int64_t end = p + segment_packets < cut.packets ? p + segment_packets : cut.packets;
    if (segment == 0) {
      if (lane < cut.head) take_one<T>(IO<T>::load1(xr + lane), scale, run);
      if (lane < cut.tail) take_one<T>(IO<T>::load1(body + cut.packets * kVec + lane), scale, run);
    }
    for (; p + kUnroll * kTPR <= end; p += kUnroll * kTPR) {
      u32x4 raw[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) raw[k] = load_packet(body + (p + k * kTPR + lane) * kVec);
#pragma unroll
      for (int k = 0; k < kUnroll; k += kTake) {
        A v[kTake][kVec];
#pragma unroll
        for (int i = 0; i < kTake; ++i) IO<T>::unpack(raw[k + i], v[i]);
        take_packets<T, kTake>(v, scale, run);
      }
    }
    if (p < end) {  // what is left, requested at once too
      u32x4 raw[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int64_t at = p + k * kTPR + lane;
        raw[k] = load_packet(body + (at < end ? at : p) * kVec);
      }
#pragma unroll
      for (int k = 0; k < kUnroll; k += kTake) {
        A v[kTake][kVec];
#pragma unroll
        for (int i = 0; i < kTake; ++i) {
          const bool on = p + (k + i) * kTPR + lane < end;
          IO<T>::unpack(raw[k + i], v[i]);
#pragma unroll
          for (int e = 0; e < kVec; ++e) v[i][e] = on ? v[i][e] : acc_neg_inf<A>();
        }
        take_packets<T, kTake>(v, scale, run);
      }
    }
    run = group_join<T, kTPR>(run, slots);
    if constexpr (kWhole) {
      row_loss = finish_row<T, IndexT, kTPR, kSlots>(row, C, inv_t, t2, x, entries, run, stats, slots + 2);
      row_count = A(1);
      if (!kReduce && lane == 0) loss[row] = row_loss;
    } else if (lane == 0) {
      pairs[item] = run;
    }
    if constexpr (kTPR > kWaveSize) __syncthreads();  // slots are reused by the next row
  }
  if constexpr (kReduce) reduce_waves(N, normalizer, row_loss, row_count, stats, loss);
}

// Joins the pairs of a row's segments and finishes the row: a wavefront per row, or a workgroup.
template <typename T, typename IndexT, int kTPR, int kSlots, bool kReduce = false>
__global__ __launch_bounds__(row_threads(kReduce)) void distill_forward_join(
    const int64_t N, const int64_t C, const int K, const int segments, const typename IO<T>::Acc inv_t,
    const typename IO<T>::Acc t2, const T* __restrict__ x, const IndexT* __restrict__ index,
    const typename IO<T>::Acc* __restrict__ teacher, typename IO<T>::Acc* __restrict__ stats,
    typename IO<T>::Acc* __restrict__ loss, const ExpSum<typename IO<T>::Acc>* __restrict__ pairs,
    const float normalizer) {
  using A = typename IO<T>::Acc;
  constexpr int kRows = row_threads(kReduce) / kTPR;
  A row_loss = A(0), row_count = A(0);
  __shared__ A slots[7][kTPR / kWaveSize];
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTPR; row < N;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    Entries<T, IndexT, kTPR, kSlots> entries;
    entries.load(row, C, K, index, teacher);
    if (!entries.any()) continue;  // written by the row's first segment, which left no pair
    ExpSum<A> run = ExpSum<A>::none();
    for (int i = lane; i < segments; i += kTPR) {
      const ExpSum<A> other = pairs[row * segments + i];
      const A m = MaxOp()(run.m, other.m);
      run = {m, run.s * ExpMath<T>::shrink(run.m - m) + other.s * ExpMath<T>::shrink(other.m - m)};
    }
    run = group_join<T, kTPR>(run, slots);
    row_loss = finish_row<T, IndexT, kTPR, kSlots>(row, C, inv_t, t2, x, entries, run, stats, slots + 2);
    row_count = A(1);
    if (!kReduce && lane == 0) loss[row] = row_loss;
    if constexpr (kTPR > kWaveSize) __syncthreads();  // slots are reused by the next row
  }
  if constexpr (kReduce) reduce_waves(N, normalizer, row_loss, row_count, stats, loss);
}

// How a row is cut into segments. A wavefront that holds the entries takes rows of up to 512 packets
// whole, and of up to 2048 where there are 2048 rows and more (fp16 [5330, 5440]: 27 us by
// workgroups, 19 by wavefronts). Workgroups take longer rows whole where enough of them fill the
// device, which saves the second launch (bf16 [4096, 32000] 50 -> 47 us, [1000, 32000] 22 -> 17).
// Other rows are cut: 2048 packets (8 per thread) at most at a time (bf16 [4096, 131072]: 153 us;
// 4096 packets 155, 1024 163, for the entries that each reads), and 1024 at least where there
// are too few rows to give every compute unit eight workgroups.
struct SegmentPlan {
  bool wave_rows;
  int64_t segments, packets;  // per row, per segment
};
inline SegmentPlan plan_segments(int64_t N, int64_t C, int64_t K, int vec) {
  const int64_t packets = ceil_div(C, vec);
  const bool waves = K <= kWaveK && packets <= (N >= 2048 ? 2048 : 512);
  const int64_t whole = N >= 2048 ? 8192 : (N >= 512 ? 4096 : 2048);
  if (waves || packets <= whole) return {waves, 1, packets};
  const int64_t fewest = ceil_div(packets, 2048), most = ceil_div(packets, 1024);
  int64_t segments = ceil_div(static_cast<int64_t>(num_cus()) * 8, N > 0 ? N : 1);
  segments = segments < fewest ? fewest : (segments > most ? most : segments);
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
  constexpr int kAtOnce = 8;  // loads in flight: the loop is all latency
  for (int64_t base = 0; base < N; base += kAtOnce * kLoopThreads) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t i = base + k * kLoopThreads + threadIdx.x;
      sum += i < N ? rows[i] : A(0);
      count += i < N && stats[i] != -acc_neg_inf<A>() ? A(1) : A(0);
    }
  }
  sum = block_allreduce<kLoopWaves>(sum, SumOp(), slots[0]);
  count = block_allreduce<kLoopWaves>(count, SumOp(), slots[1]);
  if (threadIdx.x == 0) {
    const A divisor = divisor_of(normalizer, count);
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
  const SegmentPlan plan = plan_segments(N, C, K, IO<T>::kVec);
  // Up to 16 rows that wavefronts finish: one workgroup has them all, and reduces them in the same
  // launch (a call for bf16 [8, 32000]: 17.1 us in three launches, 13.4 in two; for fp32 [16, 2000]
  // 12.9 in two, 9.6 in one).
  const bool reduce = normalizer != 0.f;
  const bool fused = reduce && N > 0 && N <= kRowWaves && K <= kWaveK && (plan.wave_rows || plan.segments > 1);
  ExpSum<A>* pairs = static_cast<ExpSum<A>*>(scratch);
  A* total = static_cast<A*>(loss);
  A* rows = reduce ? static_cast<A*>(scratch) + 2 * N * plan.segments : total;
  const T* xp = static_cast<const T*>(x);
  const IndexT* ip = static_cast<const IndexT*>(index);
  const A* tp = static_cast<const A*>(teacher);
  A* sp = static_cast<A*>(stats);
  const A inv_t = A(1) / A(temperature), t2 = A(temperature) * A(temperature);
  const int k = static_cast<int>(K);
  if (N > 0) {
    const dim3 block(kSegmentThreads), waves(row_grid(N, kSegmentThreads / kWaveSize));
    const dim3 grid(row_grid(N * plan.segments, 1)), one(1), all(row_threads(true));
    const uint32_t segments = static_cast<uint32_t>(plan.segments);
    // GRID, BLOCK, where the losses go, then the kernel's last template arguments
#define SEGMENTS(GRID, BLOCK, LOSSES, ...)                                                             \
  hipLaunchKernelGGL((distill_forward_segments<T, IndexT, __VA_ARGS__>), GRID, BLOCK, 0, stream, N, C, \
                     k, segments, plan.packets, inv_t, t2, xp, ip, tp, sp, LOSSES, pairs, normalizer);
#define JOIN(GRID, BLOCK, LOSSES, ...)                                                                 \
  hipLaunchKernelGGL((distill_forward_join<T, IndexT, __VA_ARGS__>), GRID, BLOCK, 0, stream, N, C, k,  \
                     static_cast<int>(plan.segments), inv_t, t2, xp, ip, tp, sp, LOSSES, pairs, normalizer);
    if (plan.wave_rows) {
      if (fused && K <= 64) SEGMENTS(one, all, total, 64, 1, true, true)
      else if (fused) SEGMENTS(one, all, total, 64, 4, true, true)
      else if (K <= 64) SEGMENTS(waves, block, rows, 64, 1, true)
      else SEGMENTS(waves, block, rows, 64, 4, true)
    } else if (plan.segments == 1) {
      if (K <= kSegmentThreads) SEGMENTS(grid, block, rows, 256, 1, true)
      else SEGMENTS(grid, block, rows, 256, 4, true)
    } else {
      if (K <= kSegmentThreads) SEGMENTS(grid, block, rows, 256, 1, false)
      else SEGMENTS(grid, block, rows, 256, 4, false)
      if (fused && K <= 64) JOIN(one, all, total, 64, 1, true)
      else if (fused) JOIN(one, all, total, 64, 4, true)
      else if (K <= 64) JOIN(waves, block, rows, 64, 1)
      else if (K <= kWaveK) JOIN(waves, block, rows, 64, 4)
      else JOIN(dim3(row_grid(N, 1)), block, rows, 256, 4)
    }
#undef SEGMENTS
#undef JOIN
  }
  if (reduce && !fused) {
    hipLaunchKernelGGL((distill_reduce<A>), dim3(1), dim3(kLoopThreads), 0, stream, N, normalizer, rows,
                       sp, total);
  } else if (N == 0) {
    hipLaunchKernelGGL((distill_no_reduction<A>), dim3(1), dim3(1), 0, stream, N, sp);
  }
  return status_of_launch();
}

// ------------------------------------------------------------------ gradient

// Orders what the threads of a row's group wrote: a workgroup's barrier, or, where the group is one
// wavefront, whose memory operations stay in order, a fence for the compiler.
template <int kTPR>
__device__ __forceinline__ void group_sync() {
  if constexpr (kTPR == kWaveSize) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// The teacher's shares by the threads of a row's group, through its LDS (classes and shares of the K
// entries, padded to a multiple of 4): share[i] is that of the class of the thread's entry i, which
// is the share of every entry of it, four entries at a time, where wanted[i]. It comes back behind a
// barrier of the group.
template <typename T, typename IndexT, int kTPR, int kSlots>
__device__ __forceinline__ void sum_shares(const Entries<T, IndexT, kTPR, kSlots>& entries,
                                           const typename IO<T>::Acc inv_t, const int padded,
                                           const bool (&wanted)[kSlots], int* classes,
                                           typename IO<T>::Acc* shares,
                                           typename IO<T>::Acc (*slots)[kTPR / kWaveSize],
                                           typename IO<T>::Acc (&kept)[kSlots],
                                           typename IO<T>::Acc (&share)[kSlots]) {
  using A = typename IO<T>::Acc;
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  const ExpSum<A> t = entries.sum(inv_t, slots);
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int k = i * kTPR + lane;
    if (k < padded) {
      classes[k] = entries.cls[i];
      shares[k] = entries.cls[i] >= 0 ? acc_exp(entries.offset(i, t.m, inv_t)) / t.s : A(0);
    }
    // its logit has arrived before another thread may write over it
    asm volatile("" : "+v"(kept[i]));
  }
  group_sync<kTPR>();
  bool some = false;
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    some |= wanted[i];
    share[i] = A(0);
  }
  if (some) {
#pragma unroll 2
    for (int k = 0; k < padded; k += 4) {
      int cls[4];
      A of[4];
      const u32x4 packed = *reinterpret_cast<const u32x4_any*>(classes + k);
      cls[0] = packed.x, cls[1] = packed.y, cls[2] = packed.z, cls[3] = packed.w;
#pragma unroll
      for (int j = 0; j < 4; j += 16 / static_cast<int>(sizeof(A))) {
        A part[16 / sizeof(A)];
        IO<A>::unpack(*reinterpret_cast<const u32x4_any*>(shares + k + j), part);
#pragma unroll
        for (int e = 0; e < static_cast<int>(16 / sizeof(A)); ++e) of[j + e] = part[e];
      }
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) share[i] += cls[j] == entries.cls[i] ? of[j] : A(0);
    }
  }
}

// The gradient of a row whose log-sum is so large that its rounding would show in the exponentials: its
// largest logit and sum are found anew, and one group takes the whole row, which no other reads or
// writes, so that dx may lie on x.
template <typename T, typename IndexT, int kTPR, int kSlots>
__device__ __forceinline__ void far_row(const T* in, T* out, const int64_t C, const int padded,
                                        const Entries<T, IndexT, kTPR, kSlots>& entries,
                                        const typename IO<T>::Acc inv_t, const typename IO<T>::Acc w,
                                        int* classes, typename IO<T>::Acc* shares,
                                        typename IO<T>::Acc (*slots)[kTPR / kWaveSize]) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  const int lane = static_cast<int>(threadIdx.x) % kTPR;
  A kept[kSlots], share[kSlots];
  bool here[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    here[i] = entries.cls[i] >= 0;
    kept[i] = here[i] ? IO<T>::load1(in + entries.cls[i]) : A(0);
  }
  sum_shares<T, IndexT, kTPR, kSlots>(entries, inv_t, padded, here, classes, shares, slots, kept, share);
  const ExpSum<A> own = far_sum<T, kTPR>(in, C, inv_t, slots + 2);
  const A inv_s = A(1) / own.s;
#pragma unroll 1
  for (int64_t col = static_cast<int64_t>(lane) * kVec; col < C; col += kTPR * kVec) {
    const int n = span_of(C - col, kVec);
    A v[kVec];
    load_span<T>(in + col, n, A(0), v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = w * (acc_exp((v[e] - own.m) * inv_t) * inv_s);
    store_span<T>(out + col, n, v);
  }
  group_sync<kTPR>();  // the second store of a listed class comes behind the first
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    if (here[i])
      IO<T>::store1(out + entries.cls[i], w * (acc_exp((kept[i] - own.m) * inv_t) * inv_s - share[i]));
  }
  group_sync<kTPR>();  // the entries' LDS is reused by the next item
}

// A group of kTPR threads holds a segment of a row, kVPT packets each, and writes its gradient:
// the softmax everywhere, then the listed classes of the segment again with the teacher's share
// taken off. The segment is requested before the teacher's side is computed, which hides behind
// it, and every logit is read before the first store, so that dx may lie on x. Small segments, of
// neighbouring workgroups, keep what is read and written at a time close together in memory:
// [4096, 131072] bf16 took 374 and 354 us in segments of 4096 and 2048 packets, 346 in segments of
// 1024 and 339 of 512 (a plain copy of its size by workgroups of this shape: 330), and 543 of 256,
// where the teacher's side outweighs the segment. Taking the shares off in the registers of the
// packets' owners instead of storing those classes again took 341 to 393 us, for more work
// between the loads and the stores.
template <typename T, typename IndexT, int kTPR, int kVPT, int kSlots>
__global__ __launch_bounds__(kSegmentThreads) void distill_backward_segments(
    const int64_t N, const int64_t C, const int K, const uint32_t segments, const int64_t segment_packets,
    const typename IO<T>::Acc inv_t, const typename IO<T>::Acc temperature, const bool per_row, const T* x,
    const IndexT* index, const typename IO<T>::Acc* teacher, const typename IO<T>::Acc* stats,
    const typename IO<T>::Acc* dl, T* dx) {
  using A = typename IO<T>::Acc;
  using Math = ExpMath<T>;
  constexpr int kVec = IO<T>::kVec, kRows = kSegmentThreads / kTPR;
  __shared__ A slots[4][kTPR / kWaveSize];
  extern __shared__ u32x4 entry_lds[];  // per group: the shares of K entries, then their classes
  const int lane = static_cast<int>(threadIdx.x) % kTPR, group = static_cast<int>(threadIdx.x) / kTPR;
  const int padded = (K + 3) / 4 * 4;
  A* shares = reinterpret_cast<A*>(entry_lds) + static_cast<int64_t>(group) * padded;
  int* classes = reinterpret_cast<int*>(reinterpret_cast<A*>(entry_lds) + kRows * padded) + group * padded;
  const A scale = Math::scale(inv_t);
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kRows + group; item < N * segments;
       item += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t row = item / segments;
    const uint32_t segment = static_cast<uint32_t>(item - row * segments);
    const A lse = stats[row];
    T* out = dx + row * C;
    const T* in = x + row * C;
    const RowCut<T> cut(out, C);  // stores are aligned; loads are where x and dx lie alike
    const bool first = segment == 0;
    const int64_t tail_at = cut.head + cut.packets * kVec + lane;
    const int64_t begin = segment * segment_packets;
    const int64_t end = begin + segment_packets < cut.packets ? begin + segment_packets : cut.packets;
    if (lse == -acc_neg_inf<A>()) {  // ignored
      A zero[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) zero[e] = A(0);
      if (first && lane < cut.head) IO<T>::store1(out + lane, A(0));
      if (first && lane < cut.tail) IO<T>::store1(out + tail_at, A(0));
      for (int64_t p = begin + lane; p < end; p += kTPR) pack_store<T>(out + cut.head + p * kVec, zero);
      continue;
    }
    if (fabs(lse) > A(kFar / 2)) {
      if (!first) continue;
      Entries<T, IndexT, kTPR, kSlots> entries;
      entries.load(row, C, K, index, teacher);
      const A divisor = stats[N];
      const A w = dl[per_row ? row : 0] * temperature / (divisor > A(0.5) ? divisor : A(0.5));
      far_row<T, IndexT, kTPR, kSlots>(in, out, C, padded, entries, inv_t, w, classes, shares, slots);
      continue;
    }
    u32x4 raw[kVPT];
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      const int64_t p = begin + s * kTPR + lane;
      if (p < end) {
        raw[s] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4_unaligned*>(in + cut.head + p * kVec));
      }
    }
    A head = A(0), tail = A(0);
    if (first && lane < cut.head) head = IO<T>::load1(in + lane);
    if (first && lane < cut.tail) tail = IO<T>::load1(in + tail_at);
    // the teacher's shares
    Entries<T, IndexT, kTPR, kSlots> entries;
    entries.load(row, C, K, index, teacher);
    const A divisor = stats[N];
    const A w = dl[per_row ? row : 0] * temperature / (divisor > A(0.5) ? divisor : A(0.5));
    const A base = Math::from_log(lse);
    // the listed classes of this segment; the row's head and tail are the first segment's
    A kept[kSlots];
    bool here[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int64_t cls = entries.cls[i];
      const bool edge = cls < cut.head || cls >= cut.head + cut.packets * kVec;
      here[i] = cls >= 0 && (edge ? first : cls >= cut.head + begin * kVec && cls < cut.head + end * kVec);
      kept[i] = here[i] ? IO<T>::load1(in + cls) : A(0);
    }
    A share[kSlots];
    sum_shares<T, IndexT, kTPR, kSlots>(entries, inv_t, padded, here, classes, shares, slots, kept, share);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) kept[i] = w * (Math::term(kept[i], scale, base) - share[i]);
    if (first && lane < cut.head) IO<T>::store1(out + lane, w * Math::term(head, scale, base));
    if (first && lane < cut.tail) IO<T>::store1(out + tail_at, w * Math::term(tail, scale, base));
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      const int64_t p = begin + s * kTPR + lane;
      if (p < end) {
        A v[kVec];
        IO<T>::unpack(raw[s], v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = w * Math::term(v[e], scale, base);
        pack_store<T>(out + cut.head + p * kVec, v);
      }
    }
    group_sync<kTPR>();  // the second store of a listed class comes behind the first
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (here[i]) IO<T>::store1(out + entries.cls[i], kept[i]);
    }
    group_sync<kTPR>();  // the entries' LDS is reused by the next item
  }
}

template <typename T, typename IndexT>
int launch_backward(int64_t N, int64_t C, int64_t K, float temperature, float normalizer, const void* x,
                    const void* index, const void* teacher, const void* stats, const void* dl, void* dx,
                    hipStream_t stream) {
  using A = typename IO<T>::Acc;
  const int64_t packets = ceil_div(C, IO<T>::kVec);
  const size_t lds = static_cast<size_t>((K + 3) / 4 * 4) * (sizeof(A) + sizeof(int));
#define LAUNCH(TPR, VPT, SLOTS, SEGMENTS, PACKETS)                                                   \
  {                                                                                                  \
    const int64_t segments = SEGMENTS;                                                               \
    constexpr int kRows = kSegmentThreads / TPR;                                                     \
    hipLaunchKernelGGL((distill_backward_segments<T, IndexT, TPR, VPT, SLOTS>),                             \
                       dim3(row_grid(N * segments, kRows)), dim3(kSegmentThreads), lds * kRows, stream, \
                       N, C, static_cast<int>(K), static_cast<uint32_t>(segments),                   \
                       static_cast<int64_t>(PACKETS), A(1) / A(temperature), A(temperature),         \
                       normalizer == 0.f, static_cast<const T*>(x), static_cast<const IndexT*>(index), \
                       static_cast<const A*>(teacher), static_cast<const A*>(stats),                 \
                       static_cast<const A*>(dl), static_cast<T*>(dx));                              \
  }
  // rows of up to 512 packets by a wavefront, if it holds the entries; longer ones in equal segments
  // of 512 packets at most, or of 1024 where each of them reads more than 64 entries
  if (packets <= 256 && K <= 64) LAUNCH(64, 4, 1, 1, packets)
  else if (packets <= 512 && K <= 64) LAUNCH(64, 8, 1, 1, packets)
  else if (packets <= 256 && K <= kWaveK) LAUNCH(64, 4, 4, 1, packets)
  else if (packets <= 512 && K <= kWaveK) LAUNCH(64, 8, 4, 1, packets)
  else if (K <= 64) LAUNCH(256, 2, 1, ceil_div(packets, 512), ceil_div(packets, segments))
  else if (K <= 256) LAUNCH(256, 4, 1, ceil_div(packets, 1024), ceil_div(packets, segments))
  else LAUNCH(256, 4, 4, ceil_div(packets, 1024), ceil_div(packets, segments))
#undef LAUNCH
  return status_of_launch();
}

inline bool index_dtype_ok(int t) { return t == DRAGON_HIP_I32 || t == DRAGON_HIP_I64; }
inline bool dtype_ok(int d) { return d >= DRAGON_HIP_F16 && d <= DRAGON_HIP_F64; }
inline bool sizes_ok(int64_t N, int64_t C, int64_t K, float temperature, float normalizer) {
  // a temperature or a normalizer that is NaN fails every comparison; beyond these bounds the
  // temperature's reciprocal or square is no 32-bit number
  return N >= 0 && N < INT_MAX && C > 0 && C <= INT_MAX && K > 0 && K <= kMaxK && temperature > 1e-18f &&
      temperature < 1e18f && normalizer == normalizer;
}

// What both calls are given; `loss` is the loss or its gradient.
struct Tensors {
  Span x, index, teacher, stats, loss;
};
inline Tensors tensors_of(int dtype, int index_dtype, int64_t N, int64_t C, int64_t K, const void* x, const void* index,
                          const void* teacher, const void* stats, const void* loss, float normalizer) {
  const int element = dtype == DRAGON_HIP_F64 ? 8 : (dtype == DRAGON_HIP_F32 ? 4 : 2);
  const int acc = dtype == DRAGON_HIP_F64 ? 8 : 4, one = index_dtype == DRAGON_HIP_I32 ? 4 : 8;
  return {{x, bytes_of(element, N, C)}, {index, bytes_of(one, N, K)}, {teacher, bytes_of(acc, N, K)},
          {stats, bytes_of(acc, N + 1)}, {loss, bytes_of(acc, normalizer == 0.f ? N : 1)}};
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
  return static_cast<size_t>(N) * (2 * plan_segments(N, C, kMaxK, vec).segments + 1) * acc;
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
  const Tensors t = tensors_of(dtype, index_dtype, N, C, K, x, index, teacher, stats, loss, normalizer);
  const Span W = {scratch, need};
  if (!apart(t.stats, {t.x, t.index, t.teacher, t.loss}) || !apart(t.loss, {t.x, t.index, t.teacher}) ||
      !apart(W, {t.x, t.index, t.teacher, t.stats, t.loss}))
    return DRAGON_HIP_EINVAL;
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
  const Tensors t = tensors_of(dtype, index_dtype, N, C, K, x, index, teacher, stats, dl, normalizer);
  const Span DX = {dx, t.x.bytes};
  if (!on_or_apart(DX, {t.x}) || !apart(DX, {t.index, t.teacher, t.stats, t.loss})) return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_INDEXED(dtype, index_dtype, launch_backward, N, C, K, temperature, normalizer, x,
                              index, teacher, stats, dl, dx, s);
}

} // extern "C"
