// Verification of drafted tokens against the target's probabilities, for gfx950.
//
// Position i of a sequence is accepted while u_i q_i(d_i) < p_i(d_i); at the first refusal n one
// token is drawn from max(p_n - q_n, 0) by the inverse of its running sum, so that the accepted
// tokens and the drawn one together follow the target's distribution. Per sequence one row of
// the target and at most one of the draft is read, whatever K: the rest are single elements.
//
// Tokens are whole numbers and must not depend on the order of sums: u q and p are compared in
// 64 bits (exact for 32- and 16-bit probabilities: 24 + 24 bits), and running sums are held in
// 64 bits, where another order moves them by parts in 10^16.
#include <climits>

#include "row_loop.h"
#include "row_tile.h"
#include "span.h"

namespace dragon_hip {
namespace {

// A probability: anything negative or not finite counts as 0 (the maximum drops NaN).
template <typename A>
__device__ __forceinline__ double weight_of(A p) {
  const A v = MaxOp()(p, A(0));
  return static_cast<double>(v < -acc_neg_inf<A>() ? v : A(0));
}

// How many of a sequence's drafted tokens pass, found by one wavefront, 64 positions at a time:
// the first lane that refuses ends it.
template <typename T, typename IndexT>
__device__ __forceinline__ int64_t count_accepted(const int64_t b, const int64_t K, const int64_t C,
                                                  const int64_t len, const T* target, const T* draft,
                                                  const IndexT* drafted, const float* u_accept) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  for (int64_t first = 0; first < len; first += kWaveSize) {
    const int64_t i = first + lane;
    bool refuse = false;
    if (i < len) {
      const int64_t d = static_cast<int64_t>(drafted[b * K + i]);
      refuse = true;
      if (d >= 0 && d < C) {
        const double p = weight_of(IO<T>::load1(target + (b * (K + 1) + i) * C + d));
        const double q =
            draft ? weight_of(IO<T>::load1(draft + (b * K + i) * C + d)) : 1.0;
        refuse = !(static_cast<double>(u_accept[b * K + i]) * q < p);
      }
    }
    const unsigned long long refused = __ballot(refuse);
    if (refused) return first + __builtin_ctzll(refused);
  }
  return len;
}

// The row that a sequence's token is drawn from: max(p - q, 0), with q a row of the draft, or all
// of the probability on the class `spike` (-1: nothing is taken off).
template <typename T>
struct SampleRow {
  using A = typename IO<T>::Acc;
  static constexpr int kVec = IO<T>::kVec;
  const T* p;
  const T* q;
  int64_t spike;
  // The kVec classes from `col`: their weights, and what the target alone gives them.
  __device__ __forceinline__ void weigh(int64_t col, const A (&a)[kVec], const A (&b)[kVec],
                                        double (&w)[kVec], double (&plain)[kVec]) const {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      plain[e] = weight_of(a[e]);
      const double d = plain[e] - weight_of(b[e]);
      w[e] = col + e == spike ? 0.0 : (d > 0.0 ? d : 0.0);
    }
  }
  // A packet of them that may reach behind `end`, where there are none.
  __device__ __forceinline__ void weights(int64_t col, int64_t end, double (&w)[kVec],
                                          double (&plain)[kVec]) const {
    A a[kVec], b[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) a[e] = b[e] = A(0);
    if (col < end) {
      const int n = span_of(end - col, kVec);
      load_span<T>(p + col, n, A(0), a);
      if (q) load_span<T>(q + col, n, A(0), b);
    }
    weigh(col, a, b, w, plain);
  }
};
template <typename T>
__device__ __forceinline__ SampleRow<T> plain_row(const SampleRow<T>& r) {
  return {r.p, nullptr, -1};
}

// Inclusive sums over a wavefront's lanes.
__device__ __forceinline__ double wave_scan(double v) {
  const int lane = threadIdx.x & (kWaveSize - 1);
#pragma unroll
  for (int o = 1; o < kWaveSize; o <<= 1) {
    const double up = __shfl_up(v, o, kWaveSize);
    if (lane >= o) v += up;
  }
  return v;
}

// A workgroup of 1024 threads reads a part of a row in steps of 1024 packets and keeps the sum of
// each wavefront's 64 packets of each step: kMaxSteps * 16 runs in the order of the classes. The
// run that holds the level is then read once more, out of the L2, by one wavefront.
constexpr int kMaxSteps = 64;
constexpr int kRuns = kMaxSteps * kLoopWaves;
template <typename T>
constexpr int64_t step_classes() { return static_cast<int64_t>(kLoopThreads) * IO<T>::kVec; }

// Sums of the runs of [begin, end), at most kMaxSteps steps, into `runs`; their total, and that of
// the target alone, for every thread. Holds barriers; `runs` and `slots` may be read behind it.
struct Totals {
  double weight, plain;
};
template <typename T>
__device__ __forceinline__ Totals sum_runs(const SampleRow<T>& row, int64_t begin, int64_t end,
                                           double* runs, double (*slots)[kLoopWaves]) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  // steps requested before the first is summed: 64 and 128 KB per workgroup; with four of eight
  // classes a thread spills
  constexpr int kAtOnce = kVec == 8 ? 2 : 4;
  constexpr int64_t kStep = step_classes<T>();
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  double weight = 0.0, plain = 0.0;
  int step = 0;
  auto take = [&](int at_step, const double(&w)[kVec], const double(&pl)[kVec]) {
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      sum += w[e];
      plain += pl[e];
    }
    sum = wave_allreduce(sum, SumOp());
    weight += sum;
    if (lane == 0) runs[at_step * kLoopWaves + wave] = sum;
  };
  int64_t at = begin + static_cast<int64_t>(threadIdx.x) * kVec;
  for (; begin + kAtOnce * kStep <= end; begin += kAtOnce * kStep, at += kAtOnce * kStep, step += kAtOnce) {
    u32x4 rp[kAtOnce], rq[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      rp[k] = load_packet_unaligned(row.p + at + k * kStep);
      if (row.q) rq[k] = load_packet_unaligned(row.q + at + k * kStep);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      A a[kVec], b[kVec];
      IO<T>::unpack(rp[k], a);
      if (row.q) {
        IO<T>::unpack(rq[k], b);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) b[e] = A(0);
      }
      double w[kVec], pl[kVec];
      row.weigh(at + k * kStep, a, b, w, pl);
      take(step + k, w, pl);
      __builtin_amdgcn_sched_barrier(0);  // one packet's 64-bit values at a time
    }
  }
  for (; begin < end; begin += kStep, at += kStep, ++step) {
    double w[kVec], pl[kVec];
    row.weights(at, end, w, pl);
    take(step, w, pl);
  }
  weight = block_allreduce<kLoopWaves>(lane == 0 ? weight : 0.0, SumOp(), slots[0]);
  return {weight, block_allreduce<kLoopWaves>(plain, SumOp(), slots[1])};
}

// The lowest class of [begin, end) whose running sum, from `before` at begin, exceeds `level`; the
// last class of non-zero weight where rounding leaves none; -1 where there is no weight. Called
// by the first wavefront, behind sum_runs of the same part.
template <typename T>
__device__ __forceinline__ int64_t pick_class(const SampleRow<T>& row, int64_t begin, int64_t end,
                                              double before, const double level, const double* runs) {
  constexpr int kVec = IO<T>::kVec;
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int64_t steps = ceil_div_device(end - begin, step_classes<T>());
  const int count = static_cast<int>(steps) * kLoopWaves;
  // the first run behind which the sum exceeds the level, else the last one with weight
  int chosen = -1, last = -1;
  double at = before, chosen_before = before, last_before = before;
  for (int first = 0; first < count && chosen < 0; first += kWaveSize) {
    const double mine = first + lane < count ? runs[first + lane] : 0.0;
    const double upto = wave_scan(mine);
    const unsigned long long hit = __ballot(mine > 0.0 && at + upto > level);
    const unsigned long long any = __ballot(mine > 0.0);
    const int l = hit ? __builtin_ctzll(hit) : (any ? 63 - __builtin_clzll(any) : 0);
    const double from = at + __shfl(upto - mine, l, kWaveSize);
    if (hit) chosen = first + l, chosen_before = from;
    else if (any) last = first + l, last_before = from;
    at += __shfl(upto, kWaveSize - 1, kWaveSize);
  }
  if (chosen < 0) {
    if (last < 0) return -1;
    chosen = last, chosen_before = last_before;
  }
  const int64_t col = begin + (static_cast<int64_t>(chosen) * kWaveSize + lane) * kVec;
  double w[kVec], plain[kVec];
  row.weights(col, end, w, plain);
  double mine = 0.0;
  int64_t held = -1;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    mine += w[e];
    if (w[e] > 0.0) held = col + e;
  }
  double run = chosen_before + (wave_scan(mine) - mine);
  int64_t found = -1;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    run += w[e];
    if (found < 0 && w[e] > 0.0 && run > level) found = col + e;
  }
  const unsigned long long hit = __ballot(found >= 0);
  if (hit) return __shfl(found, __builtin_ctzll(hit), kWaveSize);
  const unsigned long long any = __ballot(held >= 0);
  return any ? __shfl(held, 63 - __builtin_clzll(any), kWaveSize) : -1;
}

template <typename IndexT>
__device__ __forceinline__ int64_t length_of(const IndexT* lengths, int64_t b, int64_t K) {
  if (!lengths) return K;
  const int64_t len = static_cast<int64_t>(lengths[b]);
  return len < 0 ? 0 : (len > K ? K : len);
}
template <typename T, typename IndexT>
__device__ __forceinline__ SampleRow<T> sample_row(int64_t b, int64_t K, int64_t C, int64_t n, int64_t len,
                                                   const T* target, const T* draft, const IndexT* drafted) {
  SampleRow<T> row = {target + (b * (K + 1) + n) * C, nullptr, -1};
  if (n < len) {
    if (draft) row.q = draft + (b * K + n) * C;
    else row.spike = static_cast<int64_t>(drafted[b * K + n]);
  }
  return row;
}
__device__ __forceinline__ double level_of(float u, double total) {
  return u > 0.f ? static_cast<double>(u) * total : 0.0;
}

// A sequence by one workgroup: rows of one part.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kLoopThreads) void draft_verify_rows(
    const int64_t B, const int64_t K, const int64_t C, const T* __restrict__ target,
    const T* __restrict__ draft, const IndexT* __restrict__ drafted, const IndexT* __restrict__ lengths,
    const float* __restrict__ u_accept, const float* __restrict__ u_sample, IndexT* __restrict__ tokens,
    IndexT* __restrict__ accepted) {
  __shared__ double runs[kRuns];
  __shared__ double slots[2][kLoopWaves];
  __shared__ int64_t count;
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    const int64_t len = length_of(lengths, b, K);
    if (threadIdx.x < kWaveSize) {
      const int64_t n = count_accepted(b, K, C, len, target, draft, drafted, u_accept);
      if (threadIdx.x == 0) count = n;
    }
    __syncthreads();
    const int64_t n = count;
    SampleRow<T> row = sample_row(b, K, C, n, len, target, draft, drafted);
    double total = sum_runs(row, 0, C, runs, slots).weight;
    if (!(total > 0.0) && (row.q || row.spike >= 0)) {  // a residual without weight gives way to the target
      __syncthreads();
      row = plain_row(row);
      total = sum_runs(row, 0, C, runs, slots).weight;
    }
    if (threadIdx.x < kWaveSize) {
      const int64_t token = pick_class(row, 0, C, 0.0, level_of(u_sample[b], total), runs);
      if (threadIdx.x == 0) {
        tokens[b * (K + 1) + n] = static_cast<IndexT>(token);
        accepted[b] = static_cast<IndexT>(n);
      }
    }
    for (int64_t i = threadIdx.x; i <= K; i += kLoopThreads) {
      if (i != n) tokens[b * (K + 1) + i] = i < n ? drafted[b * K + i] : IndexT(-1);
    }
    __syncthreads();  // runs, slots and count are reused by the next sequence
  }
}

// Rows cut into parts, for long rows of few sequences: first the totals of every part, of the
// residual and of the target itself, then a workgroup per sequence finds the part that holds the
// level and does as above with it.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kLoopThreads) void draft_verify_parts(
    const int64_t B, const int64_t K, const int64_t C, const int64_t part, const T* __restrict__ target,
    const T* __restrict__ draft, const IndexT* __restrict__ drafted, const IndexT* __restrict__ lengths,
    const float* __restrict__ u_accept, IndexT* __restrict__ accepted, Totals* __restrict__ totals) {
  __shared__ double runs[kRuns];
  __shared__ double slots[2][kLoopWaves];
  __shared__ int64_t count;
  const int64_t begin = blockIdx.y * part;
  const int64_t end = begin + part < C ? begin + part : C;
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    const int64_t len = length_of(lengths, b, K);
    if (threadIdx.x < kWaveSize) {
      const int64_t n = count_accepted(b, K, C, len, target, draft, drafted, u_accept);
      if (threadIdx.x == 0) count = n;
    }
    __syncthreads();
    const int64_t n = count;
    const SampleRow<T> row = sample_row(b, K, C, n, len, target, draft, drafted);
    const Totals total = sum_runs(row, begin, end, runs, slots);
    if (threadIdx.x == 0) {
      totals[b * gridDim.y + blockIdx.y] = total;
      if (blockIdx.y == 0) accepted[b] = static_cast<IndexT>(n);
    }
    __syncthreads();
  }
}
template <typename T, typename IndexT>
__global__ __launch_bounds__(kLoopThreads) void draft_verify_join(
    const int64_t B, const int64_t K, const int64_t C, const int64_t part, const int parts,
    const T* __restrict__ target, const T* __restrict__ draft, const IndexT* __restrict__ drafted,
    const IndexT* __restrict__ lengths, const float* __restrict__ u_sample, IndexT* __restrict__ tokens,
    const IndexT* __restrict__ accepted, const Totals* __restrict__ totals) {
  __shared__ double runs[kRuns];
  __shared__ double slots[2][kLoopWaves];
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    const int64_t len = length_of(lengths, b, K);
    const int64_t n = static_cast<int64_t>(accepted[b]);
    SampleRow<T> row = sample_row(b, K, C, n, len, target, draft, drafted);
    const Totals* sums = totals + b * parts;
    double total = 0.0;
    for (int i = 0; i < parts; ++i) total += sums[i].weight;
    const bool plain = !(total > 0.0);  // a residual without weight gives way to the target
    if (plain) {
      row = plain_row(row);
      total = 0.0;
      for (int i = 0; i < parts; ++i) total += sums[i].plain;
    }
    const double level = level_of(u_sample[b], total);
    // the part that holds the level, else the last one with weight
    int chosen = -1, last = 0;
    double at = 0.0, before = 0.0, last_before = 0.0;
    for (int i = 0; i < parts && chosen < 0; ++i) {
      const double sum = plain ? sums[i].plain : sums[i].weight;
      if (sum > 0.0) {
        last = i, last_before = at;
        if (at + sum > level) chosen = i, before = at;
      }
      at += sum;
    }
    if (chosen < 0) chosen = last, before = last_before;
    const int64_t begin = chosen * part;
    const int64_t end = begin + part < C ? begin + part : C;
    sum_runs(row, begin, end, runs, slots);
    int64_t token = -1;
    if (threadIdx.x < kWaveSize) token = pick_class(row, begin, end, before, level, runs);
    if (threadIdx.x == 0) tokens[b * (K + 1) + n] = static_cast<IndexT>(token);
    for (int64_t i = threadIdx.x; i <= K; i += kLoopThreads) {
      if (i != n) tokens[b * (K + 1) + i] = i < n ? drafted[b * K + i] : IndexT(-1);
    }
    __syncthreads();
  }
}

// Parts of a row: one where a workgroup's runs hold it and there are sequences enough to fill the
// device, or the row is short; else parts of at least four steps (the loads that a workgroup has
// in flight at once), twice as many workgroups as compute units at most.
struct PartPlan {
  int64_t parts, classes;  // per row, per part
};
template <typename T>
PartPlan plan_parts(int64_t B, int64_t C) {
  const int64_t steps = ceil_div(C, step_classes<T>());
  const int64_t fewest = ceil_div(steps, kMaxSteps);
  int64_t parts = ceil_div(static_cast<int64_t>(num_cus()) * 2, B > 0 ? B : 1);
  if (parts > steps / 4) parts = steps / 4;
  if (B * 2 > num_cus() || parts < 1) parts = 1;
  if (parts < fewest) parts = fewest;
  const int64_t each = ceil_div(steps, parts);
  return {ceil_div(steps, each), each * step_classes<T>()};
}

template <typename T, typename IndexT>
int launch_verify(int64_t B, int64_t K, int64_t C, const void* target, const void* draft,
                  const void* drafted, const void* lengths, const void* u_accept, const void* u_sample,
                  void* tokens, void* accepted, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  const T* tp = static_cast<const T*>(target);
  const T* qp = static_cast<const T*>(draft);
  const IndexT* dp = static_cast<const IndexT*>(drafted);
  const IndexT* lp = static_cast<const IndexT*>(lengths);
  const float* ua = static_cast<const float*>(u_accept);
  const float* us = static_cast<const float*>(u_sample);
  IndexT* op = static_cast<IndexT*>(tokens);
  IndexT* ap = static_cast<IndexT*>(accepted);
  const PartPlan plan = plan_parts<T>(B, C);
  const unsigned grid = row_grid(B, 1);
  if (plan.parts == 1) {
    hipLaunchKernelGGL((draft_verify_rows<T, IndexT>), dim3(grid), dim3(kLoopThreads), 0, stream, B, K, C,
                       tp, qp, dp, lp, ua, us, op, ap);
  } else {
    Totals* totals = static_cast<Totals*>(scratch);
    if (!totals || scratch_bytes < static_cast<size_t>(B * plan.parts) * sizeof(Totals))
      return DRAGON_HIP_ESCRATCH;
    hipLaunchKernelGGL((draft_verify_parts<T, IndexT>), dim3(grid, static_cast<unsigned>(plan.parts)),
                       dim3(kLoopThreads), 0, stream, B, K, C, plan.classes, tp, qp, dp, lp, ua, ap, totals);
    hipLaunchKernelGGL((draft_verify_join<T, IndexT>), dim3(grid), dim3(kLoopThreads), 0, stream, B, K, C,
                       plan.classes, static_cast<int>(plan.parts), tp, qp, dp, lp, us, op, ap, totals);
  }
  return status_of_launch();
}

template <typename T>
int launch_verify_index(int index_dtype, int64_t B, int64_t K, int64_t C, const void* target,
                        const void* draft, const void* drafted, const void* lengths,
                        const void* u_accept, const void* u_sample, void* tokens, void* accepted,
                        void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (index_dtype == DRAGON_HIP_I32)
    return launch_verify<T, int32_t>(B, K, C, target, draft, drafted, lengths, u_accept, u_sample, tokens,
                                     accepted, scratch, scratch_bytes, stream);
  return launch_verify<T, int64_t>(B, K, C, target, draft, drafted, lengths, u_accept, u_sample, tokens,
                                   accepted, scratch, scratch_bytes, stream);
}

template <typename T>
size_t verify_scratch_bytes(int64_t B, int64_t C) {
  const PartPlan plan = plan_parts<T>(B, C);
  return plan.parts == 1 ? 0 : static_cast<size_t>(B * plan.parts) * sizeof(Totals);
}

} // namespace
} // namespace dragon_hip

extern "C" {

using namespace dragon_hip;

size_t dragon_hip_draft_verify_scratch_bytes(int dtype, int64_t B, int64_t K, int64_t C) {
  if (B <= 0 || B > INT_MAX || K < 0 || C <= 0 || C > INT_MAX) return 0;
  switch (dtype) {
    case DRAGON_HIP_F16: return verify_scratch_bytes<f16_t>(B, C);
    case DRAGON_HIP_BF16: return verify_scratch_bytes<bf16_t>(B, C);
    case DRAGON_HIP_F32: return verify_scratch_bytes<float>(B, C);
    case DRAGON_HIP_F64: return verify_scratch_bytes<double>(B, C);
    default: return 0;
  }
}

int dragon_hip_draft_verify(int dtype, int index_dtype, int64_t B, int64_t K, int64_t C,
                            const void* target, const void* draft, const void* drafted,
                            const void* lengths, const void* u_accept, const void* u_sample,
                            void* tokens, void* accepted, void* scratch, size_t scratch_bytes,
                            void* stream) {
  if (index_dtype != DRAGON_HIP_I32 && index_dtype != DRAGON_HIP_I64) return DRAGON_HIP_EDTYPE;
  if (B < 0 || B > INT_MAX || K < 0 || K >= INT_MAX || C <= 0 || C > INT_MAX) return DRAGON_HIP_EINVAL;
  if (B == 0) return DRAGON_HIP_OK;
  if (!target || !u_sample || !tokens || !accepted || (K > 0 && (!drafted || !u_accept)))
    return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_DTYPE(dtype, launch_verify_index, index_dtype, B, K, C, target, draft, drafted,
                            lengths, u_accept, u_sample, tokens, accepted, scratch, scratch_bytes, s);
}

} // extern "C"
