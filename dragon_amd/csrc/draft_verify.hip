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

#include "row_tile.h"
#include "span.h"

namespace dragon_hip {
namespace {

// A probability: anything negative or not finite counts as 0. One test for the class of positive
// normal and subnormal numbers.
__device__ __forceinline__ double weight_of(float p) {
  return static_cast<double>(__builtin_amdgcn_classf(p, 0x180) ? p : 0.f);
}
__device__ __forceinline__ double weight_of(double p) { return __builtin_amdgcn_class(p, 0x180) ? p : 0.0; }

template <typename IndexT>
__device__ __forceinline__ int64_t length_of(const IndexT* lengths, int64_t b, int64_t K) {
  if (!lengths) return K;
  const int64_t len = static_cast<int64_t>(lengths[b]);
  return len < 0 ? 0 : (len > K ? K : len);
}

// How many of a sequence's drafted tokens pass, and how many there are. Found by one wavefront, 64
// positions at a time: the first lane that refuses ends it. What a position is decided by is
// requested beside the length, not behind it.
struct Prefix {
  int64_t n, len;
};
template <typename T, typename IndexT>
__device__ __forceinline__ Prefix accepted_prefix(const int64_t b, const int64_t K, const int64_t C,
                                                  const T* target, const T* draft, const IndexT* drafted,
                                                  const IndexT* lengths, const float* u_accept) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  int64_t len = K;
  for (int64_t first = 0; first < K; first += kWaveSize) {
    const int64_t i = first + lane;
    int64_t d = -1;
    float u = 0.f;
    if (i < K) {
      d = static_cast<int64_t>(drafted[b * K + i]);
      u = u_accept[b * K + i];
    }
    if (first == 0) len = length_of(lengths, b, K);
    bool refuse = true;
    if (d >= 0 && d < C) {
      const double p = weight_of(IO<T>::load1(target + (b * (K + 1) + i) * C + d));
      const double q = draft ? weight_of(IO<T>::load1(draft + (b * K + i) * C + d)) : 1.0;
      refuse = !(static_cast<double>(u) * q < p);
    }
    const unsigned long long refused = __ballot(refuse || i >= len);
    if (refused) return {first + __builtin_ctzll(refused), len};
  }
  return {K, len};
}

// A packet that is read once: streams gain a tenth from the non-temporal hint.
template <typename T>
__device__ __forceinline__ u32x4 load_packet_once(const T* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_unaligned*>(p));
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
  // The packet of classes from `at`. One that would reach behind the row's end is moved back to end
  // with it: its first `dup` classes belong to the packet before and weigh nothing here.
  struct Piece {
    int64_t col;
    int dup;
    bool on;
  };
  static __device__ __forceinline__ Piece piece(int64_t at, int64_t end) {
    const bool on = at < end;
    const int64_t col = at + kVec > end && end >= kVec ? end - kVec : at;
    return {on ? col : 0, on ? static_cast<int>(at - col) : kVec, on};
  }
  static __device__ __forceinline__ u32x4 packet(const T* row, const Piece& at, int64_t end) {
    if (end < kVec) {  // rows shorter than a packet
      A v[kVec];
      load_span<T>(row, static_cast<int>(end), A(0), v);
      return IO<T>::pack(v);
    }
    return load_packet_unaligned(row + at.col);
  }
  // The weights of a piece, given its packets. 9 operations per class, three of them in 64 bits, which
  // the 8 bytes per class of 32-bit rows leave time for.
  __device__ __forceinline__ void weigh(int64_t col, const u32x4 tp, const u32x4 tq, double (&w)[kVec]) const {
    A a[kVec], b[kVec];
    IO<T>::unpack(tp, a);
    if (q) {
      IO<T>::unpack(tq, b);
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = MaxOp()(weight_of(a[e]) - weight_of(b[e]), 0.0);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = weight_of(a[e]);
    }
    if (spike >= col && spike < col + kVec) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = col + e == spike ? 0.0 : w[e];
    }
  }
  __device__ __forceinline__ void weigh(const Piece& at, const u32x4 tp, const u32x4 tq, double (&w)[kVec]) const {
    weigh(at.col, tp, tq, w);
#pragma unroll
    for (int e = 0; e < kVec; ++e) w[e] = e >= at.dup ? w[e] : 0.0;
  }
};

// Sum of a 64-bit value over a wavefront, for every lane, in a fixed order: four steps inside rows
// of 16 lanes by the data-parallel moves of the vector unit, then the four rows' results. A third of
// the latency of six shuffles through LDS, which are what short rows wait for.
template <int kCtrl>
__device__ __forceinline__ double dpp_add(double v) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), kCtrl, 0xf, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), kCtrl, 0xf, 0xf, false);
  return v + __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(bits), lane);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), lane);
  return __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
  v = dpp_add<0xB1>(v);   // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);   // quad_perm [2,3,0,1]
  v = dpp_add<0x141>(v);  // row_half_mirror
  v = dpp_add<0x140>(v);  // row_mirror
  return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
// Inclusive sums over a wavefront's lanes, by the same moves: within rows of 16 lanes, then the last
// lane of a row to the next row, then lane 31 to the upper half.
template <int kCtrl, int kRows>
__device__ __forceinline__ double dpp_scan_step(double v) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), kCtrl, kRows, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), kCtrl, kRows, 0xf, false);
  return v + __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = dpp_scan_step<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = dpp_scan_step<0x112, 0xf>(v);
  v = dpp_scan_step<0x114, 0xf>(v);
  v = dpp_scan_step<0x118, 0xf>(v);
  v = dpp_scan_step<0x142, 0xa>(v);  // row_bcast 15, to rows 1 and 3
  v = dpp_scan_step<0x143, 0xc>(v);  // row_bcast 31, to rows 2 and 3
  return v;
}

// A run is 64 packets of classes, a wavefront's reading. Workgroups sum the runs of a row in steps of
// one run per wavefront; whoever picks the class finds the run that holds the level among the
// sums, and only that run is read again.
template <typename T>
constexpr int64_t run_classes() { return static_cast<int64_t>(kWaveSize) * IO<T>::kVec; }

// Sums the runs of [begin, end): f(run, sum) is called by every lane of the wavefront that read it.
// `kWaves` wavefronts take runs in turn, kAtOnce of them requested before the first is summed; the
// last step may reach runs behind the end, of sum 0.
template <int kWaves, int kAtOnce, typename T, typename F>
__device__ __forceinline__ void sum_runs(const SampleRow<T>& row, const int64_t begin, const int64_t end,
                                         F&& f) {
  constexpr int kVec = IO<T>::kVec;
  constexpr int64_t kStep = kWaves * run_classes<T>();
  int64_t run = threadIdx.x / kWaveSize;
  for (int64_t at = begin + static_cast<int64_t>(threadIdx.x) * kVec, base = begin; base < end;
       base += kAtOnce * kStep, at += kAtOnce * kStep) {
    u32x4 rp[kAtOnce], rq[kAtOnce];
    double sum[kAtOnce];
    if (base + kAtOnce * kStep <= end) {
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        rp[k] = load_packet_once(row.p + at + k * kStep);
        if (row.q) rq[k] = load_packet_once(row.q + at + k * kStep);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        double w[kVec];
        row.weigh(at + k * kStep, rp[k], rq[k], w);
        sum[k] = w[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) sum[k] += w[e];
        __builtin_amdgcn_sched_barrier(0);  // one packet's 64-bit values at a time
      }
    } else {
      typename SampleRow<T>::Piece piece[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        piece[k] = row.piece(at + k * kStep, end);
        rp[k] = row.packet(row.p, piece[k], end);
        if (row.q) rq[k] = row.packet(row.q, piece[k], end);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        double w[kVec];
        row.weigh(piece[k], rp[k], rq[k], w);
        sum[k] = w[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) sum[k] += w[e];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) sum[k] = wave_sum(sum[k]);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k, run += kWaves) f(run, sum[k]);
  }
}

// Picks the class by the sums of a row's `count` runs: the lowest one whose running sum exceeds
// u * total; the last class of non-zero weight where rounding (or u >= 1) leaves none; -1 where
// there is no weight. A residual without weight gives way to the target, whose runs are summed
// here and take the others' place. By a workgroup of kWaves wavefronts, each thread of which
// takes a stretch of the runs; the class is returned to the first wavefront.
template <int kWaves, typename T>
__device__ __forceinline__ int64_t pick_class(SampleRow<T> row, const int64_t C, const int64_t count,
                                              double* runs, const float u) {
  constexpr int kVec = IO<T>::kVec, kThreads = kWaves * kWaveSize;
  __shared__ double waves[kWaves];
  __shared__ int64_t hits[kWaves], lasts[kWaves];
  __shared__ double hit_before[kWaves], last_before[kWaves];
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  const int64_t stretch = ceil_div_device(count, kThreads);
  const int64_t from = threadIdx.x * stretch < count ? threadIdx.x * stretch : count;
  const int64_t to = from + stretch < count ? from + stretch : count;
  double mine, upto, total;
  for (;;) {
    mine = 0.0;
    for (int64_t r = from; r < to; ++r) mine += runs[r];
    upto = wave_scan(mine);
    if (lane == kWaveSize - 1) waves[wave] = upto;
    __syncthreads();
    total = 0.0;
    double before = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i == wave) before = total;
      total += waves[i];
    }
    upto += before;
    if (total > 0.0 || (!row.q && row.spike < 0)) break;
    row.q = nullptr, row.spike = -1;
    __syncthreads();  // every thread has read the sums
    sum_runs<kWaves, 2>(row, 0, C, [&](int64_t run, double sum) {
      if (lane == 0 && run < count) runs[run] = sum;
    });
    __syncthreads();
  }
  // from u = 1 on no sum exceeds it: a partial sum may round above a total that was added in another order
  const double level = u > 0.f ? (u < 1.f ? static_cast<double>(u) * total : __builtin_inf()) : 0.0;
  // the first run of the stretch behind which the sum exceeds the level, and the last with weight
  int64_t hit = -1, last = -1;
  double run = upto - mine, at_hit = 0.0, at_last = 0.0;
  if (mine > 0.0) {
    for (int64_t r = from; r < to; ++r) {
      const double w = runs[r];
      if (w > 0.0) {
        if (hit < 0 && run + w > level) hit = r, at_hit = run;
        last = r, at_last = run;
      }
      run += w;
    }
  }
  const unsigned long long hit_lanes = __ballot(hit >= 0), last_lanes = __ballot(last >= 0);
  const int h = hit_lanes ? __builtin_ctzll(hit_lanes) : 0;
  const int l = last_lanes ? 63 - __builtin_clzll(last_lanes) : 0;
  if (lane == h) hits[wave] = hit, hit_before[wave] = at_hit;
  if (lane == l) lasts[wave] = last, last_before[wave] = at_last;
  __syncthreads();
  if (wave != 0) return -1;
  int64_t chosen = -1;
  double before = 0.0;
#pragma unroll
  for (int i = kWaves - 1; i >= 0; --i)
    if (hits[i] >= 0) chosen = hits[i], before = hit_before[i];
  if (chosen < 0) {
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
      if (lasts[i] >= 0) chosen = lasts[i], before = last_before[i];
    if (chosen < 0) return -1;
  }
  const typename SampleRow<T>::Piece piece = row.piece(chosen * run_classes<T>() + lane * kVec, C);
  const int64_t col = piece.col;
  double w[kVec];
  const u32x4 none = {0u, 0u, 0u, 0u};
  row.weigh(piece, row.packet(row.p, piece, C), row.q ? row.packet(row.q, piece, C) : none, w);
  double sum = w[0];
  int64_t held = -1, found = -1;
#pragma unroll
  for (int e = 1; e < kVec; ++e) sum += w[e];
  run = before + (wave_scan(sum) - sum);
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    run += w[e];
    if (w[e] > 0.0) {
      held = col + e;
      if (found < 0 && run > level) found = col + e;
    }
  }
  const unsigned long long found_lanes = __ballot(found >= 0), held_lanes = __ballot(held >= 0);
  if (found_lanes) return __shfl(found, __builtin_ctzll(found_lanes), kWaveSize);
  return held_lanes ? __shfl(held, 63 - __builtin_clzll(held_lanes), kWaveSize) : -1;
}

template <typename T, typename IndexT>
__device__ __forceinline__ SampleRow<T> sample_row(int64_t b, int64_t K, int64_t C, const Prefix& v,
                                                   const T* target, const T* draft, const IndexT* drafted) {
  SampleRow<T> row = {target + (b * (K + 1) + v.n) * C, nullptr, -1};
  if (v.n < v.len) {
    if (draft) row.q = draft + (b * K + v.n) * C;
    else row.spike = static_cast<int64_t>(drafted[b * K + v.n]);
  }
  return row;
}

// A sequence by one workgroup, the sums of its runs in LDS: one launch. Sixteen wavefronts, or eight
// where packets hold eight classes, whose 64-bit values do not fit the registers of sixteen (bf16
// [1, 5, 32000]: 10.2 us a call against 11.8).
template <typename T>
constexpr int rows_waves() { return IO<T>::kVec == 8 ? 8 : 16; }
constexpr int kMaxRuns = 1024;
template <typename T, typename IndexT>
__global__ __launch_bounds__(rows_waves<T>() * kWaveSize) void draft_verify_rows(
    const int64_t B, const int64_t K, const int64_t C, const T* __restrict__ target,
    const T* __restrict__ draft, const IndexT* __restrict__ drafted, const IndexT* __restrict__ lengths,
    const float* __restrict__ u_accept, const float* __restrict__ u_sample, IndexT* __restrict__ tokens,
    IndexT* __restrict__ accepted) {
  constexpr int kRowsWaves = rows_waves<T>();
  __shared__ double runs[kMaxRuns];
  __shared__ Prefix prefix;
  const int lane = threadIdx.x & (kWaveSize - 1);
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    const float u = u_sample[b];
    if (threadIdx.x < kWaveSize) {
      const Prefix v = accepted_prefix(b, K, C, target, draft, drafted, lengths, u_accept);
      if (threadIdx.x == 0) prefix = v;
    }
    __syncthreads();
    const Prefix v = prefix;
    const SampleRow<T> row = sample_row(b, K, C, v, target, draft, drafted);
    sum_runs<kRowsWaves, 2>(row, 0, C, [&](int64_t run, double sum) {
      if (lane == 0 && run < kMaxRuns) runs[run] = sum;
    });
    __syncthreads();
    const int64_t token = pick_class<kRowsWaves>(row, C, ceil_div_device(C, run_classes<T>()), runs, u);
    if (threadIdx.x == 0) {
      tokens[b * (K + 1) + v.n] = static_cast<IndexT>(token);
      accepted[b] = static_cast<IndexT>(v.n);
    }
    for (int64_t i = threadIdx.x; i <= K; i += kRowsWaves * kWaveSize) {
      if (i != v.n) tokens[b * (K + 1) + i] = i < v.n ? drafted[b * K + i] : IndexT(-1);
    }
    __syncthreads();  // the LDS is reused by the next sequence
  }
}

// Long rows: workgroups of four wavefronts sum the runs of a part of a row each, and a second launch
// picks the classes, a workgroup per sequence.
constexpr int kPartWaves = 4;
template <typename T, typename IndexT>
__global__ __launch_bounds__(kPartWaves * kWaveSize) void draft_verify_runs(
    const int64_t B, const int64_t K, const int64_t C, const uint32_t parts, const int64_t part_runs,
    const int64_t row_runs, const T* __restrict__ target, const T* __restrict__ draft,
    const IndexT* __restrict__ drafted, const IndexT* __restrict__ lengths,
    const float* __restrict__ u_accept, IndexT* __restrict__ accepted, double* __restrict__ sums) {
  __shared__ Prefix prefix;
  const int lane = threadIdx.x & (kWaveSize - 1);
  for (int64_t item = blockIdx.x; item < B * parts; item += gridDim.x) {
    const int64_t b = item / parts, part = item - b * parts;
    if (threadIdx.x < kWaveSize) {
      const Prefix v = accepted_prefix(b, K, C, target, draft, drafted, lengths, u_accept);
      if (threadIdx.x == 0) {
        prefix = v;
        if (part == 0) accepted[b] = static_cast<IndexT>(v.n);
      }
    }
    __syncthreads();
    const SampleRow<T> row = sample_row(b, K, C, prefix, target, draft, drafted);
    const int64_t first = part * part_runs, last = first + part_runs < row_runs ? first + part_runs : row_runs;
    const int64_t begin = first * run_classes<T>();
    const int64_t end = last * run_classes<T>() < C ? last * run_classes<T>() : C;
    double* out = sums + b * row_runs + first;
    sum_runs<kPartWaves, IO<T>::kVec == 8 ? 2 : 4>(row, begin, end, [&](int64_t run, double sum) {
      if (lane == 0 && first + run < last) out[run] = sum;
    });
    __syncthreads();  // the prefix is overwritten by the next item's
  }
}
template <typename T, typename IndexT>
__global__ __launch_bounds__(kPartWaves * kWaveSize) void draft_verify_pick(
    const int64_t B, const int64_t K, const int64_t C, const int64_t row_runs, const T* __restrict__ target,
    const T* __restrict__ draft, const IndexT* __restrict__ drafted, const IndexT* __restrict__ lengths,
    const float* __restrict__ u_sample, IndexT* __restrict__ tokens, const IndexT* __restrict__ accepted,
    double* __restrict__ sums) {
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    const Prefix v = {static_cast<int64_t>(accepted[b]), length_of(lengths, b, K)};
    const SampleRow<T> row = sample_row(b, K, C, v, target, draft, drafted);
    const int64_t token = pick_class<kPartWaves>(row, C, row_runs, sums + b * row_runs, u_sample[b]);
    if (threadIdx.x == 0) tokens[b * (K + 1) + v.n] = static_cast<IndexT>(token);
    for (int64_t i = threadIdx.x; i <= K; i += kPartWaves * kWaveSize) {
      if (i != v.n) tokens[b * (K + 1) + i] = i < v.n ? drafted[b * K + i] : IndexT(-1);
    }
    __syncthreads();  // the LDS of pick_class is reused by the next sequence
  }
}

// One workgroup takes a row whole up to 32768 classes, and where there are two sequences and more per
// compute unit; others are cut, for a second launch (3.5 us). The limit counts classes, not bytes: what one
// compute unit spends is its 64-bit work per class. Sampled drafts, us a call, whole / cut:
//            [1, 5, C]: 16384    32768    65536     131072      [64, 5, C]: 32768   65536    [512, 5, C]: 65536
//   bf16         10.3/14.3   10.4/14.3  13.2/14.1  26.7/14.4       12.6/14.5  19.0/14.3        36.7/33.2
//   fp32         10.4/14.1   10.8/14.1  15.6/14.1  29.4/14.3       13.7/14.1  20.0/14.5        43.1/43.6
//   fp64         10.6/14.2   14.4/14.2  24.0/14.1  55.8/14.3       20.9/14.6  35.7/17.3        79.5/73.4
// Between the columns of 32768 and 65536 the two cross for one sequence; fp64, which has half the packets' classes,
// loses above 16384 with several. Beyond two sequences per compute unit neither side is ahead by more than a fifth, and
// whole rows need no scratch. Rows are cut into parts of 4 to 64 runs per wavefront, as many as 16
// workgroups per compute unit make of them: short streams, of neighbouring workgroups, lie close
// together in memory (fp32 [192, 6, 131072]: 47 us with 5 workgroups per compute unit, 38 with 16,
// 37 with 48).
struct PartPlan {
  int64_t parts, part_runs, row_runs;  // parts = 0: whole rows
};
template <typename T>
PartPlan plan_parts(int64_t B, int64_t C) {
  const int64_t runs = ceil_div(C, run_classes<T>());
  if (C <= 32768 || (B >= 2 * num_cus() && runs <= kMaxRuns)) return {0, runs, runs};
  int64_t parts = static_cast<int64_t>(num_cus()) * 16 / B;
  const int64_t most = ceil_div(runs, kPartWaves * 4), fewest = ceil_div(runs, kPartWaves * 64);
  parts = parts > most ? most : (parts < fewest ? fewest : parts);
  const int64_t each = ceil_div(ceil_div(runs, parts), kPartWaves) * kPartWaves;
  return {ceil_div(runs, each), each, runs};
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
  const size_t need = plan.parts == 0 ? 0 : static_cast<size_t>(B * plan.row_runs) * sizeof(double);
  // several workgroups read the inputs of a sequence whose outputs one of them writes
  const Span P = {target, bytes_of(sizeof(T), B, K + 1, C)}, Q = {draft, bytes_of(sizeof(T), B, K, C)};
  const Span D = {drafted, bytes_of(sizeof(IndexT), B, K)}, L = {lengths, bytes_of(sizeof(IndexT), B)};
  const Span U = {u_accept, bytes_of(4, B, K)}, V = {u_sample, bytes_of(4, B)};
  const Span O = {tokens, bytes_of(sizeof(IndexT), B, K + 1)}, N = {accepted, bytes_of(sizeof(IndexT), B)};
  const Span W = {scratch, need};
  if (!apart(O, {P, Q, D, L, U, V, N}) || !apart(N, {P, Q, D, L, U, V}) || !apart(W, {P, Q, D, L, U, V, O, N}))
    return DRAGON_HIP_EINVAL;
  if (plan.parts == 0) {
    hipLaunchKernelGGL((draft_verify_rows<T, IndexT>), dim3(row_grid(B, 1)), dim3(rows_waves<T>() * kWaveSize), 0,
                       stream, B, K, C, tp, qp, dp, lp, ua, us, op, ap);
  } else {
    double* sums = static_cast<double*>(scratch);
    if (!sums || scratch_bytes < need) return DRAGON_HIP_ESCRATCH;
    const dim3 block(kPartWaves * kWaveSize);
    hipLaunchKernelGGL((draft_verify_runs<T, IndexT>), dim3(row_grid(B * plan.parts, 1)), block, 0, stream,
                       B, K, C, static_cast<uint32_t>(plan.parts), plan.part_runs, plan.row_runs, tp, qp, dp,
                       lp, ua, ap, sums);
    hipLaunchKernelGGL((draft_verify_pick<T, IndexT>), dim3(row_grid(B, 1)), block, 0, stream, B, K, C,
                       plan.row_runs, tp, qp, dp, lp, us, op, ap, sums);
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
  return plan.parts == 0 ? 0 : static_cast<size_t>(B * plan.row_runs) * sizeof(double);
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
