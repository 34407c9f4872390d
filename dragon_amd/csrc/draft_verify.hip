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

// A probability: anything negative or not finite counts as 0.
__device__ __forceinline__ double weight_of(double p) {
  return p > 0.0 && p < __builtin_inf() ? p : 0.0;
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
        const double p = weight_of(static_cast<double>(IO<T>::load1(target + (b * (K + 1) + i) * C + d)));
        const double q =
            draft ? weight_of(static_cast<double>(IO<T>::load1(draft + (b * K + i) * C + d))) : 1.0;
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
  const T* p;
  const T* q;
  int64_t spike;
  __device__ __forceinline__ void weights(int64_t col, int n, double (&w)[IO<T>::kVec]) const {
    using A = typename IO<T>::Acc;
    constexpr int kVec = IO<T>::kVec;
    A a[kVec];
    load_span<T>(p + col, n, A(0), a);
#pragma unroll
    for (int e = 0; e < kVec; ++e) w[e] = weight_of(static_cast<double>(a[e]));
    if (q) {
      A b[kVec];
      load_span<T>(q + col, n, A(0), b);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const double d = w[e] - weight_of(static_cast<double>(b[e]));
        w[e] = d > 0.0 ? d : 0.0;
      }
    }
    if (spike >= col && spike < col + kVec) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = col + e == spike ? 0.0 : w[e];
    }
  }
};

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

// The lowest class of [begin, end) whose running sum, started at `before`, exceeds `level`; the
// last class of non-zero weight where none does; -1 where there is no weight. One wavefront.
template <typename T>
__device__ __forceinline__ int64_t find_class(const SampleRow<T>& row, int64_t begin, int64_t end,
                                              double before, const double level) {
  constexpr int kVec = IO<T>::kVec;
  const int lane = threadIdx.x & (kWaveSize - 1);
  int64_t last = -1;
  for (int64_t base = begin; base < end; base += kWaveSize * kVec) {
    const int64_t col = base + lane * kVec;
    const int n = col < end ? span_of(end - col, kVec) : 0;
    double w[kVec];
    double mine = 0.0;
    int64_t found = -1, seen = -1;
    if (n > 0) {
      row.weights(col, n, w);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (e < n) {
          mine += w[e];
          if (w[e] > 0.0) seen = col + e;
        }
      }
    }
    const double upto = wave_scan(mine);
    double run = before + (upto - mine);
    if (n > 0) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (e < n) {
          run += w[e];
          if (found < 0 && w[e] > 0.0 && run > level) found = col + e;
        }
      }
    }
    const unsigned long long hit = __ballot(found >= 0);
    if (hit) return __shfl(found, __builtin_ctzll(hit), kWaveSize);
    const unsigned long long any = __ballot(seen >= 0);
    if (any) last = __shfl(seen, 63 - __builtin_clzll(any), kWaveSize);
    before += __shfl(upto, kWaveSize - 1, kWaveSize);
  }
  return last;
}

// A workgroup per sequence. Each wavefront sums a contiguous part of the row; the one whose part
// holds the level walks it again, out of the L2, for the class.
template <typename T, typename IndexT>
__global__ __launch_bounds__(kLoopThreads) void draft_verify_rows(
    const int64_t B, const int64_t K, const int64_t C, const T* __restrict__ target,
    const T* __restrict__ draft, const IndexT* __restrict__ drafted, const IndexT* __restrict__ lengths,
    const float* __restrict__ u_accept, const float* __restrict__ u_sample, IndexT* __restrict__ tokens,
    IndexT* __restrict__ accepted) {
  constexpr int kVec = IO<T>::kVec;
  __shared__ double sums[kLoopWaves];
  __shared__ int64_t count;
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  const int64_t part = ceil_div_device(ceil_div_device(C, kVec), kLoopWaves) * kVec;
  const int64_t begin = wave * part < C ? wave * part : C;
  const int64_t end = begin + part < C ? begin + part : C;
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    int64_t len = K;
    if (lengths) {
      len = static_cast<int64_t>(lengths[b]);
      len = len < 0 ? 0 : (len > K ? K : len);
    }
    if (wave == 0) {
      const int64_t n = count_accepted(b, K, C, len, target, draft, drafted, u_accept);
      if (lane == 0) count = n;
    }
    __syncthreads();
    const int64_t n = count;
    SampleRow<T> row = {target + (b * (K + 1) + n) * C, nullptr, -1};
    if (n < len) {
      if (draft) {
        row.q = draft + (b * K + n) * C;
      } else {
        row.spike = static_cast<int64_t>(drafted[b * K + n]);
      }
    }
    double total = 0.0;
    for (int again = 0; again < 2; ++again) {
      double mine = 0.0;
      for (int64_t col = begin + lane * kVec; col < end; col += kWaveSize * kVec) {
        const int n_here = span_of(end - col, kVec);
        double w[kVec];
        row.weights(col, n_here, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) mine += e < n_here ? w[e] : 0.0;
      }
      mine = wave_allreduce(mine, SumOp());
      if (lane == 0) sums[wave] = mine;
      __syncthreads();
      total = 0.0;
      for (int i = 0; i < kLoopWaves; ++i) total += sums[i];
      if (total > 0.0 || (!row.q && row.spike < 0)) break;
      row.q = nullptr, row.spike = -1;  // a residual without weight gives way to the target
      __syncthreads();
    }
    const float u = u_sample[b];
    const double level = u > 0.f ? static_cast<double>(u) * total : 0.0;
    int chosen = -1, last = 0;
    double before = 0.0, at = 0.0;
    for (int i = 0; i < kLoopWaves; ++i) {
      if (sums[i] > 0.0) last = i;
      if (chosen < 0 && before + sums[i] > level) {
        chosen = i;
        at = before;
      }
      before += sums[i];
    }
    if (chosen < 0) {  // u >= 1, or no weight at all
      chosen = last;
      at = 0.0;
    }
    if (wave == chosen) {
      const bool beyond = !(total > level);
      const int64_t token = find_class(row, begin, end, at, beyond ? __builtin_inf() : level);
      if (lane == 0) tokens[b * (K + 1) + n] = static_cast<IndexT>(token);
    }
    for (int64_t i = threadIdx.x; i <= K; i += kLoopThreads) {
      if (i != n) tokens[b * (K + 1) + i] = i < n ? drafted[b * K + i] : IndexT(-1);
    }
    if (threadIdx.x == 0) accepted[b] = static_cast<IndexT>(n);
    __syncthreads();  // sums and count are reused by the next sequence
  }
}

template <typename T, typename IndexT>
int launch_verify(int64_t B, int64_t K, int64_t C, const void* target, const void* draft,
                  const void* drafted, const void* lengths, const void* u_accept, const void* u_sample,
                  void* tokens, void* accepted, hipStream_t stream) {
  hipLaunchKernelGGL((draft_verify_rows<T, IndexT>), dim3(loop_grid(B)), dim3(kLoopThreads), 0, stream, B,
                     K, C, static_cast<const T*>(target), static_cast<const T*>(draft),
                     static_cast<const IndexT*>(drafted), static_cast<const IndexT*>(lengths),
                     static_cast<const float*>(u_accept), static_cast<const float*>(u_sample),
                     static_cast<IndexT*>(tokens), static_cast<IndexT*>(accepted));
  return status_of_launch();
}

template <typename T>
int launch_verify_index(int index_dtype, int64_t B, int64_t K, int64_t C, const void* target,
                        const void* draft, const void* drafted, const void* lengths,
                        const void* u_accept, const void* u_sample, void* tokens, void* accepted,
                        hipStream_t stream) {
  if (index_dtype == DRAGON_HIP_I32)
    return launch_verify<T, int32_t>(B, K, C, target, draft, drafted, lengths, u_accept, u_sample, tokens,
                                     accepted, stream);
  return launch_verify<T, int64_t>(B, K, C, target, draft, drafted, lengths, u_accept, u_sample, tokens,
                                   accepted, stream);
}

} // namespace
} // namespace dragon_hip

extern "C" {

using namespace dragon_hip;

size_t dragon_hip_draft_verify_scratch_bytes(int dtype, int64_t B, int64_t K, int64_t C) {
  return 0;
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
                            lengths, u_accept, u_sample, tokens, accepted, s);
}

} // extern "C"
