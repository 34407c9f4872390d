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

// The codes of a tile's packet, v times `inv`, but for the first `skip`: those of a packet that was
// moved back into a group of another scale.
template <bool kRagged, int kVec>
__device__ __forceinline__ void tile_codes(uint8_t* p, int skip, bool on, float inv, const float (&v)[kVec]) {
  float w[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) w[e] = v[e] * inv;
  if (!on) return;
  if (kRagged && skip > 0) {
    const uint32_t lo = e4m3x4(w[0], w[1], w[2], w[3]);
    uint32_t hi = 0;
    if constexpr (kVec == 8) hi = e4m3x4(w[4], w[5], w[6], w[7]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (e >= skip) p[e] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
  } else {
    store_codes<kVec>(p, kVec, w);
  }
}

// All-reduce over `lanes` neighbouring lanes (4 to 64, a power of two, aligned) by the vector unit's own
// moves: inside rows of 16 lanes, then the rows' results. Shuffles go through LDS, whose latency the
// rows wait for: fp32 [13106, 2560] in groups of 128 columns takes 104 us with them, 73 without.
template <typename Op>
__device__ __forceinline__ float cluster_reduce(float v, int lanes, Op op) {
  v = dpp_step<0xB1>(v, op);                    // quad_perm [1,0,3,2]
  v = dpp_step<0x4E>(v, op);                    // quad_perm [2,3,0,1]
  if (lanes >= 8) v = dpp_step<0x141>(v, op);   // row_half_mirror
  if (lanes >= 16) v = dpp_step<0x140>(v, op);  // row_mirror
  if (lanes >= 32) {
    auto row = [&](int lane) {
      return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    };
    const float low = op(row(0), row(16)), high = op(row(32), row(48));
    if (lanes == 64) v = op(low, high);
    else v = (threadIdx.x & 32) ? high : low;
  }
  return v;
}
template <typename Op>
__device__ __forceinline__ double cluster_reduce(double v, int lanes, Op op) {
  for (int o = 1; o < lanes; o <<= 1) v = op(v, __shfl_xor(v, o, kWaveSize));
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
          top = MaxOp()(cluster_reduce(top, group / kVec, MaxOp()), kAmaxFloor);
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

// ------------------------------------------------------------------ rows held in registers

// Workgroup sizes: rows of up to a wavefront's threads share one of 256 threads.
constexpr int tile_threads(int tpr) { return tpr < 256 ? 256 : tpr; }

// The packets of a row that a thread of a group of kTPR holds: packet s * kTPR + lane in slot s.
// Where rows are not whole aligned packets (kRagged), a row's last packet is moved back to end
// with the row: every access is a whole packet inside the row, and the `dup` elements it shares
// with the packet before it are left out of sums and written twice with the same values.
template <typename T, int kTPR, int kVPT, bool kRagged>
struct RowPackets {
  static constexpr int kVec = IO<T>::kVec;
  int col[kVPT], dup[kVPT];
  bool on[kVPT];
  __device__ __forceinline__ explicit RowPackets(int C) {
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      const int nominal = (s * kTPR + static_cast<int>(threadIdx.x) % kTPR) * kVec;
      on[s] = nominal < C;
      col[s] = on[s] ? nominal : 0;
      dup[s] = 0;
      if (kRagged && on[s] && nominal + kVec > C) {
        col[s] = C - kVec;
        dup[s] = nominal - col[s];
      }
    }
  }
  __device__ __forceinline__ bool counts(int s, int e) const { return !kRagged || e >= dup[s]; }
  // Slots without a packet hold the row's first: they are masked where they are used. Packets that
  // straddle cache lines share them with the neighbouring wavefronts' packets: with the
  // non-temporal hint of whole lines fp32 [9870, 1001] takes 30 us forward, without 26 (the
  // gradient, which reads three tensors for one that it writes, 32 and 32.5: kOnce there).
  template <bool kOnce>
  __device__ __forceinline__ void load(const T* row, u32x4 (&p)[kVPT]) const {
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      if constexpr (kRagged && !kOnce) {
        p[s] = load_packet_unaligned(row + col[s]);
      } else if constexpr (kRagged) {
        p[s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_unaligned*>(row + col[s]));
      } else {
        p[s] = load_packet(row + col[s]);
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int s, const typename IO<T>::Acc (&v)[kVec]) const {
    if constexpr (kRagged) {
      store_packet_unaligned(row + col[s], IO<T>::pack(v));
    } else {
      store_packet(row + col[s], IO<T>::pack(v));
    }
  }
  __device__ __forceinline__ void params(const typename IO<T>::Acc* gamma, int s,
                                         typename IO<T>::Acc (&g)[kVec]) const {
    if constexpr (kRagged) {
      load_params_ragged<kVec>(gamma + col[s], kVec, g);
    } else {
      load_params<kVec>(gamma + col[s], g);
    }
  }
};

// All-reduce over the kTPR threads of a row: lanes of one wavefront, or whole wavefronts through
// LDS with one barrier. Rows alternate between two sets of `slots`, so that the barrier of one
// row keeps the next but one from overwriting what is still being read.
template <int kTPR, typename A, typename Op>
__device__ __forceinline__ A row_allreduce(A v, Op op, A* slots) {
  if constexpr (kTPR < kWaveSize) {
    return cluster_reduce(v, kTPR, op);
  } else {
    v = wave_allreduce(v, op);
    if constexpr (kTPR == kWaveSize) return v;
    constexpr int kWaves = kTPR / kWaveSize;
    A* mine = slots + threadIdx.x / kTPR * kWaves;
    if ((threadIdx.x & (kWaveSize - 1)) == 0) mine[threadIdx.x % kTPR / kWaveSize] = v;
    __syncthreads();
    A r = mine[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) r = op(r, mine[i]);
    return r;
  }
}

enum RmsOut { kPlain = 0, kRowScale = 1, kGroupScale = 2 };

// One read of x and residual, one write of h and y. Workgroups stay and walk the rows, so that
// gamma is loaded once into registers (of tiles of up to two packets per thread), and the next
// row is requested before the current one is summed. Every element of a row is loaded before the
// row's first store: outputs may lie on inputs.
template <typename T, int kTPR, int kVPT, bool kRagged, bool kResidual, int kOut>
__global__ __launch_bounds__(tile_threads(kTPR)) void rms_norm_rows(
    const int64_t N, const int C, const typename IO<T>::Acc eps, const T* x, const T* residual,
    const typename IO<T>::Acc* gamma, T* h, typename IO<T>::Acc* rsig, T* y, const int group,
    const int groups, uint8_t* q, float* scale) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  constexpr int kThreads = tile_threads(kTPR), kRows = kThreads / kTPR;
  constexpr bool kAhead = kVPT <= 2;  // wider tiles leave no registers for gamma and the next row
  __shared__ A slots[2][2][kThreads / kWaveSize];
  const RowPackets<T, kTPR, kVPT, kRagged> tile(C);
  const A inv_c = A(1) / A(C);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTPR;
  u32x4 px[kVPT], pr[kVPT];
  tile.template load<false>(x + (row < N ? row : 0) * C, px);
  if constexpr (kResidual) tile.template load<false>(residual + (row < N ? row : 0) * C, pr);
  A g[kVPT][kVec];
  if constexpr (kAhead) {
#pragma unroll
    for (int s = 0; s < kVPT; ++s) tile.params(gamma, s, g[s]);
  }
  int turn = 0;
  // the trip count is the same for every row of a workgroup: the reductions hold barriers
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < N; base += step) {
    const bool valid = row < N;
    A v[kVPT][kVec];
    A sum = A(0);
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      IO<T>::unpack(px[s], v[s]);
      if constexpr (kResidual) {
        A r[kVec];
        IO<T>::unpack(pr[s], r);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[s][e] += r[e];
      }
      A part = A(0);
#pragma unroll
      for (int e = 0; e < kVec; ++e) part += tile.counts(s, e) ? v[s][e] * v[s][e] : A(0);
      sum += tile.on[s] ? part : A(0);
    }
    const int64_t next = row + step;
    if constexpr (kAhead) {
      tile.template load<false>(x + (next < N ? next : 0) * C, px);
      if constexpr (kResidual) tile.template load<false>(residual + (next < N ? next : 0) * C, pr);
    }
    sum = row_allreduce<kTPR>(sum, SumOp(), slots[turn][0]);
    const A rs = acc_rsqrt_exact(sum * inv_c + eps);
    if (valid && threadIdx.x % kTPR == 0 && rsig) rsig[row] = rs;
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      if (h && valid && tile.on[s]) tile.store(h + row * C, s, v[s]);
      if constexpr (!kAhead) tile.params(gamma, s, g[s]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[s][e] = v[s][e] * rs * g[s][e];
      if constexpr (kOut == kPlain) {
        if (valid && tile.on[s]) tile.store(y + row * C, s, v[s]);
      } else {
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < kVec; ++e) part = MaxOp()(part, tile.counts(s, e) ? fabsf(v[s][e]) : 0.f);
        part = tile.on[s] ? part : 0.f;
        if constexpr (kOut == kRowScale) {
          top = MaxOp()(top, part);
        } else {
          // a group wider than the row stays inside the row's own lanes
          const int lanes = group / kVec < kTPR ? group / kVec : kTPR;
          const float amax = MaxOp()(cluster_reduce(part, lanes, MaxOp()), kAmaxFloor);
          const int nominal = tile.col[s] + tile.dup[s];
          const bool leads = nominal % group == 0;  // its group
          if (valid && tile.on[s] && leads) scale[row * groups + nominal / group] = amax / kFp8Max;
          tile_codes<kRagged>(q + row * C + tile.col[s], leads ? tile.dup[s] : 0, valid && tile.on[s], kFp8Max / amax, v[s]);
        }
      }
    }
    if constexpr (kOut == kRowScale) {
      const float amax = MaxOp()(row_allreduce<kTPR>(top, MaxOp(), slots[turn][1]), kAmaxFloor);
      if (valid && threadIdx.x % kTPR == 0) scale[row] = amax / kFp8Max;
#pragma unroll
      for (int s = 0; s < kVPT; ++s)
        tile_codes<kRagged>(q + row * C + tile.col[s], 0, valid && tile.on[s], kFp8Max / amax, v[s]);
    }
    row = next;
    turn ^= 1;
    if constexpr (!kAhead) {
      tile.template load<false>(x + (row < N ? row : 0) * C, px);
      if constexpr (kResidual) tile.template load<false>(residual + (row < N ? row : 0) * C, pr);
    }
  }
}

// Calls LAUNCH(threads per row, packets per thread) for rows of `packets`: the fewest threads
// that hold the row with up to two packets each, four on the largest workgroup. Powers of two up to 512
// threads, where half-empty slots cost next to nothing (steps of a wavefront: bf16 [13106, 5120] 88.7 us
// against 89.1); beyond them bf16 [7280, 9216] takes 94.5 us by 1024 threads, 89.6 by 640, with e4m3
// codes 86.0 and 77.0.
#define DRAGON_HIP_RMS_SWITCH_2(packets, LAUNCH)  \
  if (packets <= 8) LAUNCH(8, 1)                  \
  else if (packets <= 16) LAUNCH(16, 1)           \
  else if (packets <= 32) LAUNCH(32, 1)           \
  else if (packets <= 64) LAUNCH(64, 1)           \
  else if (packets <= 128) LAUNCH(64, 2)          \
  else if (packets <= 256) LAUNCH(128, 2)         \
  else if (packets <= 512) LAUNCH(256, 2)         \
  else if (packets <= 1024) LAUNCH(512, 2)        \
  else if (packets <= 1280) LAUNCH(640, 2)        \
  else if (packets <= 1536) LAUNCH(768, 2)        \
  else LAUNCH(1024, 2)
#define DRAGON_HIP_RMS_SWITCH(packets, LAUNCH) \
  if (packets > 2048) LAUNCH(1024, 4)          \
  else DRAGON_HIP_RMS_SWITCH_2(packets, LAUNCH)
constexpr int64_t kMaxTilePackets = 4096;

// Workgroups that walk the rows: eight wavefronts per compute unit, each with its next row's packets
// in flight. Measured with four, eight and as many wavefronts as fit (sixteen to
// twenty-four): bf16 [8192, 8192] with a residual 109 us at four, 91 at eight, 92 at twenty-four, 99
// with a workgroup per row; its gradient at [8192, 4096] 49 us at eight, 53 at sixteen, 58 at
// thirty-two. More streams at a time are further apart in memory, and leave more partial sums.
// Quantised rows compute more per byte and wait for more reductions; those that leave a sixteenth of the
// tile's slots and more empty take twice as many, in workgroups of up to 512 threads: in groups of 128
// columns bf16 [58254, 1152] 95.9 us at eight, 82.4 at sixteen, [9362, 7168] 85.7 and 77.7, [10922, 6144]
// 73.8 and 76.3; fuller rows lose by it (bf16 [16384, 4096] 75.3 and 78.2, fp32 [33520, 1001] 78.6 and
// 87.5), and rows that are not quantised (bf16 [29127, 1152] 90.2 and 101.7).
inline int64_t rms_grid(int threads) {
  return static_cast<int64_t>(num_cus()) * (threads < 512 ? 512 / threads : 1);
}

template <typename T, int kTPR, int kVPT, bool kRagged, bool kResidual, int kOut>
int launch_rms_tile(int64_t N, int64_t C, float eps, const void* x, const void* residual,
                    const void* gamma, void* h, void* rsig, void* y, int64_t group, int64_t groups,
                    void* q, void* scale, hipStream_t stream) {
  using A = typename IO<T>::Acc;
  constexpr int kThreads = tile_threads(kTPR);
  const int64_t want = ceil_div(N, kThreads / kTPR);
  const bool more = kOut != kPlain && kThreads <= 512 && ceil_div(C, IO<T>::kVec) * 16 < kTPR * kVPT * 15;
  const int64_t most = rms_grid(kThreads) * (more ? 2 : 1);
  note_number("threads_per_row", kTPR);
  note_number("packets", kVPT);
  hipLaunchKernelGGL((rms_norm_rows<T, kTPR, kVPT, kRagged, kResidual, kOut>),
                     dim3(static_cast<unsigned>(want < most ? want : most)), dim3(kThreads), 0,
                     stream, N, static_cast<int>(C), A(eps), static_cast<const T*>(x),
                     static_cast<const T*>(residual), static_cast<const A*>(gamma), static_cast<T*>(h),
                     static_cast<A*>(rsig), static_cast<T*>(y), static_cast<int>(group),
                     static_cast<int>(groups), static_cast<uint8_t*>(q), static_cast<float*>(scale));
  return status_of_launch();
}

template <typename T, bool kRagged, bool kResidual, int kOut>
int launch_rms_tiles(int64_t N, int64_t C, float eps, const void* x, const void* residual,
                     const void* gamma, void* h, void* rsig, void* y, int64_t group, int64_t groups,
                     void* q, void* scale, hipStream_t stream) {
  const int64_t packets = ceil_div(C, IO<T>::kVec);
#define LAUNCH(TPR, VPT)                                                                            \
  return launch_rms_tile<T, TPR, VPT, kRagged, kResidual, kOut>(N, C, eps, x, residual, gamma, h, rsig, \
                                                                y, group, groups, q, scale, stream);
  DRAGON_HIP_RMS_SWITCH(packets, LAUNCH)
#undef LAUNCH
}

// Whether rows of C elements fit the tiles: up to 4096 packets, and one at least where the last
// packet is moved back.
template <typename T>
bool rms_tiles_fit(int64_t C) {
  return C >= IO<T>::kVec && ceil_div(C, IO<T>::kVec) <= kMaxTilePackets;
}

template <typename T, int kOut>
int launch_rms_rows(int64_t N, int64_t C, float eps, const void* x, const void* residual,
                    const void* gamma, void* h, void* rsig, void* y, int64_t group, int64_t groups,
                    void* q, void* scale, hipStream_t stream) {
  // a null pointer counts as aligned; codes are written 8 or 4 bytes at a time
  const bool regular = C % IO<T>::kVec == 0 && aligned16(x) && aligned16(residual) && aligned16(gamma) &&
      aligned16(h) && aligned16(y) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
#define LAUNCH(RAGGED, RESIDUAL)                                                                     \
  return launch_rms_tiles<T, RAGGED, RESIDUAL, kOut>(N, C, eps, x, residual, gamma, h, rsig, y, group, \
                                                     groups, q, scale, stream);
  if (regular) {
    if (residual) LAUNCH(false, true) else LAUNCH(false, false)
  } else {
    if (residual) LAUNCH(true, true) else LAUNCH(true, false)
  }
#undef LAUNCH
}

template <typename T>
int launch_rms_norm(int64_t N, int64_t C, float eps, const void* x, const void* residual,
                    const void* gamma, void* h, void* rsig, void* y, hipStream_t stream) {
  using A = typename IO<T>::Acc;
  if (rms_tiles_fit<T>(C)) {
    return launch_rms_rows<T, kPlain>(N, C, eps, x, residual, gamma, h, rsig, y, 0, 0, nullptr, nullptr,
                                      stream);
  }
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
  const int64_t groups = group ? ceil_div(C, group) : static_cast<int64_t>(1);
  if (rms_tiles_fit<T>(C)) {
    if (group == 0)
      return launch_rms_rows<T, kRowScale>(N, C, eps, x, residual, gamma, h, rsig, nullptr, group, groups,
                                           q, scale, stream);
    return launch_rms_rows<T, kGroupScale>(N, C, eps, x, residual, gamma, h, rsig, nullptr, group, groups,
                                           q, scale, stream);
  }
  hipLaunchKernelGGL((rms_norm_rows_looped<T, true>), dim3(loop_grid(N)), dim3(kLoopThreads), 0,
                     stream, N, C, eps, static_cast<const T*>(x), static_cast<const T*>(residual),
                     static_cast<const float*>(gamma), static_cast<T*>(h), static_cast<float*>(rsig),
                     static_cast<T*>(nullptr), static_cast<int>(group),
                     groups, static_cast<uint8_t*>(q), static_cast<float*>(scale));
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

// One read of h, dy and dh, one write of dx, and the column sums in the registers of workgroups
// that stay and walk the rows: a thread owns the same columns of every row it meets. The groups
// of a workgroup add theirs in LDS, in order, and each workgroup leaves one row of partial sums.
constexpr int grad_threads(int tpr) { return tpr <= 512 ? 512 : tpr; }
template <typename T, int kTPR, int kVPT, bool kRagged, bool kThrough>
__global__ __launch_bounds__(grad_threads(kTPR)) void rms_norm_grad_rows(
    const int64_t N, const int C, const T* h, const typename IO<T>::Acc* rsig,
    const typename IO<T>::Acc* gamma, const T* dy, const T* dh, typename IO<T>::Acc* partial, T* dx) {
  using A = typename IO<T>::Acc;
  constexpr int kVec = IO<T>::kVec;
  constexpr int kThreads = grad_threads(kTPR), kRows = kThreads / kTPR;
  constexpr bool kAhead = kVPT <= 2;
  __shared__ A slots[2][kThreads / kWaveSize];
  // gamma of the thread's columns, then the sums of the workgroup's groups: 16-byte words, those of
  // neighbouring lanes side by side
  constexpr int kPer = 16 / sizeof(A), kWords = kVec / kPer;
  __shared__ u32x4 shared[kVPT * kWords * kTPR];
  const RowPackets<T, kTPR, kVPT, kRagged> tile(C);
  const A inv_c = A(1) / A(C);
  const int lane = static_cast<int>(threadIdx.x) % kTPR, mine = static_cast<int>(threadIdx.x) / kTPR;
  auto word_at = [&](int s, int w) -> u32x4& { return shared[(s * kWords + w) * kTPR + lane]; };
  auto read_words = [&](int s, A(&v)[kVec]) {
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      A part[kPer];
      IO<A>::unpack(word_at(s, w), part);
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[w * kPer + e] = part[e];
    }
  };
  auto write_words = [&](int s, const A(&v)[kVec]) {
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      A part[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) part[e] = v[w * kPer + e];
      word_at(s, w) = IO<A>::pack(part);
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTPR;
  u32x4 ph[kVPT], py[kVPT], pd[kVPT];
  A rs_next;
  auto request = [&](int64_t r) {
    r = r < N ? r : 0;
    tile.template load<true>(h + r * C, ph);
    tile.template load<true>(dy + r * C, py);
    if constexpr (kThrough) tile.template load<true>(dh + r * C, pd);
    rs_next = rsig[r];
  };
  request(row);  // the first row comes while gamma is laid out
  A acc[kVPT][kVec];
#pragma unroll
  for (int s = 0; s < kVPT; ++s) {
    if (mine == 0) {
      A g[kVec];
      tile.params(gamma, s, g);
      write_words(s, g);
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[s][e] = A(0);
  }
  __syncthreads();
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < N; base += step) {
    const bool valid = row < N;
    const A rs = rs_next;
    u32x4 ch[kVPT], cy[kVPT], cd[kVPT];
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      ch[s] = ph[s], cy[s] = py[s];
      if constexpr (kThrough) cd[s] = pd[s];
    }
    A dot = A(0);
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      A a[kVec], b[kVec], g[kVec];
      IO<T>::unpack(ch[s], a);
      IO<T>::unpack(cy[s], b);
      read_words(s, g);
      A part = A(0);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const A t = b[e] * a[e];
        part += tile.counts(s, e) ? t * g[e] : A(0);
        acc[s][e] += valid ? t * rs : A(0);  // what is shared with another packet is not written
      }
      dot += tile.on[s] ? part : A(0);
    }
    const int64_t next = row + step;
    if constexpr (kAhead) request(next);
    if constexpr (kRagged && kThrough) {
      // dh has arrived before another wavefront may write dx over elements that both hold
#pragma unroll
      for (int s = 0; s < kVPT; ++s) asm volatile("" : "+v"(cd[s]));
    }
    dot = row_allreduce<kTPR>(dot, SumOp(), slots[turn]);
    const A c = dot * inv_c * rs * rs;
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      A a[kVec], b[kVec], d[kVec], g[kVec];
      IO<T>::unpack(ch[s], a);
      IO<T>::unpack(cy[s], b);
      read_words(s, g);
      if constexpr (kThrough) {
        IO<T>::unpack(cd[s], d);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) d[e] = A(0);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) d[e] += rs * (b[e] * g[e] - a[e] * c);
      if (valid && tile.on[s]) tile.store(dx + row * C, s, d);
    }
    row = next;
    turn ^= 1;
    if constexpr (!kAhead) request(row);
  }
  // the rows of a wavefront first: lanes that own the same columns
#pragma unroll
  for (int o = kTPR; o < kWaveSize; o <<= 1) {
#pragma unroll
    for (int s = 0; s < kVPT; ++s)
#pragma unroll
      for (int e = 0; e < kVec; ++e) acc[s][e] += __shfl_xor(acc[s][e], o, kWaveSize);
  }
  // then one wavefront (or group of them) after the other adds its sums; the last holds the
  // workgroup's
  constexpr int kOwners = kTPR < kWaveSize ? kThreads / kWaveSize : kRows;
  const int owner = kTPR < kWaveSize ? static_cast<int>(threadIdx.x) / kWaveSize : mine;
  const bool first_rows = static_cast<int>(threadIdx.x) % kWaveSize < kTPR;  // of a wavefront's
  for (int r = 0; kOwners > 1 && r < kOwners; ++r) {
    __syncthreads();
    if (owner != r || !first_rows) continue;
#pragma unroll
    for (int s = 0; s < kVPT; ++s) {
      if (r > 0) {
        A before[kVec];
        read_words(s, before);
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[s][e] += before[e];
      }
      if (r + 1 < kOwners) write_words(s, acc[s]);
    }
  }
  if (owner != kOwners - 1 || !first_rows) return;
  A* out = partial + static_cast<int64_t>(blockIdx.x) * C;
#pragma unroll
  for (int s = 0; s < kVPT; ++s) {
    if (!tile.on[s]) continue;
    if (!kRagged || tile.dup[s] == 0) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        A part[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) part[e] = acc[s][w * kPer + e];
        *reinterpret_cast<u32x4_unaligned*>(out + tile.col[s] + w * kPer) = IO<A>::pack(part);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (e >= tile.dup[s]) out[tile.col[s] + e] = acc[s][e];
      }
    }
  }
}

// dgamma = the sums of the partial rows: 16 words of a row by each of 64 groups of threads, which
// take every 64th row and are then added in order.
constexpr int kJoinThreads = 1024, kJoinWords = 16, kJoinGroups = kJoinThreads / kJoinWords;
template <typename A>
__global__ __launch_bounds__(kJoinThreads) void rms_norm_grad_join(const int64_t C, const int64_t rows,
                                                                   const A* __restrict__ partial,
                                                                   A* __restrict__ dgamma) {
  __shared__ A lds[kJoinGroups][kJoinWords + 1];
  const int word = threadIdx.x % kJoinWords, group = threadIdx.x / kJoinWords;
  const int w = threadIdx.x / kWaveSize, lane = threadIdx.x % kWaveSize;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kJoinWords; base < C;
       base += static_cast<int64_t>(gridDim.x) * kJoinWords) {
    const int64_t col = base + word;
    A sum = A(0);
    if (col < C) {
#pragma unroll 4
      for (int64_t p = group; p < rows; p += kJoinGroups) sum += partial[p * C + col];
    }
    lds[group][word] = sum;
    __syncthreads();
    // a wavefront per word (16 of them): lane g holds the sum of group g
    const A total = wave_allreduce(lds[lane][w], SumOp());
    if (lane == 0 && base + w < C) dgamma[base + w] = total;
    __syncthreads();
  }
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

// Rows that the register tiles hold: their workgroups, each of which leaves a row of partial sums.
// Four packets of 16-bit elements per thread (three tensors' and as many sums) do not fit the
// registers of 1024 threads.
template <typename T>
bool grad_tiles_fit(int64_t C) {
  return C >= IO<T>::kVec && ceil_div(C, IO<T>::kVec) <= (sizeof(T) == 2 ? kMaxTilePackets / 2 : kMaxTilePackets);
}
template <typename T>
int64_t grad_grid(int64_t N, int64_t C) {
  const int64_t packets = ceil_div(C, IO<T>::kVec);
  int tpr = 0;
#define TAKE(TPR, VPT) tpr = TPR;
  DRAGON_HIP_RMS_SWITCH(packets, TAKE)
#undef TAKE
  const int threads = grad_threads(tpr);
  const int64_t want = ceil_div(N, threads / tpr);
  const int64_t most = rms_grid(threads);
  return want < most ? want : most;
}

template <typename T>
size_t grad_scratch_bytes(int64_t N, int64_t C) {
  using A = typename IO<T>::Acc;
  if (grad_tiles_fit<T>(C)) return static_cast<size_t>(grad_grid<T>(N, C)) * C * sizeof(A);
  const GradCols p = plan_grad_cols(N, C, IO<T>::kVec);
  return static_cast<size_t>(N + p.chunks * C) * sizeof(A);
}

template <typename T, bool kRagged, bool kThrough>
void launch_grad_tiles(int64_t N, int64_t C, unsigned grid, const T* h, const typename IO<T>::Acc* rsig,
                       const typename IO<T>::Acc* gamma, const T* dy, const T* dh,
                       typename IO<T>::Acc* partial, T* dx, hipStream_t stream) {
  const int64_t packets = ceil_div(C, IO<T>::kVec);
#define LAUNCH(TPR, VPT)                                                                            \
  {                                                                                                 \
    hipLaunchKernelGGL((rms_norm_grad_rows<T, TPR, VPT, kRagged, kThrough>), dim3(grid),            \
                       dim3(grad_threads(TPR)), 0, stream, N, static_cast<int>(C), h, rsig, gamma, dy, \
                       dh, partial, dx);                                                            \
  }
  if constexpr (sizeof(T) == 2) {
    DRAGON_HIP_RMS_SWITCH_2(packets, LAUNCH)
  } else {
    DRAGON_HIP_RMS_SWITCH(packets, LAUNCH)
  }
#undef LAUNCH
}

template <typename T>
int launch_rms_norm_grad(int64_t N, int64_t C, const void* h, const void* rsig, const void* gamma,
                         const void* dy, const void* dh, void* dgamma, void* dx, void* scratch,
                         size_t scratch_bytes, hipStream_t stream) {
  using A = typename IO<T>::Acc;
  const size_t need = N > 0 ? grad_scratch_bytes<T>(N, C) : 0;
  const uint64_t bytes = bytes_of(sizeof(T), N, C);
  const Span H = {h, bytes}, S = {rsig, bytes_of(sizeof(A), N)}, G = {gamma, bytes_of(sizeof(A), C)}, DY = {dy, bytes};
  const Span DH = {dh, bytes}, DG = {dgamma, bytes_of(sizeof(A), C)}, DX = {dx, bytes}, W = {scratch, need};
  if (!on_or_apart(DX, {DY, DH}) || !apart(DX, {H, S, G}) || !apart(DG, {H, S, G, DY, DH, DX}) ||
      !apart(W, {H, S, G, DY, DH, DG, DX}))
    return DRAGON_HIP_EINVAL;
  if (need > 0 && (!scratch || scratch_bytes < need)) return DRAGON_HIP_ESCRATCH;
  const T* hp = static_cast<const T*>(h);
  const T* yp = static_cast<const T*>(dy);
  const T* dp = static_cast<const T*>(dh);
  const A* rp = static_cast<const A*>(rsig);
  const A* gp = static_cast<const A*>(gamma);
  T* xp = static_cast<T*>(dx);
  A* partial = static_cast<A*>(scratch);
  int64_t rows = 0;  // of partial sums
  if (N > 0 && grad_tiles_fit<T>(C)) {
    rows = grad_grid<T>(N, C);
    const unsigned grid = static_cast<unsigned>(rows);
    const bool regular = C % IO<T>::kVec == 0 && aligned16(h) && aligned16(gamma) && aligned16(dy) &&
        aligned16(dh) && aligned16(dx);
    if (regular && dh) launch_grad_tiles<T, false, true>(N, C, grid, hp, rp, gp, yp, dp, partial, xp, stream);
    else if (regular) launch_grad_tiles<T, false, false>(N, C, grid, hp, rp, gp, yp, dp, partial, xp, stream);
    else if (dh) launch_grad_tiles<T, true, true>(N, C, grid, hp, rp, gp, yp, dp, partial, xp, stream);
    else launch_grad_tiles<T, true, false>(N, C, grid, hp, rp, gp, yp, dp, partial, xp, stream);
  } else if (N > 0) {
    const GradCols p = plan_grad_cols(N, C, IO<T>::kVec);
    A* coef = partial;
    partial += N;
    rows = p.chunks;
    hipLaunchKernelGGL((rms_norm_grad_dots<T>), dim3(loop_grid(N)), dim3(kLoopThreads), 0, stream, N, C,
                       hp, rp, gp, yp, coef);
    const dim3 grid(static_cast<unsigned>(ceil_div(C, static_cast<int64_t>(IO<T>::kVec) * kColThreads)),
                    static_cast<unsigned>(p.chunks));
    hipLaunchKernelGGL((rms_norm_grad_cols<T>), grid, dim3(kColThreads), 0, stream, N, C,
                       p.rows_per_chunk, hp, rp, gp, yp, dp, coef, partial, xp);
  }
  hipLaunchKernelGGL((rms_norm_grad_join<A>), dim3(row_grid(C, kJoinWords)),
                     dim3(kJoinThreads), 0, stream, C, rows, partial, static_cast<A*>(dgamma));
  return status_of_launch();
}

inline int element_bytes(int dtype) {
  return dtype == DRAGON_HIP_F64 ? 8 : (dtype == DRAGON_HIP_F32 ? 4 : 2);
}
inline int acc_bytes(int dtype) { return dtype == DRAGON_HIP_F64 ? 8 : 4; }
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
  const uint64_t bytes = bytes_of(element_bytes(dtype), N, C);
  if (!x || !gamma || !y) return DRAGON_HIP_EINVAL;
  const Span X = {x, bytes}, R = {residual, bytes}, G = {gamma, bytes_of(acc_bytes(dtype), C)};
  const Span H = {h, bytes}, S = {rsig, bytes_of(acc_bytes(dtype), N)}, Y = {y, bytes};
  if (!on_or_apart(Y, {X, R}) || !on_or_apart(H, {X, R}) || !apart(Y, {H, G, S}) || !apart(H, {G, S}) ||
      !apart(S, {X, R, G}))
    return DRAGON_HIP_EINVAL;
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
  const uint64_t bytes = bytes_of(element_bytes(dtype), N, C);
  const Span X = {x, bytes}, R = {residual, bytes}, G = {gamma, bytes_of(4, C)}, H = {h, bytes};
  const Span S = {rsig, bytes_of(4, N)}, Q = {q, bytes_of(1, N, C)};
  const Span scales = {scale, bytes_of(4, N, group ? ceil_div(C, group) : 1)};
  if (!on_or_apart(H, {X, R}) || !apart(H, {G, S}) || !apart(S, {X, R, G}) || !apart(Q, {X, R, G, H, S}) ||
      !apart(scales, {X, R, G, H, S, Q}))
    return DRAGON_HIP_EINVAL;
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
  if (!dgamma || (N > 0 && (!h || !rsig || !gamma || !dy || !dx))) return DRAGON_HIP_EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DRAGON_HIP_DISPATCH_DTYPE(dtype, launch_rms_norm_grad, N, C, h, rsig, gamma, dy, dh, dgamma, dx,
                            scratch, scratch_bytes, s);
}

} // extern "C"
