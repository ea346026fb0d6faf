// selective_scan.cuh -- the selective state space scan: what its forward, its VJP
// and its single-token step share.
//
// For x, delta, z [batch, length, dim], A [dim, N] and B, C [batch, length, N]:
//   dt = softplus(delta + delta_bias)
//   h_t[d, n] = exp(dt_t[d] A[d, n]) h_{t-1}[d, n] + dt_t[d] x_t[d] B_t[n]
//   inner_t[d] = sum_n C_t[n] h_t[d, n] + D[d] x_t[d]
//   y = inner silu(z)    (y = inner without z)
// with all arithmetic and the state in f32.  Where starts[t] is set a new sequence
// begins at t: the state before it counts as zero (selected, not multiplied).
//
// VJP, with e = dy silu(z), lam_t the gradient of h_t and mu_t = a_t lam_t (0 where
// starts[t]), a_t = exp(dt_t A):
//   lam_t = C_t e_t + mu_{t+1}                         (lam_{T-1} also has dlast)
//   through_t[d] = sum_n lam B,   rate_t[d] = sum_n mu h_{t-1} A
//   dx = dt through + D e,  ddt = x through + rate,  ddelta = ddt sigmoid(raw)
//   dA = sum_{b,t} dt mu h_{t-1},  dD = sum e x,  ddelta_bias = sum ddelta
//   dB_t[n] = sum_d lam dt x,  dC_t[n] = sum_d h e,  dz = dy inner silu'(z)
//
// A thread keeps SPT states of each of two channels in registers, LPC threads side
// by side share a channel, and the CTA's threads walk through the tokens in tiles
// of kTile: the tile's operands are staged in shared memory in f32 (dt and dt x
// once per token and channel), sums over n are made across the LPC threads and
// sums over d across the warp's other lanes, its warps and the CTAs.  The VJP gets
// the state before each tile from the forward (`carry`) and goes through the tiles
// from the last to the first: it runs the recurrence forward through a tile,
// keeping the state every kBack tokens, and from the last of these backwards again
// with the decays and states of kBack tokens in registers.
//
// Where batch and dim leave the GPU idle, the sequence is cut into segments.  A
// first kernel finds what each does to the state (its decay, exp(A sum dt), and the
// state it ends with from zero), and the segments then start from the composition
// of those before them (in the VJP, after them).
#pragma once

#include <algorithm>
#include <type_traits>

#include "typed.cuh"

namespace oxc {

constexpr int kTile = 16;     // tokens; the states that the VJP needs are saved as often
constexpr int kBack = 4;      // tokens whose states the VJP holds in registers
constexpr int kMaxState = 128;
constexpr int kMaxSegments = 32;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

// A [batch, length, n] operand: the last dim dense, strides in elements.
template <typename T>
struct SeqArg {
  const T* p;
  int64_t sb, st;
};

template <typename T>
struct SelectiveArgs {
  SeqArg<T> x, delta, z, B, C, dy;
  const float *A, *D, *delta_bias, *h0, *dlast;
  const uint8_t* starts;
  T* y;
  float* last;
  float* carry;  // [batch, tiles, dim, N]
  T *dx, *ddelta, *dz;
  float* dh0;
  float* sums;   // [batch * segments][dim * N + 2 dim]: dA, dD, ddelta_bias
  float* rows;   // [channel tiles][batch * length][2 N]: dB, dC
  // what the segments do, forward or backward: [batch, segments, dim]
  float* seg_state;  // [.., N]
  float* seg_time;   // sum of dt; negative if a sequence starts in it
  int64_t batch, length, dim;
  int N, segments, seg_tiles;  // tiles per segment
  unsigned int ctiles;
};

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_pair(float2 t) { return make_float2(ex2(t.x), ex2(t.y)); }

__device__ __forceinline__ float softplus(float v) {
  return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// Sums v over the lanes that differ in the bits FROM .. TO / 2 of their number, each
// lane keeping a part of the values: halves are exchanged while the count is even.
// Afterwards v[0 .. kKept) holds the values from `first` on, the same in lanes that
// differ in the bits from kUsed on only.
template <int V, int FROM, int TO>
struct LaneSum {
  static constexpr bool kSplit = V % 2 == 0;
  using Next = LaneSum<kSplit ? V / 2 : V, FROM * 2, TO>;
  static constexpr int kKept = Next::kKept;
  static constexpr int kUsed = kSplit ? Next::kUsed : FROM;
  template <int M>
  static __device__ __forceinline__ void run(float (&v)[M], int lane, int& first) {
    if constexpr (kSplit) {
      const bool up = lane & FROM;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float keep = up ? v[i + V / 2] : v[i], send = up ? v[i] : v[i + V / 2];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, FROM);
      }
      first += up ? V / 2 : 0;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], FROM);
    }
    Next::run(v, lane, first);
  }
};
template <int V, int TO>
struct LaneSum<V, TO, TO> {
  static constexpr int kKept = V, kUsed = TO;
  template <int M>
  static __device__ __forceinline__ void run(float (&)[M], int, int&) {}
};

// SPT states (pairs) of a row in shared memory.
template <int SPT>
__device__ __forceinline__ void load_states(float2 (&v)[SPT / 2], const float* p) {
  if constexpr (SPT == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(t.x, t.y);
    v[1] = make_float2(t.z, t.w);
  } else {
#pragma unroll
    for (int i = 0; i < SPT / 2; ++i) v[i] = reinterpret_cast<const float2*>(p)[i];
  }
}

template <typename T, int SPT_, int LPC_>
struct Layout {
  static constexpr int SPT = SPT_, LPC = LPC_, P = SPT / 2;
  static constexpr int kWarps = 8, kThreads = kWarps * 32;
  static constexpr int kChannels = kWarps * 64 / LPC;  // a CTA's
  static constexpr int NP = SPT * LPC;                 // states with their padding
};

// Where a thread's states are.
template <class L>
struct Place {
  int sl, ch;    // its lane among a channel's, its first channel in the tile
  int64_t d;     // and in the tensor
  __device__ __forceinline__ Place(int64_t d0) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    sl = lane % L::LPC;
    ch = (warp * (32 / L::LPC) + lane / L::LPC) * 2;
    d = d0 + ch;
  }
  static __device__ __forceinline__ bool vectors(const float* p, int N) {
    return (N & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  }
  // states of channel c in a [.., dim, N] array, zero where there is none
  __device__ __forceinline__ void load(float2 (&v)[L::P], const float* p, int c, int64_t row,
                                       int64_t dim, int N) const {
    const bool on = p && d + c < dim;
    const float* q = p + (row * dim + d + c) * N + sl * L::SPT;
    if (L::SPT == 4 && vectors(p, N)) {
      float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (on && sl * L::SPT < N) t = *reinterpret_cast<const float4*>(q);
      v[0] = make_float2(t.x, t.y);
      v[1] = make_float2(t.z, t.w);
      return;
    }
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      const int n = sl * L::SPT + 2 * i;
      v[i].x = on && n < N ? q[2 * i] : 0.0f;
      v[i].y = on && n + 1 < N ? q[2 * i + 1] : 0.0f;
    }
  }
  __device__ __forceinline__ void store(const float2 (&v)[L::P], float* p, int c, int64_t row,
                                        int64_t dim, int N) const {
    if (!p || d + c >= dim) return;
    float* q = p + (row * dim + d + c) * N + sl * L::SPT;
    if (L::SPT == 4 && vectors(p, N)) {
      if (sl * L::SPT < N)
        *reinterpret_cast<float4*>(q) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      return;
    }
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      const int n = sl * L::SPT + 2 * i;
      if (n < N) q[2 * i] = v[i].x;
      if (n + 1 < N) q[2 * i + 1] = v[i].y;
    }
  }
};

// Four (VEC) or one consecutive elements, kept in the caches: the end of a tile reads
// them again.
template <int VW, typename T>
__device__ __forceinline__ void load_vec(float (&v)[VW], const T* p) {
  if constexpr (VW == 4 && sizeof(T) == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else if constexpr (VW == 4) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(t.x); v[1] = bf16_hi(t.x); v[2] = bf16_lo(t.y); v[3] = bf16_hi(t.y);
  } else {
    v[0] = to_f32(p[0]);
  }
}

// Runs f(token of the tile, first channel of the tile, how many tokens in) for the
// thread's vectors of a [kTile, kChannels] tile.
template <class L, int VW, typename F>
__device__ __forceinline__ void each_vec(F f) {
  constexpr int kPer = L::kChannels / VW;
#pragma unroll 4
  for (int i = threadIdx.x; i < kTile * kPer; i += L::kThreads) f(i / kPer, i % kPer * VW);
}

// The rows of B or C of a tile in f32, zero beyond N and the sequence.
template <class L, typename T>
__device__ __forceinline__ void stage_rows(float* s, const SeqArg<T>& v, int64_t b, int64_t t0,
                                           int64_t length, int N) {
  for (int i = threadIdx.x; i < kTile * L::NP; i += L::kThreads) {
    const int t = i / L::NP, n = i % L::NP;
    s[i] = n < N && t0 + t < length ? to_f32(v.p[b * v.sb + (t0 + t) * v.st + n]) : 0.0f;
  }
}

// The tile's tokens at which a sequence starts, a bit each (the same in all threads).
__device__ __forceinline__ unsigned int tile_starts(const uint8_t* starts, int64_t row, int64_t t0,
                                                   int64_t length) {
  if (!starts) return 0u;
  const int lane = threadIdx.x & 31;
  const bool s = lane < kTile && t0 + lane < length && starts[row * length + t0 + lane];
  return __ballot_sync(0xffffffffu, s);
}

__device__ __forceinline__ float bounded(float v) { return v < -1e30f ? -1e30f : v > 1e30f ? 1e30f : v; }

template <class L, typename T>
__device__ __forceinline__ void load_decay(float2 (&A2)[2][L::P], const Place<L>& at,
                                           const SelectiveArgs<T>& a) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    at.load(A2[c], a.A, c, 0, a.dim, a.N);
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      // an infinite rate times a step of zero, as of a padded token, is zero too
      A2[c][i].x = bounded(A2[c][i].x * kLog2e);
      A2[c][i].y = bounded(A2[c][i].y * kLog2e);
    }
  }
}

// Takes a state from one end of segment `seg` to the other.
template <class L, typename T>
__device__ __forceinline__ void through_segment(float2 (&h)[2][L::P], const float2 (&A2)[2][L::P],
                                                const Place<L>& at, const SelectiveArgs<T>& a, int64_t b,
                                                int seg) {
  const int64_t row = b * a.segments + seg;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float time = at.d + c < a.dim ? a.seg_time[row * a.dim + at.d + c] : 0.0f;
    float2 own[L::P];
    at.load(own, a.seg_state, c, row, a.dim, a.N);
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      const float2 e = exp2_pair(__fmul2_rn(A2[c][i], both(time)));
      h[c][i] = time < 0.0f ? own[i] : __ffma2_rn(e, h[c][i], own[i]);
    }
  }
}

// ---- host ------------------------------------------------------------------------------

inline int64_t selective_tiles(int64_t length) { return (length + kTile - 1) / kTile; }

// Calls f(states per thread, lanes per channel): as few padded states as these leave.
template <typename F>
inline auto by_state(int64_t N, F f) {
#define OXC_CASE(SPT, LPC) f(std::integral_constant<int, SPT>{}, std::integral_constant<int, LPC>{})
  if (N <= 8) return OXC_CASE(4, 2);
  if (N <= 12) return OXC_CASE(6, 2);
  if (N <= 16) return OXC_CASE(4, 4);
  if (N <= 24) return OXC_CASE(6, 4);
  if (N <= 32) return OXC_CASE(4, 8);
  if (N <= 48) return OXC_CASE(6, 8);
  if (N <= 64) return OXC_CASE(4, 16);
  if (N <= 96) return OXC_CASE(6, 16);
  return OXC_CASE(4, 32);
#undef OXC_CASE
}

inline int64_t channel_tile(int64_t N) {
  return by_state(N, [](auto spt, auto lpc) {
    return (int64_t)Layout<float, decltype(spt)::value, decltype(lpc)::value>::kChannels;
  });
}

struct Plan {
  int64_t ctiles;
  int segments, seg_tiles;
};

inline Plan selective_plan(int64_t batch, int64_t length, int64_t dim, int64_t N) {
  Plan p;
  const int64_t per = channel_tile(N);
  p.ctiles = (dim + per - 1) / per;
  const int64_t tiles = std::max<int64_t>(1, selective_tiles(length));
  int64_t segments = (2 * sm_count()) / std::max<int64_t>(1, batch * p.ctiles);
  segments = std::max<int64_t>(1, std::min<int64_t>({segments, kMaxSegments, tiles / 4}));
  p.seg_tiles = (int)((tiles + segments - 1) / segments);
  p.segments = (int)((tiles + p.seg_tiles - 1) / p.seg_tiles);
  return p;
}

template <typename T>
inline bool seq_vec(const SeqArg<T>& v) {
  return !v.p || (aligned_to(v.p, 4 * sizeof(T)) && v.sb % 4 == 0 && v.st % 4 == 0);
}

// Raises the dynamic shared memory of a kernel to `bytes` where that needs asking.
inline cudaError_t allow_smem(const void* kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename... KArgs, typename... Args>
inline cudaError_t launch_scan(void (*kernel)(KArgs...), unsigned int grid, int block, size_t smem,
                          bool dependent, cudaStream_t s, Args... args) {
  cudaError_t e = allow_smem((const void*)kernel, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline oxc_status selective_check(const char* what, int32_t dtype, int64_t batch, int64_t length,
                             int64_t dim, int64_t N) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: unknown dtype %d", what, dtype);
  if (batch < 0 || length < 0 || dim < 0 || N < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: negative shape", what);
  if (N > kMaxState)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: more than %d states a channel, got %lld",
                what, kMaxState, (long long)N);
  if (length > ((int64_t)1 << 34))
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: a sequence of %lld tokens", what,
                (long long)length);
  const int64_t ctiles = (dim + 15) / 16;  // the narrowest channel tiles
  if (ctiles > 0 && batch > 0x7fffffff / kMaxSegments / ctiles)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: batch %lld of %lld channels", what,
                (long long)batch, (long long)dim);
  return OXC_OK;
}

// A segment's map: the states, then the sums of dt.
inline size_t map_floats(const Plan& p, int64_t batch, int64_t dim, int64_t N) {
  return p.segments > 1 ? (size_t)batch * p.segments * (size_t)dim * (size_t)(N + 1) : 0;
}

template <typename T>
inline void selective_segments(SelectiveArgs<T>& a, const Plan& p, float* workspace) {
  a.segments = p.segments;
  a.seg_tiles = p.seg_tiles;
  a.ctiles = (unsigned int)p.ctiles;
  a.seg_state = workspace;
  a.seg_time = workspace + (size_t)a.batch * p.segments * a.dim * a.N;
}

// Defined for each type by a file of its own.
template <typename T>
oxc_status selective_bwd_launch(const SelectiveArgs<T>& a, float* out_sums, T* dB, T* dC, cudaStream_t s);

}  // namespace oxc
