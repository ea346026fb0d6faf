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
// A thread keeps SPT states of each of CPT channels in registers, LPC lanes of a warp
// share a channel, and the CTA's threads walk through the tokens in tiles of kTile.
// Eight more warps, the helpers, prepare the tiles: they copy the operands to shared
// memory a tile or two ahead, turn them into f32 steps (dt, dt x) there, once per token
// and channel, and finish and store a tile's outputs, while the others walk through the
// next one.  (Without helpers, and with the copies a tile ahead, f32 [4, 2048, 4096] with
// 16 states took 408 us forward and 1135 VJP, half of it the tiles' preparation.)  Sums
// over n are made across the LPC lanes, sums over d across the warp's other lanes, its
// warps and the CTAs.  The VJP gets the state before each tile from the
// forward (`carry`) and goes through the tiles from the last to the first: it runs the
// recurrence forward through a tile, keeping the state every few tokens, and from the last
// of these backwards again with the decays and states of those few tokens in registers.
//
// What bounds it, at f32 [4, 2048, 4096] with 16 states, 2^29 exponentials: at 16 a cycle
// and SM they take 120 us forward and 210 in the VJP (1.75 for each state), the operands
// 82 and 143 us of HBM.  Shared memory, which hands the operands around (26 of its cycles
// for 256 states forward, 49 in the VJP), and the issue of instructions (99 and 228 of
// them, 4 a cycle) are as busy as the exponentials, and the CTAs are 256 and 128 for 148
// SMs: 279 us forward (294 with the states saved), 777 VJP; bf16 the same.
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
constexpr int kMaxState = 128;
constexpr int kMaxSegments = 64;
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
  unsigned int ctiles, map_ctiles;  // of the VJP, and of its first kernel
};

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_pair(float2 t) { return make_float2(ex2(t.x), ex2(t.y)); }

__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float sigmoid(float v) { return rcp(1.0f + ex2(-kLog2e * v)); }

// log(1 + exp(v)) = max(v, 0) + log(1 + e), e = exp(-|v|).  e = 2^t exp(n - t ln 2) with
// n = -|v| and t = n log2(e) rounded, the second factor to first order.  log(1 + e) = 2
// artanh(s), s = e / (2 + e) <= 1/3, by the series in s^2 (2 s^17 / 17 is below 2^-26 of
// it), so a small e keeps its relative accuracy.
__device__ __forceinline__ float softplus(float v) {
  float n = -fabsf(v);
  n = n < -100.0f ? -100.0f : n;  // (a NaN stays)
  const float t = n * kLog2e;
  float e = ex2(t);
  e = fmaf(e, fmaf(t, -kLn2, n), e);
  const float s = e * rcp(2.0f + e), w = s * s;
  float p = 2.0f / 15.0f;
  p = fmaf(p, w, 2.0f / 13.0f);
  p = fmaf(p, w, 2.0f / 11.0f);
  p = fmaf(p, w, 2.0f / 9.0f);
  p = fmaf(p, w, 2.0f / 7.0f);
  p = fmaf(p, w, 2.0f / 5.0f);
  p = fmaf(p, w, 2.0f / 3.0f);
  return fmaf(s, fmaf(p, w, 2.0f), v > 0.0f ? v : 0.0f);
}

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

template <int SPT_, int LPC_, int CPT_, int WARPS>
struct Layout {
  static constexpr int SPT = SPT_, LPC = LPC_, CPT = CPT_, P = SPT / 2;
  static constexpr int kWarps = WARPS, kThreads = kWarps * 32;
  static constexpr int kLanes = 32 / LPC;               // of a warp, side by side over channels
  static constexpr int kWarpChannels = kLanes * CPT;
  static constexpr int kChannels = kWarps * kWarpChannels;  // a CTA's
  static constexpr int NP = SPT * LPC;                  // states with their padding
};

// One element if `on`, else 0.  The load is predicated rather than branched around or
// selected from, so that nothing waits for it before its value is used.
__device__ __forceinline__ float load_if(const float* p, bool on) {
  float v = 0.0f;
  asm("{.reg .pred p; setp.ne.s32 p, %2, 0; @p ld.global.nc.f32 %0, [%1];}" : "+f"(v) : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ uint16_t load_if(const bf16* p, bool on) {
  uint16_t v = 0;
  asm("{.reg .pred p; setp.ne.s32 p, %2, 0; @p ld.global.nc.u16 %0, [%1];}" : "+h"(v) : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ float4 load_if(const float4* p, bool on) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  asm("{.reg .pred p; setp.ne.s32 p, %5, 0; @p ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];}"
      : "+f"(v.x), "+f"(v.y), "+f"(v.z), "+f"(v.w) : "l"(p), "r"((int)on));
  return v;
}
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// Where a thread's states are.
template <class L>
struct Place {
  int sl, cl;    // its lane among a channel's, and over channels
  int ch;        // its first channel in the tile; the others are kLanes apart
  int64_t d;     // and in the tensor
  // Neighbouring lanes have the same states of neighbouring channels: they read the
  // same 16 bytes of B and C, which costs 2.4 cycles of the SM's shared memory a load
  // where four addresses taking turns (lane % 4) cost 4.
  __device__ __forceinline__ Place(int64_t d0) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    sl = lane / L::kLanes;
    cl = lane % L::kLanes;
    ch = warp * L::kWarpChannels + cl;
    d = d0 + ch;
  }
  static __device__ __forceinline__ bool vectors(const float* p, int N) {
    return (N & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  }
  // states of channel c in a [.., dim, N] array, zero where there is none
  __device__ __forceinline__ void load(float2 (&v)[L::P], const float* p, int c, int64_t row,
                                       int64_t dim, int N) const {
    const int64_t dc = d + c * L::kLanes;
    const bool on = p && dc < dim;
    const float* q = p + (row * dim + dc) * N + sl * L::SPT;
    if (L::SPT == 4 && vectors(p, N)) {
      const float4 t = load_if(reinterpret_cast<const float4*>(q), on && sl * L::SPT < N);
      v[0] = make_float2(t.x, t.y);
      v[1] = make_float2(t.z, t.w);
      return;
    }
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      const int n = sl * L::SPT + 2 * i;
      v[i].x = load_if(q + 2 * i, on && n < N);
      v[i].y = load_if(q + 2 * i + 1, on && n + 1 < N);
    }
  }
  // Asks L2 for what load will take.
  __device__ __forceinline__ void ask(const float* p, int c, int64_t row, int64_t dim, int N) const {
    const int64_t dc = d + c * L::kLanes;
    if (dc < dim && sl * L::SPT < N)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p + (row * dim + dc) * N + sl * L::SPT));
  }
  __device__ __forceinline__ void store(const float2 (&v)[L::P], float* p, int c, int64_t row,
                                        int64_t dim, int N) const {
    const int64_t dc = d + c * L::kLanes;
    if (!p || dc >= dim) return;
    float* q = p + (row * dim + dc) * N + sl * L::SPT;
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

// 4, 8 or 16 bytes to shared memory without passing the registers; zeros unless `on`.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool on) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(on ? 16 : 0) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(src), "r"(on ? 8 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(src), "r"(on ? 4 : 0) : "memory");
}

// Barriers between the warps that prepare tiles and those that walk through them, one
// pair for the even tiles and one for the odd: `full` when a tile is prepared, `done`
// when it is walked through.  Who waits syncs, who goes on arrives.
__device__ __forceinline__ void tile_sync(int id, int threads) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void tile_arrive(int id, int threads) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
constexpr int kFull = 1, kDone = 3;  // + the tile's parity

// The threads that prepare tiles, behind those that walk through them.  (With 128, whose
// chains of dependent operations then were what the others waited for: bf16 [3, 4097,
// 1001] with 24 states 390 us forward and 943 VJP instead of 280 and 719; now 264 and 709.)
constexpr int kHelpers = 256;

// Deals out the registers that a CTA is launched with: the warps that walk through tiles
// need more of them than the helpers.  The shares have to add up to no more than those
// at the launch, or the first of these would wait for ever.
template <int REGISTERS, bool MORE>
__device__ __forceinline__ void take_registers() {
  if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGISTERS));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGISTERS));
}

// A tile's operands as they are in memory, TENSORS of them DEPTH times over: helper i's
// vectors lie where only helper i looks, so no barrier stands between its copies and
// its reads.  A [kTile, kChannels] tile is cut into vectors of VW channels, dealt to the
// helpers token by token, kTurn tokens at a time: a thread's vectors are of the same
// channels.  Where vectors are shorter than the 4 bytes that can be copied without
// passing the registers, they wait there if they are few (up to 24: with the VJP's 32 of
// bf16 [3, 4097, 1001], 16 states, 459 us for 426); if not, L2 is asked for them and the
// copy made when the tile begins.  Both ask for the next tile as soon as one has landed
// (as late as the copies of vectors, whose place has to be free: forward there 250 us for
// 200).  DIR is 1 or -1, the direction through the tiles.
template <class L, typename T, int VW, int TENSORS, int DIR, int DEPTH>
struct Raw {
  static constexpr int kDepth = DEPTH;
  static constexpr bool kAsync = VW * sizeof(T) >= 4;
  static constexpr int kPer = L::kChannels / VW;  // vectors of a token
  static constexpr int kVecs = kTile * kPer;
  static constexpr int kMine = (kVecs + kHelpers - 1) / kHelpers;
  static constexpr int kTurn = kVecs < kHelpers ? kTile : kHelpers / kPer;
  static constexpr int kPitch = (kVecs < kHelpers ? kVecs : kHelpers) * VW;
  static constexpr int kElements = kDepth * TENSORS * kMine * kPitch;
  static constexpr bool kHold = !kAsync && TENSORS * kMine <= 24;
  static_assert(kVecs < kHelpers || (kHelpers % kPer == 0 && kVecs % kHelpers == 0),
                "a turn is a whole number of tokens");
  T* s;
  int me;      // the helper's number
  int t, ch;   // the first vector's token in the tile, and its channel there
  bool has;    // whether the thread has vectors at all
  bool in;     // and whether their channels exist
  const T* p[TENSORS];  // it, in the tile to be fetched next
  int64_t step[TENSORS];
  uint16_t held[kHold ? TENSORS : 1][kHold ? kMine : 1];
  __device__ __forceinline__ Raw(T* s, int me, int64_t d0, int64_t dim)
      : s(s), me(me), t(me / kPer), ch(me % kPer * VW), has(kVecs >= kHelpers || me < kVecs),
        in(has && d0 + ch < dim) {}
  __device__ __forceinline__ void open(int which, const SeqArg<T>& v, int64_t b, int64_t t0, int64_t d0) {
    step[which] = v.st;
    p[which] = v.p ? v.p + b * v.sb + (t0 + t) * v.st + d0 + ch : nullptr;
  }
  __device__ __forceinline__ T* at(int buffer, int which, int k) const {
    return s + ((buffer * TENSORS + which) * kMine + k) * kPitch + me * VW;
  }
  // Whether the thread's k-th vector is one of `left` tokens.
  __device__ __forceinline__ bool on(int k, int left) const { return in && t + k * kTurn < left; }
  // Asks for the next tile, `left` tokens of which are there (none: the last was asked
  // for already); zeros for the others.
  __device__ __forceinline__ void fetch(int buffer, int left) {
#pragma unroll
    for (int w = 0; w < TENSORS; ++w) {
      if (!p[w]) continue;
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const bool here = on(k, left);
        const T* q = p[w] + k * kTurn * step[w];
        if constexpr (kAsync) {
          if (has && left > 0) copy_async<VW * (int)sizeof(T)>(at(buffer, w, k), here ? q : p[w], here);
        } else if constexpr (kHold) {
          held[w][k] = load_if(q, here);
        } else {
          if (here && (me & 15) == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
        }
      }
      if (kAsync || kHold) p[w] += DIR * kTile * step[w];
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The oldest tile asked for becomes readable, of kDepth - 1 that are on the way (held
  // ones: of one).
  __device__ __forceinline__ void land(int buffer, int left) {
    if constexpr (kAsync) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
    } else {
      uint16_t v[TENSORS][kMine];
#pragma unroll
      for (int w = 0; w < TENSORS; ++w) {
        if (!p[w]) continue;
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          if constexpr (kHold) v[w][k] = held[w][k];
          else v[w][k] = load_if(p[w] + k * kTurn * step[w], on(k, left));
        }
      }
#pragma unroll
      for (int w = 0; w < TENSORS; ++w) {
        if (!p[w]) continue;
        if (!kHold) p[w] += DIR * kTile * step[w];
#pragma unroll
        for (int k = 0; k < kMine; ++k)
          if (has) *reinterpret_cast<uint16_t*>(at(buffer, w, k)) = v[w][k];
      }
    }
  }
  __device__ __forceinline__ void read(float (&f)[VW], int buffer, int which, int k) const {
    const T* q = at(buffer, which, k);
    if constexpr (VW == 4 && sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(q);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else if constexpr (VW == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(q);
      f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
    } else {
      f[0] = to_f32(q[0]);
    }
  }
};

// VW floats in shared memory.
template <int VW>
__device__ __forceinline__ void load_floats(float (&v)[VW], const float* p) {
  if constexpr (VW == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
    v[0] = p[0];
  }
}
template <int VW>
__device__ __forceinline__ void store_floats(float* p, const float (&v)[VW]) {
  if constexpr (VW == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else p[0] = v[0];
}

// VW entries of a [dim] vector from channel d on, 0 where there is none.
template <int VW>
__device__ __forceinline__ void load_channels(float (&v)[VW], const float* p, int64_t d, bool in) {
#pragma unroll
  for (int i = 0; i < VW; ++i) v[i] = p && in ? p[d + i] : 0.0f;
}

// The rows of B or C of a tile on the way to shared memory, zero beyond N and the
// sequence: in the helpers' registers from one tile to the next.
template <class L, typename T, int DIR>
struct Rows {
  static constexpr int kMine = (kTile * L::NP + kHelpers - 1) / kHelpers;
  decltype(load_if((const T*)nullptr, true)) v[kMine];
  const T* p;
  int64_t step;
  int me, t, n;
  __device__ __forceinline__ Rows(int me, const SeqArg<T>& a, int64_t b, int64_t t0)
      : p(a.p + b * a.sb + t0 * a.st), step(a.st), me(me), t(me / L::NP), n(me % L::NP) {}
  __device__ __forceinline__ void load(int left, int N) {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      if constexpr (kHelpers % L::NP == 0) {
        const int tk = t + k * (kHelpers / L::NP);
        v[k] = load_if(p + tk * step + n, n < N && tk < left);
      } else {
        const int i = k * kHelpers + me, tk = i / L::NP, nk = i % L::NP;
        v[k] = load_if(p + tk * step + nk, nk < N && tk < left);
      }
    }
    p += DIR * kTile * step;
  }
  __device__ __forceinline__ void put(float* s) const {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = k * kHelpers + me;
      if (kTile * L::NP % kHelpers == 0 || i < kTile * L::NP) s[i] = as_f32(v[k]);
    }
  }
};

// Runs f(std::true_type) where any of the tile's tokens starts a sequence, else
// f(std::false_type), whose loops need no selects.
template <typename F>
__device__ __forceinline__ void by_fresh(unsigned int starts, F f) {
  if (starts) f(std::true_type{});
  else f(std::false_type{});
}

// A tile's tokens at which a sequence starts, a bit each (the same in all of a warp's
// threads): read a tile ahead.
struct Starts {
  const uint8_t* row;
  int64_t length;
  uint8_t next;
  __device__ __forceinline__ Starts(const uint8_t* starts, int64_t b, int64_t length, int64_t tile)
      : row(starts ? starts + b * length : nullptr), length(length), next(0) {
    load(tile);
  }
  __device__ __forceinline__ void load(int64_t tile) {
    const int lane = threadIdx.x & 31;
    const int64_t t = tile * kTile + lane;
    if (row) next = lane < kTile && t >= 0 && t < length ? row[t] : (uint8_t)0;
  }
  // Those of the tile loaded last, and loads another.
  __device__ __forceinline__ unsigned int bits(int64_t then) {
    if (!row) return 0u;
    const unsigned int b = __ballot_sync(0xffffffffu, next != 0);
    load(then);
    return b;
  }
};

// A rate (times log2(e)): an infinite one times a step of zero, as of a padded token, is
// then zero too.
__device__ __forceinline__ float bounded(float v) { return v < -1e30f ? -1e30f : v > 1e30f ? 1e30f : v; }

template <class L, typename T>
__device__ __forceinline__ void load_decay(float2 (&A2)[L::CPT][L::P], const Place<L>& at,
                                           const SelectiveArgs<T>& a) {
#pragma unroll
  for (int c = 0; c < L::CPT; ++c) {
    at.load(A2[c], a.A, c, 0, a.dim, a.N);
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      A2[c][i].x = bounded(A2[c][i].x * kLog2e);
      A2[c][i].y = bounded(A2[c][i].y * kLog2e);
    }
  }
}

// Takes a state from one end of segment `seg` to the other.  Where rates above zero take
// the decay beyond f32, the state may still be small or zero: two factors of half the
// time, and a zero stays one.
template <class L, typename T>
__device__ __forceinline__ void through_segment(float2 (&h)[L::CPT][L::P], const float2 (&A2)[L::CPT][L::P],
                                                const Place<L>& at, const SelectiveArgs<T>& a, int64_t b,
                                                int seg) {
  const int64_t row = b * a.segments + seg;
#pragma unroll
  for (int c = 0; c < L::CPT; ++c) {
    const int64_t d = at.d + c * L::kLanes;
    const float time = d < a.dim ? a.seg_time[row * a.dim + d] : 0.0f;
    // plain loads: the kernel before this one wrote them, so none may move above the wait
    const float* q = a.seg_state + (row * a.dim + d) * a.N + at.sl * L::SPT;
    const int there = d < a.dim ? a.N - at.sl * L::SPT : 0;
#pragma unroll
    for (int i = 0; i < L::P; ++i) {
      const float2 own = make_float2(2 * i < there ? q[2 * i] : 0.0f, 2 * i + 1 < there ? q[2 * i + 1] : 0.0f);
      const float2 e = exp2_pair(__fmul2_rn(A2[c][i], both(0.5f * time)));
      const float2 to = __ffma2_rn(e, __fmul2_rn(e, h[c][i]), own);
      h[c][i].x = time < 0.0f || h[c][i].x == 0.0f ? own.x : to.x;
      h[c][i].y = time < 0.0f || h[c][i].y == 0.0f ? own.y : to.y;
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

template <int SPT, int LPC>
using Forward = Layout<SPT, LPC, (LPC <= 4 ? 1 : 2), 8>;
// In the VJP 4 states a thread, the lanes a power of two.
template <int LPC>
using Backward = Layout<4, LPC, (LPC == 2 ? 1 : 2), 8>;
template <typename F>
inline auto by_lanes(int64_t N, F f) {
  if (N <= 8) return f(std::integral_constant<int, 2>{});
  if (N <= 16) return f(std::integral_constant<int, 4>{});
  if (N <= 32) return f(std::integral_constant<int, 8>{});
  if (N <= 64) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 32>{});
}

struct Plan {
  int64_t ctiles;
  int segments, seg_tiles;
};

inline Plan selective_plan(int64_t batch, int64_t length, int64_t dim, int64_t N, bool backward) {
  Plan p;
  const int64_t per =
      backward ? by_lanes(N, [](auto lpc) { return (int64_t)Backward<decltype(lpc)::value>::kChannels; })
               : by_state(N, [](auto spt, auto lpc) {
                   return (int64_t)Forward<decltype(spt)::value, decltype(lpc)::value>::kChannels;
                 });
  p.ctiles = (dim + per - 1) / per;
  const int64_t tiles = std::max<int64_t>(1, selective_tiles(length));
  const int64_t work = std::max<int64_t>(1, batch * p.ctiles), slots = (backward ? 1 : 2) * sm_count();
  // the fewest segments for which the rounds of the grid, and the first kernel's work
  // beside the other's, come to the least
  const double map = backward ? 0.3 : 0.6;
  double best = 0.0;
  for (int64_t want = 1; want <= std::min<int64_t>(kMaxSegments, std::max<int64_t>(1, tiles / 4)); ++want) {
    const int64_t each = (tiles + want - 1) / want, k = (tiles + each - 1) / each;
    const int64_t rounds = (work * k + slots - 1) / slots;
    const double cost = (double)(rounds * each) * (1.0 + map * (double)(k - 1) / (double)k);
    if (want == 1 || cost < best * 0.98) {
      best = cost;
      p.seg_tiles = (int)each;
      p.segments = (int)k;
    }
  }
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
oxc_status selective_fwd_launch(const SelectiveArgs<T>& a, cudaStream_t s);
template <typename T>
oxc_status selective_bwd_launch(const SelectiveArgs<T>& a, float* out_sums, T* dB, T* dC, cudaStream_t s);

}  // namespace oxc
