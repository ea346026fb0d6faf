// causal_conv.cu -- a short causal convolution over the sequence, channel by
// channel, with an optional SiLU, its VJP, and its single-token step.
//
//   u_t = bias + sum_k w_k x_{t-W+1+k},  k = 0 .. W-1,  y_t = silu(u_t) or u_t
//
// for x [batch, length, dim] and w [dim, W].  Tokens before the first come from
// x0 [batch, W-1, dim] (zero without it).  Where starts[t] is set a new sequence
// begins at t: taps that reach before it are left out (selected, not multiplied
// by zero, so a NaN of the sequence before does not pass).
//
// VJP: du_t = dy_t act'(u_t) with u recomputed from x, and
//   dx_s = sum_k w_{W-1-k} du_{s+k}   (over the taps that y_{s+k} had)
//   dw_{W-1-k} = sum_t du_t x_{t-k},  dbias = sum_t du_t
//
// A warp takes 128 channels, four a lane in two pairs, and a run of tokens; the taps are
// a window of registers that moves along it, so each input is read once, and the W-1
// tokens before a run (and in the VJP after it) a second time, from L2.  A few tokens are
// loaded ahead of those that are worked on.  Weight gradients are summed along the run in
// registers, over the CTA's warps in shared memory and over CTAs by a second kernel, each
// in a fixed order.
//
// Bound by HBM in f32 (2 elements a token and channel forward, 3 in the VJP), by the issue
// of instructions and the two special functions of a SiLU in bf16.  At [4, 2048, 4096] with
// four taps and SiLU: f32 51 us forward (80% of the copy bandwidth) and 83 VJP (74%), bf16 32
// and 67 (64% and 46%); with eight taps, whose windows leave one CTA an SM, 44 and 102.
#include <algorithm>
#include <type_traits>

#include "typed.cuh"

namespace oxc {

constexpr int kConvWarps = 8;
constexpr int kConvMaxWidth = 8;

// Pairs of channels a lane and tokens a step, with as many registers as two CTAs an SM
// leave (up to four taps).  Measured at [4, 2048, 4096] in runs of 64 tokens, forward: 2
// pairs and 8 tokens 34 us in bf16 and 50 in f32; 2 and 4 39 and 54; 1 and 8 41 and 53.
// VJP in bf16: 2 and 4 70 us, 2 and 8 78, 1 and 8 78; single elements (4095 channels) 1
// and 4 88, 2 and 4 232; in f32 1 and 8 87, 1 and 4 97, 2 and 4 150.
constexpr int kConvFwdPairs = 2, kConvFwdStep = 8;
template <typename T, bool VEC>
struct ConvBwd {
  static constexpr int kPairs = sizeof(T) == 2 && VEC ? 2 : 1, kStep = sizeof(T) == 2 ? 4 : 8;
};

// A lane's four channels as they are in memory: consecutive ones, in one access (VEC),
// or 32 apart.  Loads are predicated, so that nothing waits for one before its use.
template <typename T, bool VEC, int NP>
struct ConvRaw;
template <bool VEC, int NP>
struct ConvRaw<float, VEC, NP> {
  float v[2 * NP];
  __device__ __forceinline__ void load(const float* p, int live) {
#pragma unroll
    for (int k = 0; k < 2 * NP; ++k) v[k] = 0.0f;
    if constexpr (VEC && NP == 1) {
      asm("{.reg .pred p; setp.gt.s32 p, %3, 0; @p ld.global.v2.f32 {%0, %1}, [%2];}"
          : "+f"(v[0]), "+f"(v[1]) : "l"(p), "r"(live));
    } else if constexpr (VEC) {
      asm("{.reg .pred p; setp.gt.s32 p, %5, 0; @p ld.global.v4.f32 {%0, %1, %2, %3}, [%4];}"
          : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]) : "l"(p), "r"(live));
    } else {
#pragma unroll
      for (int k = 0; k < 2 * NP; ++k)
        asm("{.reg .pred p; setp.gt.s32 p, %2, %3; @p ld.global.f32 %0, [%1];}"
            : "+f"(v[k]) : "l"(p + 32 * k), "r"(live), "r"(k));
    }
  }
  __device__ __forceinline__ float2 pair(int j) const { return make_float2(v[2 * j], v[2 * j + 1]); }
};
template <bool VEC, int NP>
struct ConvRaw<bf16, VEC, NP> {
  uint32_t w[VEC ? NP : 2 * NP];
  __device__ __forceinline__ void load(const bf16* p, int live) {
#pragma unroll
    for (int k = 0; k < (VEC ? NP : 2 * NP); ++k) w[k] = 0u;
    if constexpr (VEC && NP == 1) {
      asm("{.reg .pred p; setp.gt.s32 p, %2, 0; @p ld.global.u32 %0, [%1];}"
          : "+r"(w[0]) : "l"(p), "r"(live));
    } else if constexpr (VEC) {
      asm("{.reg .pred p; setp.gt.s32 p, %3, 0; @p ld.global.v2.u32 {%0, %1}, [%2];}"
          : "+r"(w[0]), "+r"(w[1]) : "l"(p), "r"(live));
    } else {
#pragma unroll
      for (int k = 0; k < 2 * NP; ++k)
        asm("{.reg .pred p; setp.gt.s32 p, %2, %3; @p ld.global.u16 %0, [%1];}"
            : "+r"(w[k]) : "l"(p + 32 * k), "r"(live), "r"(k));
    }
  }
  __device__ __forceinline__ float2 pair(int j) const {
    if constexpr (VEC) return make_float2(bf16_lo(w[j]), bf16_hi(w[j]));
    else return make_float2(bf16_lo(w[2 * j]), bf16_lo(w[2 * j + 1]));
  }
};

template <typename T, bool VEC, int NP>
struct ConvLane {
  static constexpr int kMine = 2 * NP, kChannels = 32 * kMine;  // a lane's and a warp's
  int64_t d;  // the first channel
  int live;   // how many exist
  __device__ __forceinline__ ConvLane(int64_t d0, int64_t dim) {
    const int lane = threadIdx.x & 31;
    d = VEC ? d0 + lane * kMine : d0 + lane;
    live = 0;
#pragma unroll
    for (int k = 0; k < kMine; ++k) live += d + at(k) < dim;
  }
  static __device__ __forceinline__ int at(int k) { return VEC ? k : 32 * k; }
  __device__ __forceinline__ void store(T* row, const float2 (&v)[NP]) const {
    float f[kMine];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      f[2 * j] = v[j].x;
      f[2 * j + 1] = v[j].y;
    }
    if constexpr (VEC) {
      if (live) store_from_f32<kMine>(row + d, f);
    } else {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const float one[1] = {f[k]};
        if (k < live) store_from_f32<1>(row + d + 32 * k, one);
      }
    }
  }
};

template <typename T>
struct ConvArgs {
  const T* x;  // strides in elements
  int64_t x_sb, x_st;
  const float* w;
  const float* bias;
  const T* x0;
  const uint8_t* starts;
  T* y;
  T* last;
  // VJP
  const T* dy;
  int64_t dy_sb, dy_st;
  const T* dlast;
  T* dx;
  T* dx0;
  float* parts;  // [batch * groups of runs, dim * (W + 1)]
  int64_t batch, length, dim;
  int run;  // tokens that a warp goes through
  unsigned int ctiles, groups;  // channel tiles, groups of kConvWarps runs
};

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float rcp(float t) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float sigmoid_f32(float v) { return rcp(1.0f + ex2(-1.44269504f * v)); }
// The tokens at which a sequence starts, a bit each: bit l is token t - (W - 1) + l, of the
// W - 1 tokens before a step of U tokens and the step.
template <int W, int U>
struct ConvStarts {
  const uint8_t* row;
  int64_t length;
  uint8_t next;
  __device__ __forceinline__ ConvStarts(const uint8_t* starts, int64_t row, int64_t length)
      : row(starts ? starts + row : nullptr), length(length), next(0) {}
  __device__ __forceinline__ void load(int64_t t) {
    const int lane = threadIdx.x & 31;
    const int64_t at = t - (W - 1) + lane;
    if (row) next = lane < W - 1 + U && at >= 0 && at < length ? row[at] : (uint8_t)0;
  }
  __device__ __forceinline__ unsigned int bits() const {
    return row ? __ballot_sync(0xffffffffu, next != 0) : 0u;
  }
};
// Tokens since the sequence of the step's i-th token began, at most W - 1 (also where
// none of the last W - 1 starts one: what lies before token 0 belongs to its sequence).
template <int W>
__device__ __forceinline__ int conv_age(unsigned int bits, int i) {
  const unsigned int before = bits << (31 - (W - 1 + i));
  return before ? min(W - 1, __clz(before)) : W - 1;
}
// Runs f(std::true_type) if any bit is set, else f(std::false_type), whose taps need no
// tests.
template <typename F>
__device__ __forceinline__ void by_fresh(unsigned int bits, F f) {
  if (bits) f(std::true_type{});
  else f(std::false_type{});
}

// The weights and the bias of a lane's channels, in pairs.
template <int W, bool VEC, int NP, typename T>
__device__ __forceinline__ void conv_weights(float2 (&w)[W][NP], float2 (&bias)[NP], const ConvArgs<T>& a,
                                             const ConvLane<T, VEC, NP>& lane) {
#pragma unroll
  for (int c = 0; c < 2 * NP; ++c) {
    const bool on = c < lane.live;
    const int64_t d = lane.d + lane.at(c);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float v = on ? a.w[d * W + k] : 0.0f;
      if (c & 1) w[k][c / 2].y = v;
      else w[k][c / 2].x = v;
    }
    const float v = on && a.bias ? a.bias[d] : 0.0f;
    if (c & 1) bias[c / 2].y = v;
    else bias[c / 2].x = v;
  }
}

// Token t of a batch row, one of x0 if t is negative.
template <int W, bool VEC, int NP, typename T>
__device__ __forceinline__ void conv_token(ConvRaw<T, VEC, NP>& r, const ConvArgs<T>& a,
                                           const ConvLane<T, VEC, NP>& lane, int64_t b, int64_t t) {
  if (t >= 0) r.load(a.x + b * a.x_sb + t * a.x_st + lane.d, t < a.length ? lane.live : 0);
  else r.load(a.x0 + (b * (W - 1) + t + W - 1) * a.dim + lane.d, a.x0 ? lane.live : 0);
}

template <typename T, int W, bool VEC, bool SILU>
__global__ void __launch_bounds__(kConvWarps * 32, W <= 4 ? 2 : 1) conv_fwd_kernel(ConvArgs<T> a) {
  constexpr int U = kConvFwdStep, NP = kConvFwdPairs;
  using Raw = ConvRaw<T, VEC, NP>;
  const unsigned int tile = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.groups;
  const int64_t t0 = ((int64_t)(rest % a.groups) * kConvWarps + (threadIdx.x >> 5)) * a.run;
  if (t0 >= a.length && t0 > 0) return;
  using Lane = ConvLane<T, VEC, NP>;
  const Lane lane((int64_t)tile * Lane::kChannels, a.dim);
  const int left = (int)max((int64_t)0, min(a.length - t0, (int64_t)a.run));
  float2 w[W][NP], bias[NP];
  conv_weights<W, VEC, NP>(w, bias, a, lane);
  float2 xs[W - 1 + U][NP];  // token t - (W - 1) first
  Raw raw[U];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    Raw r;
    conv_token<W, VEC, NP>(r, a, lane, b, t0 - (W - 1) + k);
#pragma unroll
    for (int c = 0; c < NP; ++c) xs[k][c] = r.pair(c);
  }
  ConvStarts<W, U> ahead(a.starts, b * a.length, a.length);
  ahead.load(t0);
  const T* px = a.x + b * a.x_sb + t0 * a.x_st + lane.d;
#pragma unroll
  for (int i = 0; i < U; ++i) raw[i].load(px + i * a.x_st, i < left ? lane.live : 0);
  T* py = a.y + (b * a.length + t0) * a.dim;
  for (int t = 0; t < left; t += U) {
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int c = 0; c < NP; ++c) xs[W - 1 + i][c] = raw[i].pair(c);
    const unsigned int bits = ahead.bits();
    px += U * a.x_st;
#pragma unroll
    for (int i = 0; i < U; ++i) raw[i].load(px + i * a.x_st, t + U + i < left ? lane.live : 0);
    ahead.load(t0 + t + U);
    by_fresh(bits, [&](auto some) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int age = decltype(some)::value ? conv_age<W>(bits, i) : W - 1;
        float2 u[NP];
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          u[c] = bias[c];
#pragma unroll
          for (int k = 0; k < W; ++k)  // tap k, W - 1 - k tokens back
            if (!decltype(some)::value || W - 1 - k <= age) u[c] = __ffma2_rn(w[k][c], xs[i + k][c], u[c]);
          if (SILU) u[c] = make_float2(u[c].x * sigmoid_f32(u[c].x), u[c].y * sigmoid_f32(u[c].y));
        }
        if (t + i < left) lane.store(py + i * a.dim, u);
      }
    });
    py += U * a.dim;
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int c = 0; c < NP; ++c) xs[k][c] = xs[U + k][c];
  }
  if (a.last && t0 + left == a.length) {  // the run of the last token
    // bit l of the ballot: a start at token length - 1 - l
    const int64_t at = a.length - 1 - (threadIdx.x & 31);
    const unsigned int starts = __ballot_sync(
        0xffffffffu, a.starts && at >= 0 && (threadIdx.x & 31) < W - 1 && a.starts[b * a.length + at]);
    const int age = starts ? __ffs(starts) - 1 : W - 1;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      Raw r;
      conv_token<W, VEC, NP>(r, a, lane, b, a.length - (W - 1) + k);
      float2 v[NP];
#pragma unroll
      for (int c = 0; c < NP; ++c) v[c] = W - 2 - k > age ? make_float2(0.0f, 0.0f) : r.pair(c);
      lane.store(a.last + (b * (W - 1) + k) * a.dim, v);
    }
  }
}

// A run of the VJP owns R = a.run - (W - 1) tokens and goes through the W - 1
// after them too, whose du its last tokens need.
template <typename T, int W, bool VEC, bool SILU>
__global__ void __launch_bounds__(kConvWarps * 32, W <= 4 ? 2 : 1) conv_bwd_kernel(ConvArgs<T> a) {
  constexpr int NP = ConvBwd<T, VEC>::kPairs, U = ConvBwd<T, VEC>::kStep;
  using Raw = ConvRaw<T, VEC, NP>;
  __shared__ float sums[kConvWarps][64 * NP];
  const unsigned int tile = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.groups;
  const int warp = threadIdx.x >> 5, R = a.run - (W - 1);
  const int64_t t0 = ((int64_t)(rest % a.groups) * kConvWarps + warp) * R;
  using Lane = ConvLane<T, VEC, NP>;
  const Lane lane((int64_t)tile * Lane::kChannels, a.dim);
  float2 dw[W][NP], db[NP];
#pragma unroll
  for (int c = 0; c < NP; ++c) {
    db[c] = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][c] = make_float2(0.0f, 0.0f);
  }
  if (t0 < a.length || t0 == 0) {
    // tokens from t0 on that are there, that the run owns and that it goes through
    const int there = (int)max((int64_t)0, min(a.length - t0, (int64_t)a.run));
    const int own = min(there, R), through = (int)min(a.length + W - 1 - t0, (int64_t)a.run);
    float2 w[W][NP], bias[NP];
    conv_weights<W, VEC, NP>(w, bias, a, lane);
    float2 xs[W - 1 + U][NP];   // token t - (W - 1) first
    float2 acc[W - 1 + U][NP];  // and its gradient
    Raw rx[U], rd[U];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      Raw r;
      conv_token<W, VEC, NP>(r, a, lane, b, t0 - (W - 1) + k);
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        xs[k][c] = r.pair(c);
        acc[k][c] = make_float2(0.0f, 0.0f);
      }
    }
    ConvStarts<W, U> ahead(a.starts, b * a.length, a.length);
    ahead.load(t0);
    const T* px = a.x + b * a.x_sb + t0 * a.x_st + lane.d;
    const T* pd = a.dy + b * a.dy_sb + t0 * a.dy_st + lane.d;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      rx[i].load(px + i * a.x_st, i < there ? lane.live : 0);
      rd[i].load(pd + i * a.dy_st, i < there && a.dy ? lane.live : 0);
    }
    // token s from t0 on, whose gradient is complete but for dlast's share
    auto emit = [&](int s, const float2 (&v)[NP]) {
      if (s >= own || s < (t0 == 0 ? 1 - W : 0)) return;
      float2 o[NP];
#pragma unroll
      for (int c = 0; c < NP; ++c) o[c] = v[c];
      if (a.dlast && t0 + s >= a.length - (W - 1)) {
        const int back = (int)(a.length - 1 - t0 - s);  // tokens before the last
        bool same = true;  // no sequence starts after it
        for (int k = 0; k < back && a.starts; ++k) same = same && !(a.length - 1 - k >= 0 && a.starts[(b + 1) * a.length - 1 - k]);
        Raw e;
        e.load(a.dlast + (b * (W - 1) + W - 2 - back) * a.dim + lane.d, same ? lane.live : 0);
#pragma unroll
        for (int c = 0; c < NP; ++c) o[c] = __fadd2_rn(o[c], e.pair(c));
      }
      if (t0 + s >= 0) lane.store(a.dx + (b * a.length + t0 + s) * a.dim, o);
      else if (a.dx0) lane.store(a.dx0 + (b * (W - 1) + s + W - 1) * a.dim, o);
    };
    for (int t = 0; t < through; t += U) {
      Raw dy[U];
#pragma unroll
      for (int i = 0; i < U; ++i) dy[i] = rd[i];
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          xs[W - 1 + i][c] = rx[i].pair(c);
          acc[W - 1 + i][c] = make_float2(0.0f, 0.0f);
        }
      const unsigned int bits = ahead.bits();
      px += U * a.x_st;
      pd += U * a.dy_st;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        rx[i].load(px + i * a.x_st, t + U + i < there ? lane.live : 0);
        rd[i].load(pd + i * a.dy_st, t + U + i < there && a.dy ? lane.live : 0);
      }
      ahead.load(t0 + t + U);
      by_fresh(bits, [&](auto some) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int age = decltype(some)::value ? conv_age<W>(bits, i) : W - 1;
          float2 u[NP], mine[NP];
#pragma unroll
          for (int c = 0; c < NP; ++c) {
            u[c] = bias[c];
#pragma unroll
            for (int k = 0; k < W; ++k)
              if (!decltype(some)::value || W - 1 - k <= age) u[c] = __ffma2_rn(w[k][c], xs[i + k][c], u[c]);
            if (SILU) {  // (u s)' = s + u s (1 - s)
              const float2 s = make_float2(sigmoid_f32(u[c].x), sigmoid_f32(u[c].y)), us = __fmul2_rn(u[c], s);
              const float2 rest = make_float2(1.0f - s.x, 1.0f - s.y);
              u[c] = __fmul2_rn(dy[i].pair(c), __ffma2_rn(us, rest, s));
            } else {
              u[c] = dy[i].pair(c);
            }
            // (0 beyond the sequence, as dy is)
            mine[c] = t + i < own ? u[c] : make_float2(0.0f, 0.0f);
            db[c] = __fadd2_rn(db[c], mine[c]);
          }
#pragma unroll
          for (int k = 0; k < W; ++k)
            if (!decltype(some)::value || W - 1 - k <= age) {
#pragma unroll
              for (int c = 0; c < NP; ++c) {
                acc[i + k][c] = __ffma2_rn(w[k][c], u[c], acc[i + k][c]);
                dw[k][c] = __ffma2_rn(mine[c], xs[i + k][c], dw[k][c]);
              }
            }
        }
      });
      const int first = t - (W - 1);
      if (first >= 0 && first + U <= own && (!a.dlast || t0 + first + U <= a.length - (W - 1))) {
        T* to = a.dx + (b * a.length + t0 + first) * a.dim;
#pragma unroll
        for (int i = 0; i < U; ++i) lane.store(to + i * a.dim, acc[i]);
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i) emit(first + i, acc[i]);
      }
#pragma unroll
      for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          xs[k][c] = xs[U + k][c];
          acc[k][c] = acc[U + k][c];
        }
    }
  }
  // over the warps, then one row of partial sums a CTA: [dim][W], then [dim]
  float* part = a.parts + (int64_t)rest * a.dim * (W + 1);
  const int first = VEC ? (threadIdx.x & 31) * 2 * NP : threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
#pragma unroll
    for (int c = 0; c < NP; ++c) {
      const float2 v = k < W ? dw[k < W ? k : 0][c] : db[c];
      sums[warp][first + Lane::at(2 * c)] = v.x;
      sums[warp][first + Lane::at(2 * c + 1)] = v.y;
    }
    __syncthreads();
    const int64_t d = (int64_t)tile * Lane::kChannels + threadIdx.x;
    if (threadIdx.x < Lane::kChannels && d < a.dim) {
      float s = sums[0][threadIdx.x];
#pragma unroll
      for (int i = 1; i < kConvWarps; ++i) s += sums[i][threadIdx.x];
      part[k < W ? d * W + k : a.dim * W + d] = s;
    }
    __syncthreads();
  }
  pdl_launch_dependents();
}

// One token: y from the W - 1 inputs kept in `state` and x; `out` keeps the next.
template <typename T, int W>
__global__ void __launch_bounds__(128) conv_step_kernel(const T* __restrict__ x, int64_t x_sb,
                                                        const float* __restrict__ w,
                                                        const float* __restrict__ bias,
                                                        const T* state, T* out, T* __restrict__ y,
                                                        int64_t n, int64_t dim, int silu) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t b = i / dim, d = i - b * dim;
  T v[W];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) v[k] = state[(b * (W - 1) + k) * dim + d];
  v[W - 1] = x[b * x_sb + d];
  float u = bias ? bias[d] : 0.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) u = fmaf(w[d * W + k], to_f32(v[k]), u);
  y[i] = from_f32<T>(silu ? u * sigmoid_f32(u) : u);
#pragma unroll
  for (int k = 1; k < W; ++k) out[(b * (W - 1) + k - 1) * dim + d] = v[k];
}

template <typename T>
static bool conv_vector(const T* p, int64_t sb, int64_t st, int channels) {
  return !p || (aligned_to(p, channels * sizeof(T)) && sb % channels == 0 && st % channels == 0);
}

// Calls f with the width as a compile-time number.
template <typename F>
static void by_width(int64_t width, F f) {
  switch (width) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 5: f(std::integral_constant<int, 5>{}); break;
    case 6: f(std::integral_constant<int, 6>{}); break;
    case 7: f(std::integral_constant<int, 7>{}); break;
    default: f(std::integral_constant<int, 8>{}); break;
  }
}

// How a call is cut: tokens that a warp goes through, and groups of warps along a row.
struct ConvCut {
  int run;
  int64_t ctiles, groups;
};

// The longest run among those whose grid takes the least time: its rounds on the GPU, at
// a run's tokens each and some for its beginning.  (Against runs of 64, bf16, four taps:
// [1, 512, 2048] 6.5 us instead of 12.6 forward and 12.4 instead of 25 VJP; [4, 2048, 4096]
// 31.7 instead of 35 and 66 instead of 72; f32 there 51.5 instead of 50.6, HBM-bound, and 82
// instead of 88.  At most 128 tokens: the VJPs 70 and 88.  At least 32: [1, 512, 2048] 8.5
// and 16.6.)
static ConvCut conv_cut(int64_t batch, int64_t length, int64_t dim, int64_t width, int channels,
                        bool backward) {
  constexpr int kLeast = 16, kMost = 256, kBeginning = 24;
  ConvCut best{0, (dim + 32 * channels - 1) / (32 * channels), 1};
  const int64_t slots = (width <= 4 ? 2 : 1) * sm_count(), tiles = batch * best.ctiles;
  int64_t least = 0;
  for (int run = kLeast; run <= kMost; run += 8) {
    const int64_t per = (backward ? run - (width - 1) : run) * kConvWarps;
    const int64_t groups = std::max<int64_t>(1, (length + per - 1) / per);
    const int64_t cost = (tiles * groups + slots - 1) / slots * (run + kBeginning);
    if (!best.run || cost <= least) {
      least = cost;
      best.run = run;
      best.groups = groups;
    }
  }
  return best;
}

template <typename T>
static oxc_status conv_launch(ConvArgs<T> a, int64_t width, bool silu, bool backward, cudaStream_t s,
                              int64_t* sums = nullptr) {
  // a lane's channels where it reads vectors
  const int wide = 2 * (backward ? ConvBwd<T, true>::kPairs : kConvFwdPairs);
  const bool vec = a.dim % wide == 0 && conv_vector(a.x, a.x_sb, a.x_st, wide) &&
                   conv_vector(a.dy, a.dy_sb, a.dy_st, wide) && conv_vector(a.x0, 0, 0, wide) &&
                   conv_vector(a.dlast, 0, 0, wide) && conv_vector<T>(a.y, 0, 0, wide) &&
                   conv_vector<T>(a.last, 0, 0, wide) && conv_vector<T>(a.dx, 0, 0, wide) &&
                   conv_vector<T>(a.dx0, 0, 0, wide);
  const int channels = vec || !backward ? wide : 2 * ConvBwd<T, false>::kPairs;
  const ConvCut cut = conv_cut(a.batch, a.length, a.dim, width, channels, backward);
  if (cut.ctiles * cut.groups > 0x7fffffff / std::max<int64_t>(a.batch, 1))
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: causal_conv: more than 2^31 blocks");
  a.run = cut.run;
  a.ctiles = (unsigned int)cut.ctiles;
  a.groups = (unsigned int)cut.groups;
  if (sums) *sums = a.batch * cut.groups;
  const unsigned int grid = (unsigned int)(a.batch * cut.ctiles * cut.groups);
  by_width(width, [&](auto w) {
    constexpr int W = decltype(w)::value;
    auto kernel = backward ? (silu ? (vec ? conv_bwd_kernel<T, W, true, true> : conv_bwd_kernel<T, W, false, true>)
                                   : (vec ? conv_bwd_kernel<T, W, true, false> : conv_bwd_kernel<T, W, false, false>))
                           : (silu ? (vec ? conv_fwd_kernel<T, W, true, true> : conv_fwd_kernel<T, W, false, true>)
                                   : (vec ? conv_fwd_kernel<T, W, true, false> : conv_fwd_kernel<T, W, false, false>));
    kernel<<<grid, kConvWarps * 32, 0, s>>>(a);
  });
  return check_launch("oxc_causal_conv");
}

static oxc_status conv_check(const char* what, int64_t batch, int64_t length, int64_t dim,
                             int64_t width, int32_t dtype) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: unknown dtype %d", what, dtype);
  if (batch < 0 || length < 0 || dim < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: negative shape", what);
  if (width < 1)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: width %lld", what, (long long)width);
  if (width > kConvMaxWidth)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: more than %d taps, got %lld", what,
                kConvMaxWidth, (long long)width);
  return OXC_OK;
}

template <typename T>
static oxc_status conv_step_launch(const void* x, int64_t x_stride, const float* w,
                                   const float* bias, const void* state, void* out, void* y,
                                   int64_t batch, int64_t dim, int64_t width, int32_t silu,
                                   cudaStream_t s) {
  const int64_t n = batch * dim;
  by_width(width, [&](auto tag) {
    constexpr int W = decltype(tag)::value;
    conv_step_kernel<T, W><<<(unsigned int)((n + 127) / 128), 128, 0, s>>>(
        static_cast<const T*>(x), x_stride, w, bias, static_cast<const T*>(state),
        static_cast<T*>(out), static_cast<T*>(y), n, dim, silu);
  });
  return check_launch("oxc_causal_conv_step");
}

}  // namespace oxc

using namespace oxc;

extern "C" {

oxc_status oxc_causal_conv_fwd(const void* x, int64_t x_sb, int64_t x_st, const float* w,
                               const float* bias, const void* x0, const uint8_t* starts, void* y,
                               void* last, int64_t batch, int64_t length, int64_t dim,
                               int64_t width, int32_t silu, int32_t dtype, void* stream) {
  const oxc_status st = conv_check("causal_conv", batch, length, dim, width, dtype);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  if (!w || (length > 0 && (!x || !y)))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: causal_conv: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    ConvArgs<T> a{};
    a.x = static_cast<const T*>(x);
    a.x_sb = x_sb;
    a.x_st = x_st;
    a.w = w;
    a.bias = bias;
    a.x0 = static_cast<const T*>(x0);
    a.starts = starts;
    a.y = static_cast<T*>(y);
    a.last = width > 1 ? static_cast<T*>(last) : nullptr;
    a.batch = batch;
    a.length = length;
    a.dim = dim;
    return conv_launch<T>(a, width, silu != 0, false, s);
  };
  return dtype == OXC_BF16 ? go(bf16{}) : go(0.0f);
}

size_t oxc_causal_conv_bwd_workspace_size(int64_t batch, int64_t length, int64_t dim, int64_t width) {
  if (batch <= 0 || length < 0 || dim <= 0 || width < 1 || width > kConvMaxWidth) return 0;
  int64_t groups = 1;
  for (int pairs = 1; pairs <= 2; ++pairs)  // of every ConvBwd
    groups = std::max(groups, conv_cut(batch, length, dim, width, 2 * pairs, true).groups);
  return sizeof(float) * (size_t)(batch * groups) * (size_t)(dim * (width + 1));
}

oxc_status oxc_causal_conv_bwd(const void* x, int64_t x_sb, int64_t x_st, const float* w,
                               const float* bias, const void* x0, const uint8_t* starts,
                               const void* dy, int64_t dy_sb, int64_t dy_st, const void* dlast,
                               void* dx, void* dx0, float* dw, int64_t batch, int64_t length,
                               int64_t dim, int64_t width, int32_t silu, int32_t dtype,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const oxc_status st = conv_check("causal_conv backward", batch, length, dim, width, dtype);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dim == 0) return OXC_OK;
  if (!dw || !w || (batch > 0 && length > 0 && (!x || !dx)))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: causal_conv backward: null pointer");
  const int64_t cols = dim * (width + 1);
  if (batch == 0) {
    const cudaError_t e = cudaMemsetAsync(dw, 0, sizeof(float) * cols, s);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_causal_conv_bwd");
  }
  if (!workspace || workspace_bytes < oxc_causal_conv_bwd_workspace_size(batch, length, dim, width))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: causal_conv backward: workspace too small");
  int64_t sums = 0;  // rows of partial sums
  auto go = [&](auto zero) {
    using T = decltype(zero);
    ConvArgs<T> a{};
    a.x = static_cast<const T*>(x);
    a.x_sb = x_sb;
    a.x_st = x_st;
    a.w = w;
    a.bias = bias;
    a.x0 = static_cast<const T*>(x0);
    a.starts = starts;
    a.dy = static_cast<const T*>(dy);
    a.dy_sb = dy_sb;
    a.dy_st = dy_st;
    a.dlast = width > 1 ? static_cast<const T*>(dlast) : nullptr;
    a.dx = static_cast<T*>(dx);
    a.dx0 = width > 1 ? static_cast<T*>(dx0) : nullptr;
    a.parts = static_cast<float*>(workspace);
    a.batch = batch;
    a.length = length;
    a.dim = dim;
    return conv_launch<T>(a, width, silu != 0, true, s, &sums);
  };
  const oxc_status r = dtype == OXC_BF16 ? go(bf16{}) : go(0.0f);
  if (r) return r;
  launch_colsum_partials(static_cast<const float*>(workspace), (int)sums, cols, dw, s);
  return check_launch("oxc_causal_conv_bwd (sums)");
}

oxc_status oxc_causal_conv_step(const void* x, int64_t x_stride, const float* w, const float* bias,
                                const void* state, void* state_out, void* y, int64_t batch,
                                int64_t dim, int64_t width, int32_t silu, int32_t dtype,
                                void* stream) {
  const oxc_status st = conv_check("causal_conv_step", batch, 1, dim, width, dtype);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  if (!x || !w || !y || (width > 1 && (!state || !state_out)))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: causal_conv_step: null pointer");
  if (dim > (int64_t)0x7fffffff * 128 / batch)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: causal_conv_step: more than 2^31 blocks");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == OXC_BF16
             ? conv_step_launch<bf16>(x, x_stride, w, bias, state, state_out, y, batch, dim, width, silu, s)
             : conv_step_launch<float>(x, x_stride, w, bias, state, state_out, y, batch, dim, width, silu, s);
}

}  // extern "C"
