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
// A warp takes 128 channels, four a lane, and a run of tokens; the taps are a
// window of registers that moves along it, so each input is read once, and the
// W-1 tokens before a run (and in the VJP after it) a second time, from L2.
// Weight gradients are summed along the run in registers, over the CTA's warps in
// shared memory and over CTAs by a second kernel, each in a fixed order.  Bound by
// HBM.
#include <algorithm>
#include <type_traits>

#include "typed.cuh"

namespace oxc {

constexpr int kConvWarps = 8;
constexpr int kConvLaneCh = 4;                  // channels a lane
constexpr int kConvChannels = 32 * kConvLaneCh;  // a warp
constexpr int kConvStep = 4;                    // tokens loaded at a time
constexpr int kConvRun = 64;                    // tokens of a forward run
constexpr int kConvMaxWidth = 8;

// A lane's four channels: consecutive ones, in one access (VEC), or 32 apart.
template <typename T, bool VEC>
struct ConvLane {
  int64_t d;
  int live;
  __device__ __forceinline__ ConvLane(int64_t d0, int64_t dim) {
    const int lane = threadIdx.x & 31;
    d = VEC ? d0 + lane * kConvLaneCh : d0 + lane;
    live = 0;
#pragma unroll
    for (int k = 0; k < kConvLaneCh; ++k) live += d + at(k) < dim;
  }
  static __device__ __forceinline__ int at(int k) { return VEC ? k : 32 * k; }
  __device__ __forceinline__ void load(float (&v)[kConvLaneCh], const T* row, bool on) const {
    if constexpr (VEC) {
      if (on && live) load_as_f32<kConvLaneCh>(v, row + d);
      else
#pragma unroll
        for (int k = 0; k < kConvLaneCh; ++k) v[k] = 0.0f;
    } else {
#pragma unroll
      for (int k = 0; k < kConvLaneCh; ++k) {
        float one[1] = {0.0f};
        if (on && k < live) load_as_f32<1>(one, row + d + 32 * k);
        v[k] = one[0];
      }
    }
  }
  __device__ __forceinline__ void store(T* row, const float (&v)[kConvLaneCh]) const {
    if constexpr (VEC) {
      if (live) store_from_f32<kConvLaneCh>(row + d, v);
    } else {
#pragma unroll
      for (int k = 0; k < kConvLaneCh; ++k) {
        const float one[1] = {v[k]};
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
  int silu;
  unsigned int ctiles, groups;  // channel tiles, groups of kConvWarps runs
};

__device__ __forceinline__ float sigmoid_f32(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// Tokens since the sequence of token t began, at most W - 1 (also where none of the
// last W - 1 starts one: what lies before token 0 belongs to its sequence).
template <int W>
__device__ __forceinline__ int conv_age(const uint8_t* starts, int64_t row, int64_t t) {
  int age = W - 1;
  if (starts) {
#pragma unroll
    for (int k = W - 2; k >= 0; --k)
      if (t - k >= 0 && starts[row + t - k]) age = k;
  }
  return age;
}

// Reads token t of a batch row, one of x0 if t is negative, zero at the end.
template <typename T, int W, bool VEC>
__device__ __forceinline__ void conv_token(const ConvArgs<T>& a, const ConvLane<T, VEC>& lane,
                                           int64_t b, int64_t t, float (&v)[kConvLaneCh]) {
  if (t >= 0) lane.load(v, a.x + b * a.x_sb + t * a.x_st, t < a.length);
  else lane.load(v, a.x0 + (b * (W - 1) + t + W - 1) * a.dim, a.x0 != nullptr);
}

template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(kConvWarps * 32) conv_fwd_kernel(ConvArgs<T> a) {
  constexpr int C = kConvLaneCh, U = kConvStep;
  const unsigned int tile = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.groups;
  const int64_t t0 = ((int64_t)(rest % a.groups) * kConvWarps + (threadIdx.x >> 5)) * kConvRun;
  if (t0 >= a.length && t0 > 0) return;
  const ConvLane<T, VEC> lane((int64_t)tile * kConvChannels, a.dim);
  const int64_t row = b * a.length, end = min(a.length, t0 + kConvRun);
  float w[W][C], bias[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const bool on = c < lane.live;
    const int64_t d = lane.d + lane.at(c);
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][c] = on ? a.w[d * W + k] : 0.0f;
    bias[c] = on && a.bias ? a.bias[d] : 0.0f;
  }
  float xs[W - 1 + U][C];  // token t0 - (W - 1) first
#pragma unroll
  for (int k = 0; k < W - 1; ++k) conv_token<T, W, VEC>(a, lane, b, t0 - (W - 1) + k, xs[k]);
  for (int64_t t = t0; t < end; t += U) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      lane.load(xs[W - 1 + i], a.x + b * a.x_sb + (t + i) * a.x_st, t + i < end);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int age = a.starts && t + i < end ? conv_age<W>(a.starts, row, t + i) : W - 1;
      float u[C];
#pragma unroll
      for (int c = 0; c < C; ++c) u[c] = bias[c];
#pragma unroll
      for (int k = 0; k < W; ++k)  // tap k, W - 1 - k tokens back
        if (W - 1 - k <= age) {
#pragma unroll
          for (int c = 0; c < C; ++c) u[c] = fmaf(w[k][c], xs[i + k][c], u[c]);
        }
      if (a.silu) {
#pragma unroll
        for (int c = 0; c < C; ++c) u[c] *= sigmoid_f32(u[c]);
      }
      if (t + i < end) lane.store(a.y + (row + t + i) * a.dim, u);
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int c = 0; c < C; ++c) xs[k][c] = xs[U + k][c];
  }
  if (a.last && end == a.length && (end > t0 || t0 == 0)) {  // the run of the last token
    const int age = a.length > 0 ? conv_age<W>(a.starts, row, a.length - 1) : W - 1;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      float v[C];
      conv_token<T, W, VEC>(a, lane, b, a.length - (W - 1) + k, v);
      if (W - 2 - k > age) {
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = 0.0f;
      }
      lane.store(a.last + (b * (W - 1) + k) * a.dim, v);
    }
  }
}

// A run of the VJP owns R = kConvRun - (W - 1) tokens and goes through the W - 1
// after them too, whose du its last tokens need.
template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(kConvWarps * 32) conv_bwd_kernel(ConvArgs<T> a) {
  constexpr int C = kConvLaneCh, U = kConvStep, R = kConvRun - (W - 1);
  __shared__ float sums[kConvWarps][kConvChannels];
  const unsigned int tile = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.groups;
  const int warp = threadIdx.x >> 5;
  const int64_t t0 = ((int64_t)(rest % a.groups) * kConvWarps + warp) * R;
  const ConvLane<T, VEC> lane((int64_t)tile * kConvChannels, a.dim);
  const int64_t row = b * a.length, own = min(a.length, t0 + R);
  float w[W][C], bias[C], dw[W][C], db[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const bool on = c < lane.live;
    const int64_t d = lane.d + lane.at(c);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      w[k][c] = on ? a.w[d * W + k] : 0.0f;
      dw[k][c] = 0.0f;
    }
    bias[c] = on && a.bias ? a.bias[d] : 0.0f;
    db[c] = 0.0f;
  }
  if (t0 < a.length || t0 == 0) {
    float xs[W - 1 + U][C];   // token t - (W - 1) first
    float acc[W - 1 + U][C];  // and its gradient
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      conv_token<T, W, VEC>(a, lane, b, t0 - (W - 1) + k, xs[k]);
#pragma unroll
      for (int c = 0; c < C; ++c) acc[k][c] = 0.0f;
    }
    const int last_age = a.dlast && a.length > 0 ? conv_age<W>(a.starts, row, a.length - 1) : W - 1;
    // token s, whose gradient is complete but for dlast's share
    auto emit = [&](int64_t s, float (&v)[C]) {
      if (s < (t0 == 0 ? 1 - W : t0) || s >= own) return;
      const int back = (int)min(a.length - 1 - s, (int64_t)W);  // tokens before the last
      if (a.dlast && back < W - 1 && back <= last_age) {
        float e[C];
        lane.load(e, a.dlast + (b * (W - 1) + W - 2 - back) * a.dim, true);
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] += e[c];
      }
      if (s >= 0) lane.store(a.dx + (row + s) * a.dim, v);
      else if (a.dx0) lane.store(a.dx0 + (b * (W - 1) + s + W - 1) * a.dim, v);
    };
    for (int64_t t = t0; t < t0 + kConvRun && t < a.length + W - 1; t += U) {
      float dy[U][C];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        lane.load(xs[W - 1 + i], a.x + b * a.x_sb + (t + i) * a.x_st, t + i < a.length);
        lane.load(dy[i], a.dy + b * a.dy_sb + (t + i) * a.dy_st, t + i < a.length && a.dy);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[W - 1 + i][c] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (t + i >= a.length) continue;
        const int age = a.starts ? conv_age<W>(a.starts, row, t + i) : W - 1;
        float u[C];
#pragma unroll
        for (int c = 0; c < C; ++c) u[c] = bias[c];
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (W - 1 - k <= age) {
#pragma unroll
            for (int c = 0; c < C; ++c) u[c] = fmaf(w[k][c], xs[i + k][c], u[c]);
          }
        if (a.silu) {  // (u s)' = s + u s (1 - s)
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float s = sigmoid_f32(u[c]);
            u[c] = dy[i][c] * fmaf(u[c] * s, 1.0f - s, s);
          }
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c) u[c] = dy[i][c];
        }
        const bool mine = t + i < own;
#pragma unroll
        for (int c = 0; c < C; ++c) db[c] += mine ? u[c] : 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (W - 1 - k <= age) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
              acc[i + k][c] = fmaf(w[k][c], u[c], acc[i + k][c]);
              if (mine) dw[k][c] = fmaf(u[c], xs[i + k][c], dw[k][c]);
            }
          }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) emit(t + i - (W - 1), acc[i]);
#pragma unroll
      for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          xs[k][c] = xs[U + k][c];
          acc[k][c] = acc[U + k][c];
        }
    }
  }
  // over the warps, then one row of partial sums a CTA: [dim][W], then [dim]
  float* part = a.parts + (int64_t)rest * a.dim * (W + 1);
#pragma unroll
  for (int k = 0; k <= W; ++k) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      sums[warp][VEC ? (threadIdx.x & 31) * C + c : (threadIdx.x & 31) + 32 * c] =
          k < W ? dw[k < W ? k : 0][c] : db[c];
    __syncthreads();
    const int64_t d = (int64_t)tile * kConvChannels + threadIdx.x;
    if (threadIdx.x < kConvChannels && d < a.dim) {
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
static bool conv_vector(const T* p, int64_t sb, int64_t st) {
  constexpr size_t n = kConvLaneCh * sizeof(T);
  return !p || (aligned_to(p, n) && sb % kConvLaneCh == 0 && st % kConvLaneCh == 0);
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

static int64_t conv_groups(int64_t length, int64_t run) {
  const int64_t per = run * kConvWarps;
  return std::max<int64_t>(1, (length + per - 1) / per);
}

template <typename T>
static oxc_status conv_launch(ConvArgs<T> a, int64_t width, bool backward, cudaStream_t s) {
  const bool vec = a.dim % kConvLaneCh == 0 && conv_vector(a.x, a.x_sb, a.x_st) &&
                   conv_vector(a.dy, a.dy_sb, a.dy_st) && conv_vector(a.x0, 0, 0) &&
                   conv_vector(a.dlast, 0, 0) && conv_vector<T>(a.y, 0, 0) &&
                   conv_vector<T>(a.last, 0, 0) && conv_vector<T>(a.dx, 0, 0) &&
                   conv_vector<T>(a.dx0, 0, 0);
  const int64_t run = backward ? kConvRun - (width - 1) : kConvRun;
  const int64_t ctiles = (a.dim + kConvChannels - 1) / kConvChannels;
  const int64_t groups = conv_groups(a.length, run);
  if (ctiles * groups > 0x7fffffff / std::max<int64_t>(a.batch, 1))
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: causal_conv: more than 2^31 blocks");
  a.ctiles = (unsigned int)ctiles;
  a.groups = (unsigned int)groups;
  const unsigned int grid = (unsigned int)(a.batch * ctiles * groups);
  by_width(width, [&](auto w) {
    constexpr int W = decltype(w)::value;
    if (backward) {
      if (vec) conv_bwd_kernel<T, W, true><<<grid, kConvWarps * 32, 0, s>>>(a);
      else conv_bwd_kernel<T, W, false><<<grid, kConvWarps * 32, 0, s>>>(a);
    } else {
      if (vec) conv_fwd_kernel<T, W, true><<<grid, kConvWarps * 32, 0, s>>>(a);
      else conv_fwd_kernel<T, W, false><<<grid, kConvWarps * 32, 0, s>>>(a);
    }
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
    a.silu = silu;
    return conv_launch<T>(a, width, false, s);
  };
  return dtype == OXC_BF16 ? go(bf16{}) : go(0.0f);
}

size_t oxc_causal_conv_bwd_workspace_size(int64_t batch, int64_t length, int64_t dim, int64_t width) {
  if (batch <= 0 || length < 0 || dim <= 0 || width < 1 || width > kConvMaxWidth) return 0;
  return sizeof(float) * (size_t)(batch * conv_groups(length, kConvRun - (width - 1))) *
         (size_t)(dim * (width + 1));
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
    a.silu = silu;
    return conv_launch<T>(a, width, true, s);
  };
  const oxc_status r = dtype == OXC_BF16 ? go(bf16{}) : go(0.0f);
  if (r) return r;
  launch_colsum_partials(static_cast<const float*>(workspace),
                         (int)(batch * conv_groups(length, kConvRun - (width - 1))), cols, dw, s);
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
