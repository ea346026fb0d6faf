// add_rms_norm.cu -- the residual's addition followed by RMSNorm, its VJP, and
// the same norm written in 8 bits with scales.
//
//   r = x + residual          (f32, the new residual stream)
//   inv = 1 / sqrt(mean_row(r^2) + eps)
//   y = r * inv * w           (rounded once to x's type)
//
// VJP, with dy and dr the gradients of y and r, g = dy * w, u = r * inv:
//   dresidual = dr + inv * g                          OXC_GRAD_REF (inv a constant)
//   dresidual = dr + inv * (g - u * mean_row(g * u))  OXC_GRAD_EXACT
//   dx = dresidual rounded to x's type,  dw = sum_rows dy * u
//
// The residual stream, the weight and every sum are f32 whatever x's type, so
// the stream loses nothing as layers add to it and the VJP sees the r that the
// forward normalised.
//
// 8-bit output: per row, each block of `block` columns has the scale
// s = max(amax(|y|) / 448, 2^-126) and q = e4m3(y / s), 448 being e4m3's
// largest value.  y is not rounded to x's type in between, and its f32 product is
// the one that the forward rounds.
//
// All are bound by HBM traffic: 8 + 2 sizeof(T) bytes an element forward, 9 +
// sizeof(T) with the 8-bit output, 12 + sizeof(T) (and 2 more at 16 bits) for the
// VJP.  A row is held in registers by a group of 1 to 32 warps (as many as its
// width needs at 4 vectors a thread, 2 in the VJP; narrow rows share a CTA), all
// of its loads issued before the first is used.  Measured, of the copy bandwidth:
// [16384, 4096] f32 162 us forward (100%), 173 us VJP (95%), bf16 8-bit output 122
// us (92%); bf16 [8192, 5001] 85, 124 and 111 us (88%, 81%, 62%: the blocks of 128
// columns of such a row lie across warps).
//
// Vectors are 4 elements at addresses that are multiples of 4 elements.  Where the
// columns are not a multiple of 4, a row starts `o` = 0 to 3 elements after such an
// address, the same in every tensor (row_shift); the row's first and last vectors
// are then partial ones, read and written by element.  Tensors that differ in
// that take the kernels for single elements, as do rows of 32766 and 32767 columns.
#include <cuda_fp8.h>

#include <algorithm>

#include "rowvec.cuh"
#include "typed.cuh"

namespace oxc {

constexpr int kQuantMaxBlocks = 32768 / 128;

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint32_t to_e4m3x4(float2 a, float2 b) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// A block's scale from the bits of its largest |y|, which order like the values,
// NaN above infinity: a NaN in a block makes its scale NaN.
__device__ __forceinline__ float quant_scale(uint32_t amax) {
  const float a = __uint_as_float(amax);
  return a != a ? a : fmaxf(__fdiv_rn(a, 448.0f), 1.17549435e-38f);
}

// y / s for a pair of columns, rounded to nearest: z = y * RN(1 / s) is off by up to 1.5
// ulp, y - z s is exact in one fma, and a second fma adds what it is worth (Markstein,
// IBM J. Res. Dev. 34, 1990).  Two packed operations more than z alone, whose code is
// the other one beside a tie in some 10 of 24 million elements; __fdiv_rn gives the
// same codes at 3 to 19% more of the kernel's time instead of 2 to 8%.  An infinite scale
// has no remainder: 0 for finite y, NaN for infinite.  (Where y is near the smallest
// normal number the remainder may lie under 2^-149, and z stands.)
struct Divisor {
  float minus_s, rcp;
};
__device__ __forceinline__ Divisor divisor(float s) {
  return {s == INFINITY ? 0.0f : -s, __fdiv_rn(1.0f, s)};
}
__device__ __forceinline__ float2 quotients(float2 y, const Divisor& a, const Divisor& b) {
  const float2 rcp = make_float2(a.rcp, b.rcp);
  const float2 z = __fmul2_rn(y, rcp);
  return __ffma2_rn(__ffma2_rn(z, make_float2(a.minus_s, b.minus_s), y), rcp, z);
}

// ---- rows in groups of warps ------------------------------------------------------------

// Four elements as loaded: 16 bytes of f32, 8 of bf16.
__device__ __forceinline__ float4 load_raw(const float* p) { return ld_stream(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ uint2 load_raw(const bf16* p) { return __ldcs(reinterpret_cast<const uint2*>(p)); }
__device__ __forceinline__ void raw_f32(float (&d)[4], const float4& t) {
  d[0] = t.x; d[1] = t.y; d[2] = t.z; d[3] = t.w;
}
__device__ __forceinline__ void raw_f32(float (&d)[4], const uint2& t) {
  d[0] = bf16_lo(t.x); d[1] = bf16_hi(t.x); d[2] = bf16_lo(t.y); d[3] = bf16_hi(t.y);
}
template <typename T>
using raw_t = decltype(load_raw(static_cast<const T*>(nullptr)));

// A thread's place in its row: vector i covers columns [e(i), e(i) + 4) of which
// those outside [0, cols) do not exist.  Without EDGE the shift is 0 and a vector
// exists whole or not at all.  With it the row's first and last vectors are loaded
// whole like the others and then masked: what they hold beside the row is memory of
// the rows before and after it, or between them -- except after the last row, whose
// last vector is read by element.
template <bool EDGE>
struct RowSlots {
  int cols, o, first, step;  // columns; shift; the thread's first vector, from one to the next
  __device__ __forceinline__ int e(int i) const { return 4 * (first + i * step) - (EDGE ? o : 0); }
  __device__ __forceinline__ bool partial(int e) const { return EDGE && (e < 0 || e + 4 > cols); }
  // the nearest vector that can be loaded: somewhere to load from without a branch
  __device__ __forceinline__ int near(int e, bool last_row) const {
    if constexpr (!EDGE) return min(e, cols - 4);
    return min(e, ((cols + o + (last_row ? 0 : 3)) & ~3) - 4 - o);
  }
  template <typename T>
  __device__ __forceinline__ void take(float (&d)[4], const raw_t<T>& raw, const T* row, int e,
                                       bool last_row) const {
    raw_f32(d, raw);
    if (!EDGE) {
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = e < cols ? d[k] : 0.0f;
    } else if (partial(e)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = e + k >= 0 && e + k < cols ? d[k] : 0.0f;
      if (last_row && e < cols && e + 4 > cols) {
#pragma unroll
        for (int k = 0; k < 3; ++k) d[k] = e + k < cols ? to_f32(row[e + k]) : 0.0f;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void put(T* row, int e, const float (&d)[4]) const {
    if (!partial(e)) {
      store_from_f32<4>(row + e, d);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k >= 0 && e + k < cols) row[e + k] = from_f32<T>(d[k]);
    }
  }
  // a [cols] parameter, 16-byte aligned
  __device__ __forceinline__ void weights(float (&d)[4], const float* w, int e) const {
    if (!EDGE || (o == 0 && !partial(e))) {
      raw_f32(d, __ldg(reinterpret_cast<const float4*>(w + near(e, true))));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = __ldg(w + min(max(e + k, 0), cols - 1));
    }
  }
};

// Barrier and sum over a group of warps; `scratch` has a place for each of its
// warps and is not written again before the group's next barrier.
__device__ __forceinline__ void group_sync(int group, int warps) {
  if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * warps) : "memory");
  else __syncwarp();
}
__device__ __forceinline__ float group_total(float v, float* scratch, int group, int warps) {
  v = warp_sum(v);
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - group * warps;
  if (lane == 0) scratch[warp] = v;
  group_sync(group, warps);
  return warp_sum(lane < warps ? scratch[lane] : 0.0f);
}

constexpr int kMaxGroups = 8;  // per CTA

template <typename T, int VPT, int MAXT, bool QUANT, bool EDGE>
__global__ void __launch_bounds__(MAXT, 1024 / MAXT) add_rms_fwd_rows_kernel(
    const T* __restrict__ x, int64_t x_stride, const float* __restrict__ res, int64_t res_stride,
    const float* __restrict__ w, T* __restrict__ y, uint8_t* __restrict__ q,
    float* __restrict__ scale, int block_shift, float* __restrict__ r, float* __restrict__ rstd,
    int64_t rows, int cols, float eps, int group_warps) {
  __shared__ float scratch[32];
  __shared__ uint32_t amax[!QUANT ? 1 : EDGE ? kQuantMaxBlocks + 1 : 32];  // of blocks or warps
  __shared__ Divisor divisors[QUANT && EDGE ? kQuantMaxBlocks + 1 : 1];
  const int lane = threadIdx.x & 31, group = (threadIdx.x >> 5) / group_warps;
  const int in_group = threadIdx.x - group * group_warps * 32;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / (32 * group_warps)) + group;
  if (row >= rows) return;  // the whole group
  const RowSlots<EDGE> s{cols, EDGE ? (int)((row * cols) & 3) : 0, in_group, group_warps * 32};
  const T* xr = x + row * x_stride;
  const float* rr = res + row * res_stride;
  const bool last_row = row == rows - 1;
  raw_t<T> rx[VPT];
  float4 rv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = s.near(s.e(i), last_row);
    rx[i] = load_raw(xr + e);
    rv[i] = load_raw(rr + e);
  }
  const int blocks = QUANT && EDGE ? ((cols - 1) >> block_shift) + 1 : 0;
  uint32_t* am = amax + group * blocks;
  if constexpr (QUANT && EDGE) {
    for (int b = in_group; b < blocks; b += 32 * group_warps) am[b] = 0u;
  }
  float v[VPT][4];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = s.e(i);
    float a[4];
    s.take(a, rx[i], xr, e, last_row);
    s.take(v[i], rv[i], rr, e, last_row);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[i][k] += a[k];
      ss = fmaf(v[i][k], v[i][k], ss);
    }
    if (e < cols) s.put(r + row * (int64_t)cols, e, v[i]);
  }
  ss = group_total(ss, scratch + group * group_warps, group, group_warps);
  const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)cols) + eps));
  if constexpr (!QUANT) {
    if (in_group == 0) rstd[row] = inv;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.e(i);
      if (e < cols) {
        float wv[4], o[4];
        s.weights(wv, w, e);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = v[i][k] * inv * wv[k];
        s.put(y + row * (int64_t)cols, e, o);
      }
    }
  } else if constexpr (!EDGE) {  // a block of 128 columns is a warp's own affair
    const bool by_block = block_shift == 7;
    uint32_t m[VPT], all = 0u;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.e(i);
      float wv[4];
      s.weights(wv, w, e);
      m[i] = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[i][k] = v[i][k] * inv * wv[k];
        m[i] = max(m[i], e < cols ? __float_as_uint(fabsf(v[i][k])) : 0u);
      }
      m[i] = __reduce_max_sync(0xffffffffu, m[i]);
      all = max(all, m[i]);
    }
    if (!by_block && group_warps > 1) {
      if (lane == 0) amax[threadIdx.x >> 5] = all;
      group_sync(group, group_warps);
      all = __reduce_max_sync(0xffffffffu, lane < group_warps ? amax[group * group_warps + lane] : 0u);
    }
    uint8_t* qr = q + row * (int64_t)cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.e(i);
      const float sc = quant_scale(by_block ? m[i] : all);
      const Divisor by = divisor(sc);
      if (e < cols) {
        *reinterpret_cast<uint32_t*>(qr + e) = to_e4m3x4(quotients(make_float2(v[i][0], v[i][1]), by, by),
                                                         quotients(make_float2(v[i][2], v[i][3]), by, by));
        if (lane == 0 && (by_block || e == 0)) scale[by_block ? row * ((cols + 127) / 128) + e / 128 : row] = sc;
      }
    }
  } else {  // with a shift the blocks lie across warps
    uint32_t m[VPT];
    if (group_warps == 1) __syncwarp();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.e(i);
      float wv[4];
      s.weights(wv, w, e);
      uint32_t before = 0u;  // of the columns of the block before the warp's
      m[i] = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[i][k] = v[i][k] * inv * wv[k];
        const bool in = e + k >= 0 && e + k < cols;
        const uint32_t u = in ? __float_as_uint(fabsf(v[i][k])) : 0u;
        if (lane == 0 && k < s.o) before = max(before, u);
        else m[i] = max(m[i], u);
      }
      m[i] = __reduce_max_sync(0xffffffffu, m[i]);
      const int e0 = __shfl_sync(0xffffffffu, e, 0) + s.o;  // a multiple of 128
      if (lane == 0 && e0 < cols + s.o) {
        if (e0 < cols) atomicMax(&am[e0 >> block_shift], m[i]);
        if (s.o && e0 > 0) atomicMax(&am[(e0 - 1) >> block_shift], before);
      }
    }
    group_sync(group, group_warps);
    // each block's scale and reciprocal once
    Divisor* by = divisors + group * blocks;
    for (int b = in_group; b < blocks; b += 32 * group_warps) {
      const float sc = quant_scale(am[b]);
      scale[row * blocks + b] = sc;
      by[b] = divisor(sc);
    }
    group_sync(group, group_warps);
    uint8_t* qr = q + row * (int64_t)cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.e(i);
      if (e >= cols) continue;
      // at most two blocks meet in a vector
      const int b0 = max(e, 0) >> block_shift, b1 = min(e + 3, cols - 1) >> block_shift;
      const Divisor d0 = by[b0], d1 = by[b1];
      auto of = [&](int k) { return (max(e + k, 0) >> block_shift) == b0 ? d0 : d1; };
      const uint32_t o = to_e4m3x4(quotients(make_float2(v[i][0], v[i][1]), of(0), of(1)),
                                   quotients(make_float2(v[i][2], v[i][3]), of(2), of(3)));
      if (!s.partial(e)) {
        *reinterpret_cast<uint32_t*>(qr + e) = o;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (e + k >= 0 && e + k < cols) qr[e + k] = (uint8_t)(o >> (8 * k));
      }
    }
  }
}

// Asks L2 for n elements, but those that share 16 bytes with what lies after them.
template <typename T>
__device__ __forceinline__ void ask_row(const T* p, int n) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15;
  const uint32_t bytes = (uint32_t)(reinterpret_cast<uintptr_t>(p + n) - from) & ~15u;
  if (bytes)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(bytes) : "memory");
}

// CTAs of the VJP on an SM.
__host__ __device__ constexpr int bwd_ctas(int vpt, bool edge, int threads) {
  const int n = vpt >= 4 ? 1 : (edge && vpt == 2 ? 768 : 1024) / threads;
  return n > 1 ? n : 1;
}

// Persistent VJP.  Rows whose shift is equal (`period` apart) belong to one CTA, so
// a thread's columns, and with them its dw sums, stay the same; the CTA's groups
// are added in shared memory, in order, into its partial parts[b][cols].
template <typename T, int VPT, int MAXT, int MODE, bool EDGE>
__global__ void __launch_bounds__(MAXT, bwd_ctas(VPT, EDGE, MAXT)) add_rms_bwd_rows_kernel(
    const float* __restrict__ r, const float* __restrict__ w, const float* __restrict__ rstd,
    const T* __restrict__ dy, int64_t dy_stride, const float* __restrict__ dr, int64_t dr_stride,
    float* __restrict__ dres, T* __restrict__ dx, float* __restrict__ parts, int64_t rows, int cols,
    int period, int group_warps) {
  pdl_launch_dependents();  // the dweight finisher waits for this grid
  __shared__ float scratch[2][32];
  extern __shared__ __align__(16) float sums[];  // by column (several groups) or by vector
  const int group = (threadIdx.x >> 5) / group_warps, groups = blockDim.x / (32 * group_warps);
  const int in_group = threadIdx.x - group * group_warps * 32;
  const int part = blockIdx.x % period;
  const int64_t ctas = (gridDim.x - part + period - 1) / period;
  const RowSlots<EDGE> s{cols, EDGE ? (int)(((int64_t)part * cols) & 3) : 0, in_group, group_warps * 32};
  // the dw sums and the weights: registers, or this thread's own vectors of shared
  // memory in wide rows (one group a CTA; beyond 4 vectors the weights are read anew
  // for each row)
  constexpr bool kShared = VPT >= 4, kOwnW = kShared && VPT <= 4;
  float4* own_sums = reinterpret_cast<float4*>(sums) + threadIdx.x;
  float4* own_w = own_sums + VPT * blockDim.x;
  float w_held[kShared ? 1 : VPT][4], acc[kShared ? 1 : VPT][4];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if constexpr (kShared) {
      own_sums[i * blockDim.x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if constexpr (kOwnW) {
        float wv[4];
        s.weights(wv, w, s.e(i));
        own_w[i * blockDim.x] = make_float4(wv[0], wv[1], wv[2], wv[3]);
      }
    } else {
      s.weights(w_held[i], w, s.e(i));
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = 0.0f;
    }
  }
  // With few threads on the SM, nobody else loads while these add up and write: L2 is
  // asked for the CTA's next row (bf16 [8192, 5000] 122 us instead of 141; with 1024
  // threads in several CTAs, [16384, 4096], 184 instead of 174).
  constexpr bool kAhead = (EDGE && VPT > 1) || MAXT > 512 || MAXT == 384;
  const float inv_n = __fdiv_rn(1.0f, (float)cols);
  int parity = 0;
  for (int64_t row = part + period * ((blockIdx.x / period) * groups + group); row < rows;
       row += period * ctas * groups, parity ^= 1) {
    const float* ur = r + row * (int64_t)cols;
    const T* gr = dy + row * dy_stride;
    const float* pr = dr ? dr + row * dr_stride : nullptr;
    const bool last_row = row == rows - 1;
    float4 ru[VPT], rd[VPT];
    raw_t<T> rg[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.near(s.e(i), last_row);
      ru[i] = load_raw(ur + e);
      rg[i] = load_raw(gr + e);
    }
    auto load_dr = [&] {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        rd[i] = pr ? load_raw(pr + s.near(s.e(i), last_row)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    if constexpr (!kShared) load_dr();
    if (kAhead && threadIdx.x == 0) {
      const int64_t next = row + period * ctas * groups;
      if (next < rows) {
        ask_row(r + next * cols, cols);
        ask_row(dy + next * dy_stride, cols);
        if (dr) ask_row(dr + next * dr_stride, cols);
      }
    }
    const float inv = __ldg(rstd + row);
    float u[VPT][4], g[VPT][4];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      s.take(u[i], ru[i], ur, s.e(i), last_row);
      s.take(g[i], rg[i], gr, s.e(i), last_row);
      float now[4], wv[4];
      if constexpr (kShared) raw_f32(now, own_sums[i * blockDim.x]);
      if constexpr (kOwnW) raw_f32(wv, own_w[i * blockDim.x]);
      else if constexpr (kShared) s.weights(wv, w, s.e(i));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        u[i][k] *= inv;
        if constexpr (kShared) now[k] = fmaf(g[i][k], u[i][k], now[k]);
        else acc[i][k] = fmaf(g[i][k], u[i][k], acc[i][k]);
        g[i][k] *= kShared ? wv[k] : w_held[kShared ? 0 : i][k];
        sum = fmaf(g[i][k], u[i][k], sum);
      }
      if constexpr (kShared) own_sums[i * blockDim.x] = make_float4(now[0], now[1], now[2], now[3]);
    }
    if constexpr (kShared) load_dr();  // all three at once would not fit the registers
    float mean = 0.0f;
    if constexpr (MODE == OXC_GRAD_EXACT)
      mean = group_total(sum, scratch[parity] + group * group_warps, group, group_warps) * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = s.e(i);
      if (e >= cols) continue;
      float d[4];
      if (pr) s.take(d, rd[i], pr, e, last_row);
      else raw_f32(d, rd[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (MODE == OXC_GRAD_EXACT) g[i][k] = fmaf(-u[i][k], mean, g[i][k]);
        d[k] = fmaf(inv, g[i][k], d[k]);
      }
      s.put(dres + row * (int64_t)cols, e, d);
      if constexpr (sizeof(T) == 2) s.put(dx + row * (int64_t)cols, e, d);
    }
  }
  float* pr = parts + (int64_t)blockIdx.x * cols;
  if constexpr (kShared) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float now[4];
      raw_f32(now, own_sums[i * blockDim.x]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = s.e(i) + k;
        if (c >= 0 && c < cols) pr[c] = now[k];
      }
    }
  } else {
    for (int gi = 0; gi < groups; ++gi) {  // one group after the other
      if (group == gi) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int c = s.e(i) + k;
            if (c < 0 || c >= cols) continue;
            const float a = gi > 0 ? sums[c] + acc[i][k] : acc[i][k];
            if (gi + 1 < groups) sums[c] = a;
            else pr[c] = a;
          }
      }
      __syncthreads();
    }
  }
}

// ---- single elements: rows that no common shift fits --------------------------------------

// One CTA per row, the row in registers: thread t holds the elements t, t +
// blockDim, ...
template <typename T, int VPT, bool QUANT>
__global__ void __launch_bounds__(1024) add_rms_fwd_kernel(
    const T* __restrict__ x, int64_t x_stride, const float* __restrict__ res, int64_t res_stride,
    const float* __restrict__ w, T* __restrict__ y, uint8_t* __restrict__ q,
    float* __restrict__ scale, int block_shift, float* __restrict__ r, float* __restrict__ rstd,
    int64_t rows, int cols, float eps) {
  __shared__ float scratch[33];
  __shared__ uint32_t amax[QUANT ? kQuantMaxBlocks : 1];
  const int blocks = QUANT ? ((cols - 1) >> block_shift) + 1 : 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * x_stride;
    const float* rr = res + row * res_stride;
    const int64_t out = row * (int64_t)cols;
    if constexpr (QUANT) {
      for (int b = threadIdx.x; b < blocks; b += blockDim.x) amax[b] = 0u;
    }
    float v[VPT];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = i * blockDim.x + threadIdx.x;
      v[i] = e < cols ? to_f32(xr[e]) + ld_stream(rr + e) : 0.0f;
      ss = fmaf(v[i], v[i], ss);
    }
    ss = block_sum(ss, scratch);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)cols) + eps));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = i * blockDim.x + threadIdx.x;
      if (e >= cols) continue;
      st_stream(r + out + e, v[i]);
      v[i] = v[i] * inv * __ldg(w + e);
      if constexpr (QUANT) atomicMax(&amax[e >> block_shift], __float_as_uint(fabsf(v[i])));
      else y[out + e] = from_f32<T>(v[i]);
    }
    if constexpr (QUANT) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = i * blockDim.x + threadIdx.x;
        if (e >= cols) continue;
        const int b = e >> block_shift;
        const float s = quant_scale(amax[b]);
        const Divisor by = divisor(s);
        q[out + e] = to_e4m3(quotients(make_float2(v[i], v[i]), by, by).x);
        if (e == b << block_shift) scale[row * blocks + b] = s;
      }
      __syncthreads();  // amax is read; the next row clears it
    } else if (threadIdx.x == 0) {
      rstd[row] = inv;
    }
  }
}

// Persistent VJP: CTA b handles rows [b * chunk, min((b + 1) * chunk, rows)) and
// writes its dw partial to parts[b][cols].
template <typename T, int VPT, int MODE>
__global__ void __launch_bounds__(1024) add_rms_bwd_kernel(
    const float* __restrict__ r, const float* __restrict__ w, const float* __restrict__ rstd,
    const T* __restrict__ dy, int64_t dy_stride, const float* __restrict__ dr, int64_t dr_stride,
    float* __restrict__ dres, T* __restrict__ dx, float* __restrict__ parts, int64_t rows, int cols,
    int64_t chunk) {
  pdl_launch_dependents();  // the dweight finisher waits for this grid
  __shared__ float scratch[33];
  const int64_t r0 = (int64_t)blockIdx.x * chunk;
  const int64_t r1 = min(rows, r0 + chunk);
  float wv[VPT], acc[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = i * blockDim.x + threadIdx.x;
    acc[i] = 0.0f;
    wv[i] = e < cols ? __ldg(w + e) : 0.0f;
  }
  const float inv_n = __fdiv_rn(1.0f, (float)cols);
  for (int64_t row = r0; row < r1; ++row) {
    const float inv = __ldg(rstd + row);
    const int64_t out = row * (int64_t)cols;
    float u[VPT], g[VPT];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = i * blockDim.x + threadIdx.x;
      u[i] = e < cols ? ld_stream(r + out + e) * inv : 0.0f;
      g[i] = e < cols ? to_f32(dy[row * dy_stride + e]) : 0.0f;
      acc[i] = fmaf(g[i], u[i], acc[i]);
      g[i] *= wv[i];
      s = fmaf(g[i], u[i], s);
    }
    float mean = 0.0f;
    if constexpr (MODE == OXC_GRAD_EXACT) mean = block_sum(s, scratch) * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = i * blockDim.x + threadIdx.x;
      if (e >= cols) continue;
      if constexpr (MODE == OXC_GRAD_EXACT) g[i] = fmaf(-u[i], mean, g[i]);
      const float d = fmaf(inv, g[i], dr ? ld_stream(dr + row * dr_stride + e) : 0.0f);
      st_stream(dres + out + e, d);
      if constexpr (sizeof(T) == 2) dx[out + e] = from_f32<T>(d);
    }
  }
  float* pr = parts + (int64_t)blockIdx.x * cols;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = i * blockDim.x + threadIdx.x;
    if (e < cols) pr[e] = acc[i];
  }
}

// Warps per row, rows per CTA and vectors per thread, for rows of `slots` vectors:
// `vpt` vectors a thread where 32 warps suffice, more beyond.
struct GroupGeom {
  int vpt, warps, groups;
  int threads() const { return 32 * warps * groups; }
  // 8 vectors a thread at most: all rows but those of 32766 and 32767 columns, whose
  // shifts touch up to 8193 vectors (the single-element kernels hold them: bf16 [2000,
  // 32766] 264 us, 1.09 ms VJP; 32765 columns 158 us and 1.02 ms, as 8 vectors spill)
  bool held() const { return vpt <= 8; }
};
static GroupGeom group_geom(int64_t cols, int vpt) {
  const int64_t slots = (cols + (cols % 4 ? 3 : 0) + 3) / 4;
  while (vpt > 1 && slots <= 32 * (vpt / 2)) vpt /= 2;
  while (slots > 32 * 32 * vpt) vpt *= 2;
  const int warps = (int)((slots + 32 * vpt - 1) / (32 * vpt));
  return {vpt, warps, warps >= kMaxGroups ? 1 : kMaxGroups / warps};
}
constexpr int kFwdVecs = 4;
// 2 vectors a thread in the VJP: its 64 registers let 1024 threads share an SM.  The
// masks of rows of odd width need about 90, or they spill: fewer threads share the SM
// (bf16 [8192, 1001]: 29 us instead of 36), and where a row alone needs more than 640
// they have 4 vectors each ([8192, 7001]: 179 us instead of 205).
static GroupGeom bwd_geom(int64_t cols) {
  const GroupGeom g = group_geom(cols, 2);
  if (cols % 4 && g.vpt == 2 && g.threads() > 640) return group_geom(cols, 4);
  return g;
}

// CTAs of the VJP: as many as are resident, at least 4 rows a group; 4 at least,
// one for each shift of the rows.
static int64_t add_rms_bwd_ctas(int64_t rows, int64_t cols) {
  const GroupGeom g = bwd_geom(cols);
  const int64_t per_sm = bwd_ctas(g.vpt, cols % 4 != 0, g.threads());
  const int64_t by_rows = (rows + 4 * g.groups - 1) / (4 * g.groups);
  return std::max<int64_t>(4, std::min<int64_t>(per_sm * sm_count(), by_rows));
}

static oxc_status add_rms_check(const char* fn, int32_t dtype, int64_t rows, int64_t cols) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: unknown dtype %d", fn, dtype);
  if (rows < 0 || cols < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: negative shape [%lld, %lld]", fn,
                (long long)rows, (long long)cols);
  if (cols > 32768)
    return fail(OXC_ERR_NOT_IMPLEMENTED,
                "not implemented: %s: rows wider than 32768 elements are not supported", fn);
  if (cols == 0 && rows > 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s over a zero-length dim", fn);
  return OXC_OK;
}

// Whether every row of x (and of the f32 tensor f) starts where the rows of the
// dense tensors do, relative to a multiple of 4 elements, and where vectors are
// partial (columns not a multiple of 4) at least 4 elements after the row before.
template <typename T>
static bool row_shift(const void* x, int64_t x_stride, const void* f, int64_t f_stride,
                      int64_t cols, int64_t rows) {
  return cols >= 8 && aligned_to(x, 4 * sizeof(T)) && aligned16(f) &&
         (rows == 1 || ((x_stride - cols) % 4 == 0 && (f_stride - cols) % 4 == 0 &&
                        (cols % 4 == 0 || std::min(x_stride, f_stride) >= 4)));
}

template <typename T, bool QUANT>
static oxc_status add_rms_fwd_launch(const char* fn, const void* x, int64_t x_stride,
                                     const float* res, int64_t res_stride, const float* w, void* y,
                                     uint8_t* q, float* scale, int block_shift, float* r,
                                     float* rstd, int64_t rows, int64_t cols, float eps,
                                     cudaStream_t s) {
  if (group_geom(cols, kFwdVecs).held() && row_shift<T>(x, x_stride, res, res_stride, cols, rows) &&
      aligned16(w) && aligned16(r) && (QUANT ? aligned_to(q, 4) : aligned_to(y, 4 * sizeof(T)))) {
    const GroupGeom g = group_geom(cols, kFwdVecs);
    const int64_t grid = (rows + g.groups - 1) / g.groups;
    if (grid > 0x7fffffff)
      return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: %lld rows", fn, (long long)rows);
#define LAUNCH(VPT, MAXT)                                                                       \
  (cols % 4 ? add_rms_fwd_rows_kernel<T, VPT, MAXT, QUANT, true>                                \
            : add_rms_fwd_rows_kernel<T, VPT, MAXT, QUANT, false>)<<<(unsigned)grid, g.threads(), 0, s>>>( \
      static_cast<const T*>(x), x_stride, res, res_stride, w, static_cast<T*>(y), q, scale,     \
      block_shift, r, rstd, rows, (int)cols, eps, g.warps)
    if (g.vpt == 1) LAUNCH(1, 256);
    else if (g.vpt == 2) LAUNCH(2, 256);
    else if (g.vpt == 4 && g.threads() <= 512) LAUNCH(4, 512);
    else if (g.vpt == 4) LAUNCH(4, 1024);
    else LAUNCH(8, 1024);
#undef LAUNCH
    return check_launch(fn);
  }
  const RowGeom g = row_geom(cols, false);
  const unsigned grid = (unsigned)std::min<int64_t>(rows, 0x7fffffff);
#define LAUNCH(VPT)                                                                             \
  add_rms_fwd_kernel<T, VPT, QUANT><<<grid, g.block, 0, s>>>(                          \
      static_cast<const T*>(x), x_stride, res, res_stride, w, static_cast<T*>(y), q, scale,     \
      block_shift, r, rstd, rows, (int)cols, eps)
  switch (g.vpt) {
    case 1: LAUNCH(1); break;
    case 2: LAUNCH(2); break;
    case 4: LAUNCH(4); break;
    case 8: LAUNCH(8); break;
    case 16: LAUNCH(16); break;
    default: LAUNCH(32); break;
  }
#undef LAUNCH
  return check_launch(fn);
}

template <typename T>
static oxc_status add_rms_bwd_launch(const float* r, const float* w, const float* rstd,
                                     const void* dy, int64_t dy_stride, const float* dr,
                                     int64_t dr_stride, float* dres, void* dx, float* dw,
                                     int64_t rows, int64_t cols, int32_t mode, float* parts,
                                     cudaStream_t s) {
  const int64_t ctas = add_rms_bwd_ctas(rows, cols);
  if (bwd_geom(cols).held() && row_shift<T>(dy, dy_stride, dr, dr ? dr_stride : cols, cols, rows) &&
      aligned16(r) && aligned16(w) && aligned16(dres) &&
      (sizeof(T) == 4 || aligned_to(dx, 4 * sizeof(T)))) {
    const GroupGeom g = bwd_geom(cols);
    const int period = cols % 4 == 0 ? 1 : cols % 2 == 0 ? 2 : 4;
    const bool edge = cols % 4 != 0, exact = mode == OXC_GRAD_EXACT;
    const size_t smem = g.vpt >= 4
                            ? (size_t)g.vpt * g.threads() * sizeof(float4) * (g.vpt <= 4 ? 2 : 1)
                        : g.groups > 1 ? (size_t)cols * sizeof(float)
                                       : 0;
#define LAUNCH(VPT, MAXT, EDGE)                                                                 \
  do {                                                                                          \
    auto kernel = exact ? add_rms_bwd_rows_kernel<T, VPT, MAXT, OXC_GRAD_EXACT, EDGE>           \
                        : add_rms_bwd_rows_kernel<T, VPT, MAXT, OXC_GRAD_REF, EDGE>;            \
    if (smem > 40 * 1024) {                                                                     \
      const cudaError_t e = cudaFuncSetAttribute(                                               \
          (const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);         \
      if (e != cudaSuccess) return cuda_fail(e, "oxc_add_rms_norm_bwd");                        \
    }                                                                                           \
    kernel<<<(unsigned)ctas, g.threads(), smem, s>>>(                                           \
        r, w, rstd, static_cast<const T*>(dy), dy_stride, dr, dr_stride, dres,                  \
        static_cast<T*>(dx), parts, rows, (int)cols, period, g.warps);                          \
  } while (0)
    const int n = g.threads();
    if (edge) {
      if (g.vpt == 1) LAUNCH(1, 256, true);
      else if (g.vpt == 2 && n <= 256) LAUNCH(2, 256, true);
      else if (g.vpt == 2 && n <= 384) LAUNCH(2, 384, true);
      else if (g.vpt == 2) LAUNCH(2, 640, true);
      else if (g.vpt == 4 && n <= 512) LAUNCH(4, 512, true);
      else if (g.vpt == 4 && n <= 768) LAUNCH(4, 768, true);
      else if (g.vpt == 4) LAUNCH(4, 1024, true);
      else LAUNCH(8, 1024, true);
    } else {
      // 352 and 384 threads: two CTAs fit an SM, a third neither at 64 registers, so
      // they take 85 ([16384, 2944] f32 120 us instead of 132, bf16 127 instead of 140)
      if (g.vpt == 1) LAUNCH(1, 256, false);
      else if (g.vpt == 2 && n <= 384 && n > 1024 / 3) LAUNCH(2, 384, false);
      else if (g.vpt == 2 && n <= 512) LAUNCH(2, 512, false);
      else if (g.vpt == 2 && n <= 640) LAUNCH(2, 640, false);
      else if (g.vpt == 2) LAUNCH(2, 1024, false);
      else if (g.vpt == 4 && n <= 768) LAUNCH(4, 768, false);
      else if (g.vpt == 4) LAUNCH(4, 1024, false);
      else LAUNCH(8, 1024, false);
    }
#undef LAUNCH
  } else {
    const RowGeom g = row_geom(cols, false, 512);
    const int64_t chunk = (rows + ctas - 1) / ctas;
#define LAUNCH(VPT)                                                                             \
  do {                                                                                          \
    if (mode == OXC_GRAD_REF)                                                                   \
      add_rms_bwd_kernel<T, VPT, OXC_GRAD_REF><<<(unsigned)ctas, g.block, 0, s>>>(     \
          r, w, rstd, static_cast<const T*>(dy), dy_stride, dr, dr_stride, dres,                \
          static_cast<T*>(dx), parts, rows, (int)cols, chunk);                                  \
    else                                                                                        \
      add_rms_bwd_kernel<T, VPT, OXC_GRAD_EXACT><<<(unsigned)ctas, g.block, 0, s>>>(   \
          r, w, rstd, static_cast<const T*>(dy), dy_stride, dr, dr_stride, dres,                \
          static_cast<T*>(dx), parts, rows, (int)cols, chunk);                                  \
  } while (0)
    switch (g.vpt) {
      case 1: LAUNCH(1); break;
      case 2: LAUNCH(2); break;
      case 4: LAUNCH(4); break;
      case 8: LAUNCH(8); break;
      case 16: LAUNCH(16); break;
      default: LAUNCH(32); break;
    }
#undef LAUNCH
  }
  oxc_status st = check_launch("oxc_add_rms_norm_bwd");
  if (st) return st;
  launch_colsum_partials(parts, (int)ctas, cols, dw, s);
  return check_launch("oxc_add_rms_norm_bwd (dw)");
}

}  // namespace oxc

using namespace oxc;

extern "C" {

oxc_status oxc_add_rms_norm_fwd(const void* x, int64_t x_stride, const float* residual,
                                int64_t residual_stride, const float* w, void* y, float* r,
                                float* rstd, int64_t rows, int64_t cols, int32_t dtype, float eps,
                                void* stream) {
  oxc_status st = add_rms_check("add_rms_norm", dtype, rows, cols);
  if (st) return st;
  if (rows == 0) return OXC_OK;
  if (!x || !residual || !w || !y || !r || !rstd)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: add_rms_norm: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == OXC_BF16)
    return add_rms_fwd_launch<bf16, false>("oxc_add_rms_norm_fwd", x, x_stride, residual,
                                           residual_stride, w, y, nullptr, nullptr, 1, r, rstd,
                                           rows, cols, eps, s);
  return add_rms_fwd_launch<float, false>("oxc_add_rms_norm_fwd", x, x_stride, residual,
                                          residual_stride, w, y, nullptr, nullptr, 1, r, rstd,
                                          rows, cols, eps, s);
}

oxc_status oxc_add_rms_norm_quant(const void* x, int64_t x_stride, const float* residual,
                                  int64_t residual_stride, const float* w, uint8_t* q,
                                  float* scale, float* r, int64_t rows, int64_t cols,
                                  int64_t block, int32_t dtype, float eps, void* stream) {
  oxc_status st = add_rms_check("add_rms_norm_quant", dtype, rows, cols);
  if (st) return st;
  if (block != 0 && block != 128)
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: add_rms_norm_quant: block must be 128 or 0 (the whole row), "
                "got %lld",
                (long long)block);
  if (rows == 0) return OXC_OK;
  if (!x || !residual || !w || !q || !scale || !r)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: add_rms_norm_quant: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int block_shift = block ? 7 : 31;  // a column's block
  if (dtype == OXC_BF16)
    return add_rms_fwd_launch<bf16, true>("oxc_add_rms_norm_quant", x, x_stride, residual,
                                          residual_stride, w, nullptr, q, scale, block_shift, r,
                                          nullptr, rows, cols, eps, s);
  return add_rms_fwd_launch<float, true>("oxc_add_rms_norm_quant", x, x_stride, residual,
                                         residual_stride, w, nullptr, q, scale, block_shift, r,
                                         nullptr, rows, cols, eps, s);
}

size_t oxc_add_rms_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)add_rms_bwd_ctas(rows, cols) * (size_t)cols * sizeof(float);
}

oxc_status oxc_add_rms_norm_bwd(const float* r, const float* w, const float* rstd, const void* dy,
                                int64_t dy_stride, const float* dr, int64_t dr_stride,
                                float* dresidual, void* dx, float* dw, int64_t rows, int64_t cols,
                                int32_t dtype, int32_t grad_mode, void* workspace,
                                size_t workspace_bytes, void* stream) {
  oxc_status st = add_rms_check("add_rms_norm backward", dtype, rows, cols);
  if (st) return st;
  if (grad_mode != OXC_GRAD_REF && grad_mode != OXC_GRAD_EXACT)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: unknown grad mode %d", grad_mode);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cols == 0) return OXC_OK;
  if (rows == 0) {
    if (!dw) return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: add_rms_norm backward: null pointer");
    cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)cols * sizeof(float), s);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_add_rms_norm_bwd");
  }
  const size_t need = oxc_add_rms_norm_bwd_workspace_size(rows, cols);
  if (!workspace || workspace_bytes < need)
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: add_rms_norm backward needs a %zu-byte workspace, got %zu", need,
                workspace_bytes);
  if (!r || !w || !rstd || !dy || !dresidual || !dw || (dtype == OXC_BF16 && !dx))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: add_rms_norm backward: null pointer");
  float* parts = static_cast<float*>(workspace);
  if (dtype == OXC_BF16)
    return add_rms_bwd_launch<bf16>(r, w, rstd, dy, dy_stride, dr, dr_stride, dresidual, dx, dw,
                                    rows, cols, grad_mode, parts, s);
  return add_rms_bwd_launch<float>(r, w, rstd, dy, dy_stride, dr, dr_stride, dresidual, dx, dw,
                                   rows, cols, grad_mode, parts, s);
}

}  // extern "C"
