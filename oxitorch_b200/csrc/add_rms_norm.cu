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
// largest value.  y is not rounded to x's type in between.
//
// All are bound by HBM traffic: 8 + 2 sizeof(T) bytes an element forward, 9 +
// sizeof(T) with the 8-bit output.
#include <cuda_fp8.h>

#include <algorithm>

#include "rowvec.cuh"
#include "typed.cuh"

namespace oxc {

constexpr int kQuantMaxBlocks = 32768 / 128;

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// One CTA per row, the row in registers: thread t holds the VPT vectors
// [(i * blockDim + t) * VW, +VW).
template <typename T, int VW, int VPT, int MAXT, bool QUANT>
__global__ void __launch_bounds__(MAXT) add_rms_fwd_kernel(
    const T* __restrict__ x, int64_t x_stride, const float* __restrict__ res, int64_t res_stride,
    const float* __restrict__ w, T* __restrict__ y, uint8_t* __restrict__ q,
    float* __restrict__ scale, int block_cols, float* __restrict__ r, float* __restrict__ rstd,
    int64_t rows, int cols, float eps) {
  __shared__ float scratch[33];
  __shared__ uint32_t amax[QUANT ? kQuantMaxBlocks : 1];
  const int blocks = QUANT ? (cols + block_cols - 1) / block_cols : 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float v[VPT][VW];
    float ss = 0.0f;
    if constexpr (QUANT) {
      for (int b = threadIdx.x; b < blocks; b += blockDim.x) amax[b] = 0u;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = (i * blockDim.x + threadIdx.x) * VW;
      if (e < cols) {
        float a[VW];
        load_as_f32<VW>(a, x + row * x_stride + e);
        load_as_f32<VW>(v[i], res + row * res_stride + e);
#pragma unroll
        for (int k = 0; k < VW; ++k) v[i][k] += a[k];
        store_from_f32<VW>(r + row * (int64_t)cols + e, v[i]);
      } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) v[i][k] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < VW; ++k) ss = fmaf(v[i][k], v[i][k], ss);
    ss = block_sum(ss, scratch);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)cols) + eps));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = (i * blockDim.x + threadIdx.x) * VW;
      if (e < cols) {
        float wv[VW];
        load_vec<VW>(wv, w + e, false);
#pragma unroll
        for (int k = 0; k < VW; ++k) v[i][k] = v[i][k] * inv * wv[k];
        if constexpr (!QUANT) store_from_f32<VW>(y + row * (int64_t)cols + e, v[i]);
      }
    }
    if constexpr (QUANT) {
      // |y|'s bits order like its values, NaN above infinity: a NaN in a block
      // makes its scale NaN
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = (i * blockDim.x + threadIdx.x) * VW;
        if (e < cols) {
          uint32_t m = 0u;
#pragma unroll
          for (int k = 0; k < VW; ++k) m = max(m, __float_as_uint(fabsf(v[i][k])));
          atomicMax(&amax[e / block_cols], m);
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = (i * blockDim.x + threadIdx.x) * VW;
        if (e < cols) {
          const int b = e / block_cols;
          const float a = __uint_as_float(amax[b]);
          const float s = a != a ? a : fmaxf(__fdiv_rn(a, 448.0f), 1.17549435e-38f);
          uint8_t o[VW];
#pragma unroll
          for (int k = 0; k < VW; ++k) o[k] = to_e4m3(__fdiv_rn(v[i][k], s));
          uint8_t* qp = q + row * (int64_t)cols + e;
          if constexpr (VW == 4)
            *reinterpret_cast<uchar4*>(qp) = make_uchar4(o[0], o[1], o[2], o[3]);
          else
            qp[0] = o[0];
          if (e == b * block_cols) scale[row * blocks + b] = s;
        }
      }
      __syncthreads();  // amax is read; the next row clears it
    } else if (threadIdx.x == 0) {
      rstd[row] = inv;
    }
  }
}

// Persistent VJP: CTA b handles rows [b * chunk, min((b + 1) * chunk, rows))
// and writes its dw partial to parts[b][cols].
template <typename T, int VW, int VPT, int MAXT, int MODE>
__global__ void __launch_bounds__(MAXT) add_rms_bwd_kernel(
    const float* __restrict__ r, const float* __restrict__ w, const float* __restrict__ rstd,
    const T* __restrict__ dy, int64_t dy_stride, const float* __restrict__ dr, int64_t dr_stride,
    float* __restrict__ dres, T* __restrict__ dx, float* __restrict__ parts, int64_t rows, int cols,
    int64_t chunk) {
  pdl_launch_dependents();  // the dweight finisher waits for this grid
  __shared__ float scratch[33];
  const int64_t r0 = (int64_t)blockIdx.x * chunk;
  const int64_t r1 = min(rows, r0 + chunk);
  float wv[VPT][VW], acc[VPT][VW];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = (i * blockDim.x + threadIdx.x) * VW;
#pragma unroll
    for (int k = 0; k < VW; ++k) { acc[i][k] = 0.0f; wv[i][k] = 0.0f; }
    if (e < cols) load_vec<VW>(wv[i], w + e, false);
  }
  const float inv_n = __fdiv_rn(1.0f, (float)cols);
  for (int64_t row = r0; row < r1; ++row) {
    float u[VPT][VW], g[VPT][VW], d[VPT][VW];
    const float inv = __ldg(rstd + row);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = (i * blockDim.x + threadIdx.x) * VW;
#pragma unroll
      for (int k = 0; k < VW; ++k) { u[i][k] = 0.0f; g[i][k] = 0.0f; d[i][k] = 0.0f; }
      if (e < cols) {
        load_vec<VW>(u[i], r + row * (int64_t)cols + e, true);
        load_as_f32<VW>(g[i], dy + row * dy_stride + e);
        if (dr) load_as_f32<VW>(d[i], dr + row * dr_stride + e);
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        u[i][k] *= inv;
        acc[i][k] = fmaf(g[i][k], u[i][k], acc[i][k]);
        g[i][k] *= wv[i][k];
        s = fmaf(g[i][k], u[i][k], s);
      }
    float mean = 0.0f;
    if constexpr (MODE == OXC_GRAD_EXACT) mean = block_sum(s, scratch) * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = (i * blockDim.x + threadIdx.x) * VW;
      if (e < cols) {
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          if constexpr (MODE == OXC_GRAD_EXACT) g[i][k] = fmaf(-u[i][k], mean, g[i][k]);
          d[i][k] = fmaf(inv, g[i][k], d[i][k]);
        }
        store_from_f32<VW>(dres + row * (int64_t)cols + e, d[i]);
        if constexpr (sizeof(T) == 2) store_from_f32<VW>(dx + row * (int64_t)cols + e, d[i]);
      }
    }
  }
  float* pr = parts + (int64_t)blockIdx.x * cols;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = (i * blockDim.x + threadIdx.x) * VW;
    if (e < cols) {
#pragma unroll
      for (int k = 0; k < VW; ++k) pr[e + k] = acc[i][k];
    }
  }
}

static int64_t add_rms_bwd_ctas(int64_t rows) {
  int64_t g = 2 * (int64_t)sm_count();
  const int64_t by_rows = (rows + 7) / 8;
  if (g > by_rows) g = by_rows;
  return g < 1 ? 1 : g;
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

// Vectors of 4 when every row of x and of the f32 tensors starts on one.
template <typename T>
static bool rows_vec4(const void* x, int64_t x_stride, const void* f, int64_t f_stride,
                      int64_t cols) {
  return cols % 4 == 0 && x_stride % 4 == 0 && f_stride % 4 == 0 &&
         aligned_to(x, 4 * sizeof(T)) && aligned16(f);
}

template <typename T, bool QUANT>
static oxc_status add_rms_fwd_launch(const char* fn, const void* x, int64_t x_stride,
                                     const float* res, int64_t res_stride, const float* w, void* y,
                                     uint8_t* q, float* scale, int block_cols, float* r,
                                     float* rstd, int64_t rows, int64_t cols, float eps,
                                     cudaStream_t s) {
  const bool v4 = rows_vec4<T>(x, x_stride, res, res_stride, cols) && aligned16(w) &&
                  aligned16(r) && (QUANT ? aligned_to(q, 4) : aligned_to(y, 4 * sizeof(T)));
  RowGeom g = row_geom(cols, v4);
  if (v4) {
    const RowGeom d = row_geom_deep(cols);
    if (d.ok && d.block <= 512) g = d;
  }
  const unsigned grid = (unsigned)std::min<int64_t>(rows, 0x7fffffff);
#define LAUNCH(VW, VPT, MAXT)                                                                   \
  add_rms_fwd_kernel<T, VW, VPT, MAXT, QUANT><<<grid, g.block, 0, s>>>(                         \
      static_cast<const T*>(x), x_stride, res, res_stride, w, static_cast<T*>(y), q, scale,     \
      block_cols, r, rstd, rows, (int)cols, eps)
  OXC_DISPATCH_ROW(g, LAUNCH);
#undef LAUNCH
  return check_launch(fn);
}

template <typename T>
static oxc_status add_rms_bwd_launch(const float* r, const float* w, const float* rstd,
                                     const void* dy, int64_t dy_stride, const float* dr,
                                     int64_t dr_stride, float* dres, void* dx, float* dw,
                                     int64_t rows, int64_t cols, int32_t mode, float* parts,
                                     cudaStream_t s) {
  const bool v4 = rows_vec4<T>(dy, dy_stride, dr, dr ? dr_stride : 0, cols) && aligned16(r) &&
                  aligned16(w) && aligned16(dres) && aligned16(parts) &&
                  (sizeof(T) == 4 || aligned_to(dx, 4 * sizeof(T)));
  const RowGeom g = row_geom(cols, v4, 512);
  const int64_t ctas = add_rms_bwd_ctas(rows);
  const int64_t chunk = (rows + ctas - 1) / ctas;
#define LAUNCH(VW, VPT, MAXT)                                                                   \
  do {                                                                                          \
    if (mode == OXC_GRAD_REF)                                                                   \
      add_rms_bwd_kernel<T, VW, VPT, MAXT, OXC_GRAD_REF><<<(unsigned)ctas, g.block, 0, s>>>(    \
          r, w, rstd, static_cast<const T*>(dy), dy_stride, dr, dr_stride, dres,                \
          static_cast<T*>(dx), parts, rows, (int)cols, chunk);                                  \
    else                                                                                        \
      add_rms_bwd_kernel<T, VW, VPT, MAXT, OXC_GRAD_EXACT><<<(unsigned)ctas, g.block, 0, s>>>(  \
          r, w, rstd, static_cast<const T*>(dy), dy_stride, dr, dr_stride, dres,                \
          static_cast<T*>(dx), parts, rows, (int)cols, chunk);                                  \
  } while (0)
  OXC_DISPATCH_ROW(g, LAUNCH);
#undef LAUNCH
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
  const int block_cols = block ? (int)block : (int)cols;
  if (dtype == OXC_BF16)
    return add_rms_fwd_launch<bf16, true>("oxc_add_rms_norm_quant", x, x_stride, residual,
                                          residual_stride, w, nullptr, q, scale, block_cols, r,
                                          nullptr, rows, cols, eps, s);
  return add_rms_fwd_launch<float, true>("oxc_add_rms_norm_quant", x, x_stride, residual,
                                         residual_stride, w, nullptr, q, scale, block_cols, r,
                                         nullptr, rows, cols, eps, s);
}

size_t oxc_add_rms_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)add_rms_bwd_ctas(rows) * (size_t)cols * sizeof(float);
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
