// rowparts.cuh -- rows of logits held in shared memory, a part in each CTA of a
// cluster: how a row is cut, and the (max, sum of exponentials) pairs that its parts
// are reduced to.  Used by the losses that write the logits' gradient in the pass
// that reads them.
#pragma once

#include "pipeline.cuh"
#include "typed.cuh"

namespace oxc {

// Records the first bad id: flag[0] = 2 (dim 1), flag[1..2] = id, flag[3] = vocab.
__device__ __forceinline__ void record_bad_id(int32_t* flag, int64_t id, int64_t vocab) {
  if (flag && atomicCAS(flag, 0, 2) == 0) {
    flag[1] = (int32_t)(uint32_t)((uint64_t)id & 0xffffffffu);
    flag[2] = (int32_t)(uint32_t)((uint64_t)id >> 32);
    flag[3] = (int32_t)vocab;
  }
}

// 2^t within 2 units of the last place; the functions of this file are each
// translation unit's own.
static __device__ __forceinline__ float ex2_approx(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
static __device__ __forceinline__ float rcp_approx(float t) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// exp(d / tau) for d = x - max <= 0, c = log2(e) / tau.  The subtraction comes
// first, so the large terms see only ex2's own error; results below 2^-126 are 0.
__device__ __forceinline__ float exp_scaled(float d, float c) { return ex2_approx(d * c); }

// Maximum over the warp, NaN ignored.
__device__ __forceinline__ float warp_max_fast(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// (max, sum of exponentials relative to it) of two sets; -inf with 0 is the empty
// one.  A sum that is not 0 beside a maximum of -inf is NaN and stays.
__device__ __forceinline__ float2 pair_merge(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x);
  const float sa = a.x == m ? a.y : a.y * exp_scaled(a.x - m, c);
  const float sb = b.x == m ? b.y : b.y * exp_scaled(b.x - m, c);
  return make_float2(m, sa + sb);
}
__device__ __forceinline__ float2 warp_merge(float2 v, float c) {
  const float m = warp_max_fast(v.x);
  return make_float2(m, warp_sum(m == -INFINITY ? v.y : v.y * exp_scaled(v.x - m, c)));
}

// A row's bytes are cut at 16-byte boundaries of memory: `body` whole vectors,
// CTA r of the cluster taking the r-th share of them, thread t the vectors t,
// t + THREADS, ... of it; the elements before the first boundary and after the
// last (fewer than a vector each) are single elements of the last CTA's warp 0.
template <typename T>
struct RowCut {
  static constexpr int kVec = 16 / (int)sizeof(T);
  const T* row;
  int head, body, v0, v1;
  __device__ __forceinline__ RowCut(const T* row, int vocab, int rank, int log_size) : row(row) {
    head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
    body = (vocab - head) / kVec;
    const int each = (body + (1 << log_size) - 1) >> log_size;
    v0 = min(body, rank * each);
    v1 = min(body, v0 + each);
  }
  __device__ __forceinline__ const T* part() const { return row + head + (int64_t)v0 * kVec; }
};

// The elements of a 16-byte vector, in pairs.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float2 (&v)[8 / (int)sizeof(T)]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
    if constexpr (sizeof(T) == 4)
      v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else
      v[i] = make_float2(bf16_lo(w[i]), bf16_hi(w[i]));
  }
}

// Folds V vectors of logits into a running (max, sum of exponentials): the maximum
// of all first (of bf16, two at a time), a rescale of the sum when it grows, then
// the terms.
template <typename T, int V>
__device__ __forceinline__ void pair_fold(float2& p, const uint4 (&q)[V], float c) {
  constexpr int kPairs = 8 / (int)sizeof(T);
  float m = p.x;
  if constexpr (sizeof(T) == 2) {
    __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&q[0].x);
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) h = __hmax2(h, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    }
    m = fmaxf(m, fmaxf(__low2float(h), __high2float(h)));
  } else {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      m = fmaxf(m, fmaxf(__uint_as_float(q[u].x), __uint_as_float(q[u].y)));
      m = fmaxf(m, fmaxf(__uint_as_float(q[u].z), __uint_as_float(q[u].w)));
    }
  }
  if (m > p.x) {
    p.y *= exp_scaled(p.x - m, c);
    p.x = m;
  }
  const float base = m == -INFINITY ? 0.0f : -m;
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < V; ++u) {
    float2 v[kPairs];
    unpack<T>(q[u], v);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 d = __fmul2_rn(__fadd2_rn(v[i], make_float2(base, base)), make_float2(c, c));
      s = __fadd2_rn(s, make_float2(ex2_approx(d.x), ex2_approx(d.y)));
    }
  }
  p.y += s.x + s.y;
}

// Sends v to `to` in CTA `rank` of the cluster, completing 8 bytes on its `bar`.
__device__ __forceinline__ void send_pair(const float2* to, uint64_t* bar, int rank, float2 v) {
  uint32_t dst, rbar;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(to)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rbar) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
               ::"r"(dst), "f"(v.x), "f"(v.y), "r"(rbar) : "memory");
}

// loss = scale * sum of row_loss, folded in f64 by one CTA in a fixed order.
static __global__ void __launch_bounds__(1024) sum_losses_kernel(const float* __restrict__ row_loss,
                                                            int64_t rows, double scale,
                                                            float* __restrict__ loss) {
  __shared__ double scratch[33];
  pdl_wait();  // row_loss is the previous kernel's output
  double acc = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) acc += (double)row_loss[r];
  const double sum = block_sum(acc, scratch);
  if (threadIdx.x == 0) loss[0] = (float)(sum * scale);
}

}  // namespace oxc
