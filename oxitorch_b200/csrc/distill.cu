// distill.cu -- distillation from a teacher's top logits: the loss and the
// student's gradient in one call.
//
// Row n has the student's logits s (vocab of them) and at most K of the
// teacher's, t_k at the ids i_k; with temperature tau
//   p = softmax(t / tau) over the row's entries,  q = softmax(s / tau)
//   loss = tau^2 / total_rows * sum_n sum_k p_k (log p_k - log q_{i_k})
//   d loss / d s_j = tau / total_rows * (q_j - sum_{k: i_k = j} p_k)
// An entry is absent when its id is negative or its logit is -inf; a row with
// no entry has loss 0 and gradient 0, whatever its logits hold.  An id listed
// twice counts twice.
#include <math.h>

#include <algorithm>

#include "typed.cuh"

namespace oxc {

constexpr int kDistillMaxTop = 4096;

// Records the first bad id: flag[0] = 2 (dim 1), flag[1..2] = id, flag[3] = vocab.
__device__ __forceinline__ void record_bad_id(int32_t* flag, int64_t id, int64_t vocab) {
  if (flag && atomicCAS(flag, 0, 2) == 0) {
    flag[1] = (int32_t)(uint32_t)((uint64_t)id & 0xffffffffu);
    flag[2] = (int32_t)(uint32_t)((uint64_t)id >> 32);
    flag[3] = (int32_t)vocab;
  }
}

// One CTA per row, three passes over it.
template <typename T>
__global__ void __launch_bounds__(512) distill_kernel(
    const T* __restrict__ logits, int64_t stride, const float* __restrict__ tl,
    const int64_t* __restrict__ ti, int top, float inv_tau, float grad_scale,
    const float* __restrict__ grad_loss, float* __restrict__ row_loss, T* __restrict__ dlogits,
    int64_t rows, int vocab, int32_t* err) {
  extern __shared__ float prob[];  // [top]
  __shared__ float scratch[33];
  const float gs = grad_loss ? grad_scale * __ldg(grad_loss) : grad_scale;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = logits + row * stride;
    T* dr = dlogits ? dlogits + row * (int64_t)vocab : nullptr;
    const float* tr = tl + row * top;
    const int64_t* ir = ti + row * top;
    // the teacher's probabilities
    float tm = -INFINITY;
    int bad = 0;
    for (int k = threadIdx.x; k < top; k += blockDim.x) {
      const int64_t id = ir[k];
      if (id >= vocab) { record_bad_id(err, id, vocab); bad = 1; }
      const float v = id >= 0 ? tr[k] : -INFINITY;
      prob[k] = v;
      tm = fmaxf(tm, v);
      if (v != v) bad = 1;
    }
    bad = __syncthreads_or(bad);
    tm = block_max(tm, scratch);
    if (tm == -INFINITY && !bad) {
      for (int c = threadIdx.x; dr && c < vocab; c += blockDim.x) dr[c] = from_f32<T>(0.0f);
      if (threadIdx.x == 0) row_loss[row] = 0.0f;
      continue;
    }
    float ts = 0.0f;
    for (int k = threadIdx.x; k < top; k += blockDim.x) ts += expf((prob[k] - tm) * inv_tau);
    ts = block_sum(ts, scratch);
    // the student's row
    float m = -INFINITY;
    for (int c = threadIdx.x; c < vocab; c += blockDim.x) m = fmaxf(m, to_f32(xr[c]));
    m = block_max(m, scratch);
    float sum = 0.0f;
    for (int c = threadIdx.x; c < vocab; c += blockDim.x) sum += expf((to_f32(xr[c]) - m) * inv_tau);
    sum = block_sum(sum, scratch);
    const float log_ts = logf(ts), log_sum = logf(sum);
    float loss = 0.0f;
    for (int k = threadIdx.x; k < top; k += blockDim.x) {
      const int64_t id = ir[k];
      const float z = (prob[k] - tm) * inv_tau;
      const float p = expf(z) / ts;
      prob[k] = p;
      if (id >= 0 && id < vocab && p > 0.0f)
        loss += p * ((z - log_ts) - ((to_f32(xr[id]) - m) * inv_tau - log_sum));
    }
    loss = block_sum(loss, scratch);
    if (threadIdx.x == 0) row_loss[row] = bad ? NAN : loss;
    if (dr) {
      const float inv_sum = 1.0f / sum;
      for (int c = threadIdx.x; c < vocab; c += blockDim.x)
        dr[c] = from_f32<T>(bad ? NAN : gs * (expf((to_f32(xr[c]) - m) * inv_tau) * inv_sum));
      __syncthreads();
      if (!bad) {
        for (int k = threadIdx.x; k < top; k += blockDim.x) {
          const int64_t id = ir[k];
          if (id < 0) continue;
          float p = 0.0f;  // all entries of this id, in order
          for (int j = 0; j < top; ++j)
            if (ir[j] == id) p += prob[j];
          dr[id] = from_f32<T>(gs * (expf((to_f32(xr[id]) - m) * inv_tau) * inv_sum - p));
        }
      }
    }
    __syncthreads();  // prob is read; the next row overwrites it
  }
}

// loss = scale * sum of row_loss, folded in f64 by one CTA in a fixed order.
__global__ void __launch_bounds__(1024) distill_loss_kernel(const float* __restrict__ row_loss,
                                                            int64_t rows, double scale,
                                                            float* __restrict__ loss) {
  __shared__ double scratch[33];
  double acc = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) acc += (double)row_loss[r];
  const double sum = block_sum(acc, scratch);
  if (threadIdx.x == 0) loss[0] = (float)(sum * scale);
}

// x *= g[0]; nothing to do, and nothing read, when g[0] is 1.
template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* __restrict__ x, int64_t n,
                                                       const float* __restrict__ g) {
  const float s = __ldg(g);
  if (s == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    x[i] = from_f32<T>(to_f32(x[i]) * s);
}

}  // namespace oxc

using namespace oxc;

extern "C" {

oxc_status oxc_distill_loss(const void* logits, int64_t logits_stride, const float* teacher_logits,
                            const int64_t* teacher_ids, int64_t top, float temperature,
                            const float* grad_loss, float* loss, float* row_loss, void* dlogits,
                            int64_t rows, int64_t vocab, int64_t total_rows, int32_t dtype,
                            int32_t* err_flag, void* stream) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: unknown dtype %d", dtype);
  if (rows < 0 || vocab < 0 || top < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: negative shape");
  if (total_rows < rows || total_rows <= 0)
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: distill_loss: total_rows %lld must cover the %lld local rows",
                (long long)total_rows, (long long)rows);
  if (!(temperature > 0.0f) || isinf(temperature))
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: distill_loss: temperature must be positive, got %g",
                (double)temperature);
  if (vocab > 0x7fffffff)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: distill_loss: rows wider than 2^31");
  if (top > kDistillMaxTop)
    return fail(OXC_ERR_NOT_IMPLEMENTED,
                "not implemented: distill_loss: more than %d teacher logits per row, got %lld",
                kDistillMaxTop, (long long)top);
  if (!loss) return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: null pointer");
  if (rows > 0 && vocab == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss over zero classes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows > 0) {
    if (!logits || !row_loss || (top > 0 && (!teacher_logits || !teacher_ids)))
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: null pointer");
    const unsigned grid = (unsigned)std::min<int64_t>(rows, (int64_t)sm_count() * 64);
    const float inv_tau = (float)(1.0 / (double)temperature);
    const float gs = (float)((double)temperature / (double)total_rows);
    const size_t smem = (size_t)top * sizeof(float);
    if (dtype == OXC_BF16)
      distill_kernel<bf16><<<grid, 512, smem, s>>>(
          static_cast<const bf16*>(logits), logits_stride, teacher_logits, teacher_ids, (int)top,
          inv_tau, gs, grad_loss, row_loss, static_cast<bf16*>(dlogits), rows, (int)vocab, err_flag);
    else
      distill_kernel<float><<<grid, 512, smem, s>>>(
          static_cast<const float*>(logits), logits_stride, teacher_logits, teacher_ids, (int)top,
          inv_tau, gs, grad_loss, row_loss, static_cast<float*>(dlogits), rows, (int)vocab,
          err_flag);
    oxc_status st = check_launch("oxc_distill_loss");
    if (st) return st;
  }
  const double scale = (double)temperature * (double)temperature / (double)total_rows;
  distill_loss_kernel<<<1, 1024, 0, s>>>(row_loss, rows, scale, loss);
  return check_launch("oxc_distill_loss (sum)");
}

oxc_status oxc_scale_by(void* x, int64_t n, int32_t dtype, const float* g, void* stream) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: scale_by: unknown dtype %d", dtype);
  if (n < 0) return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: scale_by: negative size");
  if (n == 0) return OXC_OK;
  if (!x || !g) return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: scale_by: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, (int64_t)sm_count() * 8);
  if (dtype == OXC_BF16)
    scale_by_kernel<bf16><<<grid, 256, 0, s>>>(static_cast<bf16*>(x), n, g);
  else
    scale_by_kernel<float><<<grid, 256, 0, s>>>(static_cast<float*>(x), n, g);
  return check_launch("oxc_scale_by");
}

}  // extern "C"
