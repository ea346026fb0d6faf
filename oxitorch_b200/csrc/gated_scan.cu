// gated_scan.cu -- the gated linear recurrence over a sequence, its VJP, and
// its single-token step.
//
//   a_t = sigmoid(gate_t),  h_t = a_t * h_{t-1} + (1 - a_t) * x_t
//
// per batch row and channel, the state h in f32.  Where starts[t] is set a new
// sequence begins at t: the state before it counts as zero (selected, not
// multiplied away, so nothing of the sequence before -- a NaN or an infinity
// included -- reaches it).
//
// VJP: with mu_t the gradient that flows from h_t to h_{t-1},
//   lam_t = dh_t + mu_{t+1}        (lam_{T-1} also has dlast)
//   mu_t = a_t * lam_t             (0 where starts[t])
//   dx_t = lam_t * (1 - a_t)
//   dgate_t = lam_t * (h_{t-1} - x_t) * a_t * (1 - a_t)
//   dh0 = mu_0
// h_{t-1} is recomputed in f32 from the states that the forward saves before
// each chunk of kScanChunk tokens, so the VJP does not read h back: 5 elements
// of traffic per token and channel instead of 6, and no rounding of h to bf16
// in the gradient.
#include <algorithm>

#include "typed.cuh"

namespace oxc {

constexpr int kScanChunk = 64;

// A [batch, length, dim] operand: the last dim dense, strides in elements.
template <typename T>
struct SeqView {
  const T* p;
  int64_t sb, st;
  __device__ __forceinline__ const T* at(int64_t b, int64_t t, int64_t d) const {
    return p + b * sb + t * st + d;
  }
};

// a = sigmoid(g) and b = 1 - a, both to f32 accuracy (b is not formed by
// subtraction, which would lose it for large gates).
__device__ __forceinline__ void gate_pair(float g, float& a, float& b) {
  const float e = expf(-fabsf(g));
  const float big = __frcp_rn(1.0f + e);
  const float small = e * big;
  a = g >= 0.0f ? big : small;
  b = g >= 0.0f ? small : big;
  if (g != g) a = b = g;
}

template <typename T>
__global__ void __launch_bounds__(128) scan_fwd_kernel(SeqView<T> x, SeqView<T> gate,
                                                       const uint8_t* __restrict__ starts,
                                                       const float* __restrict__ h0,
                                                       T* __restrict__ h, float* __restrict__ last,
                                                       float* __restrict__ carry, int64_t length,
                                                       int64_t dim) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t bi = blockIdx.y;
  if (d >= dim) return;
  const int64_t chunks = (length + kScanChunk - 1) / kScanChunk;
  float s = h0 ? h0[bi * dim + d] : 0.0f;
  for (int64_t t = 0; t < length; ++t) {
    if (carry && t % kScanChunk == 0) carry[(bi * chunks + t / kScanChunk) * dim + d] = s;
    float a, b;
    gate_pair(to_f32(*gate.at(bi, t, d)), a, b);
    const float v = b * to_f32(*x.at(bi, t, d));
    s = starts && starts[bi * length + t] ? v : fmaf(a, s, v);
    h[(bi * length + t) * dim + d] = from_f32<T>(s);
  }
  if (last) last[bi * dim + d] = s;
}

template <typename T>
__global__ void __launch_bounds__(128) scan_bwd_kernel(
    SeqView<T> x, SeqView<T> gate, const uint8_t* __restrict__ starts,
    const float* __restrict__ carry, SeqView<T> dh, const float* __restrict__ dlast,
    T* __restrict__ dx, T* __restrict__ dgate, float* __restrict__ dh0, int64_t length,
    int64_t dim) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t bi = blockIdx.y;
  if (d >= dim) return;
  const int64_t chunks = (length + kScanChunk - 1) / kScanChunk;
  float mu = dlast ? dlast[bi * dim + d] : 0.0f;
  for (int64_t c = chunks - 1; c >= 0; --c) {
    const int64_t t0 = c * kScanChunk, t1 = min(length, t0 + kScanChunk);
    float before[kScanChunk];  // the state before each token of the chunk
    float s = carry[(bi * chunks + c) * dim + d];
    for (int64_t t = t0; t < t1; ++t) {
      float a, b;
      gate_pair(to_f32(*gate.at(bi, t, d)), a, b);
      if (starts && starts[bi * length + t]) s = 0.0f;
      before[t - t0] = s;
      s = fmaf(a, s, b * to_f32(*x.at(bi, t, d)));
    }
    for (int64_t t = t1 - 1; t >= t0; --t) {
      float a, b;
      gate_pair(to_f32(*gate.at(bi, t, d)), a, b);
      const float lam = (dh.p ? to_f32(*dh.at(bi, t, d)) : 0.0f) + mu;
      const float db = lam * b;
      const int64_t o = (bi * length + t) * dim + d;
      dx[o] = from_f32<T>(db);
      dgate[o] = from_f32<T>(db * a * (before[t - t0] - to_f32(*x.at(bi, t, d))));
      mu = starts && starts[bi * length + t] ? 0.0f : a * lam;
    }
  }
  if (dh0) dh0[bi * dim + d] = mu;
}

// One token: state_out (which may be state itself) and h = state_out rounded.
template <typename T>
__global__ void __launch_bounds__(128) scan_step_kernel(const T* __restrict__ x, int64_t x_stride,
                                                        const T* __restrict__ gate,
                                                        int64_t gate_stride, const float* state,
                                                        float* state_out, T* __restrict__ h,
                                                        int64_t dim) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t bi = blockIdx.y;
  if (d >= dim) return;
  float a, b;
  gate_pair(to_f32(gate[bi * gate_stride + d]), a, b);
  const float s = fmaf(a, state[bi * dim + d], b * to_f32(x[bi * x_stride + d]));
  state_out[bi * dim + d] = s;
  h[bi * dim + d] = from_f32<T>(s);
}

static oxc_status scan_check(const char* fn, int32_t dtype, int64_t batch, int64_t length,
                             int64_t dim) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: %s: unknown dtype %d", fn, dtype);
  if (batch < 0 || length < 0 || dim < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: %s: negative shape [%lld, %lld, %lld]", fn, (long long)batch,
                (long long)length, (long long)dim);
  if (batch > 65535)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: batch of %lld > 65535", fn,
                (long long)batch);
  return OXC_OK;
}

static int64_t scan_chunks(int64_t length) { return (length + kScanChunk - 1) / kScanChunk; }

}  // namespace oxc

using namespace oxc;

extern "C" {

int64_t oxc_gated_scan_carry_size(int64_t batch, int64_t length, int64_t dim) {
  if (batch <= 0 || length <= 0 || dim <= 0) return 0;
  return batch * scan_chunks(length) * dim;
}

size_t oxc_gated_scan_workspace_size(int64_t batch, int64_t length, int64_t dim) {
  (void)batch; (void)length; (void)dim;
  return 0;
}

oxc_status oxc_gated_scan_fwd(const void* x, int64_t x_sb, int64_t x_st, const void* gate,
                              int64_t g_sb, int64_t g_st, const uint8_t* starts, const float* h0,
                              void* h, float* last, float* carry, int64_t batch, int64_t length,
                              int64_t dim, int32_t dtype, void* workspace, size_t workspace_bytes,
                              void* stream) {
  oxc_status st = scan_check("gated_scan", dtype, batch, length, dim);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (length == 0) {  // the state passes through
    if (!last) return OXC_OK;
    const size_t n = (size_t)batch * (size_t)dim * sizeof(float);
    cudaError_t e = h0 ? cudaMemcpyAsync(last, h0, n, cudaMemcpyDeviceToDevice, s)
                       : cudaMemsetAsync(last, 0, n, s);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_gated_scan_fwd");
  }
  if (!x || !gate || !h)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: gated_scan: null pointer");
  const dim3 grid((unsigned)((dim + 127) / 128), (unsigned)batch);
  if (dtype == OXC_BF16)
    scan_fwd_kernel<bf16><<<grid, 128, 0, s>>>({static_cast<const bf16*>(x), x_sb, x_st},
                                               {static_cast<const bf16*>(gate), g_sb, g_st},
                                               starts, h0, static_cast<bf16*>(h), last, carry,
                                               length, dim);
  else
    scan_fwd_kernel<float><<<grid, 128, 0, s>>>({static_cast<const float*>(x), x_sb, x_st},
                                                {static_cast<const float*>(gate), g_sb, g_st},
                                                starts, h0, static_cast<float*>(h), last, carry,
                                                length, dim);
  return check_launch("oxc_gated_scan_fwd");
}

oxc_status oxc_gated_scan_bwd(const void* x, int64_t x_sb, int64_t x_st, const void* gate,
                              int64_t g_sb, int64_t g_st, const uint8_t* starts,
                              const float* carry, const void* dh, int64_t dh_sb, int64_t dh_st,
                              const float* dlast, void* dx, void* dgate, float* dh0, int64_t batch,
                              int64_t length, int64_t dim, int32_t dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  oxc_status st = scan_check("gated_scan backward", dtype, batch, length, dim);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (length == 0) {
    if (!dh0) return OXC_OK;
    const size_t n = (size_t)batch * (size_t)dim * sizeof(float);
    cudaError_t e = dlast ? cudaMemcpyAsync(dh0, dlast, n, cudaMemcpyDeviceToDevice, s)
                          : cudaMemsetAsync(dh0, 0, n, s);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_gated_scan_bwd");
  }
  if (!x || !gate || !carry || !dx || !dgate)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: gated_scan backward: null pointer");
  const dim3 grid((unsigned)((dim + 127) / 128), (unsigned)batch);
  if (dtype == OXC_BF16)
    scan_bwd_kernel<bf16><<<grid, 128, 0, s>>>(
        {static_cast<const bf16*>(x), x_sb, x_st}, {static_cast<const bf16*>(gate), g_sb, g_st},
        starts, carry, {static_cast<const bf16*>(dh), dh_sb, dh_st}, dlast,
        static_cast<bf16*>(dx), static_cast<bf16*>(dgate), dh0, length, dim);
  else
    scan_bwd_kernel<float><<<grid, 128, 0, s>>>(
        {static_cast<const float*>(x), x_sb, x_st}, {static_cast<const float*>(gate), g_sb, g_st},
        starts, carry, {static_cast<const float*>(dh), dh_sb, dh_st}, dlast,
        static_cast<float*>(dx), static_cast<float*>(dgate), dh0, length, dim);
  return check_launch("oxc_gated_scan_bwd");
}

oxc_status oxc_gated_step(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride,
                          const float* state, float* state_out, void* h, int64_t batch,
                          int64_t dim, int32_t dtype, void* stream) {
  oxc_status st = scan_check("gated_step", dtype, batch, 1, dim);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  if (!x || !gate || !state || !state_out || !h)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: gated_step: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((dim + 127) / 128), (unsigned)batch);
  if (dtype == OXC_BF16)
    scan_step_kernel<bf16><<<grid, 128, 0, s>>>(static_cast<const bf16*>(x), x_stride,
                                                static_cast<const bf16*>(gate), gate_stride, state,
                                                state_out, static_cast<bf16*>(h), dim);
  else
    scan_step_kernel<float><<<grid, 128, 0, s>>>(static_cast<const float*>(x), x_stride,
                                                 static_cast<const float*>(gate), gate_stride,
                                                 state, state_out, static_cast<float*>(h), dim);
  return check_launch("oxc_gated_step");
}

}  // extern "C"
