// selective_scan.cu -- the single-token step of the selective scan and the C entries (the mathematics is in selective_scan.cuh).
#include "selective_scan.cuh"

namespace oxc {

// One token: LPC lanes a channel, four states a lane at a time.  Rates are bounded as the
// scan bounds them, so that an infinite one times a step of zero is zero here too.
template <typename T, int LPC>
__global__ void __launch_bounds__(128)
selective_step_kernel(const T* __restrict__ x, int64_t x_sb, const T* __restrict__ delta,
                      int64_t delta_sb, const float* __restrict__ A, const T* __restrict__ B,
                      int64_t B_sb, const T* __restrict__ C, int64_t C_sb,
                      const float* __restrict__ D, const T* __restrict__ z, int64_t z_sb,
                      const float* __restrict__ delta_bias, const float* state, float* out,
                      T* __restrict__ y, int64_t n, int64_t dim, int N, bool vec) {
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LPC;
  const int sl = threadIdx.x % LPC;
  const bool on = i < n;
  const int64_t b = on ? i / dim : 0, d = on ? i - b * dim : 0;
  const float xv = on ? to_f32(x[b * x_sb + d]) : 0.0f;
  const float dt = on ? softplus(to_f32(delta[b * delta_sb + d]) + (delta_bias ? delta_bias[d] : 0.0f)) : 0.0f;
  const float dtx = dt * xv;
  const T* Bb = B + b * B_sb;
  const T* Cb = C + b * C_sb;
  float sum = 0.0f;
  for (int s = sl * 4; on && s < N; s += LPC * 4) {
    const int64_t o = i * N + s;
    if (vec) {
      float4 h = *reinterpret_cast<const float4*>(state + o);
      const float4 r = __ldg(reinterpret_cast<const float4*>(A + d * N + s));
      float bv[4], cv[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bv[k] = to_f32(Bb[s + k]);
        cv[k] = to_f32(Cb[s + k]);
      }
      h.x = fmaf(ex2(dt * bounded(r.x * kLog2e)), h.x, dtx * bv[0]);
      h.y = fmaf(ex2(dt * bounded(r.y * kLog2e)), h.y, dtx * bv[1]);
      h.z = fmaf(ex2(dt * bounded(r.z * kLog2e)), h.z, dtx * bv[2]);
      h.w = fmaf(ex2(dt * bounded(r.w * kLog2e)), h.w, dtx * bv[3]);
      sum = fmaf(cv[0], h.x, fmaf(cv[1], h.y, fmaf(cv[2], h.z, fmaf(cv[3], h.w, sum))));
      *reinterpret_cast<float4*>(out + o) = h;
    } else {
      for (int k = 0; k < 4 && s + k < N; ++k) {
        const float h = fmaf(ex2(dt * bounded(A[d * N + s + k] * kLog2e)), state[o + k],
                             dtx * to_f32(Bb[s + k]));
        sum = fmaf(to_f32(Cb[s + k]), h, sum);
        out[o + k] = h;
      }
    }
  }
#pragma unroll
  for (int m = 1; m < LPC; m *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (on && sl == 0) {
    float v = D ? fmaf(D[d], xv, sum) : sum;
    if (z) {
      const float g = to_f32(z[b * z_sb + d]);
      v *= g * sigmoid(g);
    }
    y[i] = from_f32<T>(v);
  }
}

template <typename T>
static oxc_status selective_step_launch(const void* x, int64_t x_sb, const void* delta,
                                        int64_t delta_sb, const float* A, const void* B,
                                        int64_t B_sb, const void* C, int64_t C_sb, const float* D,
                                        const void* z, int64_t z_sb, const float* delta_bias,
                                        const float* state, float* out, void* y, int64_t batch,
                                        int64_t dim, int64_t N, cudaStream_t s) {
  const int64_t n = batch * dim;
  const bool vec = N % 4 == 0 && aligned16(state) && aligned16(out) && aligned16(A);
  auto go = [&](auto lanes) {
    constexpr int LPC = decltype(lanes)::value;
    selective_step_kernel<T, LPC><<<(unsigned int)((n * LPC + 127) / 128), 128, 0, s>>>(
        static_cast<const T*>(x), x_sb, static_cast<const T*>(delta), delta_sb, A,
        static_cast<const T*>(B), B_sb, static_cast<const T*>(C), C_sb, D,
        static_cast<const T*>(z), z_sb, delta_bias, state, out, static_cast<T*>(y), n, dim, (int)N,
        vec);
  };
  if (N <= 4) go(std::integral_constant<int, 1>{});
  else if (N <= 8) go(std::integral_constant<int, 2>{});
  else if (N <= 16) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 8>{});
  return check_launch("oxc_selective_step");
}

}  // namespace oxc

using namespace oxc;

extern "C" {

int64_t oxc_selective_scan_carry_size(int64_t batch, int64_t length, int64_t dim, int64_t state) {
  if (batch <= 0 || length <= 0 || dim <= 0 || state <= 0) return 0;
  return batch * selective_tiles(length) * dim * state;
}

size_t oxc_selective_scan_workspace_size(int64_t batch, int64_t length, int64_t dim, int64_t state,
                                         int32_t backward) {
  if (batch <= 0 || length <= 0 || dim <= 0 || state <= 0 || state > kMaxState) return 0;
  const Plan p = selective_plan(batch, length, dim, state, backward);
  size_t n = map_floats(p, batch, dim, state);
  if (backward)
    n += (size_t)batch * p.segments * (size_t)(dim * state + 2 * dim) +
         (size_t)p.ctiles * (size_t)(batch * length) * (size_t)(2 * state);
  return n * sizeof(float);
}

oxc_status oxc_selective_scan_fwd(const void* x, int64_t x_sb, int64_t x_st, const void* delta,
                                  int64_t delta_sb, int64_t delta_st, const float* A, const void* B,
                                  int64_t B_sb, int64_t B_st, const void* C, int64_t C_sb,
                                  int64_t C_st, const float* D, const void* z, int64_t z_sb,
                                  int64_t z_st, const float* delta_bias, const uint8_t* starts,
                                  const float* h0, void* y, float* last, float* carry,
                                  int64_t batch, int64_t length, int64_t dim, int64_t state,
                                  int32_t dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const oxc_status st = selective_check("selective_scan", dtype, batch, length, dim, state);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (state == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_scan without states");
  if (length == 0) {  // the state passes through
    if (!last) return OXC_OK;
    const size_t n = (size_t)batch * (size_t)dim * (size_t)state * sizeof(float);
    const cudaError_t e = h0 ? cudaMemcpyAsync(last, h0, n, cudaMemcpyDeviceToDevice, s)
                             : cudaMemsetAsync(last, 0, n, s);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_selective_scan_fwd");
  }
  if (!x || !delta || !A || !B || !C || !y)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_scan: null pointer");
  const size_t need = oxc_selective_scan_workspace_size(batch, length, dim, state, 0);
  if (need && (!workspace || workspace_bytes < need))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_scan: workspace too small");
  auto go = [&](auto zero) {
    using T = decltype(zero);
    SelectiveArgs<T> a{};
    a.x = {static_cast<const T*>(x), x_sb, x_st};
    a.delta = {static_cast<const T*>(delta), delta_sb, delta_st};
    a.z = {static_cast<const T*>(z), z_sb, z_st};
    a.B = {static_cast<const T*>(B), B_sb, B_st};
    a.C = {static_cast<const T*>(C), C_sb, C_st};
    a.A = A;
    a.D = D;
    a.delta_bias = delta_bias;
    a.h0 = h0;
    a.starts = starts;
    a.y = static_cast<T*>(y);
    a.last = last;
    a.carry = carry;
    a.batch = batch;
    a.length = length;
    a.dim = dim;
    a.N = (int)state;
    selective_segments(a, selective_plan(batch, length, dim, state, false), static_cast<float*>(workspace));
    return selective_fwd_launch(a, s);
  };
  return dtype == OXC_BF16 ? go(bf16{}) : go(0.0f);
}

oxc_status oxc_selective_scan_bwd(const void* x, int64_t x_sb, int64_t x_st, const void* delta,
                                  int64_t delta_sb, int64_t delta_st, const float* A, const void* B,
                                  int64_t B_sb, int64_t B_st, const void* C, int64_t C_sb,
                                  int64_t C_st, const float* D, const void* z, int64_t z_sb,
                                  int64_t z_st, const float* delta_bias, const uint8_t* starts,
                                  const float* carry, const void* dy, int64_t dy_sb, int64_t dy_st,
                                  const float* dlast, void* dx, void* ddelta, float* sums, void* dB,
                                  void* dC, void* dz, float* dh0, int64_t batch, int64_t length,
                                  int64_t dim, int64_t state, int32_t dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const oxc_status st = selective_check("selective_scan backward", dtype, batch, length, dim, state);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dim == 0) return OXC_OK;
  if (state == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_scan without states");
  if (batch == 0 || length == 0) {
    cudaError_t e = sums ? cudaMemsetAsync(sums, 0, sizeof(float) * (size_t)(dim * (state + 2)), s) : cudaSuccess;
    const size_t n = (size_t)batch * (size_t)dim * (size_t)state * sizeof(float);
    if (e == cudaSuccess && dh0 && n)
      e = dlast ? cudaMemcpyAsync(dh0, dlast, n, cudaMemcpyDeviceToDevice, s)
                : cudaMemsetAsync(dh0, 0, n, s);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_selective_scan_bwd");
  }
  if (!x || !delta || !A || !B || !C || !carry || !dx || !ddelta || !sums || !dB || !dC || (z && !dz))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_scan backward: null pointer");
  const size_t need = oxc_selective_scan_workspace_size(batch, length, dim, state, 1);
  if (!workspace || workspace_bytes < need)
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: selective_scan backward: workspace too small");
  if (batch * length > 0x7fffffffll * 256 / (2 * state))
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: selective_scan backward: %lld tokens",
                (long long)(batch * length));
  auto go = [&](auto zero) {
    using T = decltype(zero);
    SelectiveArgs<T> a{};
    a.x = {static_cast<const T*>(x), x_sb, x_st};
    a.delta = {static_cast<const T*>(delta), delta_sb, delta_st};
    a.z = {static_cast<const T*>(z), z_sb, z_st};
    a.B = {static_cast<const T*>(B), B_sb, B_st};
    a.C = {static_cast<const T*>(C), C_sb, C_st};
    a.dy = {static_cast<const T*>(dy), dy_sb, dy_st};
    a.A = A;
    a.D = D;
    a.delta_bias = delta_bias;
    a.starts = starts;
    a.carry = const_cast<float*>(carry);
    a.dlast = dlast;
    a.dx = static_cast<T*>(dx);
    a.ddelta = static_cast<T*>(ddelta);
    a.dz = static_cast<T*>(dz);
    a.dh0 = dh0;
    a.batch = batch;
    a.length = length;
    a.dim = dim;
    a.N = (int)state;
    const Plan p = selective_plan(batch, length, dim, state, true);
    float* ws = static_cast<float*>(workspace);
    a.sums = ws;  // first, as its parts of dA are read as vectors
    a.rows = a.sums + (size_t)batch * p.segments * (size_t)(dim * state + 2 * dim);
    selective_segments(a, p, a.rows + (size_t)p.ctiles * (size_t)(batch * length) * (size_t)(2 * state));
    return selective_bwd_launch<T>(a, sums, static_cast<T*>(dB), static_cast<T*>(dC), s);
  };
  return dtype == OXC_BF16 ? go(bf16{}) : go(0.0f);
}

oxc_status oxc_selective_step(const void* x, int64_t x_sb, const void* delta, int64_t delta_sb,
                              const float* A, const void* B, int64_t B_sb, const void* C,
                              int64_t C_sb, const float* D, const void* z, int64_t z_sb,
                              const float* delta_bias, const float* state_in, float* state_out,
                              void* y, int64_t batch, int64_t dim, int64_t state, int32_t dtype,
                              void* stream) {
  const oxc_status st = selective_check("selective_step", dtype, batch, 1, dim, state);
  if (st) return st;
  if (batch == 0 || dim == 0) return OXC_OK;
  if (state == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_step without states");
  if (!x || !delta || !A || !B || !C || !state_in || !state_out || !y)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: selective_step: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = dtype == OXC_BF16 ? selective_step_launch<bf16> : selective_step_launch<float>;
  return go(x, x_sb, delta, delta_sb, A, B, B_sb, C, C_sb, D, z, z_sb, delta_bias, state_in,
            state_out, y, batch, dim, state, s);
}

}  // extern "C"
