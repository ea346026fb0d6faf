// selective_scan.cu -- the forward of the selective scan, its single-token step and
// the C entries (the mathematics is in selective_scan.cuh).
#include "selective_scan.cuh"

namespace oxc {

// MAP: only finds what a segment does to the state.
template <typename T, int SPT, int LPC, bool VEC, bool MAP>
__global__ void __launch_bounds__(Layout<T, SPT, LPC>::kThreads)
selective_fwd_kernel(SelectiveArgs<T> a) {
  using L = Layout<T, SPT, LPC>;
  constexpr int P = L::P, VW = VEC ? 4 : 1;
  extern __shared__ __align__(16) float smem[];
  float* s_dt = smem;                               // [kTile][kChannels]
  float* s_dtx = s_dt + kTile * L::kChannels;       // dt x
  float* s_y = s_dtx + kTile * L::kChannels;
  float* s_B = s_y + (MAP ? 0 : kTile * L::kChannels);  // [kTile][NP]
  float* s_C = s_B + kTile * L::NP;
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int runs = MAP ? a.segments - 1 : a.segments;  // nothing follows the last
  const int64_t b = rest / runs;
  const int seg = rest % runs;
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const Place<L> at(d0);
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, tile1 = min(tiles, tile0 + a.seg_tiles);
  if (!MAP) pdl_wait();
  float2 A2[2][P], h[2][P];
  load_decay<L>(A2, at, a);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (MAP) {
#pragma unroll
      for (int i = 0; i < P; ++i) h[c][i] = both(0.0f);
    } else {
      at.load(h[c], a.h0, c, b, a.dim, a.N);
    }
  }
  if (!MAP)
    for (int k = 0; k < seg; ++k) through_segment<L>(h, A2, at, a, b, k);
  float time[2] = {0.0f, 0.0f};
  bool fresh = false;
  for (int64_t tile = tile0; tile < tile1; ++tile) {
    const int64_t t0 = tile * kTile;
    each_vec<L, VW>([&](int t, int ch) {
      const bool on = t0 + t < a.length && d0 + ch < a.dim;
      float x[VW], dt[VW];
      if (on) {
        load_vec<VW>(x, a.x.p + b * a.x.sb + (t0 + t) * a.x.st + d0 + ch);
        load_vec<VW>(dt, a.delta.p + b * a.delta.sb + (t0 + t) * a.delta.st + d0 + ch);
      }
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        // beyond the sequence dt = 0: the state stays
        dt[k] = on ? softplus(dt[k] + (a.delta_bias ? a.delta_bias[d0 + ch + k] : 0.0f)) : 0.0f;
        s_dt[t * L::kChannels + ch + k] = dt[k];
        s_dtx[t * L::kChannels + ch + k] = on ? dt[k] * x[k] : 0.0f;
      }
    });
    stage_rows<L>(s_B, a.B, b, t0, a.length, a.N);
    if (!MAP) stage_rows<L>(s_C, a.C, b, t0, a.length, a.N);
    const unsigned int starts = tile_starts(a.starts, b, t0, a.length);
    __syncthreads();
    if (!MAP && a.carry) {
#pragma unroll
      for (int c = 0; c < 2; ++c) at.store(h[c], a.carry, c, b * tiles + tile, a.dim, a.N);
    }
#pragma unroll 4
    for (int t = 0; t < kTile; ++t) {
      const float2 dt = *reinterpret_cast<const float2*>(s_dt + t * L::kChannels + at.ch);
      const float2 dtx = *reinterpret_cast<const float2*>(s_dtx + t * L::kChannels + at.ch);
      float2 B[P], C[P];
      load_states<SPT>(B, s_B + t * L::NP + at.sl * SPT);
      if (!MAP) load_states<SPT>(C, s_C + t * L::NP + at.sl * SPT);
      float2 y[2] = {both(0.0f), both(0.0f)};
      const bool start = (starts >> t) & 1u;
      if (start) fresh = true;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float2 d2 = both(c ? dt.y : dt.x), u2 = both(c ? dtx.y : dtx.x);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 e = exp2_pair(__fmul2_rn(A2[c][i], d2));
          const float2 u = __fmul2_rn(u2, B[i]);
          h[c][i] = start ? u : __ffma2_rn(e, h[c][i], u);
          if (!MAP) y[c] = __ffma2_rn(C[i], h[c][i], y[c]);
        }
      }
      if (MAP) {
        time[0] += dt.x;
        time[1] += dt.y;
      } else {
        using Sum = LaneSum<2, 1, LPC>;
        float v[2] = {y[0].x + y[0].y, y[1].x + y[1].y};
        int first = 0;
        Sum::run(v, at.sl, first);
        if (at.sl < Sum::kUsed) {
#pragma unroll
          for (int i = 0; i < Sum::kKept; ++i) s_y[t * L::kChannels + at.ch + first + i] = v[i];
        }
      }
    }
    __syncthreads();
    if (!MAP)
      each_vec<L, VW>([&](int t, int ch) {
        if (t0 + t >= a.length || d0 + ch >= a.dim) return;
        float x[VW], y[VW];
        load_vec<VW>(x, a.x.p + b * a.x.sb + (t0 + t) * a.x.st + d0 + ch);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          y[k] = s_y[t * L::kChannels + ch + k];
          if (a.D) y[k] = fmaf(a.D[d0 + ch + k], x[k], y[k]);
        }
        if (a.z.p) {
          load_vec<VW>(x, a.z.p + b * a.z.sb + (t0 + t) * a.z.st + d0 + ch);
#pragma unroll
          for (int k = 0; k < VW; ++k) y[k] *= x[k] * sigmoid(x[k]);
        }
        store_from_f32<VW>(a.y + (b * a.length + t0 + t) * a.dim + d0 + ch, y);
      });
  }
  if (MAP) {
    const int64_t row = b * a.segments + seg;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      at.store(h[c], a.seg_state, c, row, a.dim, a.N);
      if (at.sl == 0 && at.d + c < a.dim)
        a.seg_time[row * a.dim + at.d + c] = fresh ? -1.0f : time[c];
    }
    pdl_launch_dependents();
  } else if (seg == a.segments - 1 && a.last) {
#pragma unroll
    for (int c = 0; c < 2; ++c) at.store(h[c], a.last, c, b, a.dim, a.N);
  }
}

// One token: LPC lanes a channel, four states a lane at a time.
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
      h.x = fmaf(ex2(dt * (r.x * kLog2e)), h.x, dtx * bv[0]);
      h.y = fmaf(ex2(dt * (r.y * kLog2e)), h.y, dtx * bv[1]);
      h.z = fmaf(ex2(dt * (r.z * kLog2e)), h.z, dtx * bv[2]);
      h.w = fmaf(ex2(dt * (r.w * kLog2e)), h.w, dtx * bv[3]);
      sum = fmaf(cv[0], h.x, fmaf(cv[1], h.y, fmaf(cv[2], h.z, fmaf(cv[3], h.w, sum))));
      *reinterpret_cast<float4*>(out + o) = h;
    } else {
      for (int k = 0; k < 4 && s + k < N; ++k) {
        const float h = fmaf(ex2(dt * (A[d * N + s + k] * kLog2e)), state[o + k],
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
static oxc_status selective_fwd_launch(const SelectiveArgs<T>& a, cudaStream_t s) {
  const bool vec = a.dim % 4 == 0 && seq_vec(a.x) && seq_vec(a.delta) && seq_vec(a.z) &&
                   aligned_to(a.y, 4 * sizeof(T));
  const cudaError_t err = by_state(a.N, [&](auto spt, auto lpc) -> cudaError_t {
    constexpr int SPT = decltype(spt)::value, LPC = decltype(lpc)::value;
    using L = Layout<T, SPT, LPC>;
    const size_t plane = kTile * L::kChannels * sizeof(float), row = kTile * L::NP * sizeof(float);
    const unsigned int per = (unsigned int)(a.batch * a.ctiles);
    if (a.segments > 1) {
      auto map = vec ? selective_fwd_kernel<T, SPT, LPC, true, true>
                     : selective_fwd_kernel<T, SPT, LPC, false, true>;
      const cudaError_t e = launch_scan(map, per * (a.segments - 1), L::kThreads, 2 * plane + row, false, s, a);
      if (e != cudaSuccess) return e;
    }
    auto kernel = vec ? selective_fwd_kernel<T, SPT, LPC, true, false>
                      : selective_fwd_kernel<T, SPT, LPC, false, false>;
    return launch_scan(kernel, per * a.segments, L::kThreads, 3 * plane + 2 * row, a.segments > 1, s, a);
  });
  return err == cudaSuccess ? check_launch("oxc_selective_scan_fwd")
                            : cuda_fail(err, "oxc_selective_scan_fwd");
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
  const Plan p = selective_plan(batch, length, dim, state);
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
    selective_segments(a, selective_plan(batch, length, dim, state), static_cast<float*>(workspace));
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
    const Plan p = selective_plan(batch, length, dim, state);
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
