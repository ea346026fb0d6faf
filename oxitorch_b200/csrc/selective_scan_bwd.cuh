// selective_scan_bwd.cuh -- the VJP of the selective scan (the mathematics is in
// selective_scan.cuh).
#pragma once

#include "selective_scan.cuh"

namespace oxc {

// What the segments from the second on do to mu, the gradient that flows out of
// their first token.
template <typename T, int SPT, int LPC, bool VEC>
__global__ void __launch_bounds__(Layout<T, SPT, LPC>::kThreads)
selective_bwd_map_kernel(SelectiveArgs<T> a) {
  using L = Layout<T, SPT, LPC>;
  constexpr int P = L::P, VW = VEC ? 4 : 1;
  extern __shared__ __align__(16) float smem[];
  float* s_dt = smem;
  float* s_e = s_dt + kTile * L::kChannels;  // dy silu(z)
  float* s_C = s_e + kTile * L::kChannels;
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / (a.segments - 1);
  const int seg = 1 + rest % (a.segments - 1);
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const Place<L> at(d0);
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, tile1 = min(tiles, tile0 + a.seg_tiles);
  float2 A2[2][P], mu[2][P];
  load_decay<L>(A2, at, a);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < P; ++i) mu[c][i] = both(0.0f);
  float time[2] = {0.0f, 0.0f};
  bool fresh = false;
  for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
    const int64_t t0 = tile * kTile;
    each_vec<L, VW>([&](int t, int ch) {
      const bool on = t0 + t < a.length && d0 + ch < a.dim;
      float e[VW], dt[VW], z[VW];
#pragma unroll
      for (int k = 0; k < VW; ++k) e[k] = 0.0f;
      if (on) {
        load_vec<VW>(dt, a.delta.p + b * a.delta.sb + (t0 + t) * a.delta.st + d0 + ch);
        if (a.dy.p) load_vec<VW>(e, a.dy.p + b * a.dy.sb + (t0 + t) * a.dy.st + d0 + ch);
        if (a.z.p) load_vec<VW>(z, a.z.p + b * a.z.sb + (t0 + t) * a.z.st + d0 + ch);
      }
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        if (on && a.z.p) e[k] *= z[k] * sigmoid(z[k]);
        s_dt[t * L::kChannels + ch + k] =
            on ? softplus(dt[k] + (a.delta_bias ? a.delta_bias[d0 + ch + k] : 0.0f)) : 0.0f;
        s_e[t * L::kChannels + ch + k] = e[k];
      }
    });
    stage_rows<L>(s_C, a.C, b, t0, a.length, a.N);
    const unsigned int starts = tile_starts(a.starts, b, t0, a.length);
    __syncthreads();
#pragma unroll 4
    for (int t = kTile - 1; t >= 0; --t) {
      const float2 dt = *reinterpret_cast<const float2*>(s_dt + t * L::kChannels + at.ch);
      const float2 e = *reinterpret_cast<const float2*>(s_e + t * L::kChannels + at.ch);
      float2 C[P];
      load_states<SPT>(C, s_C + t * L::NP + at.sl * SPT);
      const bool start = (starts >> t) & 1u;
      if (start) fresh = true;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 decay = exp2_pair(__fmul2_rn(A2[c][i], both(c ? dt.y : dt.x)));
          const float2 lam = __ffma2_rn(C[i], both(c ? e.y : e.x), mu[c][i]);
          mu[c][i] = start ? both(0.0f) : __fmul2_rn(decay, lam);
        }
      time[0] += dt.x;
      time[1] += dt.y;
    }
    __syncthreads();
  }
  const int64_t row = b * a.segments + seg;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    at.store(mu[c], a.seg_state, c, row, a.dim, a.N);
    if (at.sl == 0 && at.d + c < a.dim)
      a.seg_time[row * a.dim + at.d + c] = fresh ? -1.0f : time[c];
  }
  pdl_launch_dependents();
}

template <typename T, int SPT, int LPC, bool VEC, bool GATED>
__global__ void __launch_bounds__(Layout<T, SPT, LPC>::kThreads)
selective_bwd_kernel(SelectiveArgs<T> a) {
  using L = Layout<T, SPT, LPC>;
  constexpr int P = L::P, VW = VEC ? 4 : 1, kPlane = kTile * L::kChannels;
  constexpr int kParts = kTile / kBack;
  extern __shared__ __align__(16) float smem[];
  float* s_dt = smem;                    // [kTile][kChannels] each
  float* s_dtx = s_dt + kPlane;
  float* s_e = s_dtx + kPlane;           // dy silu(z)
  float* s_sum = s_e + kPlane;           // through, rate / ln 2, inner - D x
  float* s_B = s_sum + (GATED ? 3 : 2) * kPlane;  // [kTile][NP]
  float* s_C = s_B + kTile * L::NP;
  float* s_rows = s_C + kTile * L::NP;   // [kWarps][kTile][2 NP]: dB, dC
  float2* s_kept = reinterpret_cast<float2*>(s_rows + L::kWarps * kTile * 2 * L::NP);
                                         // [kParts][2 P][kThreads]
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.segments;
  const int seg = rest % a.segments;
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const Place<L> at(d0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, tile1 = min(tiles, tile0 + a.seg_tiles);
  pdl_wait();
  float2 A2[2][P], mu[2][P], dA[2][P];
  load_decay<L>(A2, at, a);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    at.load(mu[c], a.dlast, c, b, a.dim, a.N);
#pragma unroll
    for (int i = 0; i < P; ++i) dA[c][i] = both(0.0f);
  }
  for (int k = a.segments - 1; k > seg; --k) through_segment<L>(mu, A2, at, a, b, k);
  // this thread's columns of dD and ddelta_bias: those of its vectors, which are the
  // same channels at every turn as a turn is a whole number of tokens
  float dD[VW], dbias[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) dD[k] = dbias[k] = 0.0f;
  constexpr int kPer = L::kChannels / VW;
  static_assert(L::kThreads % kPer == 0 || kPer % L::kThreads == 0, "turns end with a token");
  static_assert(kPer <= L::kThreads, "a turn is a token at least");
  for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
    const int64_t t0 = tile * kTile;
    float2 h[2][P];
#pragma unroll
    for (int c = 0; c < 2; ++c) at.load(h[c], a.carry, c, b * tiles + tile, a.dim, a.N);
    each_vec<L, VW>([&](int t, int ch) {
      const bool on = t0 + t < a.length && d0 + ch < a.dim;
      float x[VW], dt[VW], e[VW], z[VW];
#pragma unroll
      for (int k = 0; k < VW; ++k) e[k] = 0.0f;
      if (on) {
        load_vec<VW>(x, a.x.p + b * a.x.sb + (t0 + t) * a.x.st + d0 + ch);
        load_vec<VW>(dt, a.delta.p + b * a.delta.sb + (t0 + t) * a.delta.st + d0 + ch);
        if (a.dy.p) load_vec<VW>(e, a.dy.p + b * a.dy.sb + (t0 + t) * a.dy.st + d0 + ch);
        if (GATED) load_vec<VW>(z, a.z.p + b * a.z.sb + (t0 + t) * a.z.st + d0 + ch);
      }
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        dt[k] = on ? softplus(dt[k] + (a.delta_bias ? a.delta_bias[d0 + ch + k] : 0.0f)) : 0.0f;
        if (GATED && on) e[k] *= z[k] * sigmoid(z[k]);
        s_dt[t * L::kChannels + ch + k] = dt[k];
        s_dtx[t * L::kChannels + ch + k] = on ? dt[k] * x[k] : 0.0f;
        s_e[t * L::kChannels + ch + k] = e[k];
      }
    });
    stage_rows<L>(s_B, a.B, b, t0, a.length, a.N);
    stage_rows<L>(s_C, a.C, b, t0, a.length, a.N);
    const unsigned int starts = tile_starts(a.starts, b, t0, a.length);
    __syncthreads();
    auto kept = [&](int j, int c, int i) -> float2& {
      return s_kept[((j * 2 + c) * P + i) * L::kThreads + threadIdx.x];
    };
    // one token forward: `e` the decay, h the state after it
    auto forward = [&](int t, float2 (&e)[2][P], float2 (&h)[2][P]) {
      const float2 dt = *reinterpret_cast<const float2*>(s_dt + t * L::kChannels + at.ch);
      const float2 dtx = *reinterpret_cast<const float2*>(s_dtx + t * L::kChannels + at.ch);
      float2 B[P];
      load_states<SPT>(B, s_B + t * L::NP + at.sl * SPT);
      const bool start = (starts >> t) & 1u;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          e[c][i] = exp2_pair(__fmul2_rn(A2[c][i], both(c ? dt.y : dt.x)));
          const float2 u = __fmul2_rn(both(c ? dtx.y : dtx.x), B[i]);
          h[c][i] = start ? u : __ffma2_rn(e[c][i], h[c][i], u);
        }
    };
    for (int j = 0; j < kParts; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < P; ++i) kept(j, c, i) = h[c][i];
      if (j + 1 == kParts) break;
#pragma unroll
      for (int t = 0; t < kBack; ++t) {
        float2 e[2][P];
        forward(j * kBack + t, e, h);
      }
    }
    for (int j = kParts - 1; j >= 0; --j) {
      float2 in[2][P], decay[kBack][2][P], state[kBack][2][P];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < P; ++i) in[c][i] = h[c][i] = kept(j, c, i);
#pragma unroll
      for (int t = 0; t < kBack; ++t) {
        forward(j * kBack + t, decay[t], h);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < P; ++i) state[t][c][i] = h[c][i];
      }
#pragma unroll
      for (int back = kBack - 1; back >= 0; --back) {
        const int t = j * kBack + back;
        const float2 dt = *reinterpret_cast<const float2*>(s_dt + t * L::kChannels + at.ch);
        const float2 dtx = *reinterpret_cast<const float2*>(s_dtx + t * L::kChannels + at.ch);
        const float2 e = *reinterpret_cast<const float2*>(s_e + t * L::kChannels + at.ch);
        float2 B[P], C[P], dB[P], dC[P], through[2], rate[2], inner[2];
        load_states<SPT>(B, s_B + t * L::NP + at.sl * SPT);
        load_states<SPT>(C, s_C + t * L::NP + at.sl * SPT);
        const bool start = (starts >> t) & 1u;
#pragma unroll
        for (int i = 0; i < P; ++i) dB[i] = dC[i] = both(0.0f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 dt2 = both(c ? dt.y : dt.x), dtx2 = both(c ? dtx.y : dtx.x),
                       e2 = both(c ? e.y : e.x);
          through[c] = rate[c] = inner[c] = both(0.0f);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 lam = __ffma2_rn(C[i], e2, mu[c][i]);
            dC[i] = __ffma2_rn(state[back][c][i], e2, dC[i]);
            dB[i] = __ffma2_rn(lam, dtx2, dB[i]);
            through[c] = __ffma2_rn(lam, B[i], through[c]);
            if (GATED) inner[c] = __ffma2_rn(state[back][c][i], C[i], inner[c]);
            // selected: neither the state nor the gradient crosses a start
            const float2 before = back ? state[back ? back - 1 : 0][c][i] : in[c][i];
            mu[c][i] = start ? both(0.0f) : __fmul2_rn(decay[back][c][i], lam);
            const float2 q = start ? both(0.0f) : __fmul2_rn(mu[c][i], before);
            rate[c] = __ffma2_rn(q, A2[c][i], rate[c]);
            dA[c][i] = __ffma2_rn(q, dt2, dA[c][i]);
          }
        }
        {
          using Sum = LaneSum<4, 1, LPC>;
          float v[4] = {through[0].x + through[0].y, through[1].x + through[1].y,
                        rate[0].x + rate[0].y, rate[1].x + rate[1].y};
          int first = 0;
          Sum::run(v, at.sl, first);
          if (at.sl < Sum::kUsed) {
#pragma unroll
            for (int i = 0; i < Sum::kKept; ++i)
              s_sum[(first + i) / 2 * kPlane + t * L::kChannels + at.ch + (first + i) % 2] = v[i];
          }
        }
        if (GATED) {
          using Sum = LaneSum<2, 1, LPC>;
          float v[2] = {inner[0].x + inner[0].y, inner[1].x + inner[1].y};
          int first = 0;
          Sum::run(v, at.sl, first);
          if (at.sl < Sum::kUsed) {
#pragma unroll
            for (int i = 0; i < Sum::kKept; ++i)
              s_sum[2 * kPlane + t * L::kChannels + at.ch + first + i] = v[i];
          }
        }
        {
          using Sum = LaneSum<2 * SPT, LPC, 32>;
          float v[2 * SPT];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            v[2 * i] = dB[i].x;
            v[2 * i + 1] = dB[i].y;
            v[SPT + 2 * i] = dC[i].x;
            v[SPT + 2 * i + 1] = dC[i].y;
          }
          int first = 0;
          Sum::run(v, lane, first);
          if (lane < Sum::kUsed) {
            float* row = s_rows + (warp * kTile + t) * 2 * L::NP + at.sl * SPT;
#pragma unroll
            for (int i = 0; i < Sum::kKept; ++i) {
              const int k = first + i;
              row[k < SPT ? k : L::NP + k - SPT] = v[i];
            }
          }
        }
      }
    }
    __syncthreads();
    each_vec<L, VW>([&](int t, int ch) {
      if (t0 + t >= a.length || d0 + ch >= a.dim) return;
      const int64_t out = (b * a.length + t0 + t) * a.dim + d0 + ch;
      float x[VW], raw[VW], dx[VW], dd[VW];
      load_vec<VW>(x, a.x.p + b * a.x.sb + (t0 + t) * a.x.st + d0 + ch);
      load_vec<VW>(raw, a.delta.p + b * a.delta.sb + (t0 + t) * a.delta.st + d0 + ch);
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const int i = t * L::kChannels + ch + k;
        const float skip = a.D ? a.D[d0 + ch + k] : 0.0f;
        dx[k] = fmaf(s_dt[i], s_sum[i], skip * s_e[i]);
        const float ddt = fmaf(x[k], s_sum[i], kLn2 * s_sum[kPlane + i]);
        dd[k] = ddt * sigmoid(raw[k] + (a.delta_bias ? a.delta_bias[d0 + ch + k] : 0.0f));
        dD[k] = fmaf(s_e[i], x[k], dD[k]);
        dbias[k] += dd[k];
      }
      store_from_f32<VW>(a.dx + out, dx);
      store_from_f32<VW>(a.ddelta + out, dd);
      if (GATED) {
        float z[VW], dy[VW];
#pragma unroll
        for (int k = 0; k < VW; ++k) dy[k] = 0.0f;
        load_vec<VW>(z, a.z.p + b * a.z.sb + (t0 + t) * a.z.st + d0 + ch);
        if (a.dy.p) load_vec<VW>(dy, a.dy.p + b * a.dy.sb + (t0 + t) * a.dy.st + d0 + ch);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          const float skip = a.D ? a.D[d0 + ch + k] : 0.0f, s = sigmoid(z[k]);
          const float inner = fmaf(skip, x[k], s_sum[2 * kPlane + t * L::kChannels + ch + k]);
          z[k] = dy[k] * inner * fmaf(z[k] * s, 1.0f - s, s);
        }
        store_from_f32<VW>(a.dz + out, z);
      }
    });
    for (int i = threadIdx.x; i < kTile * 2 * L::NP; i += L::kThreads) {
      const int t = i / (2 * L::NP), k = i % (2 * L::NP), n = k % L::NP;
      if (t0 + t < a.length && n < a.N) {
        float s = s_rows[i];
#pragma unroll
        for (int w = 1; w < L::kWarps; ++w) s += s_rows[w * kTile * 2 * L::NP + i];
        a.rows[((int64_t)ct * a.batch * a.length + b * a.length + t0 + t) * 2 * a.N +
               (k < L::NP ? 0 : a.N) + n] = s;
      }
    }
    __syncthreads();
  }
  if (seg == 0) {
#pragma unroll
    for (int c = 0; c < 2; ++c) at.store(mu[c], a.dh0, c, b, a.dim, a.N);
  }
  float* sums = a.sums + (b * a.segments + seg) * (a.dim * a.N + 2 * a.dim);
#pragma unroll
  for (int c = 0; c < 2; ++c) at.store(dA[c], sums, c, 0, a.dim, a.N);
  // dD and ddelta_bias over the threads with the same channels
  constexpr int kSame = L::kThreads / kPer;  // tokens of a turn
  sums += a.dim * a.N;
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    const int ch = threadIdx.x % kPer * VW + k, turn = threadIdx.x / kPer;
    smem[turn * L::kChannels + ch] = dD[k];
    smem[(kSame + turn) * L::kChannels + ch] = dbias[k];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * L::kChannels; i += L::kThreads) {
    const int ch = i % L::kChannels, what = i / L::kChannels;
    float s = 0.0f;
    for (int k = 0; k < kSame; ++k) s += smem[(what * kSame + k) * L::kChannels + ch];
    if (d0 + ch < a.dim) sums[what * a.dim + d0 + ch] = s;
  }
  pdl_launch_dependents();
}

// dB, dC = the sums over the channel tiles, in their order.
template <typename T>
__global__ void __launch_bounds__(256) selective_rows_kernel(const float* __restrict__ rows,
                                                             int64_t tokens, int N, int ctiles,
                                                             T* __restrict__ dB,
                                                             T* __restrict__ dC) {
  pdl_wait();
  const int64_t n = tokens * 2 * N, i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.0f;
#pragma unroll 8
  for (int c = 0; c < ctiles; ++c) s += rows[c * n + i];
  const int64_t token = i / (2 * N);
  const int k = (int)(i - token * 2 * N);
  (k < N ? dB : dC)[token * N + (k < N ? k : k - N)] = from_f32<T>(s);
}

template <typename T, int SPT, int LPC, bool VEC, bool GATED>
static cudaError_t selective_bwd_one(const SelectiveArgs<T>& a, cudaStream_t s) {
  using L = Layout<T, SPT, LPC>;
  const size_t plane = kTile * L::kChannels, row = kTile * L::NP;
  const size_t smem = sizeof(float) * ((GATED ? 6 : 5) * plane + 2 * row + L::kWarps * 2 * row +
                                       2 * 2 * (kTile / kBack) * L::P * L::kThreads);
  return launch_scan(selective_bwd_kernel<T, SPT, LPC, VEC, GATED>,
                (unsigned int)(a.batch * a.ctiles) * a.segments, L::kThreads, smem,
                a.segments > 1, s, a);
}

template <typename T>
oxc_status selective_bwd_launch(const SelectiveArgs<T>& a, float* out_sums, T* dB, T* dC,
                                  cudaStream_t s) {
  const bool vec = a.dim % 4 == 0 && seq_vec(a.x) && seq_vec(a.delta) && seq_vec(a.z) &&
                   seq_vec(a.dy) && aligned_to(a.dx, 4 * sizeof(T)) &&
                   aligned_to(a.ddelta, 4 * sizeof(T)) && aligned_to(a.dz, 4 * sizeof(T));
  cudaError_t err = by_state(a.N, [&](auto spt, auto lpc) -> cudaError_t {
    constexpr int SPT = decltype(spt)::value, LPC = decltype(lpc)::value;
    using L = Layout<T, SPT, LPC>;
    if (a.segments > 1) {
      auto map = vec ? selective_bwd_map_kernel<T, SPT, LPC, true>
                     : selective_bwd_map_kernel<T, SPT, LPC, false>;
      const size_t smem = sizeof(float) * kTile * (2 * L::kChannels + L::NP);
      const cudaError_t e = launch_scan(map, (unsigned int)(a.batch * a.ctiles) * (a.segments - 1),
                                   L::kThreads, smem, false, s, a);
      if (e != cudaSuccess) return e;
    }
    if (a.z.p)
      return vec ? selective_bwd_one<T, SPT, LPC, true, true>(a, s) : selective_bwd_one<T, SPT, LPC, false, true>(a, s);
    return vec ? selective_bwd_one<T, SPT, LPC, true, false>(a, s) : selective_bwd_one<T, SPT, LPC, false, false>(a, s);
  });
  if (err != cudaSuccess) return cuda_fail(err, "oxc_selective_scan_bwd");
  const int64_t tokens = a.batch * a.length, n = tokens * 2 * a.N;
  launch_colsum_partials(a.sums, (int)(a.batch * a.segments), a.dim * a.N + 2 * a.dim, out_sums, s);
  err = launch_scan(selective_rows_kernel<T>, (unsigned int)((n + 255) / 256), 256, 0, false, s, a.rows,
               tokens, a.N, (int)a.ctiles, dB, dC);
  return err == cudaSuccess ? check_launch("oxc_selective_scan_bwd")
                            : cuda_fail(err, "oxc_selective_scan_bwd");
}

}  // namespace oxc
