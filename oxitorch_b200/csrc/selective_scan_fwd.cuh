// selective_scan_fwd.cuh -- the forward of the selective scan (the mathematics is in
// selective_scan.cuh).
#pragma once

#include "selective_scan.cuh"

namespace oxc {

// MAP: only finds what a segment does to the state.
template <typename T, int SPT, int LPC, bool VEC, bool MAP>
__global__ void __launch_bounds__(Forward<SPT, LPC>::kThreads)
selective_fwd_kernel(SelectiveArgs<T> a) {
  using L = Forward<SPT, LPC>;
  constexpr int P = L::P, CPT = L::CPT, VW = VEC ? 4 : 1;
  constexpr int kLeft = LPC < 4 ? LPC : 4;  // partial sums of y that a channel is left with
  using R = Raw<L, T, VW, MAP ? 2 : 3, 1>;  // x, delta, z
  extern __shared__ __align__(16) float smem[];
  float2* s_in = reinterpret_cast<float2*>(smem);   // [kTile][kChannels] dt, dt x
  float* s_y = smem + 2 * kTile * L::kChannels;     // [kTile][kChannels][kLeft]
  float* s_B = s_y + (MAP ? 0 : kLeft * kTile * L::kChannels);  // [kTile][NP]
  float* s_C = s_B + kTile * L::NP;
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int runs = MAP ? a.segments - 1 : a.segments;  // nothing follows the last
  const int64_t b = rest / runs;
  const int seg = rest % runs;
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const Place<L> at(d0);
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, tile1 = min(tiles, tile0 + a.seg_tiles);
  R raw(reinterpret_cast<T*>(s_C + (MAP ? 0 : kTile * L::NP)), d0, a.dim);
  raw.open(0, a.x, b, tile0 * kTile, d0);
  raw.open(1, a.delta, b, tile0 * kTile, d0);
  if (!MAP) raw.open(2 % (MAP ? 2 : 3), a.z, b, tile0 * kTile, d0);
  Rows<L, T, 1> rows_B(a.B, b, tile0 * kTile, a.N), rows_C(a.C, b, tile0 * kTile, a.N);
  auto tokens = [&](int64_t tile) { return (int)min((int64_t)kTile, a.length - tile * kTile); };
  auto fetch = [&](int64_t tile) {
    const int left = tokens(tile), buffer = (int)tile & 1;
    raw.fetch(0, buffer, left);
    raw.fetch(1, buffer, left);
    if (!MAP && a.z.p) raw.fetch(2 % (MAP ? 2 : 3), buffer, left);
    copies_sent();
    rows_B.load(left, a.N);
    if (!MAP) rows_C.load(left, a.N);
  };
  fetch(tile0);
  float bias[VW], skip[VW];  // of the thread's vectors
  load_channels(bias, a.delta_bias, d0 + raw.ch, raw.in, 0.0f);
  load_channels(skip, a.D, d0 + raw.ch, raw.in, 0.0f);
  T* out = a.y + (b * a.length + tile0 * kTile + raw.t) * a.dim + d0 + raw.ch;
  float2 A2[CPT][P], h[CPT][P];
  load_decay<L>(A2, at, a);
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    if (MAP) {
#pragma unroll
      for (int i = 0; i < P; ++i) h[c][i] = both(0.0f);
    } else {
      at.load(h[c], a.h0, c, b, a.dim, a.N);
    }
  }
  if (!MAP && a.segments > 1) {
    pdl_wait();
    for (int k = 0; k < seg; ++k) through_segment<L>(h, A2, at, a, b, k);
  }
  float time[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) time[c] = 0.0f;
  bool fresh = false;
  for (int64_t tile = tile0; tile < tile1; ++tile) {
    const int left = tokens(tile), buffer = (int)tile & 1;
    raw.land(buffer, left);
#pragma unroll
    for (int k = 0; k < R::kMine; ++k) {
      if (!raw.has) break;
      const bool on = raw.on(k, left);
      float x[VW], dt[VW];
      raw.read(x, buffer, 0, k);
      raw.read(dt, buffer, 1, k);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        // beyond the sequence dt = 0: the state stays
        dt[i] = on ? softplus(dt[i] + bias[i]) : 0.0f;
        x[i] = dt[i] * x[i];
      }
      float2* to = s_in + (raw.t + k * R::kTurn) * L::kChannels + raw.ch;
      if constexpr (VW == 4) {
        reinterpret_cast<float4*>(to)[0] = make_float4(dt[0], x[0], dt[1], x[1]);
        reinterpret_cast<float4*>(to)[1] = make_float4(dt[2], x[2], dt[3], x[3]);
      } else {
        to[0] = make_float2(dt[0], x[0]);
      }
    }
    rows_B.put(s_B);
    if (!MAP) rows_C.put(s_C);
    const unsigned int starts = tile_starts(a.starts, b, tile * kTile, a.length);
    __syncthreads();
    if (tile + 1 < tile1) fetch(tile + 1);
    if (!MAP && a.carry) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) at.store(h[c], a.carry, c, b * tiles + tile, a.dim, a.N);
    }
    if (starts) fresh = true;
    by_fresh(starts, [&](auto some) {
      // kAhead tokens at a time: all their reads before the first of their stores, which
      // the compiler cannot tell from them
      constexpr int kAhead = 4;
#pragma unroll 1
      for (int t1 = 0; t1 < kTile; t1 += kAhead) {
        float2 in[kAhead][CPT], B[kAhead][P], C[kAhead][P];
        float y[kAhead][CPT];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int t = t1 + k;
          if constexpr (CPT == 2) {
            const float4 v = *reinterpret_cast<const float4*>(s_in + t * L::kChannels + at.ch);
            in[k][0] = make_float2(v.x, v.y);
            in[k][1] = make_float2(v.z, v.w);
          } else {
            in[k][0] = s_in[t * L::kChannels + at.ch];
          }
          load_states<SPT>(B[k], s_B + t * L::NP + at.sl * SPT);
          if (!MAP) load_states<SPT>(C[k], s_C + t * L::NP + at.sl * SPT);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const bool start = decltype(some)::value && ((starts >> (t1 + k)) & 1u);
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            float2 sum = both(0.0f);
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 e = exp2_pair(__fmul2_rn(A2[c][i], both(in[k][c].x)));
              const float2 u = __fmul2_rn(both(in[k][c].y), B[k][i]);
              h[c][i] = start ? u : __ffma2_rn(e, h[c][i], u);
              if (!MAP) sum = i ? __ffma2_rn(C[k][i], h[c][i], sum) : __fmul2_rn(C[k][i], h[c][i]);
            }
            if (MAP) time[c] += in[k][c].x;
            y[k][c] = sum.x + sum.y;
          }
        }
        if (!MAP) {
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
#pragma unroll
              for (int m = kLeft; m < LPC; m *= 2) y[k][c] += __shfl_xor_sync(0xffffffffu, y[k][c], m);
              if (LPC == kLeft || at.sl < kLeft)
                s_y[((t1 + k) * L::kChannels + at.ch + c) * kLeft + at.sl] = y[k][c];
            }
        }
      }
    });
    __syncthreads();
    if (!MAP) {
#pragma unroll
      for (int k = 0; k < R::kMine; ++k) {
        if (!raw.on(k, left)) break;
        float x[VW], y[VW];
        raw.read(x, buffer, 0, k);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const float* p = s_y + ((raw.t + k * R::kTurn) * L::kChannels + raw.ch + i) * kLeft;
          if constexpr (kLeft == 4) {
            const float4 v = *reinterpret_cast<const float4*>(p);
            y[i] = (v.x + v.y) + (v.z + v.w);
          } else {
            y[i] = p[0] + p[kLeft - 1];
          }
          if (a.D) y[i] = fmaf(skip[i], x[i], y[i]);
        }
        if (a.z.p) {
          raw.read(x, buffer, 2 % (MAP ? 2 : 3), k);
#pragma unroll
          for (int i = 0; i < VW; ++i) y[i] *= x[i] * sigmoid(x[i]);
        }
        store_from_f32<VW>(out + k * R::kTurn * a.dim, y);
      }
      out += kTile * a.dim;
    }
  }
  if (MAP) {
    const int64_t row = b * a.segments + seg;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      at.store(h[c], a.seg_state, c, row, a.dim, a.N);
      if (at.sl == 0 && at.d + c < a.dim)
        a.seg_time[row * a.dim + at.d + c] = fresh ? -1.0f : time[c];
    }
    pdl_launch_dependents();
  } else if (seg == a.segments - 1 && a.last) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) at.store(h[c], a.last, c, b, a.dim, a.N);
  }
}

template <typename T>
oxc_status selective_fwd_launch(const SelectiveArgs<T>& a, cudaStream_t s) {
  const bool vec = a.dim % 4 == 0 && seq_vec(a.x) && seq_vec(a.delta) && seq_vec(a.z) &&
                   aligned_to(a.y, 4 * sizeof(T));
  const cudaError_t err = by_state(a.N, [&](auto spt, auto lpc) -> cudaError_t {
    constexpr int SPT = decltype(spt)::value, LPC = decltype(lpc)::value;
    using L = Forward<SPT, LPC>;
    const size_t plane = kTile * L::kChannels * sizeof(float), row = kTile * L::NP * sizeof(float);
    const unsigned int per = (unsigned int)(a.batch * a.ctiles);
    if (a.segments > 1) {
      const size_t raw = sizeof(T) * (vec ? Raw<L, T, 4, 2, 1>::kElements : Raw<L, T, 1, 2, 1>::kElements);
      auto map = vec ? selective_fwd_kernel<T, SPT, LPC, true, true>
                     : selective_fwd_kernel<T, SPT, LPC, false, true>;
      const cudaError_t e = launch_scan(map, per * (a.segments - 1), L::kThreads, 2 * plane + row + raw, false, s, a);
      if (e != cudaSuccess) return e;
    }
    const size_t raw = sizeof(T) * (vec ? Raw<L, T, 4, 3, 1>::kElements : Raw<L, T, 1, 3, 1>::kElements);
    auto kernel = vec ? selective_fwd_kernel<T, SPT, LPC, true, false>
                      : selective_fwd_kernel<T, SPT, LPC, false, false>;
    return launch_scan(kernel, per * a.segments, L::kThreads,
                       (2 + (LPC < 4 ? LPC : 4)) * plane + 2 * row + raw, a.segments > 1, s, a);
  });
  return err == cudaSuccess ? check_launch("oxc_selective_scan_fwd")
                            : cuda_fail(err, "oxc_selective_scan_fwd");
}

}  // namespace oxc
