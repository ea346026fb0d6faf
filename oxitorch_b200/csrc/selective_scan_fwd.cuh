// selective_scan_fwd.cuh -- the forward of the selective scan (the mathematics is in
// selective_scan.cuh).
#pragma once

#include "selective_scan.cuh"

namespace oxc {

template <class L, typename T, int VW, bool MAP>
struct ForwardShared {
  using R = Raw<L, T, VW, MAP ? 2 : 3, 1, 3>;  // x, delta, z
  static constexpr int kLeft = L::LPC < 4 ? L::LPC : 4;  // partial sums of y that a channel is left with
  static constexpr int kPlane = kTile * L::kChannels, kRow = kTile * L::NP;
  // twice each, for the even tiles and the odd
  static constexpr int kIn = 2 * kPlane;                    // [kTile][kChannels] dt, dt x
  static constexpr int kYRow = L::kChannels + (L::kLanes < 4 ? 4 : L::kLanes);  // banks apart
  static constexpr int kY = MAP ? 0 : kTile * kLeft * kYRow;  // [kTile][kLeft][kYRow]
  static constexpr int kBC = (MAP ? 1 : 2) * kRow;          // [kTile][NP]
  static constexpr int kFloats = 2 * (kIn + kY + kBC);
  static_assert(kYRow % 4 == 0 && kIn % 4 == 0 && kBC % 4 == 0, "vectors of 16 bytes");
  static constexpr size_t kBytes = sizeof(float) * kFloats + sizeof(T) * R::kElements;
};

// MAP: only finds what a segment does to the state.
template <typename T, int SPT, int LPC, bool VEC, bool MAP>
__global__ void __launch_bounds__(Forward<SPT, LPC>::kThreads + kHelpers, 2)
selective_fwd_kernel(SelectiveArgs<T> a) {
  using L = Forward<SPT, LPC>;
  constexpr int P = L::P, CPT = L::CPT, VW = VEC ? 4 : 1;
  using S = ForwardShared<L, T, VW, MAP>;
  using R = typename S::R;
  constexpr int kLeft = S::kLeft, kAll = L::kThreads + kHelpers;
  extern __shared__ __align__(16) float smem[];
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int runs = MAP ? a.segments - 1 : a.segments;  // nothing follows the last
  const int64_t b = rest / runs;
  const int seg = rest % runs;
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles;
  const int count = (int)(min(tiles, tile0 + a.seg_tiles) - tile0);
  auto s_in = [&](int i) { return reinterpret_cast<float2*>(smem + (i & 1) * S::kIn); };
  auto s_y = [&](int i) { return smem + 2 * S::kIn + (i & 1) * S::kY; };
  auto s_B = [&](int i) { return smem + 2 * (S::kIn + S::kY) + (i & 1) * S::kBC; };

  if (threadIdx.x >= L::kThreads) {
    const int me = threadIdx.x - L::kThreads;
    R raw(reinterpret_cast<T*>(smem + S::kFloats), me, d0, a.dim);
    raw.open(0, a.x, b, tile0 * kTile, d0);
    raw.open(1, a.delta, b, tile0 * kTile, d0);
    if (!MAP) raw.open(MAP ? 0 : 2, a.z, b, tile0 * kTile, d0);
    Rows<L, T, 1> rows_B(me, a.B, b, tile0 * kTile), rows_C(me, a.C, b, tile0 * kTile);
    auto tokens = [&](int i) {  // of the segment's i-th tile; none after the last
      return i < count ? (int)min((int64_t)kTile, a.length - (tile0 + i) * kTile) : 0;
    };
    constexpr int kAhead = R::kAsync ? R::kDepth - 1 : 1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) raw.fetch(i, tokens(i));
    rows_B.load(tokens(0), a.N);
    if (!MAP) rows_C.load(tokens(0), a.N);
    float bias[VW], skip[VW];  // of the thread's vectors
    load_channels(bias, a.delta_bias, d0 + raw.ch, raw.in);
    load_channels(skip, a.D, d0 + raw.ch, raw.in);
    T* out = a.y + (b * a.length + tile0 * kTile + raw.t) * a.dim + d0 + raw.ch;
    int buffer = 0, next = kAhead, before = 0;  // of R::kDepth
    for (int i = 0; i <= count; ++i) {
      if (i < count) {
        const int left = tokens(i);
        raw.land(buffer, left);
        if constexpr (!R::kAsync) raw.fetch(next, tokens(i + 1));
#pragma unroll
        for (int k = 0; k < R::kMine; ++k) {
          if (!raw.has) break;
          const bool on = raw.on(k, left);
          float x[VW], dt[VW];
          raw.read(x, buffer, 0, k);
          raw.read(dt, buffer, 1, k);
#pragma unroll
          for (int v = 0; v < VW; ++v) {
            // beyond the sequence dt = 0: the state stays
            dt[v] = on ? softplus(dt[v] + bias[v]) : 0.0f;
            x[v] = dt[v] * x[v];
          }
          float2* to = s_in(i) + (raw.t + k * R::kTurn) * L::kChannels + raw.ch;
          if constexpr (VW == 4) {
            reinterpret_cast<float4*>(to)[0] = make_float4(dt[0], x[0], dt[1], x[1]);
            reinterpret_cast<float4*>(to)[1] = make_float4(dt[2], x[2], dt[3], x[3]);
          } else {
            to[0] = make_float2(dt[0], x[0]);
          }
        }
        rows_B.put(s_B(i));
        if (!MAP) rows_C.put(s_B(i) + S::kRow);
        tile_arrive(kFull + (i & 1), kAll);
        rows_B.load(tokens(i + 1), a.N);
        if (!MAP) rows_C.load(tokens(i + 1), a.N);
      }
      if (i > 0) {
        tile_sync(kDone + ((i - 1) & 1), kAll);
        if (!MAP) {
          const int left = tokens(i - 1);
          const float* s = s_y(i - 1);
#pragma unroll
          for (int k = 0; k < R::kMine; ++k) {
            if (!raw.on(k, left)) break;
            float x[VW], y[VW], part[VW];
            raw.read(x, before, 0, k);
            const float* p = s + (raw.t + k * R::kTurn) * kLeft * S::kYRow + raw.ch;
            load_floats(y, p);
#pragma unroll
            for (int m = 1; m < kLeft; ++m) {
              load_floats(part, p + m * S::kYRow);
#pragma unroll
              for (int v = 0; v < VW; ++v) y[v] += part[v];
            }
#pragma unroll
            for (int v = 0; v < VW; ++v) {
              if (a.D) y[v] = fmaf(skip[v], x[v], y[v]);
            }
            if (a.z.p) {
              raw.read(x, before, MAP ? 0 : 2, k);
#pragma unroll
              for (int v = 0; v < VW; ++v) y[v] *= x[v] * sigmoid(x[v]);
            }
            store_from_f32<VW>(out + k * R::kTurn * a.dim, y);
          }
          out += kTile * a.dim;
        }
      }
      if constexpr (R::kAsync) raw.fetch(next, tokens(i + kAhead));  // where the tile just stored was
      before = buffer;
      buffer = buffer + 1 == R::kDepth ? 0 : buffer + 1;
      next = next + 1 == R::kDepth ? 0 : next + 1;
    }
    return;
  }

  const Place<L> at(d0);
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
  Starts ahead(a.starts, b, a.length, tile0);
  for (int tile = 0; tile < count; ++tile) {
    const unsigned int starts = ahead.bits(tile0 + tile + 1);
    if (starts) fresh = true;
    if (!MAP && a.carry) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) at.store(h[c], a.carry, c, b * tiles + tile0 + tile, a.dim, a.N);
    }
    tile_sync(kFull + (tile & 1), kAll);
    const float2* in_tile = s_in(tile) + at.ch;
    const float *B_tile = s_B(tile) + at.sl * SPT, *C_tile = B_tile + S::kRow;
    float* y_tile = s_y(tile) + at.sl * S::kYRow + at.ch;
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
#pragma unroll
          for (int c = 0; c < CPT; ++c) in[k][c] = in_tile[t * L::kChannels + c * L::kLanes];
          load_states<SPT>(B[k], B_tile + t * L::NP);
          if (!MAP) load_states<SPT>(C[k], C_tile + t * L::NP);
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
              for (int m = kLeft; m < LPC; m *= 2)
                y[k][c] += __shfl_xor_sync(0xffffffffu, y[k][c], m * L::kLanes);
              if (LPC == kLeft || at.sl < kLeft) y_tile[(t1 + k) * kLeft * S::kYRow + c * L::kLanes] = y[k][c];
            }
        }
      }
    });
    tile_arrive(kDone + (tile & 1), kAll);
  }
  if (MAP) {
    const int64_t row = b * a.segments + seg;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      at.store(h[c], a.seg_state, c, row, a.dim, a.N);
      const int64_t d = at.d + c * L::kLanes;
      if (at.sl == 0 && d < a.dim) a.seg_time[row * a.dim + d] = fresh ? -1.0f : time[c];
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
    constexpr int kAll = L::kThreads + kHelpers;
    const unsigned int per = (unsigned int)(a.batch * a.ctiles);
    if (a.segments > 1) {
      auto map = vec ? selective_fwd_kernel<T, SPT, LPC, true, true>
                     : selective_fwd_kernel<T, SPT, LPC, false, true>;
      const size_t smem = vec ? ForwardShared<L, T, 4, true>::kBytes : ForwardShared<L, T, 1, true>::kBytes;
      const cudaError_t e = launch_scan(map, per * (a.segments - 1), kAll, smem, false, s, a);
      if (e != cudaSuccess) return e;
    }
    auto kernel = vec ? selective_fwd_kernel<T, SPT, LPC, true, false>
                      : selective_fwd_kernel<T, SPT, LPC, false, false>;
    const size_t smem = vec ? ForwardShared<L, T, 4, false>::kBytes : ForwardShared<L, T, 1, false>::kBytes;
    return launch_scan(kernel, per * a.segments, kAll, smem, a.segments > 1, s, a);
  });
  return err == cudaSuccess ? check_launch("oxc_selective_scan_fwd")
                            : cuda_fail(err, "oxc_selective_scan_fwd");
}

}  // namespace oxc
