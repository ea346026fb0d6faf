// selective_scan_bwd.cuh -- the VJP of the selective scan (the mathematics is in
// selective_scan.cuh).
#pragma once

#include "selective_scan.cuh"

namespace oxc {

// What the segments from the second on do to mu, the gradient that flows out of
// their first token.
template <typename T, int SPT, int LPC, bool VEC>
__global__ void __launch_bounds__(Forward<SPT, LPC>::kThreads)
selective_bwd_map_kernel(SelectiveArgs<T> a) {
  using L = Forward<SPT, LPC>;
  constexpr int P = L::P, CPT = L::CPT, VW = VEC ? 4 : 1;
  using R = Raw<L, T, VW, 3, -1>;  // delta, dy, z
  extern __shared__ __align__(16) float smem[];
  float2* s_in = reinterpret_cast<float2*>(smem);  // [kTile][kChannels] dt, dy silu(z)
  float* s_C = smem + 2 * kTile * L::kChannels;
  const unsigned int ct = blockIdx.x % a.map_ctiles, rest = blockIdx.x / a.map_ctiles;
  const int64_t b = rest / (a.segments - 1);
  const int seg = 1 + rest % (a.segments - 1);
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const Place<L> at(d0);
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, tile1 = min(tiles, tile0 + a.seg_tiles);
  R raw(reinterpret_cast<T*>(s_C + kTile * L::NP), d0, a.dim);
  raw.open(0, a.delta, b, (tile1 - 1) * kTile, d0);
  raw.open(1, a.dy, b, (tile1 - 1) * kTile, d0);
  raw.open(2, a.z, b, (tile1 - 1) * kTile, d0);
  Rows<L, T, -1> rows_C(a.C, b, (tile1 - 1) * kTile, a.N);
  auto tokens = [&](int64_t tile) { return (int)min((int64_t)kTile, a.length - tile * kTile); };
  auto fetch = [&](int64_t tile) {
    const int left = tokens(tile), buffer = (int)tile & 1;
    raw.fetch(0, buffer, left);
    if (a.dy.p) raw.fetch(1, buffer, left);
    if (a.z.p) raw.fetch(2, buffer, left);
    copies_sent();
    rows_C.load(left, a.N);
  };
  fetch(tile1 - 1);
  float bias[VW];
  load_channels(bias, a.delta_bias, d0 + raw.ch, raw.in, 0.0f);
  float2 A2[CPT][P], mu[CPT][P];
  load_decay<L>(A2, at, a);
  float time[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    time[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) mu[c][i] = both(0.0f);
  }
  bool fresh = false;
  for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
    const int left = tokens(tile), buffer = (int)tile & 1;
    raw.land(buffer, left);
#pragma unroll
    for (int k = 0; k < R::kMine; ++k) {
      if (!raw.has) break;
      const bool on = raw.on(k, left);
      float dt[VW], e[VW], z[VW];
      raw.read(dt, buffer, 0, k);
      if (a.dy.p) raw.read(e, buffer, 1, k);
      if (a.z.p) raw.read(z, buffer, 2, k);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        if (!a.dy.p) e[i] = 0.0f;
        if (a.z.p) e[i] *= z[i] * sigmoid(z[i]);
        dt[i] = on ? softplus(dt[i] + bias[i]) : 0.0f;
        s_in[(raw.t + k * R::kTurn) * L::kChannels + raw.ch + i] = make_float2(dt[i], e[i]);
      }
    }
    rows_C.put(s_C);
    const unsigned int starts = tile_starts(a.starts, b, tile * kTile, a.length);
    __syncthreads();
    if (tile > tile0) fetch(tile - 1);
    if (starts) fresh = true;
    by_fresh(starts, [&](auto some) {
#pragma unroll 4
      for (int t = kTile - 1; t >= 0; --t) {
        float2 C[P];
        load_states<SPT>(C, s_C + t * L::NP + at.sl * SPT);
        const bool start = decltype(some)::value && ((starts >> t) & 1u);
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
          const float2 in = s_in[t * L::kChannels + at.ch + c];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 decay = exp2_pair(__fmul2_rn(A2[c][i], both(in.x)));
            const float2 lam = __ffma2_rn(C[i], both(in.y), mu[c][i]);
            mu[c][i] = start ? both(0.0f) : __fmul2_rn(decay, lam);
          }
          time[c] += in.x;
        }
      }
    });
    __syncthreads();
  }
  const int64_t row = b * a.segments + seg;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    at.store(mu[c], a.seg_state, c, row, a.dim, a.N);
    if (at.sl == 0 && at.d + c < a.dim)
      a.seg_time[row * a.dim + at.d + c] = fresh ? -1.0f : time[c];
  }
  pdl_launch_dependents();
}

// Where the sums of the VJP's kBack tokens are made, a warp by itself: every lane
// leaves its share, and the shares are added up in vectors.  A few stores and loads
// for kBack tokens in the place of a shuffle and two selects for each value and step.
template <class L, bool GATED>
struct Shares {
  static constexpr int kBlock = 2;                    // tokens at a time
  static constexpr int kSums = GATED ? 3 : 2;         // through, rate, inner
  // [kBlock][kLanes][2 NP] dB and dC, rows apart by 16 banks
  static constexpr int kRow = 2 * L::NP + (L::NP % 16 == 0 && L::kLanes > 1 ? 16 : 4);
  static constexpr int kRowFloats = L::kLanes > 1 ? kBlock * L::kLanes * kRow : 0;
  // [kBlock][LPC][kSums][kWarpChannels], rows apart by 8 banks while they are few
  static constexpr int kSum = L::LPC <= 4 ? (kSums * L::kWarpChannels + 31) / 32 * 32 + 8
                                          : kSums * L::kWarpChannels + 2;
  static constexpr int kSumFloats = (kBlock * L::LPC * kSum + 3) / 4 * 4;
  static constexpr int kFloats = kRowFloats + kSumFloats;
};

template <class L, typename T, int VW, bool GATED>
struct BackwardShared {
  using R = Raw<L, T, VW, GATED ? 4 : 3, -1>;
  using S = Shares<L, GATED>;
  static constexpr int kParts = kTile / kBack;
  static constexpr int kPlane = kTile * L::kChannels;
  static constexpr int kIn = 4 * kPlane;                       // dt, dt x, e, -; later -, rate, -, through
  static constexpr int kInner = GATED ? kPlane : 0;
  static constexpr int kRows = L::kWarps * kTile * 2 * L::NP;  // dB, dC of each warp
  static constexpr int kKept = kParts * L::CPT * L::SPT * L::kThreads;
  static constexpr int kFloats =
      kIn + kInner + 2 * kTile * L::NP + kRows + kKept + L::kWarps * S::kFloats;
  static constexpr size_t kBytes = sizeof(float) * kFloats + sizeof(T) * R::kElements;
};

template <typename T, int SPT, int LPC, bool VEC, bool GATED>
__global__ void __launch_bounds__(Backward<SPT, LPC>::kThreads)
selective_bwd_kernel(SelectiveArgs<T> a) {
  using L = Backward<SPT, LPC>;
  constexpr int P = L::P, CPT = L::CPT, VW = VEC ? 4 : 1;
  static_assert(CPT == 2, "two channels a thread");
  using M = BackwardShared<L, T, VW, GATED>;
  using R = typename M::R;  // x, delta, dy, z
  using S = typename M::S;
  constexpr int kParts = M::kParts;
  extern __shared__ __align__(16) float smem[];
  float4* s_in = reinterpret_cast<float4*>(smem);
  float* s_inner = smem + M::kIn;          // inner - D x
  float* s_B = s_inner + M::kInner;        // [kTile][NP]
  float* s_C = s_B + kTile * L::NP;
  float* s_rows = s_C + kTile * L::NP;     // [kWarps][kTile][2 NP]
  float2* s_kept = reinterpret_cast<float2*>(s_rows + M::kRows);  // [kParts][2 P][kThreads]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = lane / LPC;
  float* share_rows = s_rows + M::kRows + M::kKept + warp * S::kFloats;
  float* share_sums = share_rows + S::kRowFloats;
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.segments;
  const int seg = rest % a.segments;
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const Place<L> at(d0);
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, tile1 = min(tiles, tile0 + a.seg_tiles);
  R raw(reinterpret_cast<T*>(smem + M::kFloats), d0, a.dim);
  const int64_t end0 = (tile1 - 1) * kTile;
  raw.open(0, a.x, b, end0, d0);
  raw.open(1, a.delta, b, end0, d0);
  raw.open(2, a.dy, b, end0, d0);
  if (GATED) raw.open(GATED ? 3 : 0, a.z, b, end0, d0);
  Rows<L, T, -1> rows_B(a.B, b, end0, a.N), rows_C(a.C, b, end0, a.N);
  float2 enter[CPT][P];  // the state before the next tile
  auto tokens = [&](int64_t tile) { return (int)min((int64_t)kTile, a.length - tile * kTile); };
  auto fetch = [&](int64_t tile) {
    const int left = tokens(tile), buffer = (int)tile & 1;
    raw.fetch(0, buffer, left);
    raw.fetch(1, buffer, left);
    if (a.dy.p) raw.fetch(2, buffer, left);
    if (GATED) raw.fetch(GATED ? 3 : 0, buffer, left);
    copies_sent();
    rows_B.load(left, a.N);
    rows_C.load(left, a.N);
#pragma unroll
    for (int c = 0; c < CPT; ++c) at.load(enter[c], a.carry, c, b * tiles + tile, a.dim, a.N);
  };
  fetch(tile1 - 1);
  float bias[VW], skip[VW];  // of the thread's vectors
  load_channels(bias, a.delta_bias, d0 + raw.ch, raw.in, 0.0f);
  load_channels(skip, a.D, d0 + raw.ch, raw.in, 0.0f);
  int64_t out = (b * a.length + end0 + raw.t) * a.dim + d0 + raw.ch;
  float2 A2[CPT][P], mu[CPT][P], dA[CPT][P];
  load_decay<L>(A2, at, a);
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    at.load(mu[c], a.dlast, c, b, a.dim, a.N);
#pragma unroll
    for (int i = 0; i < P; ++i) dA[c][i] = both(0.0f);
  }
  if (a.segments > 1) {
    pdl_wait();
    for (int k = a.segments - 1; k > seg; --k) through_segment<L>(mu, A2, at, a, b, k);
  }
  // this thread's columns of dD and ddelta_bias: those of its vectors
  float dD[VW], dbias[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) dD[k] = dbias[k] = 0.0f;
  for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
    const int left = tokens(tile), buffer = (int)tile & 1;
    raw.land(buffer, left);
#pragma unroll
    for (int k = 0; k < R::kMine; ++k) {
      if (!raw.has) break;
      const bool on = raw.on(k, left);
      float x[VW], dt[VW], e[VW], z[VW];
      raw.read(x, buffer, 0, k);
      raw.read(dt, buffer, 1, k);
      if (a.dy.p) raw.read(e, buffer, 2, k);
      if (GATED) raw.read(z, buffer, GATED ? 3 : 0, k);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        if (!a.dy.p) e[i] = 0.0f;
        if (GATED) e[i] *= z[i] * sigmoid(z[i]);
        dt[i] = on ? softplus(dt[i] + bias[i]) : 0.0f;
        s_in[(raw.t + k * R::kTurn) * L::kChannels + raw.ch + i] = make_float4(dt[i], dt[i] * x[i], e[i], 0.0f);
      }
    }
    rows_B.put(s_B);
    rows_C.put(s_C);
    const unsigned int starts = tile_starts(a.starts, b, tile * kTile, a.length);
    float2 h[CPT][P];
#pragma unroll
    for (int c = 0; c < CPT; ++c)
#pragma unroll
      for (int i = 0; i < P; ++i) h[c][i] = enter[c][i];
    __syncthreads();
    if (tile > tile0) fetch(tile - 1);
    auto kept = [&](int j, int c, int i) -> float2& {
      return s_kept[((j * CPT + c) * P + i) * L::kThreads + threadIdx.x];
    };
    by_fresh(starts, [&](auto some) {
      constexpr bool kSome = decltype(some)::value;
      // the operands of kBack tokens: all read before anything is stored, as the compiler
      // cannot tell the stores from them
      float4 in[kBack][CPT];
      float2 B[kBack][P];
      auto read = [&](int t) {
#pragma unroll
        for (int k = 0; k < kBack; ++k) {
          load_states<SPT>(B[k], s_B + (t + k) * L::NP + at.sl * SPT);
#pragma unroll
          for (int c = 0; c < CPT; ++c) in[k][c] = s_in[(t + k) * L::kChannels + at.ch + c];
        }
      };
      // one token forward: `e` the decay, h the state after it
      auto forward = [&](int t, int k, float2 (&e)[CPT][P], float2 (&h)[CPT][P]) {
        const bool start = kSome && ((starts >> (t + k)) & 1u);
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
          for (int i = 0; i < P; ++i) {
            e[c][i] = exp2_pair(__fmul2_rn(A2[c][i], both(in[k][c].x)));
            const float2 u = __fmul2_rn(both(in[k][c].y), B[k][i]);
            h[c][i] = start ? u : __ffma2_rn(e[c][i], h[c][i], u);
          }
      };
#pragma unroll 1
      for (int j = 0; j + 1 < kParts; ++j) {
        read(j * kBack);
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
          for (int i = 0; i < P; ++i) kept(j, c, i) = h[c][i];
#pragma unroll
        for (int k = 0; k < kBack; ++k) {
          float2 e[CPT][P];
          forward(j * kBack, k, e, h);
        }
      }
#pragma unroll 1
      for (int j = kParts - 1; j >= 0; --j) {
        float2 enters[CPT][P], decay[kBack][CPT][P], state[kBack][CPT][P], Cs[kBack][P];
        read(j * kBack);
#pragma unroll
        for (int k = 0; k < kBack; ++k) load_states<SPT>(Cs[k], s_C + (j * kBack + k) * L::NP + at.sl * SPT);
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
          for (int i = 0; i < P; ++i) {
            if (j + 1 < kParts) h[c][i] = kept(j, c, i);
            enters[c][i] = h[c][i];
          }
#pragma unroll
        for (int k = 0; k < kBack; ++k) {
          forward(j * kBack, k, decay[k], h);
#pragma unroll
          for (int c = 0; c < CPT; ++c)
#pragma unroll
            for (int i = 0; i < P; ++i) state[k][c][i] = h[c][i];
        }
#pragma unroll
        for (int back = kBack - 1; back >= 0; --back) {
          const int t = j * kBack + back, slot = back % S::kBlock;
          float2 dB[P], dC[P], through[CPT], rate[CPT], inner[CPT];
          const bool start = kSome && ((starts >> t) & 1u);
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            const float4 v = in[back][c];
            const float2 dt2 = both(v.x), dtx2 = both(v.y), e2 = both(v.z);
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 C = Cs[back][i], lam = __ffma2_rn(C, e2, mu[c][i]);
              const float2 after = state[back][c][i];
              dC[i] = c ? __ffma2_rn(after, e2, dC[i]) : __fmul2_rn(after, e2);
              dB[i] = c ? __ffma2_rn(lam, dtx2, dB[i]) : __fmul2_rn(lam, dtx2);
              through[c] = i ? __ffma2_rn(lam, B[back][i], through[c]) : __fmul2_rn(lam, B[back][i]);
              if (GATED) inner[c] = i ? __ffma2_rn(after, C, inner[c]) : __fmul2_rn(after, C);
              // selected: neither the state nor the gradient crosses a start
              const float2 before = back ? state[back ? back - 1 : 0][c][i] : enters[c][i];
              mu[c][i] = start ? both(0.0f) : __fmul2_rn(decay[back][c][i], lam);
              const float2 q = start ? both(0.0f) : __fmul2_rn(mu[c][i], before);
              rate[c] = i ? __ffma2_rn(q, A2[c][i], rate[c]) : __fmul2_rn(q, A2[c][i]);
              dA[c][i] = __ffma2_rn(q, dt2, dA[c][i]);
            }
          }
          // this lane's shares
          float* sum = share_sums + (slot * LPC + at.sl) * S::kSum + cl * CPT;
          *reinterpret_cast<float2*>(sum) = make_float2(through[0].x + through[0].y, through[1].x + through[1].y);
          *reinterpret_cast<float2*>(sum + L::kWarpChannels) =
              make_float2(rate[0].x + rate[0].y, rate[1].x + rate[1].y);
          if (GATED)
            *reinterpret_cast<float2*>(sum + 2 * L::kWarpChannels) =
                make_float2(inner[0].x + inner[0].y, inner[1].x + inner[1].y);
          float* row = L::kLanes > 1 ? share_rows + (slot * L::kLanes + cl) * S::kRow + at.sl * SPT
                                     : s_rows + (warp * kTile + t) * 2 * L::NP + at.sl * SPT;
          if constexpr (SPT == 4) {
            *reinterpret_cast<float4*>(row) = make_float4(dB[0].x, dB[0].y, dB[1].x, dB[1].y);
            *reinterpret_cast<float4*>(row + L::NP) = make_float4(dC[0].x, dC[0].y, dC[1].x, dC[1].y);
          } else {
#pragma unroll
            for (int i = 0; i < P; ++i) {
              reinterpret_cast<float2*>(row)[i] = dB[i];
              reinterpret_cast<float2*>(row + L::NP)[i] = dC[i];
            }
          }
          if (slot) continue;
          // the sums of tokens t and t + 1
          __syncwarp();
          if constexpr (L::kLanes > 1) {
            constexpr int kQuads = 2 * L::NP / 4;
#pragma unroll
            for (int o = lane; o < S::kBlock * kQuads; o += 32) {
              const int token = o / kQuads, quad = o % kQuads;
              const float* p = share_rows + token * L::kLanes * S::kRow + quad * 4;
              float4 r = *reinterpret_cast<const float4*>(p);
              float2 lo = make_float2(r.x, r.y), hi = make_float2(r.z, r.w);
#pragma unroll
              for (int k = 1; k < L::kLanes; ++k) {
                r = *reinterpret_cast<const float4*>(p + k * S::kRow);
                lo = __fadd2_rn(lo, make_float2(r.x, r.y));
                hi = __fadd2_rn(hi, make_float2(r.z, r.w));
              }
              *reinterpret_cast<float4*>(s_rows + (warp * kTile + t + token) * 2 * L::NP + quad * 4) =
                  make_float4(lo.x, lo.y, hi.x, hi.y);
            }
          }
          constexpr int kPairs = S::kSums * L::kWarpChannels / 2;
#pragma unroll
          for (int o = lane; o < S::kBlock * kPairs; o += 32) {
            const int token = o / kPairs, pair = o % kPairs, what = pair / (L::kWarpChannels / 2),
                      ch = pair % (L::kWarpChannels / 2) * 2;
            const float* p = share_sums + token * LPC * S::kSum + what * L::kWarpChannels + ch;
            float2 r = *reinterpret_cast<const float2*>(p);
#pragma unroll
            for (int k = 1; k < LPC; ++k) r = __fadd2_rn(r, *reinterpret_cast<const float2*>(p + k * S::kSum));
            const int to = (t + token) * L::kChannels + warp * L::kWarpChannels + ch;
            if (what == 0) {  // dt x has been used
              s_in[to].w = r.x;
              s_in[to + 1].w = r.y;
            } else if (what == 1) {
              s_in[to].y = r.x;
              s_in[to + 1].y = r.y;
            } else {
              *reinterpret_cast<float2*>(s_inner + to) = r;
            }
          }
          __syncwarp();
        }
      }
    });
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R::kMine; ++k) {
      if (!raw.on(k, left)) break;
      const int at0 = (raw.t + k * R::kTurn) * L::kChannels + raw.ch;
      const int64_t to = out + k * R::kTurn * a.dim;
      float x[VW], v[VW], dx[VW], e[VW];
      raw.read(x, buffer, 0, k);
      raw.read(v, buffer, 1, k);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const float4 in = s_in[at0 + i];  // dt, rate / ln 2, e, through
        dx[i] = fmaf(in.x, in.w, skip[i] * in.z);
        const float ddt = fmaf(x[i], in.w, kLn2 * in.y);
        v[i] = ddt * sigmoid(v[i] + bias[i]);
        dD[i] = fmaf(in.z, x[i], dD[i]);
        dbias[i] += v[i];
      }
      store_from_f32<VW>(a.dx + to, dx);
      store_from_f32<VW>(a.ddelta + to, v);
      if (GATED) {
        raw.read(v, buffer, GATED ? 3 : 0, k);
        if (a.dy.p) raw.read(e, buffer, 2, k);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const float s = sigmoid(v[i]), inner = fmaf(skip[i], x[i], s_inner[at0 + i]);
          v[i] = (a.dy.p ? e[i] : 0.0f) * inner * fmaf(v[i] * s, 1.0f - s, s);
        }
        store_from_f32<VW>(a.dz + to, v);
      }
    }
    out -= kTile * a.dim;
    for (int i = threadIdx.x; i < kTile * 2 * L::NP; i += L::kThreads) {
      const int t = i / (2 * L::NP), k = i % (2 * L::NP), n = k % L::NP;
      if (t < left && n < a.N) {
        float s = s_rows[i];
#pragma unroll
        for (int w = 1; w < L::kWarps; ++w) s += s_rows[w * kTile * 2 * L::NP + i];
        a.rows[((int64_t)ct * a.batch * a.length + b * a.length + tile * kTile + t) * 2 * a.N +
               (k < L::NP ? 0 : a.N) + n] = s;
      }
    }
    __syncthreads();
  }
  if (seg == 0) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) at.store(mu[c], a.dh0, c, b, a.dim, a.N);
  }
  float* sums = a.sums + (b * a.segments + seg) * (a.dim * a.N + 2 * a.dim);
#pragma unroll
  for (int c = 0; c < CPT; ++c) at.store(dA[c], sums, c, 0, a.dim, a.N);
  // dD and ddelta_bias over the threads with the same channels
  constexpr int kSame = R::kTurn;
  sums += a.dim * a.N;
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    if (raw.t >= kSame) break;
    smem[raw.t * L::kChannels + raw.ch + k] = dD[k];
    smem[(kSame + raw.t) * L::kChannels + raw.ch + k] = dbias[k];
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
  using L = Backward<SPT, LPC>;
  constexpr size_t smem = BackwardShared<L, T, VEC ? 4 : 1, GATED>::kBytes;
  static_assert(smem <= 227 * 1024, "a CTA's shared memory");
  static_assert(sizeof(float) * 2 * L::kThreads * (VEC ? 4 : 1) <= smem, "dD and ddelta_bias fit");
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
    if (a.segments > 1) {
      using L = Forward<SPT, LPC>;
      SelectiveArgs<T> m = a;
      m.map_ctiles = (unsigned int)((a.dim + L::kChannels - 1) / L::kChannels);
      auto map = vec ? selective_bwd_map_kernel<T, SPT, LPC, true>
                     : selective_bwd_map_kernel<T, SPT, LPC, false>;
      const size_t smem = sizeof(float) * kTile * (2 * L::kChannels + L::NP) +
                          sizeof(T) * (vec ? Raw<L, T, 4, 3, -1>::kElements : Raw<L, T, 1, 3, -1>::kElements);
      const cudaError_t e = launch_scan(map, (unsigned int)a.batch * m.map_ctiles * (a.segments - 1),
                                        L::kThreads, smem, false, s, m);
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
