// selective_scan_bwd.cuh -- the VJP of the selective scan (the mathematics is in
// selective_scan.cuh).
#pragma once

#include <atomic>

#include "selective_scan.cuh"

namespace oxc {

template <class L, typename T, int VW>
struct BackwardMapShared {
  using R = Raw<L, T, VW, 3, -1, 2>;  // delta, dy, z
  static constexpr int kIn = 2 * kTile * L::kChannels;  // dt, dy silu(z); twice, for the even tiles
  static constexpr int kC = kTile * L::NP;              // and the odd, as C
  static constexpr int kFloats = 2 * (kIn + kC);
  static constexpr size_t kBytes = sizeof(float) * kFloats + sizeof(T) * R::kElements;
};

// What the segments from the second on do to mu, the gradient that flows out of
// their first token.
template <typename T, int SPT, int LPC, bool VEC>
__global__ void __launch_bounds__(Forward<SPT, LPC>::kThreads + kHelpers, 2)
selective_bwd_map_kernel(SelectiveArgs<T> a) {
  using L = Forward<SPT, LPC>;
  constexpr int P = L::P, CPT = L::CPT, VW = VEC ? 4 : 1, kAll = L::kThreads + kHelpers;
  using S = BackwardMapShared<L, T, VW>;
  using R = typename S::R;
  extern __shared__ __align__(16) float smem[];
  const unsigned int ct = blockIdx.x % a.map_ctiles, rest = blockIdx.x / a.map_ctiles;
  const int64_t b = rest / (a.segments - 1);
  const int seg = 1 + rest % (a.segments - 1);
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, end = min(tiles, tile0 + a.seg_tiles) - 1;
  const int count = (int)(end + 1 - tile0);  // tile i of them is end - i
  auto s_in = [&](int i) { return reinterpret_cast<float2*>(smem + (i & 1) * S::kIn); };
  auto s_C = [&](int i) { return smem + 2 * S::kIn + (i & 1) * S::kC; };

  if (threadIdx.x >= L::kThreads) {
    const int me = threadIdx.x - L::kThreads;
    R raw(reinterpret_cast<T*>(smem + S::kFloats), me, d0, a.dim);
    raw.open(0, a.delta, b, end * kTile, d0);
    raw.open(1, a.dy, b, end * kTile, d0);
    raw.open(2, a.z, b, end * kTile, d0);
    Rows<L, T, -1> rows_C(me, a.C, b, end * kTile);
    auto tokens = [&](int i) {
      return i < count ? (int)min((int64_t)kTile, a.length - (end - i) * kTile) : 0;
    };
    raw.fetch(0, tokens(0));
    rows_C.load(tokens(0), a.N);
    float bias[VW];
    load_channels(bias, a.delta_bias, d0 + raw.ch, raw.in);
    for (int i = 0; i < count; ++i) {
      const int left = tokens(i), buffer = i & 1;
      raw.land(buffer, left);
      raw.fetch(buffer ^ 1, tokens(i + 1));
      if (i > 1) tile_sync(kDone + (i & 1), kAll);
#pragma unroll
      for (int k = 0; k < R::kMine; ++k) {
        if (!raw.has) break;
        const bool on = raw.on(k, left);
        float dt[VW], e[VW], z[VW];
        raw.read(dt, buffer, 0, k);
        if (a.dy.p) raw.read(e, buffer, 1, k);
        if (a.z.p) raw.read(z, buffer, 2, k);
#pragma unroll
        for (int v = 0; v < VW; ++v) {
          if (!a.dy.p) e[v] = 0.0f;
          if (a.z.p) e[v] *= z[v] * sigmoid(z[v]);
          dt[v] = on ? softplus(dt[v] + bias[v]) : 0.0f;
          s_in(i)[(raw.t + k * R::kTurn) * L::kChannels + raw.ch + v] = make_float2(dt[v], e[v]);
        }
      }
      rows_C.put(s_C(i));
      tile_arrive(kFull + (i & 1), kAll);
      rows_C.load(tokens(i + 1), a.N);
    }
    return;
  }

  const Place<L> at(d0);
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
  Starts ahead(a.starts, b, a.length, end);
  for (int tile = 0; tile < count; ++tile) {
    const unsigned int starts = ahead.bits(end - tile - 1);
    if (starts) fresh = true;
    tile_sync(kFull + (tile & 1), kAll);
    const float2* in_tile = s_in(tile) + at.ch;
    const float* C_tile = s_C(tile) + at.sl * SPT;
    by_fresh(starts, [&](auto some) {
#pragma unroll 4
      for (int t = kTile - 1; t >= 0; --t) {
        float2 C[P];
        load_states<SPT>(C, C_tile + t * L::NP);
        const bool start = decltype(some)::value && ((starts >> t) & 1u);
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
          const float2 in = in_tile[t * L::kChannels + c * L::kLanes];
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
    if (tile + 2 < count) tile_arrive(kDone + (tile & 1), kAll);
  }
  const int64_t row = b * a.segments + seg;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    at.store(mu[c], a.seg_state, c, row, a.dim, a.N);
    const int64_t d = at.d + c * L::kLanes;
    if (at.sl == 0 && d < a.dim) a.seg_time[row * a.dim + d] = fresh ? -1.0f : time[c];
  }
  pdl_launch_dependents();
}

template <class L, typename T, int VW, bool GATED>
struct BackwardShared {
  using R = Raw<L, T, VW, GATED ? 4 : 3, -1, 2>;  // x, delta, dy, z
  static constexpr int kBack = 4;  // tokens whose states are held in registers
  static constexpr int kParts = kTile / kBack;
  static constexpr int kPlane = kTile * L::kChannels;
  // twice each, for the even tiles and the odd
  static constexpr int kIn = (GATED ? 4 : 3) * kPlane;         // planes [kTile][kChannels]: dt, dt x, e and
                                                               // nothing; afterwards dt, through,
                                                               // rate / ln 2, inner - D x
  static constexpr int kBC = 2 * kTile * L::NP;                // [kTile][NP]
  static constexpr int kRows = L::kWarps * kTile * 2 * L::NP;  // [kWarps][kTile][2 NP]: dB, dC, once
  static constexpr int kKept = (kParts - 1) * L::CPT * L::SPT * L::kThreads;  // [..][2 P][kThreads]
  static constexpr int kFloats = 2 * (kIn + kBC) + kRows + kKept;
  static constexpr size_t kBytes = sizeof(float) * kFloats + sizeof(T) * R::kElements;
};

constexpr int kRowsFree = 5;  // the barrier after which the rows of the tile before are read

// Registers a thread: at the launch, then of those that walk and of the helpers.  (88
// for the helpers: f32 [4, 2048, 4096] 777 us; 80: 786; 72: 812; 64, which spills: 960.)
template <class L>
struct Registers {
  static constexpr int kAll = L::kThreads + kHelpers;
  static constexpr int kLaunch = 65536 / kAll / 8 * 8;
  static constexpr bool kDeal = L::CPT == 2;
  static constexpr int kHelp = 88, kWalk = 168;
  static_assert(!kDeal || L::kThreads * kWalk + kHelpers * kHelp <= kAll * kLaunch, "more than there are");
};

template <typename T, int LPC, bool VEC, bool GATED>
__global__ void __launch_bounds__(Backward<LPC>::kThreads + kHelpers, 1)
selective_bwd_kernel(SelectiveArgs<T> a) {
  using L = Backward<LPC>;
  constexpr int SPT = L::SPT, P = L::P, CPT = L::CPT, VW = VEC ? 4 : 1, kAll = L::kThreads + kHelpers;
  using M = BackwardShared<L, T, VW, GATED>;
  using R = typename M::R;
  constexpr int kParts = M::kParts, kBack = M::kBack;
  extern __shared__ __align__(16) float smem[];
  float* s_rows = smem + 2 * (M::kIn + M::kBC);
  const unsigned int ct = blockIdx.x % a.ctiles, rest = blockIdx.x / a.ctiles;
  const int64_t b = rest / a.segments;
  const int seg = rest % a.segments;
  const int64_t d0 = (int64_t)ct * L::kChannels;
  const int64_t tiles = (a.length + kTile - 1) / kTile;
  const int64_t tile0 = (int64_t)seg * a.seg_tiles, end = min(tiles, tile0 + a.seg_tiles) - 1;
  const int count = (int)(end + 1 - tile0);  // tile i of them is end - i
  auto in_of = [&](int i) { return smem + (i & 1) * M::kIn; };
  auto B_of = [&](int i) { return smem + 2 * M::kIn + (i & 1) * M::kBC; };
  float* sums = a.sums + (b * a.segments + seg) * (a.dim * a.N + 2 * a.dim);

  if (threadIdx.x >= L::kThreads) {
    if constexpr (Registers<L>::kDeal) take_registers<Registers<L>::kHelp, false>();
    const int me = threadIdx.x - L::kThreads;
    R raw(reinterpret_cast<T*>(smem + M::kFloats), me, d0, a.dim);
    raw.open(0, a.x, b, end * kTile, d0);
    raw.open(1, a.delta, b, end * kTile, d0);
    raw.open(2, a.dy, b, end * kTile, d0);
    if (GATED) raw.open(GATED ? 3 : 0, a.z, b, end * kTile, d0);
    Rows<L, T, -1> rows_B(me, a.B, b, end * kTile), rows_C(me, a.C, b, end * kTile);
    auto tokens = [&](int i) {
      return i < count ? (int)min((int64_t)kTile, a.length - (end - i) * kTile) : 0;
    };
    raw.fetch(0, tokens(0));
    rows_B.load(tokens(0), a.N);
    rows_C.load(tokens(0), a.N);
    float bias[VW], skip[VW];      // of the thread's vectors
    float dD[VW], dbias[VW];       // and their sums
    load_channels(bias, a.delta_bias, d0 + raw.ch, raw.in);
    load_channels(skip, a.D, d0 + raw.ch, raw.in);
#pragma unroll
    for (int v = 0; v < VW; ++v) dD[v] = dbias[v] = 0.0f;
    int64_t out = (b * a.length + end * kTile + raw.t) * a.dim + d0 + raw.ch;
    float* row_out = a.rows + ((int64_t)ct * a.batch * a.length + b * a.length + end * kTile) * 2 * a.N;
    for (int i = 0; i <= count; ++i) {
      if (i < count) {
        const int left = tokens(i), buffer = i & 1;
        raw.land(buffer, left);
        if constexpr (!R::kAsync) raw.fetch(buffer ^ 1, tokens(i + 1));
#pragma unroll 1
        for (int k = 0; k < R::kMine; ++k) {
          if (!raw.has) break;
          const bool on = raw.on(k, left);
          float x[VW], dt[VW], e[VW], z[VW];
          raw.read(x, buffer, 0, k);
          raw.read(dt, buffer, 1, k);
          if (a.dy.p) raw.read(e, buffer, 2, k);
          if (GATED) raw.read(z, buffer, GATED ? 3 : 0, k);
          float* to = in_of(i) + (raw.t + k * R::kTurn) * L::kChannels + raw.ch;
#pragma unroll
          for (int v = 0; v < VW; ++v) {
            if (!a.dy.p) e[v] = 0.0f;
            if (GATED) e[v] *= z[v] * sigmoid(z[v]);
            dt[v] = on ? softplus(dt[v] + bias[v]) : 0.0f;
            x[v] *= dt[v];
          }
          store_floats(to, dt);
          store_floats(to + M::kPlane, x);
          store_floats(to + 2 * M::kPlane, e);
        }
        rows_B.put(B_of(i));
        rows_C.put(B_of(i) + kTile * L::NP);
        tile_arrive(kFull + (i & 1), kAll);
        rows_B.load(tokens(i + 1), a.N);
        rows_C.load(tokens(i + 1), a.N);
      }
      if (i > 0) {
        tile_sync(kDone + ((i - 1) & 1), kAll);
        const int left = tokens(i - 1), buffer = (i - 1) & 1;
        // dB and dC over the warps
        for (int o = me; o < kTile * L::NP / 2; o += kHelpers) {
          const int t = o / (L::NP / 2), n = o % (L::NP / 2) * 4;  // four at a time
          const float* p = s_rows + t * 2 * L::NP + n;
          float4 s = *reinterpret_cast<const float4*>(p);
#pragma unroll
          for (int w = 1; w < L::kWarps; ++w) {
            const float4 q = *reinterpret_cast<const float4*>(p + w * kTile * 2 * L::NP);
            s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
          }
          const int what = n / L::NP, first = n % L::NP;
          float* to = row_out + t * 2 * a.N + what * a.N + first;
          if (t < left) {
            if (first < a.N) to[0] = s.x;
            if (first + 1 < a.N) to[1] = s.y;
            if (first + 2 < a.N) to[2] = s.z;
            if (first + 3 < a.N) to[3] = s.w;
          }
        }
        row_out -= kTile * 2 * a.N;
        if (i < count) tile_arrive(kRowsFree, kAll);
#pragma unroll 1
        for (int k = 0; k < R::kMine; ++k) {
          if (!raw.on(k, left)) break;
          const float* from = in_of(i - 1) + (raw.t + k * R::kTurn) * L::kChannels + raw.ch;
          const int64_t to = out + k * R::kTurn * a.dim;
          float x[VW], d[VW], dx[VW], e[VW], z[VW], dz[VW], through[VW], rate[VW];
          load_floats(dx, from);  // dt
          load_floats(through, from + M::kPlane);
          load_floats(rate, from + 2 * M::kPlane);
          if (GATED) load_floats(dz, from + (GATED ? 3 : 0) * M::kPlane);  // inner - D x
          raw.read(x, buffer, 0, k);
          raw.read(d, buffer, 1, k);
          if (a.dy.p) raw.read(e, buffer, 2, k);
          if (GATED) raw.read(z, buffer, GATED ? 3 : 0, k);
#pragma unroll
          for (int v = 0; v < VW; ++v) {
            if (!a.dy.p) e[v] = 0.0f;
            if (GATED) {
              const float s = sigmoid(z[v]);
              dz[v] = e[v] * fmaf(skip[v], x[v], dz[v]) * fmaf(z[v] * s, 1.0f - s, s);
              e[v] *= z[v] * s;
            }
            dx[v] = fmaf(dx[v], through[v], skip[v] * e[v]);
            const float ddt = fmaf(x[v], through[v], kLn2 * rate[v]);
            d[v] = ddt * sigmoid(d[v] + bias[v]);
            dD[v] = fmaf(e[v], x[v], dD[v]);
            dbias[v] += d[v];
          }
          store_from_f32<VW>(a.dx + to, dx);
          store_from_f32<VW>(a.ddelta + to, d);
          if (GATED) store_from_f32<VW>(a.dz + to, dz);
        }
        out -= kTile * a.dim;
      }
      if constexpr (R::kAsync) raw.fetch((i + 1) & 1, tokens(i + 1));  // where the tile just stored was
    }
    // dD and ddelta_bias over the threads with the same channels, where tile 0 or 1 was
    float* s = smem;
    sums += a.dim * a.N;
    tile_sync(kRowsFree + 1, kHelpers);
    if (raw.has) {
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        s[raw.t * L::kChannels + raw.ch + v] = dD[v];
        s[(R::kTurn + raw.t) * L::kChannels + raw.ch + v] = dbias[v];
      }
    }
    tile_sync(kRowsFree + 1, kHelpers);
    for (int o = me; o < 2 * L::kChannels; o += kHelpers) {
      const int ch = o % L::kChannels, what = o / L::kChannels;
      float v = 0.0f;
      for (int k = 0; k < R::kTurn; ++k) v += s[(what * R::kTurn + k) * L::kChannels + ch];
      if (d0 + ch < a.dim) sums[what * a.dim + d0 + ch] = v;
    }
    pdl_launch_dependents();
    return;
  }

  if constexpr (Registers<L>::kDeal) take_registers<Registers<L>::kWalk, true>();
  const Place<L> at(d0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2* s_kept = reinterpret_cast<float2*>(s_rows + M::kRows);
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
  auto kept = [&](int j, int c, int i) -> float2& {
    return s_kept[((j * CPT + c) * P + i) * L::kThreads + threadIdx.x];
  };
  Starts ahead(a.starts, b, a.length, end);
  for (int tile = 0; tile < count; ++tile) {
    const unsigned int starts = ahead.bits(end - tile - 1);
    float2 h[CPT][P];  // the state before the tile; L2 is asked for the next one
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      at.load(h[c], a.carry, c, b * tiles + end - tile, a.dim, a.N);
      if (tile + 1 < count) at.ask(a.carry, c, b * tiles + end - tile - 1, a.dim, a.N);
    }
    float* s_in = in_of(tile) + at.ch;
    const float *s_B = B_of(tile), *s_C = s_B + kTile * L::NP;
    tile_sync(kFull + (tile & 1), kAll);
    by_fresh(starts, [&](auto some) {
      constexpr bool kSome = decltype(some)::value;
      // the operands of kBack tokens: all read before anything is stored, as the compiler
      // cannot tell the stores from them
      float2 in[kBack][CPT];
      float2 B[kBack][P];
      auto read = [&](int t) {
#pragma unroll
        for (int k = 0; k < kBack; ++k) {
          load_states<SPT>(B[k], s_B + (t + k) * L::NP + at.sl * SPT);
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            const float* p = s_in + (t + k) * L::kChannels + c * L::kLanes;
            in[k][c] = make_float2(p[0], p[M::kPlane]);
          }
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
      if (tile > 0) tile_sync(kRowsFree, kAll);
#pragma unroll 1
      for (int j = kParts - 1; j >= 0; --j) {
        float2 enters[CPT][P], decay[kBack][CPT][P], state[kBack][CPT][P], Cs[kBack][P];
        float es[kBack][CPT];
        read(j * kBack);
#pragma unroll
        for (int k = 0; k < kBack; ++k) {
          load_states<SPT>(Cs[k], s_C + (j * kBack + k) * L::NP + at.sl * SPT);
#pragma unroll
          for (int c = 0; c < CPT; ++c) es[k][c] = s_in[2 * M::kPlane + (j * kBack + k) * L::kChannels + c * L::kLanes];
        }
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
          const int t = j * kBack + back;
          float2 dB[P], dC[P], through[CPT], rate[CPT], inner[CPT];
          const bool start = kSome && ((starts >> t) & 1u);
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            const float2 dt2 = both(in[back][c].x), dtx2 = both(in[back][c].y), e2 = both(es[back][c]);
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
          float* to = s_in + t * L::kChannels;
          {
            using Sum = LaneSum<2 * CPT, L::kLanes, 32>;
            float v[2 * CPT];
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
              v[c] = through[c].x + through[c].y;
              v[CPT + c] = rate[c].x + rate[c].y;
            }
            int first = 0;
            Sum::run(v, lane, first);
            if (lane < Sum::kUsed) {  // dt x and e have been used
#pragma unroll
              for (int i = 0; i < Sum::kKept; ++i)
                to[(1 + (first + i) / CPT) * M::kPlane + (first + i) % CPT * L::kLanes] = v[i];
            }
          }
          if (GATED) {
            using Sum = LaneSum<CPT, L::kLanes, 32>;
            float v[CPT];
#pragma unroll
            for (int c = 0; c < CPT; ++c) v[c] = inner[c].x + inner[c].y;
            int first = 0;
            Sum::run(v, lane, first);
            if (lane < Sum::kUsed) {
#pragma unroll
              for (int i = 0; i < Sum::kKept; ++i)
                to[(GATED ? 3 : 0) * M::kPlane + (first + i) * L::kLanes] = v[i];
            }
          }
          {
            using Sum = LaneSum<2 * SPT, 1, L::kLanes>;
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
            if (at.cl < Sum::kUsed) {
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
    });
    tile_arrive(kDone + (tile & 1), kAll);
  }
  if (seg == 0) {
#pragma unroll
    for (int c = 0; c < CPT; ++c) at.store(mu[c], a.dh0, c, b, a.dim, a.N);
  }
#pragma unroll
  for (int c = 0; c < CPT; ++c) at.store(dA[c], sums, c, 0, a.dim, a.N);
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

template <typename T, int LPC, bool VEC, bool GATED>
static cudaError_t selective_bwd_one(const SelectiveArgs<T>& a, cudaStream_t s) {
  using L = Backward<LPC>;
  using M = BackwardShared<L, T, VEC ? 4 : 1, GATED>;
  static_assert(M::kBytes <= 227 * 1024, "a CTA's shared memory");
  static_assert(2 * M::R::kTurn * L::kChannels <= 2 * M::kIn, "dD and ddelta_bias fit");
  // those that take_registers counts on have to be there; threads may ask at once
  static std::atomic<int> known{0};
  int registers = known.load(std::memory_order_relaxed);
  if (registers == 0) {
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, selective_bwd_kernel<T, LPC, VEC, GATED>);
    if (e != cudaSuccess) return e;
    registers = attr.numRegs;
    known.store(registers, std::memory_order_relaxed);
  }
  if (Registers<L>::kDeal && registers != Registers<L>::kLaunch) return cudaErrorLaunchOutOfResources;
  return launch_scan(selective_bwd_kernel<T, LPC, VEC, GATED>,
                     (unsigned int)(a.batch * a.ctiles) * a.segments, L::kThreads + kHelpers, M::kBytes,
                     a.segments > 1, s, a);
}

template <typename T>
oxc_status selective_bwd_launch(const SelectiveArgs<T>& a, float* out_sums, T* dB, T* dC,
                                cudaStream_t s) {
  const bool vec = a.dim % 4 == 0 && seq_vec(a.x) && seq_vec(a.delta) && seq_vec(a.z) &&
                   seq_vec(a.dy) && aligned_to(a.dx, 4 * sizeof(T)) &&
                   aligned_to(a.ddelta, 4 * sizeof(T)) && aligned_to(a.dz, 4 * sizeof(T));
  cudaError_t err = cudaSuccess;
  if (a.segments > 1)
    err = by_state(a.N, [&](auto spt, auto lpc) {
      constexpr int SPT = decltype(spt)::value, LPC = decltype(lpc)::value;
      using L = Forward<SPT, LPC>;
      SelectiveArgs<T> m = a;
      m.map_ctiles = (unsigned int)((a.dim + L::kChannels - 1) / L::kChannels);
      return launch_scan(vec ? selective_bwd_map_kernel<T, SPT, LPC, true>
                             : selective_bwd_map_kernel<T, SPT, LPC, false>,
                         (unsigned int)a.batch * m.map_ctiles * (a.segments - 1), L::kThreads + kHelpers,
                         vec ? BackwardMapShared<L, T, 4>::kBytes : BackwardMapShared<L, T, 1>::kBytes,
                         false, s, m);
    });
  if (err != cudaSuccess) return cuda_fail(err, "oxc_selective_scan_bwd");
  err = by_lanes(a.N, [&](auto lpc) {
    constexpr int LPC = decltype(lpc)::value;
    if (a.z.p)
      return vec ? selective_bwd_one<T, LPC, true, true>(a, s) : selective_bwd_one<T, LPC, false, true>(a, s);
    return vec ? selective_bwd_one<T, LPC, true, false>(a, s) : selective_bwd_one<T, LPC, false, false>(a, s);
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
