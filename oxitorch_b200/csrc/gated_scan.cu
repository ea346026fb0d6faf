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
//
// Both kernels cut the sequence into chunks of 64 tokens and the channels into
// tiles, one CTA each.  h_t = a_t h_{t-1} + v_t is an affine map of the state
// and maps compose, so a CTA first reduces its chunk to one map per channel (A,
// H), publishes it, finds the state that enters the chunk, and then runs the
// recurrence from it on the values that it kept in registers: x and gate are
// read once.  The VJP's mu runs through the same A from the other end.
//
// The state that enters a chunk (Chain, below) is found by looking back, as in the
// published single-pass scans with decoupled look-back (Merrill and Garland, 2016),
// over two levels: chunks form groups of 8.  A chunk applies, one after the other,
// the maps of the chunks before it in its group to the state entering the group;
// that one in turn comes from the nearest group whose entering state is known and the
// group maps between.  So
// the number of dependent steps is length / 512, the reads per chunk are at
// most 7 maps and a few group words, and since every state is defined by one
// fixed sequence of operations -- whoever computes it, from however far back --
// the results do not depend on timing.
//
// Bound by HBM in f32: [4, 2048, 4096] 75 us forward (82% of the copy bandwidth), 125
// us VJP (82%).  At 16 bits half the bytes leave the waits for the chain and the
// issue of instructions in sight: 66 and 91 us (46%, 57%), and [1, 65537, 1024], 1025
// chunks in a row, 141 and 197 us (44%, 52%).
#include <algorithm>
#include <type_traits>

#include "pipeline.cuh"
#include "typed.cuh"

namespace oxc {

constexpr int kScanWarps = 8;
constexpr int kScanSteps = 8;                        // tokens per warp
constexpr int kScanChunk = kScanWarps * kScanSteps;  // tokens per CTA
constexpr int kScanGroup = 8;                        // chunks per group
constexpr int kScanCtas = 2;                         // resident per SM

// A [batch, length, dim] operand: the last dim dense, strides in elements.
template <typename T>
struct SeqView {
  const T* p;
  int64_t sb, st;
};

// a = sigmoid(g) and b = 1 - a for two channels, both relatively accurate: with e
// = exp(-|g|) the smaller of the two is e / (1 + e), and the larger 1 minus that,
// which rounds once (a reciprocal's error in an a close to 1 would grow with the
// hundreds of tokens that such a gate remembers).  e = 2^t exp(n - t ln 2) with n =
// -|g| and t = n log2(e) rounded; the second factor, the rounding's share, to first
// order.  Below -100 e is 0 anyway, so n stops there (and stays finite for infinite
// gates; max.NaN keeps a NaN).  Two channels at a time on the packed f32x2 pipe: at
// 16 bits the kernels are bound by the issue of instructions as much as by memory.
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float gate_arg(float g) {
  float n;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(n) : "f"(-fabsf(g)), "f"(-100.0f));
  return n;
}
__device__ __forceinline__ float ex2_approx(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float rcp_approx(float t) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ void gate_pair(float2 g, float2& a, float2& b) {
  const float2 n = make_float2(gate_arg(g.x), gate_arg(g.y));
  const float2 t = __fmul2_rn(n, f2(1.44269502f));
  float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
  e = __ffma2_rn(e, __ffma2_rn(t, f2(-0.693147181f), n), e);
  const float2 d = __fadd2_rn(e, f2(1.0f));
  const float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  const float2 q = __fmul2_rn(e, r), o = __ffma2_rn(q, f2(-1.0f), f2(1.0f));
  a = make_float2(g.x > 0.0f ? o.x : q.x, g.y > 0.0f ? o.y : q.y);
  b = make_float2(g.x > 0.0f ? q.x : o.x, g.y > 0.0f ? q.y : o.y);
}

// ---- maps of the state ---------------------------------------------------------------
//
// s -> A s + H, A a product of sigmoids and so never negative.  A = -0 marks a
// map that forgets its argument (a sequence starts inside): it is selected, not
// multiplied, and keeps its mark in compositions.
__device__ __forceinline__ bool forgets(float A) { return __float_as_uint(A) == 0x80000000u; }
// Sets the mark once a warp's tokens are composed: a NaN gate among them would have
// turned it into a NaN, and mu would reach the sequence before.
template <int P>
__device__ __forceinline__ void mark_forgets(float2 (&A)[P]) {
#pragma unroll
  for (int j = 0; j < P; ++j) A[j] = f2(-0.0f);
}
__device__ __forceinline__ float map_apply(float A, float H, float s) {
  return forgets(A) ? H : fmaf(A, s, H);
}
// (A, H) after (A1, H1); branch-free, as these run in long dependent chains
__device__ __forceinline__ void map_compose(float& A, float& H, float A1, float H1) {
  const bool f = forgets(A);
  H = f ? H : fmaf(A, H1, H);
  A = f || forgets(A1) ? -0.0f : A * A1;
}
// The composition of N maps in a column of shared memory (row stride in floats),
// the first applied first; all of them are read before the first is used.
template <int N, bool REVERSE>
__device__ __forceinline__ void map_compose_column(const float* a, const float* h, int stride,
                                                   float& A, float& H) {
  float va[N], vh[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    va[i] = a[(REVERSE ? N - 1 - i : i) * stride];
    vh[i] = h[(REVERSE ? N - 1 - i : i) * stride];
  }
  A = va[N - 1];
  H = vh[N - 1];
#pragma unroll
  for (int i = N - 2; i >= 0; --i) map_compose(A, H, va[i], vh[i]);
}
// Replaces h of the N maps by the argument each gets, starting from s.
template <int N, bool REVERSE>
__device__ __forceinline__ void map_arguments_column(const float* a, float* h, int stride, float s) {
  float va[N], vh[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    va[i] = a[(REVERSE ? N - 1 - i : i) * stride];
    vh[i] = h[(REVERSE ? N - 1 - i : i) * stride];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    h[(REVERSE ? N - 1 - i : i) * stride] = s;
    s = map_apply(va[i], vh[i], s);
  }
}

// ---- the state that enters a chunk -----------------------------------------------------
//
// Words of 64 bits, written once and read whole, so a word carries its own
// "ready": a map (A low, H high) is empty while A's bits are all ones (no A has
// them: a NaN is stored as 0x7fffffff), an entering state (tag low, state high)
// while the tag's are.  The caller's workspace is set to all ones before the
// launch.  Chunks are counted along the direction of the scan.
struct Chain {
  unsigned int* ticket;       // the next tile to hand out, less one
  unsigned long long* map;    // [chunks, batch * dim]
  unsigned long long* group;  // [groups, batch * dim] the map of a whole group
  unsigned long long* enter;  // [groups, batch * dim] the state entering it
  int64_t stride;             // batch * dim
};

__device__ __forceinline__ unsigned long long word_load(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void word_store(unsigned long long* p, float lo, float hi) {
  const unsigned long long v =
      ((unsigned long long)__float_as_uint(hi) << 32) | __float_as_uint(lo);
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ void map_store(unsigned long long* p, float A, float H) {
  word_store(p, A != A ? __uint_as_float(0x7fffffffu) : A, H);
}
__device__ __forceinline__ bool word_ready(unsigned long long w) {
  return (uint32_t)w != 0xffffffffu;
}
__device__ __forceinline__ float word_lo(unsigned long long w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ float word_hi(unsigned long long w) {
  return __uint_as_float((uint32_t)(w >> 32));
}

// Bounds a spin: false once kWaitCycles (some four seconds) have passed since the
// first call.  The SM's own clock: the global timer takes far longer to read.
constexpr long long kWaitCycles = 8000000000ll;
struct Patience {
  long long t0 = 0;
  __device__ __forceinline__ bool more() {
    const long long t = clock64();
    if (t0 == 0) t0 = t;
    if (t - t0 <= kWaitCycles) return true;
    atomicOr(&g_kernel_error, OXC_KERR_PIPELINE_TIMEOUT);
    return false;
  }
};

// The word at p once it is ready; a NaN map if that takes too long.
__device__ __forceinline__ unsigned long long word_wait(const unsigned long long* p,
                                                        unsigned long long w) {
  Patience patience;
  while (!word_ready(w)) {
    if (!patience.more()) return 0x7fffffff7fffffffull;
    w = word_load(p);
  }
  return w;
}

// The state entering group g >= 0 at channel offset `off`.
__device__ __forceinline__ float chain_enter_group(const Chain& c, int g, int64_t off,
                                                   float first) {
  constexpr int kBack = 4;
  Patience patience;
  if (g == 0) return first;
  const unsigned long long* pe = c.enter + g * c.stride + off;
  const unsigned long long* pm = c.group + (g - 1) * c.stride + off;
  for (;;) {
    unsigned long long e[kBack], m[kBack];
#pragma unroll
    for (int i = 0; i < kBack; ++i) {  // e[i]: entering g - i; m[i]: the group before it
      e[i] = g - i > 0 ? word_load(pe - i * c.stride) : 0ull;
      m[i] = g - i > 0 && i + 1 < kBack ? word_load(pm - i * c.stride) : 0ull;
    }
    int at = kBack;
#pragma unroll
    for (int i = kBack - 1; i >= 0; --i) {
      if (word_ready(e[i])) at = i;                         // nearest known state so far
      else if (at < kBack && !word_ready(m[i])) at = kBack;  // a map missing on the way
    }
    if (at < kBack) {
      float s = 0.0f;
#pragma unroll
      for (int i = kBack - 1; i >= 0; --i) {
        if (i == at) s = g - i > 0 ? word_hi(e[i]) : first;
        else if (i < at) s = map_apply(word_lo(m[i]), word_hi(m[i]), s);
      }
      return s;
    }
    if (!patience.more()) return __uint_as_float(0x7fffffffu);
  }
}

// The state entering chunk k comes together from two sets of threads, one thread
// per channel each:
// chain_maps, with the map (A, H) of chunk k, publishes what later chunks need
// and leaves the maps of the chunks before k in its group in `before` [kScanGroup -
// 1][channels], a column per channel;
// chain_enter publishes and returns the state entering the group.
// Applying the former to the latter, chain_state, gives the state.  Both are
// waits on other CTAs' words, hence side by side.
template <int CHANNELS>
__device__ __forceinline__ void chain_maps(const Chain& c, int k, int chunks, int64_t off,
                                           float A, float H, float2 (*before)[CHANNELS],
                                           int channel) {
  constexpr int kBatch = 8;  // maps in flight
  const int n = k % kScanGroup;
  const bool ends_group = n + 1 == kScanGroup;
  const unsigned long long* p = c.map + (k - n) * c.stride + off;
  if (k + 1 < chunks && !ends_group) map_store(c.map + k * c.stride + off, A, H);
#pragma unroll
  for (int j0 = 0; j0 < kScanGroup - 1; j0 += kBatch) {
    unsigned long long w[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      w[i] = j0 + i < n ? word_load(p + (j0 + i) * c.stride) : 0ull;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (j0 + i < n) {
        w[i] = word_wait(p + (j0 + i) * c.stride, w[i]);
        before[j0 + i][channel] = make_float2(word_lo(w[i]), word_hi(w[i]));
      }
    }
  }
  if (k + 1 < chunks && ends_group) {
    for (int j = n - 1; j >= 0; --j) map_compose(A, H, before[j][channel].x, before[j][channel].y);
    map_store(c.group + k / kScanGroup * c.stride + off, A, H);
  }
}

__device__ __forceinline__ float chain_enter(const Chain& c, int k, int chunks, int64_t off,
                                             float first) {
  const int g = k / kScanGroup;
  const float s = chain_enter_group(c, g, off, first);
  if (k % kScanGroup == 0 && g > 0 && k + 1 < chunks)
    word_store(c.enter + g * c.stride + off, 0.0f, s);
  return s;
}

template <int CHANNELS>
__device__ __forceinline__ float chain_state(int k, const float2 (*before)[CHANNELS],
                                             int channel, float s) {
  const int n = k % kScanGroup;
#pragma unroll
  for (int j = 0; j < kScanGroup - 1; ++j) {
    const float2 m = before[j][channel];  // (not written beyond n)
    s = j < n ? map_apply(m.x, m.y, s) : s;
  }
  return s;
}

// ---- tiles -------------------------------------------------------------------------------

struct Tile {
  int chunk, b, d0, rank;  // rank: the tile's place in the order; negative at the end
};

// Hands out tiles to persistent CTAs, in the order of the scan: every batch row
// and channel tile of a chunk before the next chunk, so whatever a tile waits
// for belongs to a tile handed out before it, and the earliest unfinished tile
// never waits.  The ticket for the next tile is drawn while the current one is
// written, not before: a CTA that held one while it still waited for its state
// delayed every later tile (238 us instead of 182 at [1, 65537, 1024] bf16).
// Without a chain (one chunk) the tiles are strided over the grid.  One thread
// draws, works out the coordinates and posts them.
struct Tiles {
  Tile* next;  // shared: the next tile, and the one a round of the grid after it
  unsigned int drawn, dtiles, per, tiles;
  int channels;

  __device__ __forceinline__ bool mine() const { return threadIdx.x == blockDim.x - 1; }
  __device__ __forceinline__ void draw(const Chain& c, unsigned int now) {
    if (mine()) drawn = c.ticket ? atomicAdd(c.ticket, 1u) + 1u : now + gridDim.x;
  }
  __device__ __forceinline__ void post() {
    if (mine()) {
      next[0] = at(drawn);
      next[1] = at(per < tiles ? drawn + gridDim.x : tiles);  // one chunk: none
    }
  }
  __device__ __forceinline__ Tile at(unsigned int rank) const {
    const unsigned int chunk = rank / per, rest = rank - chunk * per, b = rest / dtiles;
    return {(int)chunk, (int)b, (int)(rest - b * dtiles) * channels,
            rank < tiles ? (int)rank : -1};
  }
};

// Asks L2 for a tile's part of an operand.  The kernels do so for the tile a round of
// the grid ahead (someone's next one: each tile is asked for once) before they wait
// for the chain, which the loads from HBM would otherwise follow: f32 [4, 2048, 4096]
// 75 us instead of 81 and 122 instead of 135 in the VJP.  With a single chunk there
// is no wait to fill, and the VJP of bf16 [16, 64, 8192] took 27 us instead of 26.
template <int TOKENS, int CHANNELS, typename T>
__device__ __forceinline__ void ask_ahead(const SeqView<T>& v, const Tile& tile, int64_t length,
                                          int64_t dim) {
  constexpr int kPerLine = 128 / sizeof(T), kLines = CHANNELS / kPerLine;
  if (tile.rank < 0) return;
#pragma unroll
  for (int i = threadIdx.x; i < TOKENS * kLines; i += kScanWarps * 32) {
    const int64_t t = (int64_t)tile.chunk * TOKENS + i / kLines, d = tile.d0 + i % kLines * kPerLine;
    if (t < length && d < dim)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(v.p + tile.b * v.sb + t * v.st + d));
  }
}

// VW channels of one token as loaded.  VEC: consecutive ones, in one access; else
// 32 apart (lane l takes l, l + 32, ...).  load_some takes the first `live` of
// them and `fill` for the rest; its loads are predicated rather than branched
// around, so that all of a thread's loads are in flight before the first is used.
template <typename T, int VW, bool VEC>
struct Raw;

template <int VW, bool VEC>
struct __align__(VEC ? 4 * VW : 4) Raw<float, VW, VEC> {
  float v[VW];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (VEC) {
      load_as_f32<VW>(v, p);
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k) v[k] = ld_stream(p + 32 * k);
    }
  }
  __device__ __forceinline__ void load_some(const float* p, int live, float fill) {
#pragma unroll
    for (int k = 0; k < VW; ++k) v[k] = fill;
    if constexpr (VEC && VW == 4) {
      asm("{.reg .pred p; setp.gt.s32 p, %5, 0; @p ld.global.cs.v4.f32 {%0, %1, %2, %3}, [%4];}"
          : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]) : "l"(p), "r"(live));
    } else if constexpr (VEC) {
      static_assert(!VEC || VW == 2 || VW == 4, "vectors of 2 or 4 channels");
      asm("{.reg .pred p; setp.gt.s32 p, %3, 0; @p ld.global.cs.v2.f32 {%0, %1}, [%2];}"
          : "+f"(v[0]), "+f"(v[1]) : "l"(p), "r"(live));
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k)
        asm("{.reg .pred p; setp.gt.s32 p, %2, %3; @p ld.global.cs.f32 %0, [%1];}"
            : "+f"(v[k]) : "l"(p + 32 * k), "r"(live), "r"(k));
    }
  }
  __device__ __forceinline__ float2 pair(int j) const { return make_float2(v[2 * j], v[2 * j + 1]); }
};

template <int VW, bool VEC>
struct __align__(VEC ? 2 * VW : 4) Raw<bf16, VW, VEC> {
  uint32_t w[VEC ? VW / 2 : VW];  // two to a word, or one in the lower half
  __device__ __forceinline__ void load(const bf16* p) {
    if constexpr (VEC && VW == 4) {
      const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = t.x;
      w[1] = t.y;
    } else if constexpr (VEC) {
      w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k) w[k] = __ldcs(reinterpret_cast<const unsigned short*>(p + 32 * k));
    }
  }
  __device__ __forceinline__ void load_some(const bf16* p, int live, float fill) {
    const uint32_t u = __float_as_uint(fill);  // 0 or infinity: the lower half is 0
#pragma unroll
    for (int k = 0; k < (VEC ? VW / 2 : VW); ++k) w[k] = VEC ? u | (u >> 16) : u >> 16;
    if constexpr (VEC && VW == 4) {
      asm("{.reg .pred p; setp.gt.s32 p, %3, 0; @p ld.global.cs.v2.u32 {%0, %1}, [%2];}"
          : "+r"(w[0]), "+r"(w[1]) : "l"(p), "r"(live));
    } else if constexpr (VEC) {
      static_assert(!VEC || VW == 2 || VW == 4, "vectors of 2 or 4 channels");
      asm("{.reg .pred p; setp.gt.s32 p, %2, 0; @p ld.global.cs.u32 %0, [%1];}"
          : "+r"(w[0]) : "l"(p), "r"(live));
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k)
        asm("{.reg .pred p; setp.gt.s32 p, %2, %3; @p ld.global.cs.u16 %0, [%1];}"
            : "+r"(w[k]) : "l"(p + 32 * k), "r"(live), "r"(k));
    }
  }
  __device__ __forceinline__ float2 pair(int j) const {
    if constexpr (VEC) return make_float2(bf16_lo(w[j]), bf16_hi(w[j]));
    else return make_float2(bf16_lo(w[2 * j]), bf16_lo(w[2 * j + 1]));
  }
};

// A lane's channels of a tile.
template <typename T, int VW, bool VEC>
struct Lane {
  static constexpr int kChannels = 32 * VW;
  int64_t d;  // the first
  int live;   // how many exist
  __device__ __forceinline__ Lane(int64_t d0, int64_t dim) {
    const int lane = threadIdx.x & 31;
    d = VEC ? d0 + lane * VW : d0 + lane;
    live = 0;
#pragma unroll
    for (int k = 0; k < VW; ++k) live += d + (VEC ? k : 32 * k) < dim;
  }
  __device__ __forceinline__ int channel(int k) const {  // within the tile
    const int lane = threadIdx.x & 31;
    return VEC ? lane * VW + k : lane + 32 * k;
  }
  __device__ __forceinline__ void store(T* row, const float2 (&v)[VW / 2]) const {
    float f[VW];
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) { f[2 * j] = v[j].x; f[2 * j + 1] = v[j].y; }
    if constexpr (VEC) {
      if (live) store_from_f32<VW>(row + d, f);
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const float one[1] = {f[k]};
        if (k < live) store_from_f32<1>(row + d + 32 * k, one);
      }
    }
  }
  // this lane's entries of a [kChannels] row in shared memory
  __device__ __forceinline__ void put(float* row, const float2 (&v)[VW / 2]) const {
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) {
      if constexpr (VEC) {
        *reinterpret_cast<float2*>(row + channel(2 * j)) = v[j];
      } else {
        row[channel(2 * j)] = v[j].x;
        row[channel(2 * j + 1)] = v[j].y;
      }
    }
  }
  __device__ __forceinline__ void get(const float* row, float2 (&v)[VW / 2]) const {
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) {
      if constexpr (VEC) v[j] = *reinterpret_cast<const float2*>(row + channel(2 * j));
      else v[j] = make_float2(row[channel(2 * j)], row[channel(2 * j + 1)]);
    }
  }
};

// The warp's tokens at which a sequence starts, a bit each.
__device__ __forceinline__ unsigned int start_bits(const uint8_t* starts, int64_t row, int64_t t0,
                                                   int64_t length) {
  if (!starts) return 0u;
  const int lane = threadIdx.x & 31;
  const bool s = lane < kScanSteps && t0 + lane < length && starts[row * length + t0 + lane];
  return __ballot_sync(0xffffffffu, s);
}

// N pairs of a thread in shared memory.
template <int N>
struct __align__(8 * N > 16 ? 16 : 8 * N) Held {
  float2 v[N];
};

// Runs f(std::true_type) if any of the warp's tokens starts a sequence, else
// f(std::false_type), whose loops need no selects.
template <typename F>
__device__ __forceinline__ void by_fresh(unsigned int fresh, F f) {
  if (fresh) f(std::true_type{});
  else f(std::false_type{});
}

// A tile is one chunk, or two (HALVES): then the gates and values of the first
// half wait in shared memory and those of the second in registers, and the chain,
// whose waits a long sequence of few channels mostly consists of, is entered half
// as often.
// Tokens beyond the length are given an infinite gate and x = 0: a = 1, b = 0,
// the identity.  Only their loads and stores are left out.
template <typename T, int VW, bool VEC, int HALVES>
__global__ void __launch_bounds__(kScanWarps * 32, kScanCtas) scan_fwd_kernel(
    SeqView<T> x, SeqView<T> gate, const uint8_t* __restrict__ starts,
    const float* __restrict__ h0, T* __restrict__ h, float* __restrict__ last,
    float* __restrict__ carry, Chain chain, int64_t batch, int64_t length, int64_t dim,
    int tiles_long, unsigned int dtiles, unsigned int tiles) {
  using L = Lane<T, VW, VEC>;
  using R = Raw<T, VW, VEC>;
  constexpr int P = VW / 2, kMaps = HALVES * kScanWarps;
  __shared__ __align__(16) float mapA[kMaps][L::kChannels];
  __shared__ __align__(16) float mapH[kMaps][L::kChannels];
  __shared__ float2 before[kScanGroup - 1][L::kChannels];
  __shared__ float enter[L::kChannels];
  __shared__ __align__(16) Tile next[2];
  extern __shared__ __align__(16) unsigned char held_bytes[];
  auto* held = reinterpret_cast<Held<2 * P>*>(held_bytes) + threadIdx.x;
  Tiles order{next, blockIdx.x, dtiles, (unsigned int)batch * dtiles, tiles, L::kChannels};
  const int warp = threadIdx.x >> 5;
  const int64_t chunks = (length + kScanChunk - 1) / kScanChunk;
  if (chain.ticket) order.draw(chain, 0u);
  order.post();
  for (;;) {
    __syncthreads();  // `next` is posted, the maps of the tile before are read
    const Tile tile = next[0];
    if (tile.rank < 0) return;
    const L lane(tile.d0, dim);
    float2 a[kScanSteps][P], v[kScanSteps][P];
    unsigned int fresh[HALVES];
    int steps[HALVES];
    const int64_t tile_t0 = (int64_t)tile.chunk * (HALVES * kScanChunk) + warp * kScanSteps;
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      const int64_t t0 = tile_t0 + half * kScanChunk;
      steps[half] = (int)max((int64_t)0, min((int64_t)kScanSteps, length - t0));
      R rg[kScanSteps], rx[kScanSteps];
      const T* pg = gate.p + (int64_t)tile.b * gate.sb + t0 * gate.st + lane.d;
      const T* px = x.p + (int64_t)tile.b * x.sb + t0 * x.st + lane.d;
      if (steps[half] == kScanSteps && tile.d0 + L::kChannels <= dim) {
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i) {
          rg[i].load(pg);
          rx[i].load(px);
          pg += gate.st;
          px += x.st;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i) {
          const int live = i < steps[half] ? lane.live : 0;
          rg[i].load_some(pg, live, INFINITY);
          rx[i].load_some(px, live, 0.0f);
          pg += gate.st;
          px += x.st;
        }
      }
      fresh[half] = start_bits(starts, tile.b, t0, length);
      float2 A[P], H[P];
#pragma unroll
      for (int k = 0; k < P; ++k) { A[k] = f2(1.0f); H[k] = f2(0.0f); }
#pragma unroll
      for (int i = 0; i < kScanSteps; ++i)
#pragma unroll
        for (int k = 0; k < P; ++k) {
          float2 b;
          gate_pair(rg[i].pair(k), a[i][k], b);
          v[i][k] = __fmul2_rn(b, rx[i].pair(k));
        }
      by_fresh(fresh[half], [&](auto some) {
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i)
#pragma unroll
          for (int k = 0; k < P; ++k) {
            H[k] = __ffma2_rn(a[i][k], H[k], v[i][k]);
            A[k] = __fmul2_rn(A[k], a[i][k]);
            if (decltype(some)::value && ((fresh[half] >> i) & 1u)) H[k] = v[i][k];
          }
        if (decltype(some)::value) mark_forgets(A);
      });
      lane.put(mapA[half * kScanWarps + warp], A);
      lane.put(mapH[half * kScanWarps + warp], H);
      if (half + 1 < HALVES) {
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i) {
          Held<2 * P> keep;
#pragma unroll
          for (int k = 0; k < P; ++k) { keep.v[k] = a[i][k]; keep.v[P + k] = v[i][k]; }
          held[i * kScanWarps * 32] = keep;
        }
      }
    }
    Tile ahead = next[1];
    ask_ahead<HALVES * kScanChunk, L::kChannels>(gate, ahead, length, dim);
    ask_ahead<HALVES * kScanChunk, L::kChannels>(x, ahead, length, dim);
    __syncthreads();
    const int c = threadIdx.x % L::kChannels, part = threadIdx.x / L::kChannels;
    const bool mine = tile.d0 + c < dim;
    const int64_t off = tile.b * dim + tile.d0 + c;
    if (mine && part == 0 && tiles_long > 1) {
      float tA, tH;
      map_compose_column<kMaps, false>(&mapA[0][c], &mapH[0][c], L::kChannels, tA, tH);
      chain_maps(chain, tile.chunk, tiles_long, off, tA, tH, before, c);
    } else if (mine && part == 1) {
      const float s = h0 ? h0[off] : 0.0f;
      enter[c] = tiles_long > 1 ? chain_enter(chain, tile.chunk, tiles_long, off, s) : s;
    }
    __syncthreads();
    if (mine && part == 0) {
      const float s = chain_state(tile.chunk, before, c, enter[c]);
      // mapH becomes the state entering each warp
      map_arguments_column<kMaps, false>(&mapA[0][c], &mapH[0][c], L::kChannels, s);
      if (carry) {
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          const int64_t k = (int64_t)tile.chunk * HALVES + half;
          if (k < chunks)
            carry[((int64_t)tile.b * chunks + k) * dim + tile.d0 + c] = mapH[half * kScanWarps][c];
        }
      }
    }
    __syncthreads();
    order.draw(chain, tile.rank);
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
      const int64_t t0 = tile_t0 + half * kScanChunk;
      float2 s[P];
      lane.get(mapH[half * kScanWarps + warp], s);
      by_fresh(fresh[half], [&](auto some) {
        T* ph = h + (tile.b * length + t0) * dim;
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i) {
          Held<2 * P> kept;
          if (half + 1 < HALVES) kept = held[i * kScanWarps * 32];
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const float2 ai = half + 1 < HALVES ? kept.v[k] : a[i][k];
            const float2 vi = half + 1 < HALVES ? kept.v[P + k] : v[i][k];
            s[k] = __ffma2_rn(ai, s[k], vi);
            if (decltype(some)::value && ((fresh[half] >> i) & 1u)) s[k] = vi;
          }
          if (i < steps[half]) lane.store(ph, s);
          ph += dim;
        }
      });
      if (last && steps[half] > 0 && t0 + steps[half] == length) {
#pragma unroll
        for (int k = 0; k < VW; ++k)
          if (k < lane.live)
            last[tile.b * dim + tile.d0 + lane.channel(k)] = k & 1 ? s[k / 2].y : s[k / 2].x;
      }
    }
    order.post();
  }
}

// 8 or 16 bytes to shared memory without passing the registers; zeros unless `on`.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool on) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(on ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(on ? 8 : 0) : "memory");
}

// With 4 channels a thread, x and dh are staged: copied to shared memory, each
// thread's own vectors, and read there where they are needed, which leaves the
// registers to the gates.
template <typename T, int VW, bool VEC>
__global__ void __launch_bounds__(kScanWarps * 32, kScanCtas) scan_bwd_kernel(
    SeqView<T> x, SeqView<T> gate, const uint8_t* __restrict__ starts,
    const float* __restrict__ carry, SeqView<T> dh, const float* __restrict__ dlast,
    T* __restrict__ dx, T* __restrict__ dgate, float* __restrict__ dh0, Chain chain, int64_t batch,
    int64_t length, int64_t dim, int chunks, unsigned int dtiles,
    unsigned int tiles) {
  using L = Lane<T, VW, VEC>;
  using R = Raw<T, VW, VEC>;
  constexpr int P = VW / 2, kThreads = kScanWarps * 32;
  constexpr bool kStaged = VW == 4;
  constexpr bool kGapStaged = kStaged && sizeof(T) == 4;  // h_{t-1} - x_t in the place of x_t
  static_assert(!kStaged || VEC, "vectors are staged");
  // per warp: its map's A, the state's H and mu's H; then the state entering it
  // from the left and the mu from the right
  __shared__ __align__(16) float mapA[kScanWarps][L::kChannels];
  __shared__ __align__(16) float mapS[kScanWarps][L::kChannels];
  __shared__ __align__(16) float mapM[kScanWarps][L::kChannels];
  __shared__ float2 before[kScanGroup - 1][L::kChannels];
  __shared__ float enter[L::kChannels];
  __shared__ __align__(16) Tile next[2];
  extern __shared__ __align__(16) unsigned char staged_bytes[];
  R* stage_x = reinterpret_cast<R*>(staged_bytes) + threadIdx.x;
  R* stage_d = stage_x + kScanSteps * kThreads;
  Tiles order{next, blockIdx.x, dtiles, (unsigned int)batch * dtiles, tiles, L::kChannels};
  const int warp = threadIdx.x >> 5;
  if (chain.ticket) order.draw(chain, 0u);
  order.post();
  for (;;) {
    __syncthreads();  // `next` is posted, the maps of the tile before are read
    Tile tile = next[0];
    if (tile.rank < 0) return;
    tile.chunk = chunks - 1 - tile.chunk;  // from the end of the sequence
    const L lane(tile.d0, dim);
    const int64_t t0 = (int64_t)tile.chunk * kScanChunk + warp * kScanSteps;
    const int64_t row0 = tile.b * length + t0;
    const int steps = (int)max((int64_t)0, min((int64_t)kScanSteps, length - t0));
    R rg[kScanSteps], rx[kStaged ? 1 : kScanSteps], rd[kStaged ? 1 : kScanSteps];
    if constexpr (kStaged) {
      const T* pg = gate.p + (int64_t)tile.b * gate.sb + t0 * gate.st + lane.d;
      const T* px = x.p + tile.b * x.sb + t0 * x.st + lane.d;
      const T* pd = dh.p + tile.b * dh.sb + t0 * dh.st + lane.d;
#pragma unroll
      for (int i = 0; i < kScanSteps; ++i) {
        const bool on = i < steps && lane.live;
        rg[i].load_some(pg, on, INFINITY);
        copy_async<sizeof(R)>(stage_x + i * kThreads, on ? px : x.p, on);
        copy_async<sizeof(R)>(stage_d + i * kThreads, on && dh.p ? pd : x.p, on && dh.p);
        pg += gate.st;
        pd += dh.st;
        px += x.st;
      }
    } else {
      const T* pg = gate.p + (int64_t)tile.b * gate.sb + t0 * gate.st + lane.d;
      const T* px = x.p + tile.b * x.sb + t0 * x.st + lane.d;
      const T* pd = dh.p + tile.b * dh.sb + t0 * dh.st + lane.d;
      const bool whole = steps == kScanSteps && tile.d0 + L::kChannels <= dim && dh.p;
      if (whole) {
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i) {
          rg[i].load(pg);
          rd[i].load(pd);
          rx[i].load(px);
          pg += gate.st;
          pd += dh.st;
          px += x.st;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kScanSteps; ++i) {
          const int live = i < steps ? lane.live : 0;
          rg[i].load_some(pg, live, INFINITY);
          rd[i].load_some(pd, dh.p ? live : 0, 0.0f);
          rx[i].load_some(px, live, 0.0f);
          pg += gate.st;
          pd += dh.st;
          px += x.st;
        }
      }
    }
    // the i-th token's x (then h_{t-1} - x) and dh
    auto get_x = [&](int i, float2 (&o)[P]) {
      const R* r;
      if constexpr (kStaged) r = stage_x + i * kThreads;
      else r = rx + i;
#pragma unroll
      for (int j = 0; j < P; ++j) o[j] = r->pair(j);
    };
    auto get_d = [&](int i, float2 (&o)[P]) {
      const R* r;
      if constexpr (kStaged) r = stage_d + i * kThreads;
      else r = rd + i;
#pragma unroll
      for (int j = 0; j < P; ++j) o[j] = r->pair(j);
    };
    const unsigned int fresh = start_bits(starts, tile.b, t0, length);
    float2 a[kScanSteps][P], b[kScanSteps][P], A[P], S[P], M[P];
#pragma unroll
    for (int j = 0; j < P; ++j) { A[j] = f2(1.0f); S[j] = M[j] = f2(0.0f); }
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) gate_pair(rg[i].pair(j), a[i][j], b[i][j]);
    if constexpr (kStaged) asm volatile("cp.async.wait_all;" ::: "memory");
    by_fresh(fresh, [&](auto some) {
#pragma unroll
      for (int i = 0; i < kScanSteps; ++i) {
        float2 xi[P];
        get_x(i, xi);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const float2 v = __fmul2_rn(b[i][j], xi[j]);
          S[j] = __ffma2_rn(a[i][j], S[j], v);
          A[j] = __fmul2_rn(A[j], a[i][j]);
          if (decltype(some)::value && ((fresh >> i) & 1u)) S[j] = v;
        }
      }
      if (decltype(some)::value) mark_forgets(A);
#pragma unroll
      for (int i = kScanSteps - 1; i >= 0; --i) {
        float2 di[P];
        get_d(i, di);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          M[j] = __fmul2_rn(a[i][j], __fadd2_rn(di[j], M[j]));
          if (decltype(some)::value && ((fresh >> i) & 1u)) M[j] = f2(0.0f);
        }
      }
    });
    lane.put(mapA[warp], A);
    lane.put(mapS[warp], S);
    lane.put(mapM[warp], M);
    Tile ahead = next[1];
    ahead.chunk = chunks - 1 - ahead.chunk;
    ask_ahead<kScanChunk, L::kChannels>(gate, ahead, length, dim);
    ask_ahead<kScanChunk, L::kChannels>(x, ahead, length, dim);
    if (dh.p) ask_ahead<kScanChunk, L::kChannels>(dh, ahead, length, dim);
    __syncthreads();
    // the mu of the chunk after this one (two sets of threads) and the state before
    // it (a third, or the second first)
    const int c = threadIdx.x % L::kChannels, part = threadIdx.x / L::kChannels;
    constexpr int kStatePart = kScanWarps * 32 >= 3 * L::kChannels ? 2 : 1;
    const bool mine = tile.d0 + c < dim;
    const int64_t off = tile.b * dim + tile.d0 + c;
    const int k = chunks - 1 - tile.chunk;
    if (mine && part == 0 && chunks > 1) {
      float tA, tM;
      map_compose_column<kScanWarps, true>(&mapA[0][c], &mapM[0][c], L::kChannels, tA, tM);
      chain_maps(chain, k, chunks, off, tA, tM, before, c);
    }
    if (mine && part == kStatePart)
      map_arguments_column<kScanWarps, false>(
          &mapA[0][c], &mapS[0][c], L::kChannels,
          carry[((int64_t)tile.b * chunks + tile.chunk) * dim + tile.d0 + c]);
    if (mine && part == 1) {
      const float m = dlast ? dlast[off] : 0.0f;
      enter[c] = chunks > 1 ? chain_enter(chain, k, chunks, off, m) : m;
    }
    __syncthreads();
    if (mine && part == 0) {
      const float m = chain_state(k, before, c, enter[c]);
      map_arguments_column<kScanWarps, true>(&mapA[0][c], &mapM[0][c], L::kChannels, m);
    }
    __syncthreads();
    order.draw(chain, tile.rank);
    float2 s[P], m[P], gap[kGapStaged ? 1 : kScanSteps][P];  // h_{t-1} - x_t, what d h_t / d a_t is
    lane.get(mapS[warp], s);
    lane.get(mapM[warp], m);
    by_fresh(fresh, [&](auto some) {
#pragma unroll
      for (int i = 0; i < kScanSteps; ++i) {
        float2 xi[P];
        get_x(i, xi);
        [[maybe_unused]] R g;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          if (decltype(some)::value && ((fresh >> i) & 1u)) s[j] = f2(0.0f);
          const float2 q = __fadd2_rn(s[j], make_float2(-xi[j].x, -xi[j].y));
          s[j] = __ffma2_rn(a[i][j], s[j], __fmul2_rn(b[i][j], xi[j]));
          if constexpr (kGapStaged) g.v[2 * j] = q.x, g.v[2 * j + 1] = q.y;
          else gap[i][j] = q;
        }
        if constexpr (kGapStaged) stage_x[i * kThreads] = g;
      }
      T* px = dx + (row0 + kScanSteps - 1) * dim;
      T* pg = dgate + (row0 + kScanSteps - 1) * dim;
#pragma unroll
      for (int i = kScanSteps - 1; i >= 0; --i) {
        float2 ox[P], og[P], gi[P], di[P];
        if constexpr (kGapStaged) {
          get_x(i, gi);
        } else {
#pragma unroll
          for (int j = 0; j < P; ++j) gi[j] = gap[i][j];
        }
        get_d(i, di);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const float2 l = __fadd2_rn(di[j], m[j]);
          ox[j] = __fmul2_rn(l, b[i][j]);
          m[j] = __fmul2_rn(a[i][j], l);
          og[j] = __fmul2_rn(__fmul2_rn(m[j], b[i][j]), gi[j]);
          if (decltype(some)::value && ((fresh >> i) & 1u)) m[j] = f2(0.0f);
        }
        if (i < steps) {
          lane.store(px, ox);
          lane.store(pg, og);
        }
        px -= dim;
        pg -= dim;
      }
    });
    if (dh0 && tile.chunk == 0 && warp == 0) {
#pragma unroll
      for (int k = 0; k < VW; ++k)
        if (k < lane.live)
          dh0[tile.b * dim + tile.d0 + lane.channel(k)] = k & 1 ? m[k / 2].y : m[k / 2].x;
    }
    order.post();
  }
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
  float2 a, b;
  gate_pair(f2(to_f32(gate[bi * gate_stride + d])), a, b);
  const float s = fmaf(a.x, state[bi * dim + d], b.x * to_f32(x[bi * x_stride + d]));
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
  if (dim > 0x7fffffff - 1024)  // a tile's channels are counted in int, past the last one
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: %s: %lld channels", fn, (long long)dim);
  return OXC_OK;
}

static int64_t scan_chunks(int64_t length) { return (length + kScanChunk - 1) / kScanChunk; }
static int64_t scan_groups(int64_t length) {
  return (scan_chunks(length) + kScanGroup - 1) / kScanGroup;
}

// Lays the chain out in the workspace and empties it; a single chunk has none.
static oxc_status scan_chain(const char* fn, int64_t batch, int64_t length, int64_t dim, int halves,
                             void* workspace, size_t workspace_bytes, cudaStream_t s, Chain* c) {
  const size_t size = oxc_gated_scan_workspace_size(batch, length, dim);
  const int64_t tiles = (scan_chunks(length) + halves - 1) / halves;
  const int64_t groups = (tiles + kScanGroup - 1) / kScanGroup;
  *c = Chain{nullptr, nullptr, nullptr, nullptr, batch * dim};
  if (size && (!workspace || workspace_bytes < size || !aligned16(workspace)))
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: %s needs a 16-byte aligned %zu-byte workspace, got %zu", fn,
                size, workspace_bytes);
  if (tiles == 1) return OXC_OK;
  const size_t need = 16 + (size_t)((tiles + 2 * groups) * c->stride) * sizeof(unsigned long long);
  c->ticket = static_cast<unsigned int*>(workspace);
  c->map = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + 16);
  c->group = c->map + tiles * c->stride;
  c->enter = c->group + groups * c->stride;
  const cudaError_t e = cudaMemsetAsync(workspace, 0xff, need, s);
  return e == cudaSuccess ? OXC_OK : cuda_fail(e, fn);
}

// VW channels of an operand in one access.
template <typename T, int VW>
static bool seq_vec(const void* p, int64_t sb, int64_t st, int64_t dim) {
  return dim % VW == 0 && sb % VW == 0 && st % VW == 0 && aligned_to(p, VW * sizeof(T));
}

// Tiles of the tensor with `halves` chunks each, or -1 if they cannot be counted.
static int64_t scan_tiles(int64_t batch, int64_t length, int64_t dim, int channels, int halves) {
  const int64_t per = batch * ((dim + channels - 1) / channels);
  const int64_t along = (scan_chunks(length) + halves - 1) / halves;
  return along > 0x7fffffff / per ? -1 : along * per;
}

// A grid that is resident at once.
static unsigned scan_grid(const void* kernel, int64_t tiles, size_t smem) {
  return (unsigned)std::min<int64_t>(tiles, (int64_t)sm_count() * occupancy(kernel, kScanWarps * 32, smem));
}

template <typename T, int VW, int HALVES>
static oxc_status scan_fwd_launch(const void* x, int64_t x_sb, int64_t x_st, const void* gate,
                                  int64_t g_sb, int64_t g_st, const uint8_t* starts,
                                  const float* h0, void* h, float* last, float* carry,
                                  int64_t batch, int64_t length, int64_t dim, void* workspace,
                                  size_t workspace_bytes, cudaStream_t s) {
  const int64_t tiles = scan_tiles(batch, length, dim, 32 * VW, HALVES);
  if (tiles < 0)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: gated_scan: [%lld, %lld, %lld]",
                (long long)batch, (long long)length, (long long)dim);
  Chain chain;
  oxc_status st = scan_chain("gated_scan", batch, length, dim, HALVES, workspace, workspace_bytes,
                             s, &chain);
  if (st) return st;
  const bool vec = seq_vec<T, VW>(x, x_sb, x_st, dim) && seq_vec<T, VW>(gate, g_sb, g_st, dim) &&
                   seq_vec<T, VW>(h, 0, 0, dim);
  auto kernel = vec ? scan_fwd_kernel<T, VW, true, HALVES> : scan_fwd_kernel<T, VW, false, HALVES>;
  const size_t smem = (HALVES - 1) * (size_t)kScanSteps * kScanWarps * 32 * 2 * VW * sizeof(float);
  if (smem) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_gated_scan_fwd");
  }
  const int64_t dtiles = (dim + 32 * VW - 1) / (32 * VW);
  const SeqView<T> xv{static_cast<const T*>(x), x_sb, x_st};
  const SeqView<T> gv{static_cast<const T*>(gate), g_sb, g_st};
  kernel<<<scan_grid((const void*)kernel, tiles, smem), kScanWarps * 32, smem, s>>>(
      xv, gv, starts, h0, static_cast<T*>(h), last, carry, chain, batch, length, dim,
      (int)(tiles / (batch * dtiles)), (unsigned)dtiles, (unsigned)tiles);
  return check_launch("oxc_gated_scan_fwd");
}

template <typename T, int VW>
static oxc_status scan_bwd_launch(const void* x, int64_t x_sb, int64_t x_st, const void* gate,
                                  int64_t g_sb, int64_t g_st, const uint8_t* starts,
                                  const float* carry, const void* dh, int64_t dh_sb, int64_t dh_st,
                                  const float* dlast, void* dx, void* dgate, float* dh0,
                                  int64_t batch, int64_t length, int64_t dim, void* workspace,
                                  size_t workspace_bytes, cudaStream_t s) {
  const int64_t tiles = scan_tiles(batch, length, dim, 32 * VW, 1);
  if (tiles < 0)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: gated_scan backward: [%lld, %lld, %lld]",
                (long long)batch, (long long)length, (long long)dim);
  Chain chain;
  oxc_status st = scan_chain("gated_scan backward", batch, length, dim, 1, workspace,
                             workspace_bytes, s, &chain);
  if (st) return st;
  const bool vec = seq_vec<T, VW>(x, x_sb, x_st, dim) && seq_vec<T, VW>(gate, g_sb, g_st, dim) &&
                   seq_vec<T, VW>(dh, dh_sb, dh_st, dim) && seq_vec<T, VW>(dx, 0, 0, dim) &&
                   seq_vec<T, VW>(dgate, 0, 0, dim);
  auto kernel = scan_bwd_kernel<T, VW, true>;
  if constexpr (VW == 2)
    kernel = vec ? kernel : scan_bwd_kernel<T, VW, false>;
  else if (!vec)
    return fail(OXC_ERR_OTHER, "internal: gated_scan backward: operands not aligned");
  const size_t smem = VW == 4 ? 2 * kScanSteps * kScanWarps * 32 * VW * sizeof(T) : 0;
  if (smem) {
    const cudaError_t e = cudaFuncSetAttribute(
        (const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_gated_scan_bwd");
  }
  const int64_t dtiles = (dim + 32 * VW - 1) / (32 * VW);
  const SeqView<T> xv{static_cast<const T*>(x), x_sb, x_st};
  const SeqView<T> gv{static_cast<const T*>(gate), g_sb, g_st};
  const SeqView<T> dv{static_cast<const T*>(dh), dh_sb, dh_st};
  kernel<<<scan_grid((const void*)kernel, tiles, smem), kScanWarps * 32, smem, s>>>(
      xv, gv, starts, carry, dv, dlast, static_cast<T*>(dx), static_cast<T*>(dgate), dh0, chain,
      batch, length, dim, (int)(tiles / (batch * dtiles)), (unsigned)dtiles, (unsigned)tiles);
  return check_launch("oxc_gated_scan_bwd");
}

}  // namespace oxc

using namespace oxc;

extern "C" {

int64_t oxc_gated_scan_carry_size(int64_t batch, int64_t length, int64_t dim) {
  if (batch <= 0 || length <= 0 || dim <= 0) return 0;
  return batch * scan_chunks(length) * dim;
}

// The same for both directions: a ticket, a map per chunk and channel, a map and
// a state per group.
size_t oxc_gated_scan_workspace_size(int64_t batch, int64_t length, int64_t dim) {
  if (batch <= 0 || length <= kScanChunk || dim <= 0) return 0;
  return 16 + (size_t)(scan_chunks(length) + 2 * scan_groups(length)) * (size_t)batch *
                  (size_t)dim * sizeof(unsigned long long);
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
  // 4 channels a thread, half as many where a tile would be wider than the tensor.
  // Tiles of two chunks where few channels leave many chunks of one chain in flight
  // (bf16 [1, 65537, 1024]: 141 us instead of 160; with 128 tiles side by side, f32
  // [4, 2048, 4096], 81 against 75), if there are several tiles for each CTA.
  const bool narrow = dim <= 64;
  const int channels = narrow ? 64 : 128;
  const bool two = batch * ((dim + channels - 1) / channels) * 8 <= sm_count() &&
                   scan_tiles(batch, length, dim, channels, 2) >= 4 * (int64_t)sm_count();
  auto launch = dtype == OXC_BF16
                    ? (narrow ? (two ? scan_fwd_launch<bf16, 2, 2> : scan_fwd_launch<bf16, 2, 1>)
                              : (two ? scan_fwd_launch<bf16, 4, 2> : scan_fwd_launch<bf16, 4, 1>))
                    : (narrow ? (two ? scan_fwd_launch<float, 2, 2> : scan_fwd_launch<float, 2, 1>)
                              : (two ? scan_fwd_launch<float, 4, 2> : scan_fwd_launch<float, 4, 1>));
  return launch(x, x_sb, x_st, gate, g_sb, g_st, starts, h0, h, last, carry, batch, length, dim,
                workspace, workspace_bytes, s);
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
  // 2 channels a thread; 4, with x and dh staged, where vectors can be read: wider
  // tiles, so fewer entries to the chain, and less of the addressing.  At [4, 2048,
  // 4096] 94 us instead of 117 in bf16 and 135 instead of 143 in f32; in f32 not with
  // a single chunk, which enters no chain ([16, 64, 8192]: 40 us against 34).
  auto vec4 = [&](const void* p, int64_t sb, int64_t st) {
    return dtype == OXC_BF16 ? seq_vec<bf16, 4>(p, sb, st, dim) : seq_vec<float, 4>(p, sb, st, dim);
  };
  const bool wide = dim > 64 && vec4(x, x_sb, x_st) && vec4(gate, g_sb, g_st) &&
                    vec4(dh, dh_sb, dh_st) && vec4(dx, 0, 0) && vec4(dgate, 0, 0) &&
                    (dtype == OXC_BF16 || length > kScanChunk);
  auto launch = dtype == OXC_BF16
                    ? (wide ? scan_bwd_launch<bf16, 4> : scan_bwd_launch<bf16, 2>)
                    : (wide ? scan_bwd_launch<float, 4> : scan_bwd_launch<float, 2>);
  return launch(x, x_sb, x_st, gate, g_sb, g_st, starts, carry, dh, dh_sb, dh_st, dlast, dx, dgate,
                dh0, batch, length, dim, workspace, workspace_bytes, s);
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
