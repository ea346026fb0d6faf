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
//
// Bound by HBM: 2 sizeof(T) bytes a logit, the row read once and its gradient
// written once.  So a row stays in shared memory between the two, shared by a
// cluster of 1 to 8 CTAs that exchange (max, sum) pairs through distributed shared
// memory.  Rows wider than a cluster holds (1.25 MB; 1.13 MB beside the 80 KB of 4096
// entries) take the three-pass kernel, which re-reads them from L2 or HBM.  Measured,
// of the copy bandwidth: f32 [4096, 131072] 701 us (94%), [8192, 32000] 364 (88%); bf16
// [8192, 32000] 204 (78%), [8192, 131072] 863 (76%), where the issue of instructions
// and the exponentials are as busy as the memory.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "pipeline.cuh"
#include "typed.cuh"

namespace oxc {

constexpr int kDistillMaxTop = 4096;
constexpr int kDistillThreads = 256;          // per CTA at most
constexpr int kDistillCopies = 4;             // bulk copies per part of a row
constexpr int kDistillPart = 100 * 1024;      // bytes of a row per CTA, if a cluster can
constexpr int kDistillMaxPart = 160 * 1024;   // and at most
constexpr int kDistillSmem = 225 * 1024;      // a part and the teacher's side: the 227 KB
                                              // that a CTA can have, less the kernel's own
constexpr int kDistillCluster = OXC_DISTILL_PARTS;  // CTAs per row at most

// Records the first bad id: flag[0] = 2 (dim 1), flag[1..2] = id, flag[3] = vocab.
__device__ __forceinline__ void record_bad_id(int32_t* flag, int64_t id, int64_t vocab) {
  if (flag && atomicCAS(flag, 0, 2) == 0) {
    flag[1] = (int32_t)(uint32_t)((uint64_t)id & 0xffffffffu);
    flag[2] = (int32_t)(uint32_t)((uint64_t)id >> 32);
    flag[3] = (int32_t)vocab;
  }
}

__device__ __forceinline__ float ex2_approx(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float rcp_approx(float t) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// exp(d / tau) for d = x - max <= 0, c = log2(e) / tau.  The subtraction comes
// first, so the large terms see only ex2's own error; results below 2^-126 are 0.
__device__ __forceinline__ float exp_scaled(float d, float c) { return ex2_approx(d * c); }

// Maximum over the warp, NaN ignored.
__device__ __forceinline__ float warp_max_fast(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The teacher's side of a row, in shared memory: its logits, then probabilities,
// and ids (negative for entries that do not count).
struct Teacher {
  float* prob;
  int* id;
  int* table;  // hash of the ids, 2^bits entries
  int bits;
};

__host__ __device__ inline int teacher_bits(int top) {
  int b = 5;
  while ((1 << b) < 2 * top) ++b;
  return b;
}
__host__ __device__ inline size_t teacher_smem(int top) {
  return (size_t)top * 12 + (sizeof(int) << teacher_bits(top));
}

struct TeacherRow {
  float log_sum;  // of exp((t - max) / tau)
  float max;
  bool none, bad, repeated;
};

// Fills the teacher's side of one row; every thread gets the summary.
__device__ __forceinline__ TeacherRow teacher_row(const Teacher& s, const float* tl,
                                                  const int64_t* ti, int top, float c, int vocab,
                                                  int32_t* err, float* scratch) {
  TeacherRow r;
  for (int i = threadIdx.x; i < (1 << s.bits); i += blockDim.x) s.table[i] = -1;
  float tm = -INFINITY;
  int bad = 0;
  for (int k = threadIdx.x; k < top; k += blockDim.x) {
    const int64_t id = ti[k];
    const float v = id >= 0 ? tl[k] : -INFINITY;
    if (id >= vocab) { record_bad_id(err, id, vocab); bad = 1; }
    if (v != v) bad = 1;
    s.id[k] = id >= 0 && id < vocab && v != -INFINITY ? (int)id : -1;
    s.prob[k] = v;
    tm = fmaxf(tm, v);
  }
  r.bad = __syncthreads_or(bad);
  tm = block_max(tm, scratch);
  r.max = tm;
  r.none = tm == -INFINITY && !r.bad;
  r.repeated = false;
  r.log_sum = 0.0f;
  if (r.none || r.bad) return r;
  float ts = 0.0f;
  int twice = 0;
  for (int k = threadIdx.x; k < top; k += blockDim.x) {
    const float e = exp_scaled(s.prob[k] - tm, c);
    s.prob[k] = e;
    ts += e;
    const int id = s.id[k];
    if (id >= 0) {  // insert; finding the id there already means it is listed twice
      unsigned int h = ((unsigned int)id * 2654435769u) >> (32 - s.bits);
      for (int n = 0; n < (1 << s.bits); ++n) {
        const int was = atomicCAS(&s.table[h], -1, id);
        if (was == -1) break;
        if (was == id) { twice = 1; break; }
        h = (h + 1) & ((1u << s.bits) - 1);
      }
    }
  }
  ts = block_sum(ts, scratch);
  r.repeated = __syncthreads_or(twice);
  r.log_sum = logf(ts);
  const float inv = __fdiv_rn(1.0f, ts);
  for (int k = threadIdx.x; k < top; k += blockDim.x) s.prob[k] *= inv;
  __syncthreads();
  return r;
}

// The probability that all entries of s.id[k]'s token have together, 0 if an
// earlier entry is that token's; in the order of the entries.
__device__ __forceinline__ float teacher_prob(const Teacher& s, bool repeated, int k, int top,
                                              bool* first) {
  *first = true;
  if (!repeated) return s.prob[k];
  float p = 0.0f;
  for (int j = 0; j < top; ++j) {
    if (s.id[j] != s.id[k]) continue;
    if (j < k) *first = false;
    p += s.prob[j];
  }
  return p;
}

struct DistillArgs {
  const float* tl;
  const int64_t* ti;
  int top;
  float inv_tau, c;   // c = log2(e) / tau
  float grad_scale;   // tau / total_rows
  const float* grad_loss;
  float* row_loss;
  int64_t rows;
  int vocab;
  int32_t* err;
};

// (max, sum of exponentials relative to it) of two sets; -inf with 0 is the empty
// one.  A sum that is not 0 beside a maximum of -inf is NaN and stays.
__device__ __forceinline__ float2 pair_merge(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x);
  const float sa = a.x == m ? a.y : a.y * exp_scaled(a.x - m, c);
  const float sb = b.x == m ? b.y : b.y * exp_scaled(b.x - m, c);
  return make_float2(m, sa + sb);
}
__device__ __forceinline__ float2 warp_merge(float2 v, float c) {
  const float m = warp_max_fast(v.x);
  return make_float2(m, warp_sum(m == -INFINITY ? v.y : v.y * exp_scaled(v.x - m, c)));
}

// A row's bytes are cut at 16-byte boundaries of memory: `body` whole vectors,
// CTA r of the cluster taking the r-th share of them, thread t the vectors t,
// t + THREADS, ... of it; the elements before the first boundary and after the
// last (fewer than a vector each) are single elements of the last CTA's warp 0.
template <typename T>
struct RowCut {
  static constexpr int kVec = 16 / (int)sizeof(T);
  const T* row;
  int head, body, v0, v1;
  __device__ __forceinline__ RowCut(const T* row, int vocab, int rank, int log_size) : row(row) {
    head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
    body = (vocab - head) / kVec;
    const int each = (body + (1 << log_size) - 1) >> log_size;
    v0 = min(body, rank * each);
    v1 = min(body, v0 + each);
  }
  __device__ __forceinline__ const T* part() const { return row + head + (int64_t)v0 * kVec; }
};

// The elements of a 16-byte vector, in pairs.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float2 (&v)[8 / (int)sizeof(T)]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
    if constexpr (sizeof(T) == 4)
      v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else
      v[i] = make_float2(bf16_lo(w[i]), bf16_hi(w[i]));
  }
}

// Folds V vectors of logits into a running (max, sum of exponentials): the maximum
// of all first (of bf16, two at a time), a rescale of the sum when it grows, then
// the terms.
template <typename T, int V>
__device__ __forceinline__ void pair_fold(float2& p, const uint4 (&q)[V], float c) {
  constexpr int kPairs = 8 / (int)sizeof(T);
  float m = p.x;
  if constexpr (sizeof(T) == 2) {
    __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&q[0].x);
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) h = __hmax2(h, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    }
    m = fmaxf(m, fmaxf(__low2float(h), __high2float(h)));
  } else {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      m = fmaxf(m, fmaxf(__uint_as_float(q[u].x), __uint_as_float(q[u].y)));
      m = fmaxf(m, fmaxf(__uint_as_float(q[u].z), __uint_as_float(q[u].w)));
    }
  }
  if (m > p.x) {
    p.y *= exp_scaled(p.x - m, c);
    p.x = m;
  }
  const float base = m == -INFINITY ? 0.0f : -m;
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < V; ++u) {
    float2 v[kPairs];
    unpack<T>(q[u], v);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 d = __fmul2_rn(__fadd2_rn(v[i], make_float2(base, base)), make_float2(c, c));
      s = __fadd2_rn(s, make_float2(ex2_approx(d.x), ex2_approx(d.y)));
    }
  }
  p.y += s.x + s.y;
}

// Sends v to `to` in CTA `rank` of the cluster, completing 8 bytes on its `bar`.
__device__ __forceinline__ void send_pair(const float2* to, uint64_t* bar, int rank, float2 v) {
  uint32_t dst, rbar;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(to)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rbar) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
               ::"r"(dst), "f"(v.x), "f"(v.y), "r"(rbar) : "memory");
}

// Persistent clusters, a row at a time.  A CTA's part of the row arrives in
// shared memory by bulk copies; one pass over it makes the (max, sum) pair, a
// second the gradient, and then the copies of the next row's part are started,
// whose bytes L2 was asked for when the second pass began.  The teacher's side of
// a row is worked out while its logits are on the way.  The warps of a row meet
// twice: each reduces its logits to a (max, sum) pair and sends it to every CTA of
// the cluster (a cluster barrier would also wait for the gradient's stores of the
// row before); a barrier within the CTA precedes the corrections at the teacher's
// tokens.  Each CTA sums the loss over the tokens in its part:
// row_loss[row][rank].
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
distill_cluster_kernel(const T* __restrict__ logits, int64_t stride, T* __restrict__ dlogits,
                       DistillArgs a, int part_bytes) {
  namespace cg = cooperative_groups;
  using Cut = RowCut<T>;
  constexpr int kVec = Cut::kVec, kPairs = kVec / 2;
  constexpr int kWarps = THREADS / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  // by the parity of the row: a CTA that is a row ahead of another sends into the
  // set that the other is not reading
  __shared__ float2 student[2][kDistillCluster * kWarps];
  __shared__ uint64_t met[2];
  __shared__ float2 teacher[kWarps];
  __shared__ float partial[kWarps];
  __shared__ uint64_t full[kDistillCopies];
  cg::cluster_group cluster = cg::this_cluster();
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int log_size = 31 - __clz(size);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint4* buffer = reinterpret_cast<const uint4*>(smem);
  float* rest = reinterpret_cast<float*>(smem + part_bytes);
  const Teacher teach{rest, reinterpret_cast<int*>(rest) + a.top,
                      reinterpret_cast<int*>(rest) + 2 * a.top, teacher_bits(a.top)};
  float* logit_k = rest + 2 * a.top + (1 << teach.bits);  // the student's logit at id[k]
  const float gs = a.grad_loss ? a.grad_scale * __ldg(a.grad_loss) : a.grad_scale;
  const int64_t rows_apart = gridDim.x >> log_size;
  const int entry_warps = min(kWarps, (a.top + 31) / 32);  // warps with entries of the teacher

  // copy i of a part of n vectors: [i, i + 1) * copy_vecs(n) of them, whole rounds
  // of the threads
  auto copy_vecs = [](int n) {
    return (n + kDistillCopies * THREADS - 1) / (kDistillCopies * THREADS) * THREADS;
  };
  auto fetch = [&](int64_t row) {  // thread 0
    const Cut cut(logits + row * stride, a.vocab, rank, log_size);
    const int n = cut.v1 - cut.v0, each = copy_vecs(n);
#pragma unroll
    for (int i = 0; i < kDistillCopies; ++i) {
      const int from = i * each, bytes = 16 * (min(n, from + each) - from);
      if (bytes > 0) {
        mbar_arrive_expect_tx(&full[i], (uint32_t)bytes);
        bulk_g2s(smem + 16 * from, cut.part() + (int64_t)from * kVec, (uint32_t)bytes, &full[i]);
      } else {
        mbar_arrive(&full[i]);
      }
    }
  };
  int64_t row = blockIdx.x >> log_size;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < kDistillCopies; ++i) mbar_init(&full[i], 1);
    mbar_init(&met[0], 1);
    mbar_init(&met[1], 1);
    fence_barrier_init();
    if (row < a.rows) fetch(row);
  }
  if (size > 1) cluster.sync();  // nobody sends before the barriers are there
  else __syncthreads();
  // this thread's first entry of the teacher, a row ahead
  int64_t next_id = -1;
  float next_t = 0.0f;
  if ((int)threadIdx.x < a.top && row < a.rows) {
    next_id = __ldcs(a.ti + row * a.top + threadIdx.x);
    next_t = __ldcs(a.tl + row * a.top + threadIdx.x);
  }
  for (uint32_t n = 0; row < a.rows; row += rows_apart, ++n) {
    const Cut cut(logits + row * stride, a.vocab, rank, log_size);
    const int vecs = cut.v1 - cut.v0, copy = copy_vecs(vecs);
    const int edges = a.vocab - cut.body * kVec;  // before the body and after it
    const bool has_edge = rank == size - 1 && (int)threadIdx.x < edges;
    const int edge_at = (int)threadIdx.x < cut.head ? threadIdx.x : cut.body * kVec + threadIdx.x;
    const float edge = has_edge ? to_f32(cut.row[edge_at]) : -INFINITY;
    // the row's pairs: one from each warp of the cluster
    if (threadIdx.x == 0) mbar_arrive_expect_tx(&met[n & 1u], (uint32_t)(size * kWarps * sizeof(float2)));

    // the teacher's entries k with (k / 32) % kWarps == warp: absent ones get id
    // -1.  An id that is too large or a NaN logit makes the sum NaN, and with it
    // the row.
    for (int i = threadIdx.x; i < (1 << teach.bits); i += THREADS) teach.table[i] = -1;
    float2 tp = make_float2(-INFINITY, 0.0f);
    for (int k = threadIdx.x; k < a.top; k += THREADS) {
      const bool first = k < THREADS;
      const int64_t id = first ? next_id : a.ti[row * a.top + k];
      float v = first ? next_t : a.tl[row * a.top + k];
      if (id < 0) v = -INFINITY;
      if (id >= a.vocab) {
        if (rank == 0) record_bad_id(a.err, id, a.vocab);
        v = NAN;
      }
      teach.id[k] = id < a.vocab && v != -INFINITY ? (int)id : -1;
      teach.prob[k] = v;
      tp.x = fmaxf(tp.x, v);
      if (v != v) tp.y = NAN;
    }
    if (warp < entry_warps) {
      tp.x = warp_max_fast(tp.x);
      for (int k = threadIdx.x; k < a.top; k += THREADS)
        if (teach.id[k] >= 0) tp.y += exp_scaled(teach.prob[k] - tp.x, a.c);
      tp.y = warp_sum(tp.y);
      if (lane == 0) teacher[warp] = tp;
    }

    float2 sp = make_float2(edge, edge == -INFINITY ? 0.0f : edge - edge + 1.0f);
#pragma unroll
    for (int i = 0; i < kDistillCopies; ++i) {
      if (!mbar_wait(&full[i], n & 1u)) atomicOr(&g_kernel_error, OXC_KERR_PIPELINE_TIMEOUT);
      int v = i * copy + threadIdx.x;
      const int end = min(vecs, (i + 1) * copy);
      constexpr int U = 16 / kVec;  // vectors at a time
      for (; v + (U - 1) * THREADS < end; v += U * THREADS) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = buffer[v + u * THREADS];
        pair_fold<T, U>(sp, q, a.c);
      }
      for (; v < end; v += THREADS) {
        const uint4 q[1] = {buffer[v]};
        pair_fold<T, 1>(sp, q, a.c);
      }
    }
    // the student's logits at this thread's entries; ids of other CTAs' parts turn
    // negative
    for (int k = threadIdx.x; k < a.top; k += THREADS) {
      const int id = teach.id[k];
      if (id < 0) continue;
      const int v = id < cut.head ? -1 : (id - cut.head) / kVec;
      const bool in_body = v >= 0 && v < cut.body;
      if (in_body ? v < cut.v0 || v >= cut.v1 : rank != size - 1) teach.id[k] = -2 - id;
      else logit_k[k] = to_f32(in_body ? reinterpret_cast<const T*>(smem)[id - cut.head - cut.v0 * kVec] : cut.row[id]);
    }
    sp = warp_merge(sp, a.c);
    if (lane < size) send_pair(&student[n & 1u][rank * kWarps + warp], &met[n & 1u], lane, sp);
    const int64_t next = row + rows_apart;
    if (next < a.rows) {
      if (threadIdx.x == 0) {
        const Cut ahead(logits + next * stride, a.vocab, rank, log_size);
        if (ahead.v1 > ahead.v0)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(ahead.part()),
                       "r"((ahead.v1 - ahead.v0) * 16) : "memory");
      }
      if ((int)threadIdx.x < a.top) {
        next_id = __ldcs(a.ti + next * a.top + threadIdx.x);
        next_t = __ldcs(a.tl + next * a.top + threadIdx.x);
      }
    }
    __syncthreads();  // the teacher's pairs are there
    if (!mbar_wait(&met[n & 1u], (n >> 1) & 1u)) atomicOr(&g_kernel_error, OXC_KERR_PIPELINE_TIMEOUT);
    sp = make_float2(-INFINITY, 0.0f);
    for (int i = lane; i < size * kWarps; i += 32) sp = pair_merge(sp, student[n & 1u][i], a.c);
    sp = warp_merge(sp, a.c);
    tp = warp_merge(lane < entry_warps ? teacher[lane] : make_float2(-INFINITY, 0.0f), a.c);
    const bool none = tp.x == -INFINITY && tp.y == 0.0f, bad = tp.y != tp.y;
    // a row of -inf alone has no softmax: its sum counts as NaN
    if (sp.x == -INFINITY) sp.y = NAN;
    const float unit = bad ? NAN : gs * rcp_approx(sp.y);
    T* dr = dlogits ? dlogits + row * (int64_t)a.vocab : nullptr;
    if (dr) {
      T* out = dr + cut.head + (int64_t)cut.v0 * kVec;
      const bool vector = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
      const float2 shift = make_float2(-sp.x, -sp.x), c2 = make_float2(a.c, a.c),
                   unit2 = make_float2(unit, unit);
#pragma unroll 4
      for (int v = threadIdx.x; v < vecs; v += THREADS) {
        float2 f[kPairs];
        unpack<T>(buffer[v], f);
        float g[kVec];
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          const float2 d = __fmul2_rn(__fadd2_rn(f[k], shift), c2);
          const float2 o = __fmul2_rn(make_float2(ex2_approx(d.x), ex2_approx(d.y)), unit2);
          g[2 * k] = o.x;
          g[2 * k + 1] = o.y;
        }
        if (none) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) g[k] = 0.0f;
        }
        if (vector) {
          store_from_f32<kVec>(out + (int64_t)v * kVec, g);
        } else {  // the gradient's rows lie otherwise within their 16 bytes
#pragma unroll
          for (int k = 0; k < kVec; ++k) out[(int64_t)v * kVec + k] = from_f32<T>(g[k]);
        }
      }
      if (has_edge) dr[edge_at] = from_f32<T>(none ? 0.0f : exp_scaled(edge - sp.x, a.c) * unit);
    }
    // this thread's entries: the loss at those in this part, and whether an id is
    // there twice (finding it in the table already means it is)
    int twice = 0;
    if (warp < entry_warps) {
      const float t_log = logf(tp.y), s_log = logf(sp.y), t_unit = rcp_approx(tp.y);
      float loss = 0.0f;
      for (int k = threadIdx.x; k < a.top; k += THREADS) {
        const int id = teach.id[k];
        if (id < 0) continue;
        const float z = (teach.prob[k] - tp.x), p = exp_scaled(z, a.c) * t_unit;
        teach.prob[k] = p;
        if (p > 0.0f)
          loss += p * ((z * a.inv_tau - t_log) - ((logit_k[k] - sp.x) * a.inv_tau - s_log));
        unsigned int h = ((unsigned int)id * 2654435769u) >> (32 - teach.bits);
        for (int i = 0; i < (1 << teach.bits); ++i) {
          const int was = atomicCAS(&teach.table[h], -1, id);
          if (was == -1) break;
          if (was == id) { twice = 1; break; }
          h = (h + 1) & ((1u << teach.bits) - 1);
        }
      }
      loss = warp_sum(loss);
      if (lane == 0) partial[warp] = loss;
    }
    const bool repeated = __syncthreads_or(twice);
    if (threadIdx.x == 0) {
      if (next < a.rows) fetch(next);  // the part has been read twice
      float sum = 0.0f;
      for (int w = 0; w < entry_warps; ++w) sum += partial[w];
      a.row_loss[row * size + rank] = none ? 0.0f : bad || sp.y != sp.y ? NAN : sum;
    }
    // q - p over the q just written
    if (dr && !none && !bad) {
      for (int k = threadIdx.x; k < a.top; k += THREADS) {
        const int id = teach.id[k];
        if (id < 0) continue;
        bool first;
        const float p = teacher_prob(teach, repeated, k, a.top, &first);
        if (first) dr[id] = from_f32<T>(exp_scaled(logit_k[k] - sp.x, a.c) * unit - gs * p);
      }
    }
    if (repeated) __syncthreads();  // the other threads' entries are read
  }
}

// One CTA per row at a time, three passes over it: any width.
template <typename T>
__global__ void __launch_bounds__(512) distill_wide_kernel(const T* __restrict__ logits,
                                                           int64_t stride, T* __restrict__ dlogits,
                                                           DistillArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  float* rest = reinterpret_cast<float*>(smem);
  __shared__ float scratch[33];
  const Teacher teach{rest, reinterpret_cast<int*>(rest) + a.top,
                      reinterpret_cast<int*>(rest) + 2 * a.top, teacher_bits(a.top)};
  const float gs = a.grad_loss ? a.grad_scale * __ldg(a.grad_loss) : a.grad_scale;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* xr = logits + row * stride;
    T* dr = dlogits ? dlogits + row * (int64_t)a.vocab : nullptr;
    const float* tl = a.tl + row * a.top;
    const TeacherRow t = teacher_row(teach, tl, a.ti + row * a.top, a.top, a.c, a.vocab, a.err, scratch);
    if (t.none || t.bad) {
      const float f = t.none ? 0.0f : NAN;
      for (int i = threadIdx.x; dr && i < a.vocab; i += blockDim.x) dr[i] = from_f32<T>(f);
      if (threadIdx.x == 0) a.row_loss[row] = f;
      __syncthreads();
      continue;
    }
    float m = -INFINITY;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) m = fmaxf(m, to_f32(xr[i]));
    m = block_max(m, scratch);
    float sum = 0.0f;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x)
      sum += exp_scaled(to_f32(xr[i]) - m, a.c);
    sum = block_sum(sum, scratch);
    if (dr) {
      const float scale = gs * __fdiv_rn(1.0f, sum);
      for (int i = threadIdx.x; i < a.vocab; i += blockDim.x)
        dr[i] = from_f32<T>(exp_scaled(to_f32(xr[i]) - m, a.c) * scale);
      __syncthreads();
      for (int k = threadIdx.x; k < a.top; k += blockDim.x) {
        const int id = teach.id[k];
        if (id < 0) continue;
        bool first;
        const float p = teacher_prob(teach, t.repeated, k, a.top, &first);
        if (first) dr[id] = from_f32<T>(exp_scaled(to_f32(xr[id]) - m, a.c) * scale - gs * p);
      }
    }
    const float s_log = logf(sum);
    float loss = 0.0f;
    for (int k = threadIdx.x; k < a.top; k += blockDim.x) {
      const float p = teach.prob[k];
      if (teach.id[k] >= 0 && p > 0.0f)
        loss += p * (((tl[k] - t.max) * a.inv_tau - t.log_sum) -
                     ((to_f32(xr[teach.id[k]]) - m) * a.inv_tau - s_log));
    }
    loss = block_sum(loss, scratch);
    if (threadIdx.x == 0) a.row_loss[row] = loss;
    __syncthreads();  // the teacher's side is read; the next row overwrites it
  }
}

// loss = scale * sum of row_loss, folded in f64 by one CTA in a fixed order.
__global__ void __launch_bounds__(1024) distill_loss_kernel(const float* __restrict__ row_loss,
                                                            int64_t rows, double scale,
                                                            float* __restrict__ loss) {
  __shared__ double scratch[33];
  pdl_wait();  // row_loss is the previous kernel's output
  double acc = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) acc += (double)row_loss[r];
  const double sum = block_sum(acc, scratch);
  if (threadIdx.x == 0) loss[0] = (float)(sum * scale);
}

// x *= g[0]; nothing to do, and nothing read, when g[0] is 1.  A bf16 gradient is
// rounded a second time here, 2^-9 relative at most: kept for the pass over the logits
// that a factor known only in backward would otherwise cost.
template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* __restrict__ x, int64_t n,
                                                       const float* __restrict__ g) {
  const float s = __ldg(g);
  if (s == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    x[i] = from_f32<T>(to_f32(x[i]) * s);
}

// CTAs per row: parts of up to 100 KB, two or more resident on an SM, as long as a
// cluster of 8 holds the row, larger ones beyond; 0 if they would be too large, by
// themselves or beside the `teacher` bytes of a long list.
// More CTAs than the row needs while that leaves SMs idle and each has some work.
static int distill_cluster(int64_t rows, int64_t bytes, int64_t teacher) {
  int size = 1;
  while (size < kDistillCluster && bytes > (int64_t)size * kDistillPart) size *= 2;
  if (bytes > (int64_t)size * kDistillMaxPart) return 0;
  if (bytes / size + 16 + teacher > kDistillSmem) return 0;
  while (size < kDistillCluster && rows * size * 2 <= sm_count() &&
         bytes >= (int64_t)size * 2 * kDistillThreads * 16)
    size *= 2;
  return size;
}

template <typename T>
static oxc_status distill_launch(const void* logits, int64_t stride, void* dlogits,
                                 const DistillArgs& a, int* losses, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  T* d = static_cast<T*>(dlogits);
  const int size = distill_cluster(a.rows, (int64_t)a.vocab * sizeof(T), teacher_smem(a.top));
  // the largest part: its share of the row's vectors
  const int vecs = a.vocab / (16 / (int)sizeof(T)), part = size ? 16 * ((vecs + size - 1) / size) : 0;
  const size_t smem = teacher_smem(a.top) + part;
  // fewer warps where a part has few logits for each, as a row costs every warp some
  // 800 instructions: f32 [32768, 1000] 153 us instead of 262, [16384, 4000] 111 instead
  // of 159; bf16 [8192, 8000] 78 instead of 101.  (64 threads: 168, 124 and 88.)
  const int threads = part <= 128 * 16 * 8 ? 128 : 256;
  auto cluster = threads == 128 ? distill_cluster_kernel<T, 128> : distill_cluster_kernel<T, 256>;
  const void* kernel = size ? (const void*)cluster : (const void*)distill_wide_kernel<T>;
  if (smem > 40 * 1024) {  // beyond what a kernel may use unasked
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_distill_loss");
  }
  *losses = size ? size : 1;
  if (size == 0) {
    distill_wide_kernel<T><<<(unsigned)std::min<int64_t>(a.rows, (int64_t)sm_count() * 4), 512, smem, s>>>(x, stride, d, a);
    return check_launch("oxc_distill_loss");
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)size);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // as many clusters as are resident at once: with more, the rest would run as a
  // second wave (a cluster's CTAs share a GPC, so not every SM can be used)
  int64_t resident = (int64_t)sm_count() * occupancy(kernel, threads, smem) / size;
  if (size > 1 && a.rows > resident / 2) {
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_distill_loss");
    resident = n;
  }
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(a.rows, std::max<int64_t>(resident, 1)) * size));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, cluster, x, stride, d, a, part);
  return e == cudaSuccess ? check_launch("oxc_distill_loss") : cuda_fail(e, "oxc_distill_loss");
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
  if (vocab > 0x7fffffff - 1024)  // a thread's int index steps past the last token
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: distill_loss: rows wider than 2^31");
  if (top > kDistillMaxTop)
    return fail(OXC_ERR_NOT_IMPLEMENTED,
                "not implemented: distill_loss: more than %d teacher logits per row, got %lld",
                kDistillMaxTop, (long long)top);
  if (!loss) return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: null pointer");
  if (rows > 0 && vocab == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss over zero classes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int losses = 1;  // per row
  if (rows > 0) {
    if (!logits || !row_loss || (top > 0 && (!teacher_logits || !teacher_ids)))
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: null pointer");
    const double tau = (double)temperature;
    const DistillArgs a{teacher_logits, teacher_ids, (int)top, (float)(1.0 / tau),
                        (float)(1.4426950408889634 / tau), (float)(tau / (double)total_rows),
                        grad_loss, row_loss, rows, (int)vocab, err_flag};
    const oxc_status st = dtype == OXC_BF16
                              ? distill_launch<bf16>(logits, logits_stride, dlogits, a, &losses, s)
                              : distill_launch<float>(logits, logits_stride, dlogits, a, &losses, s);
    if (st) return st;
  }
  const double scale = (double)temperature * (double)temperature / (double)total_rows;
  launch_dependent(distill_loss_kernel, dim3(1), dim3(1024), s, (const float*)row_loss, rows * losses,
                   scale,
                   loss);
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
