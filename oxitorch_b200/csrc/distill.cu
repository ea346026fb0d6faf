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
// written once.  So a row stays in registers between the two: a cluster of 1 to 8
// CTAs shares it, 32 logits a thread, as exponentials relative to the CTA's own
// maximum; (max, sum) pairs are exchanged through distributed shared memory, and
// one multiplication an element remains.  Rows wider than that (262144) take the
// three-pass kernel, which re-reads them from L2 or HBM.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "typed.cuh"

namespace oxc {

constexpr int kDistillMaxTop = 4096;
constexpr int kDistillEach = 32;      // logits per thread
constexpr int kDistillCluster = 8;    // CTAs per row at most
constexpr int kDistillMaxThreads = 1024;

// Records the first bad id: flag[0] = 2 (dim 1), flag[1..2] = id, flag[3] = vocab.
__device__ __forceinline__ void record_bad_id(int32_t* flag, int64_t id, int64_t vocab) {
  if (flag && atomicCAS(flag, 0, 2) == 0) {
    flag[1] = (int32_t)(uint32_t)((uint64_t)id & 0xffffffffu);
    flag[2] = (int32_t)(uint32_t)((uint64_t)id >> 32);
    flag[3] = (int32_t)vocab;
  }
}

// exp(d / tau) for d = x - max <= 0, c = log2(e) / tau.  The subtraction comes
// first, so the large terms see only ex2's own error; results below 2^-126 are 0.
__device__ __forceinline__ float exp_scaled(float d, float c) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * c));
  return r;
}

// The teacher's side of a row, in shared memory: prob[k] (0 for absent entries)
// and id[k] (-1).
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
  return (size_t)top * 8 + (sizeof(int) << teacher_bits(top));
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
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = pair_merge(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o),
                                  __shfl_xor_sync(0xffffffffu, v.y, o)), c);
  return v;
}

// One cluster per row.  The row's bytes are cut at 16-byte boundaries of memory:
// `body` whole vectors, CTA r of the cluster taking the r-th share of them,
// thread t the vectors t, t + THREADS, ...; the elements before the first
// boundary and after the last (fewer than a vector each) are single elements of
// the last CTA's warp 0.
//
// A CTA lives for a few microseconds, so what counts beside the bytes in flight
// is how rarely its warps meet.  Each warp reduces its logits, and its share of
// the teacher's entries, to a (max, sum) pair of its own; one cluster barrier
// exchanges all pairs; the gradient is written; one more barrier, within the CTA,
// precedes the corrections at the teacher's tokens.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
distill_cluster_kernel(const T* __restrict__ logits, int64_t stride, T* __restrict__ dlogits,
                       DistillArgs a) {
  namespace cg = cooperative_groups;
  constexpr int kVec = 16 / (int)sizeof(T);
  constexpr int kVecs = kDistillEach / kVec;
  constexpr int kWarps = THREADS / 32;
  extern __shared__ float smem[];
  __shared__ float2 student[kWarps], teacher[kWarps];
  __shared__ float partial[kWarps];
  const Teacher teach{smem, reinterpret_cast<int*>(smem) + a.top,
                      reinterpret_cast<int*>(smem) + 2 * a.top, teacher_bits(a.top)};
  cg::cluster_group cluster = cg::this_cluster();
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / size;
  const T* xr = logits + row * stride;
  const int head = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / (int)sizeof(T));
  const int body = (a.vocab - head) / kVec, each = (body + size - 1) / size;
  const int v0 = min(body, rank * each), v1 = min(body, v0 + each);
  const int edges = a.vocab - body * kVec;  // head + tail
  const bool has_edge = rank == size - 1 && (int)threadIdx.x < edges;
  const int edge_at = (int)threadIdx.x < head ? threadIdx.x : body * kVec + threadIdx.x;
  uint4 raw[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = v0 + i * THREADS + threadIdx.x;
    if (v < v1) raw[i] = __ldcs(reinterpret_cast<const uint4*>(xr + head) + v);
  }
  float edge = has_edge ? to_f32(xr[edge_at]) : -INFINITY;

  // the teacher's entries k with (k / 32) % kWarps == warp: exponentials relative
  // to the warp's maximum, 0 and id -1 for absent ones.  An id that is too large
  // or a NaN logit makes the sum NaN, and with it the row.
  const float* tl = a.tl + row * a.top;
  const int64_t* ti = a.ti + row * a.top;
  for (int i = threadIdx.x; i < (1 << teach.bits); i += THREADS) teach.table[i] = -1;
  float2 tp = make_float2(-INFINITY, 0.0f);
  for (int k = threadIdx.x; k < a.top; k += THREADS) {
    const int64_t id = ti[k];
    float v = tl[k];
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
  tp.x = warp_max(tp.x);
  for (int k = threadIdx.x; k < a.top; k += THREADS) {
    const float e = teach.id[k] < 0 ? 0.0f : exp_scaled(teach.prob[k] - tp.x, a.c);
    teach.prob[k] = e;
    tp.y += e;
  }
  tp.y = warp_sum(tp.y);

  float e[kDistillEach];
  float2 sp = make_float2(edge, 0.0f);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    const bool in = v0 + i * THREADS + (int)threadIdx.x < v1;
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      float f;
      if constexpr (sizeof(T) == 4) f = __uint_as_float(w[k]);
      else f = k & 1 ? bf16_hi(w[k / 2]) : bf16_lo(w[k / 2]);
      e[i * kVec + k] = in ? f : -INFINITY;
      sp.x = fmaxf(sp.x, e[i * kVec + k]);
    }
  }
  sp.x = warp_max(sp.x);
  const float base = sp.x == -INFINITY ? 0.0f : sp.x;
  edge = has_edge ? exp_scaled(edge - base, a.c) : 0.0f;
  sp.y = edge;
#pragma unroll
  for (int i = 0; i < kDistillEach; ++i) {
    e[i] = exp_scaled(e[i] - base, a.c);
    sp.y += e[i];
  }
  sp.y = warp_sum(sp.y);
  if (lane == 0) {
    student[warp] = sp;
    teacher[warp] = tp;
  }
  if (size > 1) cluster.sync();
  else __syncthreads();
  const float own_max = sp.x;
  sp = make_float2(-INFINITY, 0.0f);
  for (int i = lane; i < size * kWarps; i += 32) {
    const float2* s = size > 1 ? cluster.map_shared_rank(student, i / kWarps) : student;
    sp = pair_merge(sp, s[i % kWarps], a.c);
  }
  if (size > 1) cluster.barrier_arrive();  // the others' pairs are read
  sp = warp_merge(sp, a.c);
  tp = warp_merge(lane < kWarps ? teacher[lane] : make_float2(-INFINITY, 0.0f), a.c);
  const bool none = tp.x == -INFINITY && tp.y == 0.0f, bad = tp.y != tp.y;
  const float gs = a.grad_loss ? a.grad_scale * __ldg(a.grad_loss) : a.grad_scale;
  // a row of -inf alone has no softmax: its sum counts as NaN
  const float unit = gs * __fdiv_rn(1.0f, sp.x == -INFINITY ? NAN : sp.y);
  float scale = own_max == -INFINITY ? unit : unit * exp_scaled(own_max - sp.x, a.c);
  if (bad) scale = NAN;
  T* dr = dlogits ? dlogits + row * (int64_t)a.vocab : nullptr;
  if (dr) {
    const bool vector = ((reinterpret_cast<uintptr_t>(dr + head) & 15) == 0);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int v = v0 + i * THREADS + threadIdx.x;
      if (v < v1) {
        float g[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) g[k] = none ? 0.0f : e[i * kVec + k] * scale;
        T* out = dr + head + (int64_t)v * kVec;
        if (vector) {
          store_from_f32<kVec>(out, g);
        } else {  // the gradient's rows lie otherwise within their 16 bytes
#pragma unroll
          for (int k = 0; k < kVec; ++k) out[k] = from_f32<T>(g[k]);
        }
      }
    }
    if (has_edge) dr[edge_at] = from_f32<T>(none ? 0.0f : edge * scale);
  }
  // this thread's entries: their part of the loss (rank 0), and whether an id is
  // there twice (finding it in the table already means it is)
  const float t_unit = __fdiv_rn(1.0f, tp.y), t_log = logf(tp.y), s_log = logf(sp.y);
  const float t_share = teacher[warp].x == -INFINITY ? 0.0f : t_unit * exp_scaled(teacher[warp].x - tp.x, a.c);
  float loss = 0.0f;
  int twice = 0;
  for (int k = threadIdx.x; k < a.top; k += THREADS) {
    const int id = teach.id[k];
    const float p = teach.prob[k] * t_share;
    teach.prob[k] = p;
    if (id < 0) continue;
    if (rank == 0 && p > 0.0f)
      loss += p * (((tl[k] - tp.x) * a.inv_tau - t_log) -
                   ((to_f32(xr[id]) - sp.x) * a.inv_tau - s_log));
    unsigned int h = ((unsigned int)id * 2654435769u) >> (32 - teach.bits);
    for (int n = 0; n < (1 << teach.bits); ++n) {
      const int was = atomicCAS(&teach.table[h], -1, id);
      if (was == -1) break;
      if (was == id) { twice = 1; break; }
      h = (h + 1) & ((1u << teach.bits) - 1);
    }
  }
  if (rank == 0) {
    loss = warp_sum(loss);
    if (lane == 0) partial[warp] = loss;
  }
  const bool repeated = __syncthreads_or(twice);
  if (rank == 0 && threadIdx.x == 0) {
    float sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) sum += partial[w];
    a.row_loss[row] = none ? 0.0f : bad || sp.x == -INFINITY ? NAN : sum;
  }
  // the teacher's tokens in this CTA's part: q - p over the q just written
  if (dr && !none && !bad) {
    for (int k = threadIdx.x; k < a.top; k += THREADS) {
      const int id = teach.id[k];
      if (id < 0) continue;
      const int v = id < head ? -1 : (id - head) / kVec;
      if (v < 0 || v >= body ? rank != size - 1 : v < v0 || v >= v1) continue;
      bool first;
      const float p = teacher_prob(teach, repeated, k, a.top, &first);
      if (first) dr[id] = from_f32<T>(exp_scaled(to_f32(xr[id]) - sp.x, a.c) * unit - gs * p);
    }
  }
  if (size > 1) cluster.barrier_wait();  // no CTA leaves while its pairs are read
}

// One CTA per row at a time, three passes over it: any width.
template <typename T>
__global__ void __launch_bounds__(512) distill_wide_kernel(const T* __restrict__ logits,
                                                           int64_t stride, T* __restrict__ dlogits,
                                                           DistillArgs a) {
  extern __shared__ float smem[];
  __shared__ float scratch[33];
  const Teacher teach{smem, reinterpret_cast<int*>(smem) + a.top,
                      reinterpret_cast<int*>(smem) + 2 * a.top, teacher_bits(a.top)};
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

// x *= g[0]; nothing to do, and nothing read, when g[0] is 1.
template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* __restrict__ x, int64_t n,
                                                       const float* __restrict__ g) {
  const float s = __ldg(g);
  if (s == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    x[i] = from_f32<T>(to_f32(x[i]) * s);
}

// Threads and CTAs per row.  CTAs of 256 threads (or fewer, for narrow rows) as
// long as a cluster of 8 holds the row, else of 512 and 1024; 0 threads: none
// does.  More CTAs than the row needs while that leaves SMs idle.
static void distill_geometry(int64_t rows, int64_t vocab, int* threads, int* size) {
  *threads = 0;
  for (int n : {64, 128, 256}) {
    if ((int64_t)n * kDistillEach >= vocab) {
      *threads = n;
      *size = 1;
      break;
    }
  }
  for (int n = 256; *threads == 0 && n <= kDistillMaxThreads; n *= 2)
    for (int k = 1; *threads == 0 && k <= kDistillCluster; k *= 2)
      if ((int64_t)n * k * kDistillEach >= vocab) {
        *threads = n;
        *size = k;
      }
  if (*threads == 0) return;
  while (*size < kDistillCluster && rows * *size < sm_count() &&
         vocab >= (int64_t)*size * 2 * *threads * 4)
    *size *= 2;
}

template <typename T>
static oxc_status distill_launch(const void* logits, int64_t stride, void* dlogits,
                                 const DistillArgs& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  T* d = static_cast<T*>(dlogits);
  const size_t smem = teacher_smem(a.top);
  int threads, size;
  distill_geometry(a.rows, a.vocab, &threads, &size);
  void (*kernel)(const T*, int64_t, T*, DistillArgs) = distill_wide_kernel<T>;
  switch (threads) {
    case 64: kernel = distill_cluster_kernel<T, 64>; break;
    case 128: kernel = distill_cluster_kernel<T, 128>; break;
    case 256: kernel = distill_cluster_kernel<T, 256>; break;
    case 512: kernel = distill_cluster_kernel<T, 512>; break;
    case 1024: kernel = distill_cluster_kernel<T, 1024>; break;
    default: break;
  }
  if (smem > 40 * 1024) {  // beyond what a kernel may use unasked
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_distill_loss");
  }
  if (threads == 0) {
    kernel<<<(unsigned)std::min<int64_t>(a.rows, (int64_t)sm_count() * 4), 512, smem, s>>>(x, stride, d, a);
    return check_launch("oxc_distill_loss");
  }
  if (a.rows > 0x7fffffff / size)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: distill_loss: %lld rows", (long long)a.rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * size));
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, x, stride, d, a);
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
  if (vocab > 0x7fffffff)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: distill_loss: rows wider than 2^31");
  if (top > kDistillMaxTop)
    return fail(OXC_ERR_NOT_IMPLEMENTED,
                "not implemented: distill_loss: more than %d teacher logits per row, got %lld",
                kDistillMaxTop, (long long)top);
  if (!loss) return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: null pointer");
  if (rows > 0 && vocab == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss over zero classes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows > 0) {
    if (!logits || !row_loss || (top > 0 && (!teacher_logits || !teacher_ids)))
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: distill_loss: null pointer");
    const double tau = (double)temperature;
    const DistillArgs a{teacher_logits, teacher_ids, (int)top, (float)(1.0 / tau),
                        (float)(1.4426950408889634 / tau), (float)(tau / (double)total_rows),
                        grad_loss, row_loss, rows, (int)vocab, err_flag};
    const oxc_status st = dtype == OXC_BF16
                              ? distill_launch<bf16>(logits, logits_stride, dlogits, a, s)
                              : distill_launch<float>(logits, logits_stride, dlogits, a, s);
    if (st) return st;
  }
  const double scale = (double)temperature * (double)temperature / (double)total_rows;
  launch_dependent(distill_loss_kernel, dim3(1), dim3(1024), s, (const float*)row_loss, rows, scale,
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
