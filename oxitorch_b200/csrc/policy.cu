// policy.cu -- the clipped policy loss of sampled tokens, with a KL term towards a
// reference, and the logits' gradient in the same call.
//
// Row n has the policy's logits s (vocab of them), a sampled token i, the
// log-probability `old` that the token had when it was sampled, its advantage A and,
// for the KL term, its log-probability `ref` under a reference.  With temperature tau
//   q = softmax(s / tau),  logp = log q_i,  r = exp(logp - old)
//   L = -min(r A, clamp(r, 1 - below, 1 + above) A) + kl (exp(ref - logp) - (ref - logp) - 1)
//   loss = sum_n L / total_rows
//   g = dL / dlogp = (0 where the clamped product is the smaller, else -r A)
//                    + kl (1 - exp(ref - logp))
//   d loss / d s_j = g / (total_rows tau) ([j = i] - q_j)
// A row with a negative token (padding) has loss 0, gradient 0 and logp 0, whatever
// its logits hold; its logits are not read.
//
// Bound by HBM: 2 sizeof(T) bytes a logit, the row read once and its gradient
// written once.  As in distill.cu a row stays in shared memory between the two,
// shared by a cluster of 1 to 8 CTAs that exchange (max, sum) pairs; rows wider
// than that take the kernel of three passes.  f32 [8192, 32000] takes 342 us, 94% of the
// copy bandwidth; bf16 [8192, 131072] 816 us, 80%: there the two exponentials a logit keep
// their unit busy for 60% of that time, and issue and barriers come to as much.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "rowparts.cuh"

namespace oxc {

constexpr int kPolicyThreads = 256;            // per CTA at most
constexpr int kPolicyCopies = 2;               // bulk copies per part of a row
constexpr int kPolicyMaxPart = 160 * 1024;     // and at most
constexpr int kPolicyCluster = 8;              // CTAs per row at most

struct PolicyArgs {
  const int64_t* tokens;
  const float *old_logp, *adv, *ref_logp;  // adv NULL: only logp is asked for
  float low, high, log_low, log_high;  // 1 - below, 1 + above and their logarithms
  double low64, high64, inv_tau64;     // as they were given
  float kl;
  float inv_tau, c;   // c = log2(e) / tau
  float grad_scale;   // 1 / (total_rows tau)
  const float* grad_loss;
  float* logp;
  float* row_loss;
  int64_t rows;
  int vocab;
  int32_t* err;
};

// The sampled token of a row and its numbers.
struct Sample {
  int64_t token;
  float old, adv, ref;
  __device__ __forceinline__ void load(const PolicyArgs& a, int64_t row) {
    token = __ldg(a.tokens + row);
    old = adv = ref = 0.0f;
    if (a.adv) {
      old = __ldg(a.old_logp + row);
      adv = __ldg(a.adv + row);
      if (a.ref_logp) ref = __ldg(a.ref_logp + row);
    }
  }
};

struct PolicyTerm {
  float logp, loss, by;  // by = d loss / d logp
};

// exp(logp - old) in 64 bits.  Not inlined, as few rows need it: the registers of log and
// exp would be those of every row.
__device__ __noinline__ double policy_ratio(float logit, float2 row, float old, double inv_tau) {
  return exp(((double)logit - (double)row.x) * inv_tau - log((double)row.y) - (double)old);
}

// From the token's logit and the row's (max, sum of exponentials).  Comparisons are
// written so that a NaN reaches both the loss and the gradient.
// In 32 bits the ratio's logarithm is off by up to 2^-24 (5 |logp| + |old| + 4): three
// roundings of the scaled logit, logf's, and those of the two differences.  Whether the
// row is clipped, and so whether it has a gradient, may hang on less: a ratio that lies
// so near to an edge is taken in 64 bits.  (Log-probability and ratio of every row in 64
// bits: f32 [8192, 32000] 361 us for 342, in sums of two floats 359; the row waits for it.)
__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& a, const Sample& s, float logit,
                                                  float2 row) {
  PolicyTerm t;
  t.logp = (logit - row.x) * a.inv_tau - logf(row.y);
  t.loss = t.by = 0.0f;
  if (!a.adv) return t;
  const float gap = t.logp - s.old;
  const float near = 0x1p-21f * (1.0f + fabsf(t.logp) + fabsf(s.old)), r = expf(gap);
  float held = (r < a.low ? a.low : r > a.high ? a.high : r) * s.adv, free = r * s.adv;
  bool clipped = free > held;
  if (__builtin_expect(fminf(fabsf(gap - a.log_low), fabsf(gap - a.log_high)) < near, 0)) {
    const double q = policy_ratio(logit, row, s.old, a.inv_tau64), f = q * (double)s.adv;
    const double h = (q < a.low64 ? a.low64 : q > a.high64 ? a.high64 : q) * (double)s.adv;
    clipped = f > h;
    free = (float)f;
    held = (float)h;
  }
  t.loss = clipped ? -held : -free;
  t.by = clipped ? 0.0f : -free;
  if (a.ref_logp) {
    const float to_ref = s.ref - t.logp, e = expm1f(to_ref);
    t.loss = fmaf(a.kl, e - to_ref, t.loss);
    t.by = fmaf(-a.kl, e, t.by);
  }
  return t;
}

// Persistent clusters, a row at a time.  A CTA's part of the row arrives in shared
// memory by bulk copies; one pass over it makes the (max, sum) pair, which every warp
// sends to every CTA of the cluster, and a second the gradient; then the copies of the
// next row's part are started, whose bytes L2 was asked for when the second pass began.
// Every thread works out the row's term by itself.
// (With registers for four CTAs of 256 threads an SM, not fewer: 334 us against 353 at f32
// [8192, 32000].  Those of 128 threads lose by it: 134 us against 122 at bf16 [16384, 8000];
// there with registers for seven 120, for six 125.)
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 4 : sizeof(T) == 2 ? 7 : 1)
policy_cluster_kernel(const T* __restrict__ logits, int64_t stride, T* __restrict__ dlogits,
                      PolicyArgs a) {
  namespace cg = cooperative_groups;
  using Cut = RowCut<T>;
  constexpr int kVec = Cut::kVec, kPairs = kVec / 2;
  constexpr int kWarps = THREADS / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  // by the parity of the row: a CTA that is a row ahead of another sends into the
  // set that the other is not reading
  __shared__ float2 pairs[2][kPolicyCluster * kWarps];
  __shared__ uint64_t met[2];
  __shared__ uint64_t full[kPolicyCopies];
  cg::cluster_group cluster = cg::this_cluster();
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int log_size = 31 - __clz(size);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint4* buffer = reinterpret_cast<const uint4*>(smem);
  const float gs = a.grad_loss ? a.grad_scale * __ldg(a.grad_loss) : a.grad_scale;
  const int64_t rows_apart = gridDim.x >> log_size;

  // copy i of a part of n vectors: [i, i + 1) * copy_vecs(n) of them, whole rounds
  // of the threads
  auto copy_vecs = [](int n) {
    return (n + kPolicyCopies * THREADS - 1) / (kPolicyCopies * THREADS) * THREADS;
  };
  auto wanted = [&](const Sample& s) { return s.token >= 0 && s.token < a.vocab; };
  auto fetch = [&](int64_t row) {  // thread 0
    const Cut cut(logits + row * stride, a.vocab, rank, log_size);
    const int n = cut.v1 - cut.v0, each = copy_vecs(n);
#pragma unroll
    for (int i = 0; i < kPolicyCopies; ++i) {
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
  Sample sample;
  sample.token = -1;
  if (row < a.rows) sample.load(a, row);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < kPolicyCopies; ++i) mbar_init(&full[i], 1);
    mbar_init(&met[0], 1);
    mbar_init(&met[1], 1);
    fence_barrier_init();
    if (row < a.rows && wanted(sample)) fetch(row);
  }
  if (size > 1) cluster.sync();  // nobody sends before the barriers are there
  else __syncthreads();
  // n counts the rows whose logits are read: the same in every CTA of the cluster
  for (uint32_t n = 0; row < a.rows;) {
    const Cut cut(logits + row * stride, a.vocab, rank, log_size);
    const int vecs = cut.v1 - cut.v0, copy = copy_vecs(vecs);
    const int edges = a.vocab - cut.body * kVec;  // before the body and after it
    const bool has_edge = rank == size - 1 && (int)threadIdx.x < edges;
    const int edge_at = (int)threadIdx.x < cut.head ? threadIdx.x : cut.body * kVec + threadIdx.x;
    const bool read = wanted(sample);
    T* dr = dlogits ? dlogits + row * (int64_t)a.vocab : nullptr;
    T* out = dr + cut.head + (int64_t)cut.v0 * kVec;
    const bool vector = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int64_t next = row + rows_apart;
    Sample ahead;
    ahead.token = -1;
    if (next < a.rows) ahead.load(a, next);
    if (!read) {  // padding, or no token at all
      const float f = sample.token < 0 ? 0.0f : NAN;
      if (dr) {
        for (int v = threadIdx.x; v < vecs; v += THREADS) {
          float g[kVec];
#pragma unroll
          for (int k = 0; k < kVec; ++k) g[k] = f;
          if (vector) {
            store_from_f32<kVec>(out + (int64_t)v * kVec, g);
          } else {
#pragma unroll
            for (int k = 0; k < kVec; ++k) out[(int64_t)v * kVec + k] = from_f32<T>(f);
          }
        }
        if (has_edge) dr[edge_at] = from_f32<T>(f);
      }
      if (rank == 0 && threadIdx.x == 0) {
        if (sample.token >= 0) record_bad_id(a.err, sample.token, a.vocab);
        a.logp[row] = f;
        if (a.row_loss) a.row_loss[row] = f;
      }
      if (threadIdx.x == 0 && next < a.rows && wanted(ahead)) fetch(next);
      row = next;
      sample = ahead;
      continue;
    }
    const float edge = has_edge ? to_f32(cut.row[edge_at]) : -INFINITY;
    const float logit = to_f32(cut.row[sample.token]);
    // the row's pairs: one from each warp of the cluster
    if (threadIdx.x == 0) mbar_arrive_expect_tx(&met[n & 1u], (uint32_t)(size * kWarps * sizeof(float2)));

    float2 sp = make_float2(edge, edge == -INFINITY ? 0.0f : edge - edge + 1.0f);
#pragma unroll
    for (int i = 0; i < kPolicyCopies; ++i) {
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
    sp = warp_merge(sp, a.c);
    if (lane < size) send_pair(&pairs[n & 1u][rank * kWarps + warp], &met[n & 1u], lane, sp);
    if (threadIdx.x == 0 && next < a.rows && wanted(ahead)) {
      const Cut there(logits + next * stride, a.vocab, rank, log_size);
      if (there.v1 > there.v0)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(there.part()),
                     "r"((there.v1 - there.v0) * 16) : "memory");
    }
    if (!mbar_wait(&met[n & 1u], (n >> 1) & 1u)) atomicOr(&g_kernel_error, OXC_KERR_PIPELINE_TIMEOUT);
    sp = make_float2(-INFINITY, 0.0f);
    for (int i = lane; i < size * kWarps; i += 32) sp = pair_merge(sp, pairs[n & 1u][i], a.c);
    sp = warp_merge(sp, a.c);
    // a row of -inf alone has no softmax: its sum counts as NaN
    if (sp.x == -INFINITY) sp.y = NAN;
    const PolicyTerm term = policy_term(a, sample, logit, sp);
    if (rank == 0 && threadIdx.x == 0) {
      a.logp[row] = term.logp;
      if (a.row_loss) a.row_loss[row] = term.loss;
    }
    if (dr) {
      const float by = term.by * gs, unit = -by * rcp_approx(sp.y);
      const int at = (int)sample.token;
      // the token's vector in this part, if it is there
      const int mine = at >= cut.head && (at - cut.head) / kVec < cut.body ? (at - cut.head) / kVec - cut.v0 : -1;
      const int which = mine >= 0 ? (at - cut.head) % kVec : 0;
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
        if (v == mine) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) g[k] += k == which ? by : 0.0f;
        }
        if (vector) {
          store_from_f32<kVec>(out + (int64_t)v * kVec, g);
        } else {  // the gradient's rows lie otherwise within their 16 bytes
#pragma unroll
          for (int k = 0; k < kVec; ++k) out[(int64_t)v * kVec + k] = from_f32<T>(g[k]);
        }
      }
      if (has_edge)
        dr[edge_at] = from_f32<T>(fmaf(exp_scaled(edge - sp.x, a.c), unit, edge_at == at ? by : 0.0f));
    }
    __syncthreads();  // the part has been read twice
    if (threadIdx.x == 0 && next < a.rows && wanted(ahead)) fetch(next);
    row = next;
    sample = ahead;
    ++n;
  }
}

// One CTA per row at a time, three passes over it: any width.
template <typename T>
__global__ void __launch_bounds__(512) policy_wide_kernel(const T* __restrict__ logits,
                                                          int64_t stride, T* __restrict__ dlogits,
                                                          PolicyArgs a) {
  __shared__ float scratch[33];
  const float gs = a.grad_loss ? a.grad_scale * __ldg(a.grad_loss) : a.grad_scale;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* xr = logits + row * stride;
    T* dr = dlogits ? dlogits + row * (int64_t)a.vocab : nullptr;
    Sample sample;
    sample.load(a, row);
    if (sample.token < 0 || sample.token >= a.vocab) {
      const float f = sample.token < 0 ? 0.0f : NAN;
      for (int i = threadIdx.x; dr && i < a.vocab; i += blockDim.x) dr[i] = from_f32<T>(f);
      if (threadIdx.x == 0) {
        if (sample.token >= 0) record_bad_id(a.err, sample.token, a.vocab);
        a.logp[row] = f;
        if (a.row_loss) a.row_loss[row] = f;
      }
      continue;
    }
    float m = -INFINITY;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) m = fmaxf(m, to_f32(xr[i]));
    m = block_max(m, scratch);
    float sum = 0.0f;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) sum += exp_scaled(to_f32(xr[i]) - m, a.c);
    sum = block_sum(sum, scratch);
    const PolicyTerm term = policy_term(a, sample, to_f32(xr[sample.token]), make_float2(m, sum));
    if (threadIdx.x == 0) {
      a.logp[row] = term.logp;
      if (a.row_loss) a.row_loss[row] = term.loss;
    }
    if (dr) {
      const float by = term.by * gs, unit = -by * __fdiv_rn(1.0f, sum);
      for (int i = threadIdx.x; i < a.vocab; i += blockDim.x)
        dr[i] = from_f32<T>(fmaf(exp_scaled(to_f32(xr[i]) - m, a.c), unit,
                                 i == sample.token ? by : 0.0f));
    }
  }
}

// CTAs per row: parts of up to 40 KB in f32 and 100 KB in bf16 as long as a cluster of 8
// holds the row, larger ones beyond; 0 if they would be too large.  ([8192, 32000]: f32
// in parts of 32 KB 344 us and of 64 KB 371, bf16 of 32 KB 224 and of 64 KB 200.)  More
// CTAs than the row needs while that leaves SMs idle and each has some work.
static int policy_cluster(int64_t rows, int64_t bytes, int64_t most) {
  int size = 1;
  while (size < kPolicyCluster && bytes > size * most) size *= 2;
  if (bytes > (int64_t)size * kPolicyMaxPart) return 0;
  while (size < kPolicyCluster && rows * size * 2 <= sm_count() &&
         bytes >= (int64_t)size * 2 * kPolicyThreads * 16)
    size *= 2;
  return size;
}

template <typename T>
static oxc_status policy_launch(const void* logits, int64_t stride, void* dlogits,
                                const PolicyArgs& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  T* d = static_cast<T*>(dlogits);
  const int size = policy_cluster(a.rows, (int64_t)a.vocab * sizeof(T), (sizeof(T) == 4 ? 40 : 100) * 1024);
  if (size == 0) {
    policy_wide_kernel<T><<<(unsigned)std::min<int64_t>(a.rows, (int64_t)sm_count() * 4), 512, 0, s>>>(x, stride, d, a);
    return check_launch("oxc_policy_loss");
  }
  // the largest part: its share of the row's vectors
  const int vecs = a.vocab / (16 / (int)sizeof(T)), part = 16 * ((vecs + size - 1) / size);
  const int threads = part <= 128 * 16 * 8 ? 128 : 256;
  auto kernel = threads == 128 ? policy_cluster_kernel<T, 128> : policy_cluster_kernel<T, 256>;
  if (part > 40 * 1024) {  // beyond what a kernel may use unasked
    // the most that any call asks for: a smaller limit, set by another thread between this
    // and the launch, would refuse it
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kPolicyMaxPart);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_policy_loss");
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)size);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)part;
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
  static thread_local struct { int device = -1, part = 0, size = 0; int64_t resident = 0; } known;
  int device = 0;
  cudaGetDevice(&device);
  if (known.device != device || known.part != part || known.size != size) {
    int64_t resident = (int64_t)sm_count() * occupancy((const void*)kernel, threads, part) / size;
    if (size > 1) {
      int n = 0;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, (const void*)kernel, &cfg);
      if (e != cudaSuccess) return cuda_fail(e, "oxc_policy_loss");
      resident = n;
    }
    known.device = device;
    known.part = part;
    known.size = size;
    known.resident = resident;
  }
  const int64_t resident = known.resident;
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(a.rows, std::max<int64_t>(resident, 1)) * size));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, x, stride, d, a);
  return e == cudaSuccess ? check_launch("oxc_policy_loss") : cuda_fail(e, "oxc_policy_loss");
}

}  // namespace oxc

using namespace oxc;

extern "C" {

oxc_status oxc_policy_loss(const void* logits, int64_t logits_stride, const int64_t* tokens,
                           const float* old_logp, const float* advantages, const float* ref_logp,
                           double clip_below, double clip_above, double kl_coef,
                           double temperature, const float* grad_loss, float* loss, float* logp,
                           float* row_loss, void* dlogits, int64_t rows, int64_t vocab,
                           int64_t total_rows, int32_t dtype, int32_t* err_flag, void* stream) {
  if (!known_dtype(dtype))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: policy_loss: unknown dtype %d", dtype);
  if (rows < 0 || vocab < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: policy_loss: negative shape");
  if (total_rows <= 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: policy_loss: total_rows %lld must be positive",
                (long long)total_rows);
  const float c = (float)(1.4426950408889634 / temperature);  // log2(e) / tau
  if (!(temperature > 0.0) || isinf((float)temperature) || isinf(c))
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: policy_loss: temperature must be positive, got %g", temperature);
  if (!(clip_below >= 0.0) || !(clip_above >= 0.0) || !(kl_coef >= 0.0) || isinf((float)kl_coef))
    return fail(OXC_ERR_INVALID_ARGUMENT,
                "invalid argument: policy_loss: clip (%g, %g) and kl_coef %g must not be negative",
                clip_below, clip_above, kl_coef);
  if (vocab > 0x7fffffff - 1024)  // a thread's int index steps past the last token
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: policy_loss: rows wider than 2^31");
  if (rows > 0 && vocab == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: policy_loss over zero classes");
  const bool term = loss != nullptr;  // else only logp is asked for
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows > 0) {
    if (!logits || !tokens || !logp || (term && (!advantages || !old_logp || !row_loss)) ||
        (!term && dlogits) || (term && kl_coef > 0.0 && !ref_logp))
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: policy_loss: null pointer");
    PolicyArgs a{};
    a.tokens = tokens;
    a.old_logp = old_logp;
    a.adv = term ? advantages : nullptr;
    a.ref_logp = kl_coef > 0.0 ? ref_logp : nullptr;
    a.low = (float)(1.0 - clip_below);
    a.high = (float)(1.0 + clip_above);
    a.log_low = clip_below < 1.0 ? (float)log1p(-clip_below) : -INFINITY;
    a.log_high = (float)log1p(clip_above);
    a.low64 = 1.0 - clip_below;
    a.high64 = 1.0 + clip_above;
    a.kl = (float)kl_coef;
    a.inv_tau = (float)(1.0 / temperature);
    a.inv_tau64 = 1.0 / temperature;
    a.c = c;
    a.grad_scale = (float)(1.0 / (temperature * (double)total_rows));
    a.grad_loss = grad_loss;
    a.logp = logp;
    a.row_loss = term ? row_loss : nullptr;
    a.rows = rows;
    a.vocab = (int)vocab;
    a.err = err_flag;
    const oxc_status st = dtype == OXC_BF16
                              ? policy_launch<bf16>(logits, logits_stride, dlogits, a, s)
                              : policy_launch<float>(logits, logits_stride, dlogits, a, s);
    if (st) return st;
  }
  if (!term) return OXC_OK;
  launch_dependent(sum_losses_kernel, dim3(1), dim3(1024), s, (const float*)row_loss, rows,
                   1.0 / (double)total_rows, loss);
  return check_launch("oxc_policy_loss (sum)");
}

}  // extern "C"
