// verify.cu -- verification of drafted tokens against the target's
// probabilities, from given random numbers.
//
// Sequence b drafted n = lengths[b] <= K tokens x_0 .. x_{n-1}, each sampled
// from the draft's probabilities q_k; p_k are the target's at the same places,
// p_n at the place after them.  Token k is kept while u_k * q_k(x_k) < p_k(x_k)
// (probability min(1, p/q) for u uniform in [0, 1)).  The token that follows
// the j kept ones is sampled from what the target holds beyond the draft,
//   w = max(p_j - q_j, 0) for j < n,  w = p_n for j = n,
// as argmax_v w_v / e_v with e exponential variates (the first of equal ones),
// which picks v with probability w_v / sum(w).  Should w be zero everywhere,
// p_j takes its place; -1 if that has no positive entry either.  Without draft
// probabilities q_k is 1 at x_k and 0 elsewhere (a draft that was not sampled).  A
// NaN probability keeps no token and is never the argmax.
//
// Each weight is one subtraction and one division in f32, correctly rounded,
// so the choice is the same on every machine and in every order of reduction.
//
// Three rows of the vocabulary are read per sequence, 12 bytes an entry.  A cluster
// of up to 8 CTAs shares a sequence, so that few sequences still use many SMs;
// every CTA works the acceptance out for itself (a few dozen loads) and the
// argmax's keys meet in distributed shared memory.  Measured: 256 sequences of
// 131072 entries 65 us (94% of the copy bandwidth), 64 of them 24 us (64%), where
// the launch, the acceptance and the meeting are not hidden by other sequences.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"

namespace oxc {

__device__ __forceinline__ void record_bad_token(int32_t* flag, int64_t id, int64_t vocab) {
  if (flag && atomicCAS(flag, 0, 1) == 0) {
    flag[1] = (int32_t)(uint32_t)((uint64_t)id & 0xffffffffu);
    flag[2] = (int32_t)(uint32_t)((uint64_t)id >> 32);
    flag[3] = (int32_t)vocab;
  }
}

// w / e as an ordered key with the index's complement below it, so the largest
// key is the largest quotient at the lowest index; 0 for no weight or a NaN (any
// other key has a nonzero low half).  A variate of zero gives a positive weight an
// infinite quotient; a token without weight never wins, whatever its variate.
__device__ __forceinline__ unsigned long long race_key(float w, float e, uint32_t v) {
  if (!(w > 0.0f)) return 0ull;
  const float s = __fdiv_rn(w, e);
  return s >= 0.0f ? ((unsigned long long)__float_as_uint(s) << 32) | (0xffffffffu - v) : 0ull;
}

__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

constexpr int kVerifyCluster = 8;
// CTAs of 256 threads per SM: capped at 64 registers for a fourth (64 x 131072 24 us,
// with three 30; 256 x 131072 65 and 95).
constexpr int kVerifyCtas = 4;

// The largest key of the vocabulary entries [v0, v1) with weights p - q (q may be null;
// token x counts 0).  The rows start anywhere: vectors where their addresses agree
// modulo 16 bytes, else single entries.
template <int THREADS>
__device__ __forceinline__ unsigned long long race_best(const float* p, const float* q,
                                                        const float* e, int64_t x, int64_t v0,
                                                        int64_t v1) {
  unsigned long long k = 0ull;
  p += v0;
  e += v0;
  if (q) q += v0;
  const uint32_t n = (uint32_t)(v1 - v0);
  const int64_t own = x - v0;
  auto one = [&](float pv, float qv, float ev, uint32_t at) {
    k = max(k, race_key(at == own ? 0.0f : __fsub_rn(pv, qv), ev, (uint32_t)(v0 + at)));
  };
  const uintptr_t o = reinterpret_cast<uintptr_t>(p) & 15;
  if (o == (reinterpret_cast<uintptr_t>(e) & 15) && (!q || o == (reinterpret_cast<uintptr_t>(q) & 15))) {
    const uint32_t from = min(n, (uint32_t)((16 - o) & 15) / 4), to = from + ((n - from) & ~3u);
    constexpr int U = 2;  // vectors in flight per row
    for (uint32_t v = from + 4 * threadIdx.x; v < to; v += 4 * U * THREADS) {
      float4 pv[U], qv[U], ev[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t at = min(v + 4 * u * THREADS, to - 4);  // twice the last is no harm
        pv[u] = ld_stream(reinterpret_cast<const float4*>(p + at));
        ev[u] = ld_stream(reinterpret_cast<const float4*>(e + at));
        qv[u] = q ? ld_stream(reinterpret_cast<const float4*>(q + at)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t at = min(v + 4 * u * THREADS, to - 4);
        one(pv[u].x, qv[u].x, ev[u].x, at);
        one(pv[u].y, qv[u].y, ev[u].y, at + 1);
        one(pv[u].z, qv[u].z, ev[u].z, at + 2);
        one(pv[u].w, qv[u].w, ev[u].w, at + 3);
      }
    }
    if (threadIdx.x < from + (n - to)) {  // before the vectors and after them
      const uint32_t at = threadIdx.x < from ? threadIdx.x : to + threadIdx.x - from;
      one(p[at], q ? q[at] : 0.0f, e[at], at);
    }
  } else {
    constexpr int S = 8;  // entries in flight per row (64 x 131071: 27 us; with 4, 32)
    for (uint32_t i = threadIdx.x; i < n; i += S * THREADS) {
      float pv[S], qv[S], ev[S];
#pragma unroll
      for (int u = 0; u < S; ++u) {
        const uint32_t at = min(i + u * THREADS, n - 1);  // twice the last is no harm
        pv[u] = ld_stream(p + at);
        ev[u] = ld_stream(e + at);
        qv[u] = q ? ld_stream(q + at) : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < S; ++u) one(pv[u], qv[u], ev[u], min(i + u * THREADS, n - 1));
    }
  }
  return k;
}

// One cluster per sequence.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_kernel(
    const float* __restrict__ target, int64_t t_sb, int64_t t_sk, const float* __restrict__ draft,
    int64_t d_sb, int64_t d_sk, const int64_t* __restrict__ tokens,
    const int64_t* __restrict__ lengths, const float* __restrict__ uniform,
    const float* __restrict__ race, int drafted, int64_t vocab, int64_t* __restrict__ out_tokens,
    int64_t* __restrict__ accepted, int32_t* err) {
  namespace cg = cooperative_groups;
  constexpr int kWarps = THREADS / 32;
  __shared__ unsigned long long best[kWarps], mine[2];
  __shared__ int first;
  cg::cluster_group cluster = cg::this_cluster();
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / size;
  const int64_t* tok = tokens + b * drafted;
  const int64_t want = lengths ? lengths[b] : drafted;
  const int n = (int)(want < 0 ? 0 : want > drafted ? drafted : want);
  if (threadIdx.x == 0) first = n;
  __syncthreads();
  for (int k = threadIdx.x; k < n; k += THREADS) {
    const int64_t x = tok[k];
    bool keep = false;
    if (x < 0 || x >= vocab) {
      if (rank == 0) record_bad_token(err, x, vocab);
    } else {
      const float p = target[b * t_sb + k * t_sk + x];
      const float q = draft ? draft[b * d_sb + k * d_sk + x] : 1.0f;
      keep = __fmul_rn(uniform[b * drafted + k], q) < p;
    }
    if (!keep) atomicMin(&first, k);
  }
  __syncthreads();
  const int j = first;
  const float* p = target + b * t_sb + j * t_sk;
  const float* e = race + b * vocab;
  // this CTA's entries: a share in multiples of 4
  const int64_t each = ((vocab + size - 1) / size + 3) & ~(int64_t)3;
  const int64_t v0 = min(vocab, rank * each), v1 = min(vocab, v0 + each);
  unsigned long long k = 0ull;
  for (int pass = 0; pass < 2; ++pass) {  // the second from p alone, if nothing was left
    const bool beyond = pass == 0 && j < n;
    k = race_best<THREADS>(p, beyond && draft ? draft + b * d_sb + j * d_sk : nullptr, e,
                  beyond && !draft ? tok[j] : -1, v0, v1);
    k = warp_max_key(k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = k;
    __syncthreads();
    k = 0ull;
    for (int w = 0; w < kWarps; ++w) k = max(k, best[w]);
    if (size > 1) {
      if (threadIdx.x == 0) mine[pass] = k;
      cluster.sync();
      k = 0ull;
      for (int r = 0; r < size; ++r) k = max(k, *cluster.map_shared_rank(&mine[pass], r));
    }
    if (k != 0ull || j == n) break;  // (the same in every CTA)
  }
  if (rank == 0) {
    const int64_t next = k ? (int64_t)(0xffffffffu - (uint32_t)k) : -1;
    for (int i = threadIdx.x; i <= drafted; i += THREADS)
      out_tokens[b * (drafted + 1) + i] = i < j ? tok[i] : i == j ? next : -1;
    if (threadIdx.x == 0) accepted[b] = j;
  }
  if (size > 1) cluster.sync();  // no CTA leaves while its key is read
}

}  // namespace oxc

using namespace oxc;

extern "C" {

oxc_status oxc_verify_draft(const float* target, int64_t target_sb, int64_t target_sk,
                            const float* draft, int64_t draft_sb, int64_t draft_sk,
                            const int64_t* tokens, const int64_t* lengths, const float* uniform,
                            const float* race, int64_t batch, int64_t drafted, int64_t vocab,
                            int64_t* out_tokens, int64_t* accepted, int32_t* err_flag,
                            void* stream) {
  if (batch < 0 || drafted < 0 || vocab < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: verify_draft: negative shape");
  if (batch == 0) return OXC_OK;
  if (vocab == 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: verify_draft over zero classes");
  if (vocab > 0x7fffffff || batch > 0x7fffffff || drafted > 65535)
    return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: verify_draft: [%lld, %lld, %lld]",
                (long long)batch, (long long)drafted, (long long)vocab);
  if (!target || !race || !out_tokens || !accepted || (drafted > 0 && (!tokens || !uniform)))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: verify_draft: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // CTAs per sequence: doubled while all of them are resident at once
  // and every CTA has a few thousand entries
  int size = 1;
  while (size < kVerifyCluster && batch * size * 2 <= kVerifyCtas * (int64_t)sm_count() &&
         vocab >= (int64_t)size * 2 * 2048)
    size *= 2;
  if (batch > 0x7fffffff / size) size = 1;
  // and larger CTAs where there are few (8 x 200003: 18 us instead of 28): as long as
  // they fill three quarters of the SMs at most, since a cluster's share a GPC, which
  // leaves some idle (16 x 131072 with a CTA an SM: 22 us instead of 18)
  int threads = 256;
  while (threads < 1024 && batch * size * threads * 2 <= 768 * (int64_t)sm_count() &&
         vocab >= (int64_t)size * threads * 2 * 4)
    threads *= 2;
  auto kernel = threads == 256 ? verify_kernel<256> : threads == 512 ? verify_kernel<512> : verify_kernel<1024>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * size));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, target, target_sb, target_sk, draft,
                                           draft_sb, draft_sk, tokens, lengths, uniform, race,
                                           (int)drafted, vocab, out_tokens, accepted, err_flag);
  if (e != cudaSuccess) return cuda_fail(e, "oxc_verify_draft");
  return check_launch("oxc_verify_draft");
}

}  // extern "C"
