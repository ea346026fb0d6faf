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
// p_j takes its place; -1 if that has no positive entry either.  Without draft probabilities q_k is 1 at x_k and 0
// elsewhere (a draft that was not sampled).  A NaN probability keeps no token
// and is never the argmax.
//
// Each weight is one subtraction and one division in f32, correctly rounded,
// so the choice is the same on every machine and in every order of reduction.
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
// key is the largest quotient at the lowest index; 0 for no weight or a NaN
// (any other key has a nonzero low half).
__device__ __forceinline__ unsigned long long race_key(float w, float e, uint32_t v) {
  if (!(w > 0.0f)) return 0ull;
  const float s = __fdiv_rn(w, e);
  if (s != s) return 0ull;
  return ((unsigned long long)__float_as_uint(s) << 32) | (0xffffffffu - v);
}

__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

// One CTA per sequence.
__global__ void __launch_bounds__(512) verify_kernel(
    const float* __restrict__ target, int64_t t_sb, int64_t t_sk, const float* __restrict__ draft,
    int64_t d_sb, int64_t d_sk, const int64_t* __restrict__ tokens,
    const int64_t* __restrict__ lengths, const float* __restrict__ uniform,
    const float* __restrict__ race, int drafted, int64_t vocab, int64_t* __restrict__ out_tokens,
    int64_t* __restrict__ accepted, int32_t* err) {
  __shared__ unsigned long long best[16];
  __shared__ int first;
  const int64_t b = blockIdx.x;
  const int64_t* tok = tokens + b * drafted;
  int64_t want = lengths ? lengths[b] : drafted;
  const int n = (int)(want < 0 ? 0 : want > drafted ? drafted : want);
  if (threadIdx.x == 0) first = n;
  __syncthreads();
  for (int k = threadIdx.x; k < n; k += blockDim.x) {
    const int64_t x = tok[k];
    bool keep = false;
    if (x < 0 || x >= vocab) {
      record_bad_token(err, x, vocab);
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
  const float* q = j < n && draft ? draft + b * d_sb + j * d_sk : nullptr;
  const int64_t x = j < n && !draft ? tok[j] : -1;
  const float* e = race + b * vocab;
  unsigned long long k = 0ull;
  for (int pass = 0; pass < 2; ++pass) {  // the second from p alone, if nothing was left
    for (int64_t v = threadIdx.x; v < vocab; v += blockDim.x) {
      float w = p[v];
      if (pass == 0) w = q ? __fsub_rn(w, q[v]) : v == x ? 0.0f : w;
      k = max(k, race_key(w, e[v], (uint32_t)v));
    }
    k = warp_max_key(k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = k;
    __syncthreads();
    k = 0ull;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) k = max(k, best[w]);
    if (k != 0ull) break;
  }
  const int64_t next = k ? (int64_t)(0xffffffffu - (uint32_t)k) : -1;
  for (int i = threadIdx.x; i <= drafted; i += blockDim.x)
    out_tokens[b * (drafted + 1) + i] = i < j ? tok[i] : i == j ? next : -1;
  if (threadIdx.x == 0) accepted[b] = j;
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
  verify_kernel<<<(unsigned)batch, 512, 0, s>>>(target, target_sb, target_sk, draft, draft_sb,
                                                draft_sk, tokens, lengths, uniform, race,
                                                (int)drafted, vocab, out_tokens, accepted,
                                                err_flag);
  return check_launch("oxc_verify_draft");
}

}  // extern "C"
