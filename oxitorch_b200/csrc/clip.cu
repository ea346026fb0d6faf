// clip.cu -- the norm over many tensors, and all of them scaled where it is too large.
//
//   norm = sqrt(sum over tensors of sum g^2)
//   g = g * (max_norm / (norm + 1e-6)) where that factor is below 1
//
// Two launches for up to kClipTensors tensors of f32 and bf16 mixed, without a host
// round trip: the tensors' addresses and sizes are kernel arguments, so a captured
// graph holds them.  Tensors are cut into chunks, the chunks dealt to a grid of
// resident CTAs.  The first kernel leaves a sum of squares per CTA in f64 (a square of
// an f32 neither overflows nor vanishes there); every CTA of the second adds up all of
// these in one order, so all have the same factor, and scales the chunks from the
// last to the first: the last ones read are still in L2.
//
// Bound by HBM: each element is read for the norm, and read again and written for the
// scaling; the second read comes from L2 as far as that goes (126 MB).  473 million f32:
// the norm 270 us, with the scaling 944 to 982, 88 to 92% of the copy bandwidth for three
// passes; 83 tensors of a small model 11 us in a captured graph (79 by the host).
#include <algorithm>
#include <new>

#include "typed.cuh"

namespace oxc {

constexpr int kClipThreads = 512;
constexpr int kClipBytes = 32768;     // of a chunk
constexpr int kClipTensors = 640;     // per launch: 18 KB of arguments

struct ClipTensor {
  const void* in;
  void* out;
  int64_t n;
};

template <int CAP>
struct ClipList {
  ClipTensor t[CAP];
  int first[CAP + 1];        // its first chunk
  unsigned int bf[(CAP + 31) / 32];  // a bit for each bf16 tensor
  int count;
  __device__ __forceinline__ bool is_bf16(int i) const { return bf[i / 32] >> (i % 32) & 1u; }
  __device__ __forceinline__ int find(int chunk) const {  // the tensor of a chunk
    int lo = 0, hi = count;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first[mid] <= chunk) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t n) {
  constexpr int kVec = 16 / sizeof(T), U = 4;
  double a[2] = {0.0, 0.0};
  auto add = [&](const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        const double v = (double)__uint_as_float(w[i]);
        a[i & 1] = fma(v, v, a[i & 1]);
      } else {
        const double lo = (double)bf16_lo(w[i]), hi = (double)bf16_hi(w[i]);
        a[0] = fma(lo, lo, a[0]);
        a[1] = fma(hi, hi, a[1]);
      }
    }
  };
  int64_t i = threadIdx.x;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const uint4* v = reinterpret_cast<const uint4*>(p);
    const int64_t nv = n / kVec;
    for (; i + (U - 1) * kClipThreads < nv; i += U * kClipThreads) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = __ldg(v + i + u * kClipThreads);
#pragma unroll
      for (int u = 0; u < U; ++u) add(q[u]);
    }
    for (; i < nv; i += kClipThreads) add(__ldg(v + i));
    i = nv * kVec + threadIdx.x;
  }
  for (; i < n; i += kClipThreads) {
    const double v = (double)to_f32(p[i]);
    a[0] = fma(v, v, a[0]);
  }
  return a[0] + a[1];
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads)
clip_squares_kernel(const __grid_constant__ ClipList<CAP> list, double* __restrict__ sums) {
  __shared__ double scratch[33];
  double s = 0.0;
  const int chunks = list.first[list.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = list.find(c);
    const ClipTensor t = list.t[i];
    const bool half = list.is_bf16(i);
    const int64_t each = kClipBytes / (half ? 2 : 4), from = (int64_t)(c - list.first[i]) * each;
    const int64_t n = min(each, t.n - from);
    s += half ? chunk_squares(static_cast<const bf16*>(t.in) + from, n)
              : chunk_squares(static_cast<const float*>(t.in) + from, n);
  }
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
  pdl_launch_dependents();
}

// The squares' total, the same in every thread of every CTA.
__device__ __forceinline__ double total_squares(const double* sums, int n, double* scratch) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) s += sums[i];
  return block_sum(s, scratch);
}

// F: float, or double for factors that f32 does not hold.
template <typename T, typename F>
__device__ __forceinline__ void chunk_scale(const T* p, T* out, int64_t n, F f) {
  constexpr int kVec = 16 / sizeof(T), U = 4;
  int64_t i = threadIdx.x;
  auto times = [f](float v) { return (float)((F)v * f); };
  auto scaled = [&](const uint4& q) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(times(__uint_as_float(w[k])));
      else w[k] = pack_bf16(times(bf16_lo(w[k])), times(bf16_hi(w[k])));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
    const uint4* v = reinterpret_cast<const uint4*>(p);
    uint4* o = reinterpret_cast<uint4*>(out);
    const int64_t nv = n / kVec;
    for (; i + (U - 1) * kClipThreads < nv; i += U * kClipThreads) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = __ldcs(v + i + u * kClipThreads);
#pragma unroll
      for (int u = 0; u < U; ++u) __stcs(o + i + u * kClipThreads, scaled(q[u]));
    }
    for (; i < nv; i += kClipThreads) __stcs(o + i, scaled(__ldcs(v + i)));
    i = nv * kVec + threadIdx.x;
  }
  for (; i < n; i += kClipThreads) out[i] = from_f32<T>(times(to_f32(p[i])));
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads)
clip_scale_kernel(const __grid_constant__ ClipList<CAP> list, const double* __restrict__ sums,
                  int nsums, double max_norm, float* __restrict__ norm_out) {
  __shared__ double scratch[33];
  pdl_wait();
  const double norm = sqrt(total_squares(sums, nsums, scratch));
  if (blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
  const double factor = max_norm / (norm + 1e-6);
  const bool scale = factor < 1.0;  // not with a NaN
  const float f = scale ? (float)factor : 1.0f;
  // large gradients clipped to a small norm: in f32 such a factor has few bits or none
  const bool tiny = factor > 0.0 && factor < 0x1p-126;
  const int chunks = list.first[list.count];
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= (int)gridDim.x) {
    const int i = list.find(c);
    const ClipTensor t = list.t[i];
    if (!scale && t.in == t.out) continue;
    const bool half = list.is_bf16(i);
    const int64_t each = kClipBytes / (half ? 2 : 4), from = (int64_t)(c - list.first[i]) * each;
    const int64_t n = min(each, t.n - from);
    auto by = [&](auto factor) {
      if (half)
        chunk_scale(static_cast<const bf16*>(t.in) + from, static_cast<bf16*>(t.out) + from, n, factor);
      else
        chunk_scale(static_cast<const float*>(t.in) + from, static_cast<float*>(t.out) + from, n, factor);
    };
    if (tiny) by(factor);
    else by(f);
  }
}

__global__ void __launch_bounds__(kClipThreads)
clip_norm_kernel(const double* __restrict__ sums, int nsums, float* __restrict__ norm_out) {
  __shared__ double scratch[33];
  pdl_wait();
  const double s = total_squares(sums, nsums, scratch);
  if (threadIdx.x == 0) norm_out[0] = (float)sqrt(s);
}

static int64_t clip_chunks(int64_t n, int32_t dtype) {
  const int64_t each = kClipBytes / (dtype == OXC_BF16 ? 2 : 4);
  return (n + each - 1) / each;
}

static int clip_ctas() { return sm_count() * 4; }  // 2048 threads an SM
static int64_t clip_launches(int64_t count) { return std::max<int64_t>(1, (count + kClipTensors - 1) / kClipTensors); }

// The arguments of a launch for tensors [from, to).
template <int CAP>
static oxc_status clip_list(ClipList<CAP>& list, const int64_t* in, const int64_t* out,
                            const int64_t* sizes, const int32_t* dtypes, int64_t from, int64_t to) {
  list.count = 0;
  int64_t chunks = 0;
  for (unsigned int& w : list.bf) w = 0u;
  for (int64_t i = from; i < to; ++i) {
    if (sizes[i] == 0) continue;
    const int k = list.count++;
    list.t[k] = {reinterpret_cast<const void*>(in[i]),
                 reinterpret_cast<void*>(out ? out[i] : in[i]), sizes[i]};
    list.first[k] = (int)chunks;
    if (dtypes[i] == OXC_BF16) list.bf[k / 32] |= 1u << (k % 32);
    chunks += clip_chunks(sizes[i], dtypes[i]);
    if (chunks > 0x7fffffff / 2)
      return fail(OXC_ERR_NOT_IMPLEMENTED, "not implemented: clip_global_norm: tensors beyond 2^30 chunks");
  }
  list.first[list.count] = (int)chunks;
  return OXC_OK;
}

template <typename... KArgs, typename... Args>
static cudaError_t clip_launch(void (*kernel)(KArgs...), int grid, bool dependent, cudaStream_t s,
                               const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kClipThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int CAP>
static oxc_status clip_run(const int64_t* in, const int64_t* out, const int64_t* sizes,
                           const int32_t* dtypes, int64_t count, bool clip, double max_norm,
                           float* norm, double* sums, cudaStream_t s) {
  static thread_local ClipList<CAP> list;  // too large for some stacks
  const int64_t launches = clip_launches(count);
  int64_t nsums = 0;
  for (int64_t l = 0; l < launches; ++l) {
    const oxc_status st = clip_list(list, in, out, sizes, dtypes, l * kClipTensors,
                                    std::min<int64_t>(count, (l + 1) * kClipTensors));
    if (st) return st;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(clip_ctas(), list.first[list.count]));
    const cudaError_t e = clip_launch(clip_squares_kernel<CAP>, grid, false, s, list, sums + nsums);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_clip_global_norm");
    nsums += grid;
  }
  if (!clip) {
    const cudaError_t e = clip_launch(clip_norm_kernel, 1, true, s, (const double*)sums, (int)nsums, norm);
    return e == cudaSuccess ? OXC_OK : cuda_fail(e, "oxc_clip_global_norm");
  }
  for (int64_t l = launches - 1; l >= 0; --l) {  // the last tensors first
    if (launches > 1) {
      const oxc_status st = clip_list(list, in, out, sizes, dtypes, l * kClipTensors,
                                      std::min<int64_t>(count, (l + 1) * kClipTensors));
      if (st) return st;
    }
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(clip_ctas(), list.first[list.count]));
    const cudaError_t e = clip_launch(clip_scale_kernel<CAP>, grid, l == launches - 1, s, list,
                                      (const double*)sums, (int)nsums, max_norm, norm);
    if (e != cudaSuccess) return cuda_fail(e, "oxc_clip_global_norm");
  }
  return check_launch("oxc_clip_global_norm");
}

struct ClipRange {
  uint64_t from, to;
};

// Refuses tensors that share memory: scaled side by side, an element of two of them
// would be written twice.  An output may be its own input.
static oxc_status clip_apart(const int64_t* in, const int64_t* out, const int64_t* sizes,
                             const int32_t* dtypes, int64_t count) {
  ClipRange* r = new (std::nothrow) ClipRange[(size_t)(2 * count + 1)];
  if (!r) return fail(OXC_ERR_OTHER, "clip_global_norm: out of host memory");
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    const uint64_t bytes = (uint64_t)sizes[i] * (dtypes[i] == OXC_BF16 ? 2 : 4);
    if (!bytes) continue;
    r[n++] = {(uint64_t)in[i], (uint64_t)in[i] + bytes};
    if (out && out[i] != in[i]) r[n++] = {(uint64_t)out[i], (uint64_t)out[i] + bytes};
  }
  std::sort(r, r + n, [](const ClipRange& a, const ClipRange& b) { return a.from < b.from; });
  bool apart = true;
  for (int64_t i = 1; i < n; ++i) apart = apart && r[i - 1].to <= r[i].from;
  delete[] r;
  return apart ? OXC_OK
               : fail(OXC_ERR_INVALID_ARGUMENT,
                      "invalid argument: clip_global_norm: tensors overlap, or one is listed twice");
}

static oxc_status clip_call(const int64_t* in, const int64_t* out, const int64_t* sizes,
                            const int32_t* dtypes, int64_t count, bool clip, double max_norm,
                            float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0)
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: %lld tensors", (long long)count);
  if (!norm || (count > 0 && (!in || !sizes || !dtypes)))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: null pointer");
  for (int64_t i = 0; i < count; ++i) {
    if (!known_dtype(dtypes[i]))
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: unknown dtype %d", dtypes[i]);
    if (sizes[i] < 0)
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: negative size");
    if (sizes[i] > 0 && (!in[i] || (out && !out[i])))
      return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: null pointer");
  }
  if (!workspace || workspace_bytes < oxc_clip_global_norm_workspace_size(count))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: workspace too small");
  if (clip) {
    const oxc_status st = clip_apart(in, out, sizes, dtypes, count);
    if (st) return st;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  double* sums = static_cast<double*>(workspace);
  // short lists as arguments of 3 KB instead of 17, copied twice by the host (83 tensors 80.6
  // us a call for 83.4, 10 tensors 26 for 28; on the device 0.1 us less)
  return count <= 96 ? clip_run<96>(in, out, sizes, dtypes, count, clip, max_norm, norm, sums, s)
                     : clip_run<kClipTensors>(in, out, sizes, dtypes, count, clip, max_norm, norm, sums, s);
}

}  // namespace oxc

using namespace oxc;

extern "C" {

size_t oxc_clip_global_norm_workspace_size(int64_t count) {
  return count < 0 ? 0 : (size_t)clip_launches(count) * (size_t)clip_ctas() * sizeof(double);
}

oxc_status oxc_global_norm(const int64_t* tensors, const int64_t* sizes, const int32_t* dtypes,
                           int64_t count, float* norm, void* workspace, size_t workspace_bytes,
                           void* stream) {
  return clip_call(tensors, nullptr, sizes, dtypes, count, false, 0.0, norm, workspace,
                   workspace_bytes, stream);
}

oxc_status oxc_clip_global_norm(const int64_t* grads, const int64_t* out, const int64_t* sizes,
                                const int32_t* dtypes, int64_t count, double max_norm, float* norm,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (!(max_norm >= 0.0))
    return fail(OXC_ERR_INVALID_ARGUMENT, "invalid argument: clip_global_norm: max_norm %g", max_norm);
  return clip_call(grads, out, sizes, dtypes, count, true, max_norm, norm, workspace,
                   workspace_bytes, stream);
}

}  // extern "C"
