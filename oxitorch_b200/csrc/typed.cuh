// typed.cuh -- f32 / bf16 element access for the layers that take both.
//
// Activations and logits may be float32 or bfloat16 (OXC_F32 / OXC_BF16); all
// arithmetic is in f32 and a bf16 result is rounded once (to nearest, ties to
// even) when it is stored.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace oxc {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

// The two bf16 values of a 32-bit word, low half first.
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// VW consecutive elements as f32, evict-first; VW > 1 needs VW * sizeof(T)
// alignment.  VW = 1, 2 or 4, and 8 for storing bf16.
template <int VW>
__device__ __forceinline__ void load_as_f32(float (&d)[VW], const float* p) {
  if constexpr (VW == 4) {
    const float4 t = ld_stream(reinterpret_cast<const float4*>(p));
    d[0] = t.x; d[1] = t.y; d[2] = t.z; d[3] = t.w;
  } else if constexpr (VW == 2) {
    const float2 t = __ldcs(reinterpret_cast<const float2*>(p));
    d[0] = t.x; d[1] = t.y;
  } else {
    static_assert(VW == 1, "f32 vectors hold 1, 2 or 4 elements");
    d[0] = ld_stream(p);
  }
}
template <int VW>
__device__ __forceinline__ void load_as_f32(float (&d)[VW], const bf16* p) {
  if constexpr (VW == 4) {
    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
    d[0] = bf16_lo(t.x); d[1] = bf16_hi(t.x); d[2] = bf16_lo(t.y); d[3] = bf16_hi(t.y);
  } else if constexpr (VW == 2) {
    const uint32_t t = __ldcs(reinterpret_cast<const uint32_t*>(p));
    d[0] = bf16_lo(t); d[1] = bf16_hi(t);
  } else {
    static_assert(VW == 1, "bf16 vectors hold 1, 2 or 4 elements");
    d[0] = bf16_lo(__ldcs(reinterpret_cast<const unsigned short*>(p)));
  }
}
template <int VW>
__device__ __forceinline__ void store_from_f32(float* p, const float (&d)[VW]) {
  if constexpr (VW == 4) {
    st_stream(reinterpret_cast<float4*>(p), make_float4(d[0], d[1], d[2], d[3]));
  } else if constexpr (VW == 2) {
    __stcs(reinterpret_cast<float2*>(p), make_float2(d[0], d[1]));
  } else {
    static_assert(VW == 1, "f32 vectors hold 1, 2 or 4 elements");
    st_stream(p, d[0]);
  }
}
template <int VW>
__device__ __forceinline__ void store_from_f32(bf16* p, const float (&d)[VW]) {
  if constexpr (VW == 8) {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack_bf16(d[0], d[1]), pack_bf16(d[2], d[3]),
                                                   pack_bf16(d[4], d[5]), pack_bf16(d[6], d[7])));
  } else if constexpr (VW == 4) {
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack_bf16(d[0], d[1]), pack_bf16(d[2], d[3])));
  } else if constexpr (VW == 2) {
    __stcs(reinterpret_cast<uint32_t*>(p), pack_bf16(d[0], d[1]));
  } else {
    static_assert(VW == 1, "bf16 vectors hold 1, 2, 4 or 8 elements");
    __stcs(reinterpret_cast<unsigned short*>(p), __bfloat16_as_ushort(__float2bfloat16_rn(d[0])));
  }
}

inline bool known_dtype(int32_t t) { return t == OXC_F32 || t == OXC_BF16; }
inline bool aligned_to(const void* p, size_t n) {
  return reinterpret_cast<uintptr_t>(p) % n == 0;
}

}  // namespace oxc
