// Element types of the training-step operators (vcb_dtype): conversion to and
// from fp32 and 4-element vector access.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "vcb.h"

namespace vcb {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Four consecutive elements; p is aligned to 4 elements.
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 t = *reinterpret_cast<const float4*>(p);
  v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
}

template <typename T>  // the 16-bit types
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  T e[4];
  *reinterpret_cast<uint2*>(e) = t;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
}

__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
}

// As store4, marked to leave L2 first.
__device__ __forceinline__ void store4_stream(float* p, const float (&v)[4]) {
  __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
}

template <typename T>
__device__ __forceinline__ void store4_stream(T* p, const float (&v)[4]) {
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
  __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(e));
}

inline bool valid_dtype(int t) { return t == VCB_F32 || t == VCB_BF16 || t == VCB_F16; }
inline int dtype_bytes(int t) { return t == VCB_F32 ? 4 : 2; }

}  // namespace vcb
