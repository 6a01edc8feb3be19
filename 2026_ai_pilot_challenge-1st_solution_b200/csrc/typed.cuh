// typed.cuh -- loads and stores of fp32 / bf16 / fp16 values as fp32, one by one or as vectors.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace f16 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <int BYTES> struct RawVec;
template <> struct RawVec<2> { typedef unsigned short type; };
template <> struct RawVec<4> { typedef unsigned type; };
template <> struct RawVec<8> { typedef uint2 type; };
template <> struct RawVec<16> { typedef uint4 type; };

// V values of type T in one register vector (V * sizeof(T) = 2, 4, 8 or 16 bytes, aligned to that).
template <typename T, int V>
union Vec {
  typedef typename RawVec<V * (int)sizeof(T)>::type raw;
  raw r;
  T e[V];
  __device__ __forceinline__ Vec() {}
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  Vec<T, V> v;
  v.r = *reinterpret_cast<const typename Vec<T, V>::raw*>(p);
  return v;
}
// Read-once data (never written while the kernel runs).
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec_nc(const T* p) {
  Vec<T, V> v;
  v.r = __ldg(reinterpret_cast<const typename Vec<T, V>::raw*>(p));
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& v) {
  *reinterpret_cast<typename Vec<T, V>::raw*>(p) = v.r;
}

inline cudaStream_t cu_stream(f16_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace f16
