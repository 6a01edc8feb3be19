// typed.cuh -- loads and stores of fp32 / bf16 / fp16 values as fp32, one by one or as vectors.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
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

// Two fp32 values in a register pair, computed with by one instruction (each rounded by itself, to nearest).
struct Two {
  unsigned long long r;
};
__device__ __forceinline__ Two two(float x, float y) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.r) : "f"(x), "f"(y));
  return t;
}
__device__ __forceinline__ Two two(float x) { return two(x, x); }
__device__ __forceinline__ void split(Two t, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(t.r)); }
__device__ __forceinline__ float2 split(Two t) {
  float2 f;
  split(t, f.x, f.y);
  return f;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two t;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(t.r) : "l"(a.r), "l"(b.r));
  return t;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two t;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.r) : "l"(a.r), "l"(b.r));
  return t;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two t;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.r) : "l"(a.r), "l"(b.r), "l"(c.r));
  return t;
}

// The pair i (values 2 i and 2 i + 1) of a register vector as fp32, and the way back (rounded to nearest).
template <typename T, int V>
__device__ __forceinline__ Two pair_of(const Vec<T, V>& v, int i) {
  const unsigned* w = reinterpret_cast<const unsigned*>(&v);
  if constexpr (std::is_same<T, float>::value) {
    return two(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  } else if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
    return two(f.x, f.y);
  } else {
    return two(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
}
template <typename T, int V>
__device__ __forceinline__ void set_pair(Vec<T, V>& v, int i, Two t) {
  const float2 f = split(t);
  unsigned* w = reinterpret_cast<unsigned*>(&v);
  if constexpr (std::is_same<T, float>::value) {
    w[2 * i] = __float_as_uint(f.x);
    w[2 * i + 1] = __float_as_uint(f.y);
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const unsigned*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const unsigned*>(&h);
  }
}

inline cudaStream_t cu_stream(f16_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace f16
