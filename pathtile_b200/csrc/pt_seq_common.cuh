// pt_seq_common.cuh -- element types, vector access and elementwise functions
// of the sequence operators' kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "pathtile_b200.h"

namespace pt {
namespace seq {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// E consecutive elements as they lie in memory: moved in words of up to 16 bytes.
template <class T, int E>
struct Pack {
  static constexpr int kBytes = E * static_cast<int>(sizeof(T));
  static constexpr int kWord = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : static_cast<int>(sizeof(T));
  alignas(kBytes >= 16 ? 16 : kWord) T v[E];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = from_f<T>(0.f);
  }
  // The first n of E elements (the others become 0); `vec`: p is aligned to kWord bytes.
  __device__ __forceinline__ void load(const T* __restrict__ p, int n, bool vec) {
    if (vec && n >= E) {
      if constexpr (kWord == 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
      } else if constexpr (kWord == 8) {
#pragma unroll
        for (int i = 0; i < kBytes / 8; ++i) reinterpret_cast<uint2*>(v)[i] = __ldg(reinterpret_cast<const uint2*>(p) + i);
      } else if constexpr (kWord == 4) {
#pragma unroll
        for (int i = 0; i < kBytes / 4; ++i)
          reinterpret_cast<unsigned*>(v)[i] = __ldg(reinterpret_cast<const unsigned*>(p) + i);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = p[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = i < n ? p[i] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(T* p, int n, bool vec) const {
    if (vec && n >= E) {
      if constexpr (kWord == 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
      } else if constexpr (kWord == 8) {
#pragma unroll
        for (int i = 0; i < kBytes / 8; ++i) reinterpret_cast<uint2*>(p)[i] = reinterpret_cast<const uint2*>(v)[i];
      } else if constexpr (kWord == 4) {
#pragma unroll
        for (int i = 0; i < kBytes / 4; ++i) reinterpret_cast<unsigned*>(p)[i] = reinterpret_cast<const unsigned*>(v)[i];
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] = v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i < n) p[i] = v[i];
    }
  }
  __device__ __forceinline__ float f(int i) const { return to_f<T>(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = from_f<T>(x); }
};

// A parameter in fp32 or in the activations' type.
template <class T>
__device__ __forceinline__ float param(const void* p, long long i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : to_f<T>(static_cast<const T*>(p)[i]);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / (1 + e^-v).  The fast division returns 0 for divisors past 2^126, where
// the quotient is below 2^-126.
__device__ __forceinline__ float sigmoidf(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }
__device__ __forceinline__ float siluf(float v) { return __fdividef(v, 1.f + __expf(-v)); }
// d silu(v) / dv, with s = sigmoid(v).
__device__ __forceinline__ float silu_grad(float v, float s) { return s * (1.f + v * (1.f - s)); }
// log(1 + e^v); past 20 the 1 is below half a step of e^v.
__device__ __forceinline__ float softplusf(float v) { return v > 20.f ? v : log1pf(__expf(v)); }

// A row's state slot: -1 where there is none to touch.  Every thread of the
// block calls it.  A slot at or past the cache's end (bit 7 of the device error
// word) or one that an earlier row of the batch names too (bit 8) has none, so
// no row writes outside the cache and no two rows write one state.
__device__ __forceinline__ int slot_of(const int* __restrict__ slots, int row, int cache_rows, unsigned* err,
                                       int thread, int threads) {
  const int s = __ldg(slots + row);
  if (s < 0) return -1;
  if (s >= cache_rows) {
    if (thread == 0) atomicOr(err, 128u);
    return -1;
  }
  int twice = 0;
  for (int i = thread; i < row; i += threads) twice |= __ldg(slots + i) == s;
  if (__syncthreads_or(twice)) {
    if (thread == 0) atomicOr(err, 256u);
    return -1;
  }
  return s;
}

// Calls fn(T()) for the element type `dtype`.
template <class F>
inline cudaError_t by_type(int dtype, F&& fn) {
  switch (dtype) {
    case PT_F32: return fn(float());
    case PT_BF16: return fn(__nv_bfloat16());
    case PT_F16: return fn(__half());
    default: return cudaErrorInvalidValue;
  }
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

}  // namespace seq
}  // namespace pt
