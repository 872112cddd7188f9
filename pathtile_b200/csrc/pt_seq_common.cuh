// pt_seq_common.cuh -- element types, vector access and elementwise functions
// of the sequence operators' kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

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

// Two floats in a 64-bit register pair, for the packed fp32 instructions.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lo2(F2 v) {
  return __uint_as_float(static_cast<unsigned>(v));
}
__device__ __forceinline__ float hi2(F2 v) {
  return __uint_as_float(static_cast<unsigned>(v >> 32));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
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
  // Elements 2 i and 2 i + 1 (of a single element: itself and 0).
  __device__ __forceinline__ F2 pair(int i) const {
    if constexpr (E == 1) {
      return pack2(to_f<T>(v[0]), 0.f);
    } else if constexpr (sizeof(T) == 4) {
      return pack2(v[2 * i], v[2 * i + 1]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const unsigned w = reinterpret_cast<const unsigned*>(v)[i];
      return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
      const float2 w = __half22float2(reinterpret_cast<const __half2*>(v)[i]);
      return pack2(w.x, w.y);
    }
  }
  __device__ __forceinline__ void set_pair(int i, F2 x) {
    if constexpr (E == 1) {
      v[0] = from_f<T>(lo2(x));
    } else if constexpr (sizeof(T) == 4) {
      v[2 * i] = lo2(x), v[2 * i + 1] = hi2(x);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      reinterpret_cast<__nv_bfloat162*>(v)[i] = __floats2bfloat162_rn(lo2(x), hi2(x));
    } else {
      reinterpret_cast<__half2*>(v)[i] = __floats2half2_rn(lo2(x), hi2(x));
    }
  }
  static constexpr int kPairs = (E + 1) / 2;
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

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ F2 ex2x2(F2 x) { return pack2(ex2(lo2(x)), ex2(hi2(x))); }
__device__ __forceinline__ F2 same2(float v) { return pack2(v, v); }
__device__ __forceinline__ float sum2(F2 v) { return lo2(v) + hi2(v); }
__device__ __forceinline__ F2 rcp2(F2 v) { return pack2(rcp(lo2(v)), rcp(hi2(v))); }

// The larger and the smaller of two; a NaN stays one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e^a for -150 <= a < 88.5.  2^m with m = a log2 e rounded is e^(m ln 2), off by a relative
// a - m ln 2 (up to |a| 2^-24): that is known to more bits than it needs, ln 2 taken as
// the sum of two floats, and given back with one more multiplication.
__device__ __forceinline__ F2 exp2x(F2 a) {
  const F2 m = mul2(a, same2(kLog2e));
  const F2 r = fma2(m, same2(1.9046543e-9f), fma2(m, same2(-kLn2), a));
  const F2 e = ex2x2(m);
  return fma2(e, r, e);
}

// What activations of type T are computed from: in fp32 to a few half steps (2^-24 of
// the value) over the whole range (the largest error of silu from -80 to 80 was 62 half
// steps without, its bound is 9 now; the scan of 8 x 2048 x 2048 channels takes 264 us for
// 258, the memory-bound kernels what they took).  For bf16 and fp16, whose outputs are
// rounded at 2^-9 or 2^-12, the exponent is rounded once: |v| 2^-24 of the value, which
// their fp32 states and streams carry too.  (Without that choice 8 x 2048 x 4096 of
// convolution training takes 172 us for 160, gated norm training 218 for 208, scan
// training 1048 for 1033; softplus alone 1037.)
template <class T>
constexpr bool kFullExp = sizeof(T) == 4;

// 1 / (1 + e^-v), 0 for v < -87.3.  The reciprocal of infinity (16-bit types), and of what is past
// 2^126, is 0, so large negative v need no care.
template <class T>
__device__ __forceinline__ F2 sigmoid2(F2 v) {
  F2 e;
  if constexpr (kFullExp<T>)
    e = exp2x(pack2(max_nan(min_nan(-lo2(v), 88.4f), -120.f), max_nan(min_nan(-hi2(v), 88.4f), -120.f)));
  else
    e = ex2x2(mul2(v, same2(-kLog2e)));
  return rcp2(add2(e, same2(1.f)));
}
template <class T>
__device__ __forceinline__ float siluf(float v) { return v * lo2(sigmoid2<T>(same2(v))); }
// d silu(v) / dv, with s = sigmoid(v): s (1 + v (1 - s)).
__device__ __forceinline__ F2 silu_grad2(F2 v, F2 s) {
  return mul2(s, fma2(v, fma2(s, same2(-1.f), same2(1.f)), same2(1.f)));
}

// log(1 + e^v).  With e = e^-|v| <= 1 it is max(v, 0) + log(1 + e), and
// log(1 + e) = 2 artanh(s), s = e / (2 + e) <= 1/3: the odd series up to s^13
// leaves s^14 / 15 < 2e-8 of the value, so small results keep their relative
// precision (log(1 + e) computed as such would not).
template <class T>
__device__ __forceinline__ F2 softplus2(F2 v) {
  F2 e;
  if constexpr (kFullExp<T>) {
    e = exp2x(pack2(max_nan(-fabsf(lo2(v)), -120.f), max_nan(-fabsf(hi2(v)), -120.f)));
  } else {
    const F2 m = mul2(v, same2(kLog2e));
    e = pack2(ex2(-fabsf(lo2(m))), ex2(-fabsf(hi2(m))));
  }
  const F2 s = mul2(e, rcp2(add2(e, same2(2.f)))), q = mul2(s, s);
  F2 p = fma2(q, same2(1.f / 13.f), same2(1.f / 11.f));
  p = fma2(p, q, same2(1.f / 9.f));
  p = fma2(p, q, same2(1.f / 7.f));
  p = fma2(p, q, same2(1.f / 5.f));
  p = fma2(p, q, same2(1.f / 3.f));
  p = fma2(p, q, same2(1.f));
  // A NaN stays one: fmaxf would drop it, e carries it.
  return fma2(add2(s, s), p, pack2(fmaxf(lo2(v), 0.f), fmaxf(hi2(v), 0.f)));
}
template <class T>
__device__ __forceinline__ float softplusf(float v) { return lo2(softplus2<T>(same2(v))); }

// Copies of 4, 8 or 16 bytes from global to shared memory that run on while the thread works.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* smem, const void* gmem) {
  const unsigned dst = static_cast<unsigned>(__cvta_generic_to_shared(smem));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(gmem) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(gmem), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// E floats of shared memory in packed pairs (16-byte aligned where E is 4 or more).
template <int E>
__device__ __forceinline__ void put_pairs(float* dst, const F2 (&v)[(E + 1) / 2]) {
  if constexpr (E == 1) {
    *dst = lo2(v[0]);
  } else if constexpr (E == 2) {
    *reinterpret_cast<F2*>(dst) = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) reinterpret_cast<ulonglong2*>(dst)[i] = make_ulonglong2(v[2 * i], v[2 * i + 1]);
  }
}
template <int E>
__device__ __forceinline__ void get_pairs(const float* src, F2 (&v)[(E + 1) / 2]) {
  if constexpr (E == 1) {
    v[0] = pack2(*src, 0.f);
  } else if constexpr (E == 2) {
    v[0] = *reinterpret_cast<const F2*>(src);
  } else {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const ulonglong2 f = reinterpret_cast<const ulonglong2*>(src)[i];
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

// A row of a batch whose slot lies past the cache, or was named by an earlier row
// too, is treated as padding and sets a bit of the device error word: no row
// writes outside the cache, and no two rows write one state.
constexpr unsigned kSlotPastCache = 1u << 7, kSlotTwice = 1u << 8;

// Whether a row before `row` names the slot as well.  Every thread of the block calls it.
// Every block of a row reads the slots of all rows before it, which grows with the square
// of the batch.  Steps of 2048 channels (16 states, 4 taps, bf16) without and with slots:
// 256 rows, scan 20.1 and 22.5 us, convolution 8.2 and 10.2; 4096 rows, 188 and 274, 35 and
// 53; 16384 rows, 723 and 1966, 117 and 295.
__device__ __forceinline__ bool named_before(const int* __restrict__ slots, int row, int slot, int thread, int threads) {
  int twice = 0;
  if (slot >= 0)
    for (int i = thread; i < row; i += threads) twice |= __ldg(slots + i) == slot;
  return __syncthreads_or(twice);
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
