// pt_seq_norm.cu -- root-mean-square norm fused with what stands around it:
//   u = x silu(gate);  r = residual + scale u;  y = r / sqrt(mean(r^2) + eps) weight
// with the mean over each of `groups` equal parts of a row; forward and backward.
//
// A block holds one part of a row in registers (V x NV elements per thread), so
// each tensor is read once and written once: the kernels are bound by memory.
// A block keeps its group of columns and walks rows, with the weights (and,
// backward, the sums of dweight and dscale) in registers.  V is a 16-byte word
// of activations where all rows and widths allow it, else one element.
//
// Backward, with hat = r rstd and v = dy weight:
//   dr = rstd (v - hat mean(v hat)) + dr_in;  dx = dr scale silu(gate), ...
// mean(r^2) and mean(v r) come from one reduction.  dweight and dscale: one
// partial sum per block, added in a fixed order by a second kernel.
//
// 16384 x 4096 in 8 groups, gated, bf16: forward 65 us (6.2 TB/s), backward 130
// (5.2 TB/s), with issue slots 70 % busy.  8191 x 1027, residual in fp32 and scale,
// single elements: 24 and 53 us.
#include <type_traits>

#include "pt_seq.h"
#include "pt_seq_common.cuh"

namespace pt {
namespace seq {
namespace {

// What is fused: the common forms have kernels of their own (registers), any
// other combination runs the general one.
enum NormForm { kGated, kResidual, kAny };

// What a thread holds of a row: NV words of V elements, `threads` words apart, as
// packed pairs (neighbours in a word; of single elements, two words' together).
// Words past the row's end are zeros.
template <int V, int NV>
struct Words {
  static_assert(V * NV % 2 == 0, "whole pairs");
  static constexpr int N = V * NV / 2;

  template <class T>
  static __device__ __forceinline__ void load(Pack<T, V> (&w)[NV], const T* row, int width) {
    const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width)
        w[k].load(row + i, V, true);
      else
        w[k].zero();
    }
  }
  template <class T>
  static __device__ __forceinline__ void store(const Pack<T, V> (&w)[NV], T* row, int width) {
    const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) w[k].store(row + i, V, true);
    }
  }
  template <class T>
  static __device__ __forceinline__ F2 get(const Pack<T, V> (&w)[NV], int q) {
    if constexpr (V > 1)
      return w[q / (V / 2)].pair(q % (V / 2));
    else
      return pack2(w[2 * q].f(0), w[2 * q + 1].f(0));
  }
  template <class T>
  static __device__ __forceinline__ void set(Pack<T, V> (&w)[NV], int q, F2 v) {
    if constexpr (V > 1)
      w[q / (V / 2)].set_pair(q % (V / 2), v);
    else
      w[2 * q].set(0, lo2(v)), w[2 * q + 1].set(0, hi2(v));
  }
  // Parameters in fp32 or the activations' type; zeros from no pointer.
  template <class T>
  static __device__ __forceinline__ void params(const void* p, int first, int width, bool f32, F2 (&out)[N]) {
    if (!p) {
#pragma unroll
      for (int q = 0; q < N; ++q) out[q] = 0;
    } else if (f32) {
      Pack<float, V> w[NV];
      load(w, static_cast<const float*>(p) + first, width);
#pragma unroll
      for (int q = 0; q < N; ++q) out[q] = get(w, q);
    } else {
      Pack<T, V> w[NV];
      load(w, static_cast<const T*>(p) + first, width);
#pragma unroll
      for (int q = 0; q < N; ++q) out[q] = get(w, q);
    }
  }
  // fp32, one row of a partial sum.
  static __device__ __forceinline__ void put(const F2 (&v)[N], float* row, int width) {
    Pack<float, V> w[NV];
#pragma unroll
    for (int q = 0; q < N; ++q) set(w, q, v[q]);
    const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) w[k].store(row + i, V, false);
    }
  }
};

// Sums of (p, q) over the block; `slot` alternates between calls, so that one
// barrier is enough.
__device__ __forceinline__ float2 block_sum(float p, float q, float2 (*buf)[32], int slot) {
#pragma unroll
  for (int m = 16; m >= 1; m /= 2) {
    p += __shfl_xor_sync(0xffffffffu, p, m);
    q += __shfl_xor_sync(0xffffffffu, q, m);
  }
  const int warps = static_cast<int>(blockDim.x) / 32;
  if (warps == 1) return make_float2(p, q);
  const int lane = static_cast<int>(threadIdx.x) & 31;
  if (lane == 0) buf[slot][threadIdx.x / 32] = make_float2(p, q);
  __syncthreads();
  const float2 v = lane < warps ? buf[slot][lane] : make_float2(0.f, 0.f);
  p = v.x, q = v.y;
#pragma unroll
  for (int m = 16; m >= 1; m /= 2) {
    p += __shfl_xor_sync(0xffffffffu, p, m);
    q += __shfl_xor_sync(0xffffffffu, q, m);
  }
  return make_float2(p, q);
}

// One part of a row as it lies in memory.
template <class T, class R, int V, int NV, int FORM>
struct NormRow {
  Pack<T, V> x[NV], gate[NV];
  Pack<R, V> res[NV];
};

template <class T, class R, int V, int NV, int FORM, int MAXT>
__global__ void __launch_bounds__(MAXT) seq_norm_fwd_kernel(pt_norm_args a, int width, long long stride) {
  using W = Words<V, NV>;
  __shared__ float2 buf[2][32];
  const int c0 = static_cast<int>(blockIdx.x % a.groups) * width;
  const bool gated = FORM == kGated || (FORM == kAny && a.gate);
  const bool resid = FORM == kResidual || (FORM == kAny && a.residual);
  const bool scaled = FORM != kGated && a.scale;
  F2 w[W::N], sc[W::N];
  W::template params<T>(a.weight, c0, width, a.param_f32, w);
  if (scaled) W::template params<T>(a.scale, c0, width, a.param_f32, sc);
  NormRow<T, R, V, NV, FORM> next;
  auto load = [&](long long row) {
    W::load(next.x, static_cast<const T*>(a.x) + row * a.x_row + c0, width);
    if (gated) W::load(next.gate, static_cast<const T*>(a.gate) + row * a.gate_row + c0, width);
    if (resid) W::load(next.res, static_cast<const R*>(a.residual) + row * a.residual_row + c0, width);
  };
  int slot = 0;
  long long row = blockIdx.x / a.groups;
  if (row < a.rows) load(row);
  for (; row < a.rows; row += stride, slot ^= 1) {
    NormRow<T, R, V, NV, FORM> in = next;
    if (row + stride < a.rows) load(row + stride);  // on its way while this row is worked on
    const long long o = row * a.dim + c0;
    F2 r[W::N], ss = 0;
#pragma unroll
    for (int q = 0; q < W::N; ++q) {
      F2 u = W::get(in.x, q);
      if (gated) {
        const F2 g = W::get(in.gate, q);
        u = mul2(u, mul2(g, sigmoid2<T>(g)));
      }
      if (scaled) u = mul2(u, sc[q]);
      if (resid) {
        // The stream that goes on is what is normalised: rounded to its type first.
        W::set(in.res, q, add2(W::get(in.res, q), u));
        u = W::get(in.res, q);
      }
      r[q] = u;
      ss = fma2(u, u, ss);
    }
    if (resid) W::store(in.res, static_cast<R*>(a.r) + o, width);
    const float rstd = rsqrtf(block_sum(sum2(ss), 0.f, buf, slot).x / static_cast<float>(width) + a.eps);
    Pack<T, V> out[NV];
#pragma unroll
    for (int q = 0; q < W::N; ++q) W::set(out, q, mul2(mul2(r[q], same2(rstd)), w[q]));
    W::store(out, static_cast<T*>(a.y) + o, width);
  }
}

template <class T, class R, int V, int NV, int FORM>
struct NormGradRow {
  Pack<T, V> dy[NV], x[NV], gate[NV];
  Pack<R, V> r[NV], dr[NV];
};

template <class T, class R, int V, int NV, int FORM, int MAXT>
__global__ void __launch_bounds__(MAXT) seq_norm_bwd_kernel(pt_norm_args a, float* part, int width, long long stride) {
  using W = Words<V, NV>;
  __shared__ float2 buf[2][32];
  const int c0 = static_cast<int>(blockIdx.x % a.groups) * width;
  const bool gated = FORM == kGated || (FORM == kAny && a.gate);
  const bool resid = FORM == kResidual || (FORM == kAny && a.residual);
  const bool scaled = FORM != kGated && a.scale;
  const bool need_x = !resid || gated || (scaled && a.dscale);
  const bool more = FORM != kGated && a.dr;
  F2 w[W::N], sc[W::N], dw[W::N], ds[W::N];
#pragma unroll
  for (int q = 0; q < W::N; ++q) dw[q] = ds[q] = 0;
  W::template params<T>(a.weight, c0, width, a.param_f32, w);
  if (scaled) W::template params<T>(a.scale, c0, width, a.param_f32, sc);
  NormGradRow<T, R, V, NV, FORM> next;
  auto load = [&](long long row) {
    W::load(next.dy, static_cast<const T*>(a.dy) + row * a.dy_row + c0, width);
    if (need_x) W::load(next.x, static_cast<const T*>(a.x) + row * a.x_row + c0, width);
    if (gated) W::load(next.gate, static_cast<const T*>(a.gate) + row * a.gate_row + c0, width);
    if (resid) W::load(next.r, static_cast<const R*>(a.r) + row * a.dim + c0, width);
    if (more) W::load(next.dr, static_cast<const R*>(a.dr) + row * a.dr_row + c0, width);
  };
  int slot = 0;
  long long row = blockIdx.x / a.groups;
  if (row < a.rows) load(row);
  for (; row < a.rows; row += stride, slot ^= 1) {
    const NormGradRow<T, R, V, NV, FORM> in = next;
    if (row + stride < a.rows) load(row + stride);  // on its way while this row is worked on
    const long long o = row * a.dim + c0;
    F2 r[W::N], ss = 0, sv = 0;
#pragma unroll
    for (int q = 0; q < W::N; ++q) {
      F2 u;
      if (resid) {
        u = W::get(in.r, q);
      } else {
        u = W::get(in.x, q);
        if (gated) {
          const F2 g = W::get(in.gate, q);
          u = mul2(u, mul2(g, sigmoid2<T>(g)));
        }
        if (scaled) u = mul2(u, sc[q]);
      }
      r[q] = u;
      ss = fma2(u, u, ss);
      sv = fma2(mul2(W::get(in.dy, q), w[q]), u, sv);
    }
    const float2 sums = block_sum(sum2(ss), sum2(sv), buf, slot);
    const float inv = 1.f / static_cast<float>(width);
    const float rstd = rsqrtf(fmaf(sums.x, inv, a.eps)), mean = sums.y * inv * rstd;  // mean(v hat)
    Pack<T, V> ox[NV], og[NV];
    Pack<R, V> ores[NV];
#pragma unroll
    for (int q = 0; q < W::N; ++q) {
      const F2 hat = mul2(r[q], same2(rstd)), y = W::get(in.dy, q);
      dw[q] = fma2(y, hat, dw[q]);
      F2 d = mul2(same2(rstd), fma2(hat, same2(-mean), mul2(y, w[q])));
      if (more) d = add2(d, W::get(in.dr, q));
      if (resid) W::set(ores, q, d);
      F2 sig = 0, gv = 0, open = same2(1.f);
      if (gated) gv = W::get(in.gate, q), sig = sigmoid2<T>(gv), open = mul2(gv, sig);
      if (scaled) {
        if (need_x) ds[q] = fma2(d, mul2(W::get(in.x, q), open), ds[q]);
        d = mul2(d, sc[q]);
      }
      W::set(ox, q, mul2(d, open));
      if (gated) W::set(og, q, mul2(mul2(d, W::get(in.x, q)), silu_grad2(gv, sig)));
    }
    if (a.dx) W::store(ox, static_cast<T*>(a.dx) + o, width);
    if (gated && a.dgate) W::store(og, static_cast<T*>(a.dgate) + o, width);
    if (resid && a.dresidual) W::store(ores, static_cast<R*>(a.dresidual) + o, width);
  }
  float* mine = part + static_cast<long long>(blockIdx.x / a.groups) * 2 * a.dim + c0;
  W::put(dw, mine, width);
  if (a.dscale) W::put(ds, mine + a.dim, width);
}

// Words per thread and the most threads of a block, which fix the registers
// (64 Ki over the threads).  Rows of up to 512 words (single elements: 2048) keep
// everything in registers, or all but a few words of the general form.  Up to twice
// that so does the forward pass; backward, 16-bit rows spill 0.1 to 1.5 KB per thread.
// Longer rows spill 2 to 4.5 KB and are bound by it.  64 Mi elements, gated, forward
// and backward: bf16 4096 wide 73 and 148 us, 5120 69 and 282, 8192 70 and 247, 16384
// 494 and 1359; fp32 4096 wide 130 and 215, 8192 799 and 1889.
template <int V, int NV, int MAXT>
struct NormSize {
  static constexpr int kV = V, kNV = NV, kMaxT = MAXT;
};

struct NormPlan {
  bool wide;
  int size, threads, blocks;  // size: 0, 1, 2 as above; blocks: per group of columns
};

template <class T, class R>
NormPlan norm_size(const pt_norm_args& a) {
  constexpr int W = 16 / static_cast<int>(sizeof(T));
  const int width = a.dim / a.groups;
  auto ok = [&](const void* p, long long s) { return aligned(p, 16) && (!p || s % W == 0); };
  NormPlan p;
  p.wide = width % W == 0 && ok(a.x, a.x_row) && ok(a.gate, a.gate_row) && ok(a.residual, a.residual_row) &&
           ok(a.weight, 0) && ok(a.scale, 0) && ok(a.y, 0) && ok(a.r, 0) && ok(a.dy, a.dy_row) && ok(a.dr, a.dr_row) &&
           ok(a.dx, 0) && ok(a.dgate, 0) && ok(a.dresidual, 0);
  const int v = p.wide ? W : 1;
  const int words = static_cast<int>(cdiv(width, v)), one = p.wide ? 1 : 4;
  p.size = words <= 512 * one ? 0 : words <= 1024 * one ? 1 : 2;
  const int nv = p.size == 0 ? one : p.size == 1 ? 2 * one : p.wide ? PT_NORM_MAX_WIDTH / 1024 / W : 32;
  p.threads = static_cast<int>(cdiv(cdiv(words, nv), 32)) * 32;
  return p;
}

// Calls fn(size, form) with both as constants.
template <class T, class R, class F>
cudaError_t by_plan(const pt_norm_args& a, const NormPlan& p, F&& fn) {
  constexpr int W = 16 / static_cast<int>(sizeof(T));
  auto sized = [&](auto form) -> cudaError_t {
    if (p.wide) {
      if (p.size == 0) return fn(NormSize<W, 1, 512>(), form);
      if (p.size == 1) return fn(NormSize<W, 2, 512>(), form);
    } else {
      if (p.size == 0) return fn(NormSize<1, 4, 512>(), form);
      if (p.size == 1) return fn(NormSize<1, 8, 512>(), form);
    }
    return cudaErrorInvalidValue;
  };
  if (p.size == 2) {
    constexpr auto any = std::integral_constant<int, kAny>();
    if (p.wide) return fn(NormSize<W, PT_NORM_MAX_WIDTH / 1024 / W, 1024>(), any);
    return fn(NormSize<1, 32, 1024>(), any);
  }
  if (a.gate && !a.residual && !a.scale) return sized(std::integral_constant<int, kGated>());
  if (a.residual && !a.gate) return sized(std::integral_constant<int, kResidual>());
  return sized(std::integral_constant<int, kAny>());
}

template <class T, class R, class Z, int FORM>
const void* norm_kernel(bool backward) {
  return backward ? reinterpret_cast<const void*>(&seq_norm_bwd_kernel<T, R, Z::kV, Z::kNV, FORM, Z::kMaxT>)
                  : reinterpret_cast<const void*>(&seq_norm_fwd_kernel<T, R, Z::kV, Z::kNV, FORM, Z::kMaxT>);
}

// One wave: as many blocks as fit on the SMs, so that all walk about as many rows.
template <class T, class R>
cudaError_t norm_plan(const pt_norm_args& a, int sm_count, bool backward, NormPlan& p) {
  p = norm_size<T, R>(a);
  p.blocks = static_cast<int>(a.rows < sm_count ? a.rows : sm_count);
  if (a.rows * a.groups <= sm_count) return cudaSuccess;
  int per_sm = 1;
  const cudaError_t e = by_plan<T, R>(a, p, [&](auto size, auto form) {
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(
        &per_sm, norm_kernel<T, R, decltype(size), decltype(form)::value>(backward), p.threads, 0);
  });
  const long long want = cdiv(static_cast<long long>(sm_count) * (per_sm > 0 ? per_sm : 1), a.groups);
  p.blocks = static_cast<int>(a.rows < want ? a.rows : want);
  return e;
}

template <class T, class R>
cudaError_t norm_fwd(const pt_norm_args& a, int sm_count, cudaStream_t stream) {
  NormPlan p;
  cudaError_t e = norm_plan<T, R>(a, sm_count, false, p);
  if (e != cudaSuccess) return e;
  return by_plan<T, R>(a, p, [&](auto size, auto form) {
    using Z = decltype(size);
    seq_norm_fwd_kernel<T, R, Z::kV, Z::kNV, decltype(form)::value, Z::kMaxT>
        <<<static_cast<unsigned>(p.blocks * a.groups), p.threads, 0, stream>>>(a, a.dim / a.groups, p.blocks);
    return cudaGetLastError();
  });
}

template <class T, class R>
cudaError_t norm_bwd(const pt_norm_args& a, float* ws, int sm_count, cudaStream_t stream) {
  NormPlan p;
  cudaError_t e = norm_plan<T, R>(a, sm_count, true, p);
  if (e != cudaSuccess) return e;
  e = by_plan<T, R>(a, p, [&](auto size, auto form) {
    using Z = decltype(size);
    seq_norm_bwd_kernel<T, R, Z::kV, Z::kNV, decltype(form)::value, Z::kMaxT>
        <<<static_cast<unsigned>(p.blocks * a.groups), p.threads, 0, stream>>>(a, ws, a.dim / a.groups, p.blocks);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  const int out = a.param_f32 ? PT_F32 : a.dtype;
  return launch_reduce(ws, p.blocks, {{a.dweight, a.dim, out}, {a.dscale, a.dim, out}, {nullptr, 0, out}}, stream);
}

// Calls fn(T(), R()): R, the residual's type, is T or float.
template <class F>
cudaError_t by_types(const pt_norm_args& a, F&& fn) {
  return by_type(a.dtype, [&](auto t) -> cudaError_t {
    if (a.residual && a.residual_f32) return fn(t, float());
    return fn(t, t);
  });
}

struct ReduceArgs {
  ReduceOut out[3];
  long long end[3];  // first element behind each output
};

// One block: 32 columns x 8 threads that each add every eighth chunk.
__global__ void __launch_bounds__(256) seq_reduce_kernel(const float* part, long long chunks, ReduceArgs a) {
  __shared__ float buf[8][32];
  const int tx = static_cast<int>(threadIdx.x), ty = static_cast<int>(threadIdx.y);
  const long long i = static_cast<long long>(blockIdx.x) * 32 + tx, stride = a.end[2];
  const int k = i < a.end[0] ? 0 : i < a.end[1] ? 1 : 2;
  const bool in = i < stride && a.out[k].out;
  float s = 0.f;
  if (in) {
    long long c = ty;
    for (; c + 24 < chunks; c += 32) {
      const float* p = part + c * stride + i;
      const float v0 = p[0], v1 = p[8 * stride], v2 = p[16 * stride], v3 = p[24 * stride];
      s += (v0 + v1) + (v2 + v3);
    }
    for (; c < chunks; c += 8) s += part[c * stride + i];
  }
  buf[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && in) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += buf[r][tx];
    const long long j = k ? i - a.end[k - 1] : i;
    if (a.out[k].dtype == PT_F32)
      static_cast<float*>(a.out[k].out)[j] = s;
    else if (a.out[k].dtype == PT_BF16)
      static_cast<__nv_bfloat16*>(a.out[k].out)[j] = from_f<__nv_bfloat16>(s);
    else
      static_cast<__half*>(a.out[k].out)[j] = from_f<__half>(s);
  }
}

}  // namespace

cudaError_t launch_reduce(const float* part, long long chunks, const ReduceOut (&outs)[3], cudaStream_t stream) {
  ReduceArgs a;
  long long end = 0;
  bool any = false;
  for (int k = 0; k < 3; ++k) {
    a.out[k] = outs[k];
    a.end[k] = end += outs[k].m;
    any |= outs[k].out && outs[k].m > 0;
  }
  if (!any) return cudaSuccess;
  seq_reduce_kernel<<<static_cast<unsigned>(cdiv(end, 32)), dim3(32, 8), 0, stream>>>(part, chunks, a);
  return cudaGetLastError();
}

cudaError_t launch_norm_fwd(const pt_norm_args& a, int sm_count, cudaStream_t stream) {
  return by_types(a, [&](auto t, auto r) { return norm_fwd<decltype(t), decltype(r)>(a, sm_count, stream); });
}
cudaError_t launch_norm_bwd(const pt_norm_args& a, float* ws, int sm_count, cudaStream_t stream) {
  return by_types(a, [&](auto t, auto r) { return norm_bwd<decltype(t), decltype(r)>(a, ws, sm_count, stream); });
}
size_t norm_bwd_workspace(const pt_norm_args& a, int sm_count) {
  NormPlan p;
  const cudaError_t e = by_types(a, [&](auto t, auto r) { return norm_plan<decltype(t), decltype(r)>(a, sm_count, true, p); });
  return e == cudaSuccess ? sizeof(float) * 2 * a.dim * static_cast<size_t>(p.blocks) : 0;
}

}  // namespace seq
}  // namespace pt
