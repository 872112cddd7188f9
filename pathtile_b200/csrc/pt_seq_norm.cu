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
#include <type_traits>

#include "pt_seq.h"
#include "pt_seq_common.cuh"

namespace pt {
namespace seq {
namespace {

constexpr int kNormMaxThreads = 1024;

// V parameters from index i on.
template <class T, int V>
__device__ __forceinline__ void load_param(const void* p, int i, int n, bool f32, float (&out)[V]) {
  if (f32) {
    Pack<float, V> w;
    w.load(static_cast<const float*>(p) + i, n, true);
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = w.f(v);
  } else {
    Pack<T, V> w;
    w.load(static_cast<const T*>(p) + i, n, true);
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = w.f(v);
  }
}

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

template <class T, class R, int V, int NV>
__global__ void __launch_bounds__(kNormMaxThreads) seq_norm_fwd_kernel(pt_norm_args a, int width, long long stride) {
  __shared__ float2 buf[2][32];
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
  const int c0 = static_cast<int>(blockIdx.x % a.groups) * width;
  float w[NV][V], sc[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * threads + tid) * V;
    if (i < width) {
      load_param<T, V>(a.weight, c0 + i, V, a.param_f32, w[k]);
      if (a.scale) load_param<T, V>(a.scale, c0 + i, V, a.param_f32, sc[k]);
    }
  }
  int slot = 0;
  for (long long row = blockIdx.x / a.groups; row < a.rows; row += stride, slot ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_row + c0;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + row * a.gate_row + c0 : nullptr;
    const R* res = a.residual ? static_cast<const R*>(a.residual) + row * a.residual_row + c0 : nullptr;
    const long long o = row * a.dim + c0;
    Pack<T, V> px[NV], pg[NV];
    Pack<R, V> pr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) {
        px[k].load(x + i, V, true);
        if (gate) pg[k].load(gate + i, V, true);
        if (res) pr[k].load(res + i, V, true);
      }
    }
    float r[NV][V], ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float u = px[k].f(v);
          if (gate) u *= siluf(pg[k].f(v));
          if (a.scale) u *= sc[k][v];
          if (res) {
            // The stream that goes on is what is normalised: rounded to its type first.
            pr[k].set(v, pr[k].f(v) + u);
            u = pr[k].f(v);
          }
          r[k][v] = u;
          ss = fmaf(u, u, ss);
        }
        if (res) pr[k].store(static_cast<R*>(a.r) + o + i, V, true);
      }
    }
    const float rstd = rsqrtf(block_sum(ss, 0.f, buf, slot).x / static_cast<float>(width) + a.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) {
        Pack<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) out.set(v, r[k][v] * rstd * w[k][v]);
        out.store(static_cast<T*>(a.y) + o + i, V, true);
      }
    }
  }
}

template <class T, class R, int V, int NV>
__global__ void __launch_bounds__(kNormMaxThreads)
    seq_norm_bwd_kernel(pt_norm_args a, float* part, int width, long long stride) {
  __shared__ float2 buf[2][32];
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
  const int c0 = static_cast<int>(blockIdx.x % a.groups) * width;
  const bool need_x = !a.residual || a.gate || (a.scale && a.dscale);
  float dw[NV][V], ds[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) dw[k][v] = ds[k][v] = 0.f;
  int slot = 0;
  for (long long row = blockIdx.x / a.groups; row < a.rows; row += stride, slot ^= 1) {
    const long long o = row * a.dim + c0;
    const T* x = static_cast<const T*>(a.x) + row * a.x_row + c0;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + row * a.gate_row + c0 : nullptr;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_row + c0;
    const R* dr = a.dr ? static_cast<const R*>(a.dr) + row * a.dr_row + c0 : nullptr;
    Pack<T, V> px[NV], pg[NV], py[NV];
    Pack<R, V> pr[NV], pd[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) {
        py[k].load(dy + i, V, true);
        if (need_x) px[k].load(x + i, V, true);
        if (gate) pg[k].load(gate + i, V, true);
        if (a.residual) pr[k].load(static_cast<const R*>(a.r) + o + i, V, true);
        if (dr) pd[k].load(dr + i, V, true);
      }
    }
    float r[NV][V], ss = 0.f, sv = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) {
        float w[V], sc[V];
        load_param<T, V>(a.weight, c0 + i, V, a.param_f32, w);
        if (a.scale && !a.residual) load_param<T, V>(a.scale, c0 + i, V, a.param_f32, sc);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float u;
          if (a.residual) {
            u = pr[k].f(v);
          } else {
            u = px[k].f(v);
            if (gate) u *= siluf(pg[k].f(v));
            if (a.scale) u *= sc[v];
          }
          r[k][v] = u;
          ss = fmaf(u, u, ss);
          sv = fmaf(py[k].f(v) * w[v], u, sv);
        }
      }
    }
    const float2 sums = block_sum(ss, sv, buf, slot);
    const float inv = 1.f / static_cast<float>(width);
    const float rstd = rsqrtf(fmaf(sums.x, inv, a.eps)), mean = sums.y * inv * rstd;  // mean(v hat)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * threads + tid) * V;
      if (i < width) {
        float w[V], sc[V];
        load_param<T, V>(a.weight, c0 + i, V, a.param_f32, w);
        if (a.scale) load_param<T, V>(a.scale, c0 + i, V, a.param_f32, sc);
        Pack<T, V> ox, og;
        Pack<R, V> ores;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float hat = r[k][v] * rstd, y = py[k].f(v);
          dw[k][v] = fmaf(y, hat, dw[k][v]);
          float d = rstd * (y * w[v] - hat * mean);
          if (dr) d += pd[k].f(v);
          if (a.residual) ores.set(v, d);
          float sig = 0.f, gv = 0.f, open = 1.f;
          if (gate) gv = pg[k].f(v), sig = sigmoidf(gv), open = gv * sig;
          if (a.scale) {
            if (need_x) ds[k][v] = fmaf(d, px[k].f(v) * open, ds[k][v]);
            d *= sc[v];
          }
          ox.set(v, d * open);
          if (gate) og.set(v, d * px[k].f(v) * silu_grad(gv, sig));
        }
        if (a.dx) ox.store(static_cast<T*>(a.dx) + o + i, V, true);
        if (a.dgate) og.store(static_cast<T*>(a.dgate) + o + i, V, true);
        if (a.dresidual) ores.store(static_cast<R*>(a.dresidual) + o + i, V, true);
      }
    }
  }
  float* mine = part + static_cast<long long>(blockIdx.x / a.groups) * 2 * a.dim;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * threads + tid) * V;
    if (i < width) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        mine[c0 + i + v] = dw[k][v];
        if (a.dscale) mine[a.dim + c0 + i + v] = ds[k][v];
      }
    }
  }
}

struct NormPlan {
  bool wide;
  int nv, threads, blocks;  // blocks: per group of columns
};

template <class T, class R>
NormPlan norm_plan(const pt_norm_args& a, int sm_count, bool backward) {
  constexpr int W = 16 / static_cast<int>(sizeof(T));
  const int width = a.dim / a.groups;
  auto ok = [&](const void* p, long long s) { return aligned(p, 16) && (!p || s % W == 0); };
  NormPlan p;
  p.wide = width % W == 0 && ok(a.x, a.x_row) && ok(a.gate, a.gate_row) && ok(a.residual, a.residual_row) &&
           ok(a.weight, 0) && ok(a.scale, 0) && ok(a.y, 0) && ok(a.r, 0) && ok(a.dy, a.dy_row) && ok(a.dr, a.dr_row) &&
           ok(a.dx, 0) && ok(a.dgate, 0) && ok(a.dresidual, 0);
  const int v = p.wide ? W : 1;
  const int words = static_cast<int>(cdiv(width, v));
  // One word per thread up to 1024 threads (single elements: four), more beyond.
  if (p.wide)
    p.nv = words <= 1024 ? 1 : words <= 2048 ? 2 : 8 / (W / 4);
  else
    p.nv = words <= 4096 ? 4 : 32;
  p.threads = static_cast<int>(cdiv(cdiv(words, p.nv), 32)) * 32;
  // Forward one wave of the SMs' 2048 threads, twice; backward one (each block writes a partial sum).
  const long long want = cdiv(static_cast<long long>(sm_count) * (backward ? 1024 : 4096) / p.threads, a.groups);
  p.blocks = static_cast<int>(a.rows < want ? a.rows : want);
  return p;
}

template <class T, class R, class F>
cudaError_t by_plan(const NormPlan& p, F&& fn) {
  constexpr int W = 16 / static_cast<int>(sizeof(T));
  if (p.wide) {
    if (p.nv == 1) return fn(std::integral_constant<int, W>(), std::integral_constant<int, 1>());
    if (p.nv == 2) return fn(std::integral_constant<int, W>(), std::integral_constant<int, 2>());
    return fn(std::integral_constant<int, W>(), std::integral_constant<int, 8 / (W / 4)>());
  }
  if (p.nv == 4) return fn(std::integral_constant<int, 1>(), std::integral_constant<int, 4>());
  return fn(std::integral_constant<int, 1>(), std::integral_constant<int, 32>());
}

template <class T, class R>
cudaError_t norm_fwd(const pt_norm_args& a, int sm_count, cudaStream_t stream) {
  const NormPlan p = norm_plan<T, R>(a, sm_count, false);
  return by_plan<T, R>(p, [&](auto vc, auto nc) {
    seq_norm_fwd_kernel<T, R, decltype(vc)::value, decltype(nc)::value>
        <<<static_cast<unsigned>(p.blocks * a.groups), p.threads, 0, stream>>>(a, a.dim / a.groups, p.blocks);
    return cudaGetLastError();
  });
}

template <class T, class R>
cudaError_t norm_bwd(const pt_norm_args& a, float* ws, int sm_count, cudaStream_t stream) {
  const NormPlan p = norm_plan<T, R>(a, sm_count, true);
  cudaError_t e = by_plan<T, R>(p, [&](auto vc, auto nc) {
    seq_norm_bwd_kernel<T, R, decltype(vc)::value, decltype(nc)::value>
        <<<static_cast<unsigned>(p.blocks * a.groups), p.threads, 0, stream>>>(a, ws, a.dim / a.groups, p.blocks);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  const int out = a.param_f32 ? PT_F32 : a.dtype;
  if (a.dweight && (e = launch_reduce(ws, p.blocks, 2LL * a.dim, a.dim, a.dweight, out, stream)) != cudaSuccess) return e;
  if (a.dscale) return launch_reduce(ws + a.dim, p.blocks, 2LL * a.dim, a.dim, a.dscale, out, stream);
  return cudaSuccess;
}

// Calls fn(T(), R()): R, the residual's type, is T or float.
template <class F>
cudaError_t by_types(const pt_norm_args& a, F&& fn) {
  return by_type(a.dtype, [&](auto t) -> cudaError_t {
    if (a.residual && a.residual_f32) return fn(t, float());
    return fn(t, t);
  });
}

// One block: 32 columns x 8 threads that each add every eighth chunk.
template <class O>
__global__ void __launch_bounds__(256)
    seq_reduce_kernel(const float* part, int chunks, long long stride, long long m, O* out) {
  __shared__ float buf[8][32];
  const int tx = static_cast<int>(threadIdx.x), ty = static_cast<int>(threadIdx.y);
  const long long i = static_cast<long long>(blockIdx.x) * 32 + tx;
  float s = 0.f;
  if (i < m) {
    int c = ty;
    for (; c + 24 < chunks; c += 32) {
      const float* p = part + c * stride + i;
      const float v0 = p[0], v1 = p[8 * stride], v2 = p[16 * stride], v3 = p[24 * stride];
      s += (v0 + v1) + (v2 + v3);
    }
    for (; c < chunks; c += 8) s += part[c * stride + i];
  }
  buf[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && i < m) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += buf[r][tx];
    out[i] = from_f<O>(s);
  }
}

}  // namespace

cudaError_t launch_reduce(const float* part, int chunks, long long stride, long long m, void* out, int dtype,
                          cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    using O = decltype(t);
    seq_reduce_kernel<O><<<static_cast<unsigned>(cdiv(m, 32)), dim3(32, 8), 0, stream>>>(part, chunks, stride, m,
                                                                                         static_cast<O*>(out));
    return cudaGetLastError();
  });
}

cudaError_t launch_norm_fwd(const pt_norm_args& a, int sm_count, cudaStream_t stream) {
  return by_types(a, [&](auto t, auto r) { return norm_fwd<decltype(t), decltype(r)>(a, sm_count, stream); });
}
cudaError_t launch_norm_bwd(const pt_norm_args& a, float* ws, int sm_count, cudaStream_t stream) {
  return by_types(a, [&](auto t, auto r) { return norm_bwd<decltype(t), decltype(r)>(a, ws, sm_count, stream); });
}
size_t norm_bwd_workspace(const pt_norm_args& a, int sm_count) {
  size_t n = 0;
  by_types(a, [&](auto t, auto r) {
    n = sizeof(float) * 2 * a.dim * static_cast<size_t>(norm_plan<decltype(t), decltype(r)>(a, sm_count, true).blocks);
    return cudaSuccess;
  });
  return n;
}

}  // namespace seq
}  // namespace pt
