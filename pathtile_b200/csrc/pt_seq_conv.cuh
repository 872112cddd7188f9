// pt_seq_conv.cuh -- causal depthwise convolution of a few taps (1..8) over
// [batch, len, dim]: forward, backward and the single-token step.
//
// A thread owns V neighbouring channels of one batch row and walks TS steps;
// the last K-1 inputs and the taps stay in registers, so every input is read
// once from memory (plus K-1 steps of overlap per thread) and the kernel is
// bound by the two (backward: three) streams it moves.  V is the widest word
// (up to 16 bytes forward, 8 backward) that every pointer, stride and row
// length allows; loads of U steps are issued together so that enough bytes are
// in flight.  Channels are the fast axis of the block, steps the slow one.
//
// Backward, walking forward in time: g[t] = dy[t] act'(pre[t]) with pre
// recomputed from the window, dx[t-K+1] = sum_j w[j] g[t-j] from the window of
// the last K g's, dw[j] += g[t] x[t-K+1+j].  A block adds its threads' dw in a
// fixed order and writes one partial sum; a second kernel adds the partials.
#pragma once

#include "pt_seq.h"
#include "pt_seq_common.cuh"

namespace pt {
namespace seq {

constexpr int kConvThreads = 128;
constexpr int kConvBwdTx = 32, kConvBwdTy = kConvThreads / kConvBwdTx;

__device__ __forceinline__ int row_length(const int* lengths, int b, int len) {
  if (!lengths) return len;
  const int n = __ldg(lengths + b);
  return n < 0 ? 0 : n > len ? len : n;
}

template <class T, int K, int V>
struct ConvRow {
  const T* x;
  const T* state;  // [K-1, dim] rows before x, or null
  long long step;
  int dim, len;  // valid steps
  // Input at step t: x, before it the state, 0 elsewhere.
  __device__ __forceinline__ void load(Pack<T, V>& p, int t) const {
    if (t >= 0) {
      if (t < len)
        p.load(x + t * step, V, true);
      else
        p.zero();
    } else if (state && t >= 1 - K) {
      p.load(state + static_cast<long long>(t + K - 1) * dim, V, true);
    } else {
      p.zero();
    }
  }
};

template <class T, int K, int V>
__device__ __forceinline__ void conv_params(const pt_conv_args& a, int c, float (&w)[K][V], float (&bias)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][v] = param<T>(a.w, static_cast<long long>(c + v) * K + j, a.param_f32);
    bias[v] = a.bias ? param<T>(a.bias, c + v, a.param_f32) : 0.f;
  }
}

template <class T, int K, int V>
__global__ void __launch_bounds__(kConvThreads)
    seq_conv_fwd_kernel(pt_conv_args a, int cblocks, int tblocks, int steps) {
  constexpr int U = 4;  // steps whose loads are in flight together
  const int cb = static_cast<int>(blockIdx.x) % cblocks;
  const int rest = static_cast<int>(blockIdx.x) / cblocks;
  const int tb = rest % tblocks, b = rest / tblocks;
  const int c = (cb * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * V;
  if (c >= a.dim) return;
  const int len = row_length(a.lengths, b, a.len);
  ConvRow<T, K, V> row{static_cast<const T*>(a.x) + b * a.x_batch + c,
                       a.state_in ? static_cast<const T*>(a.state_in) + static_cast<long long>(b) * (K - 1) * a.dim + c
                                  : nullptr,
                       a.x_step, a.dim, len};
  if (K > 1 && a.state_out && tb == 0 && threadIdx.y == 0) {
    T* out = static_cast<T*>(a.state_out) + static_cast<long long>(b) * (K - 1) * a.dim + c;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      Pack<T, V> p;
      row.load(p, len - (K - 1) + j);
      p.store(out + static_cast<long long>(j) * a.dim, V, true);
    }
  }
  const int t0 = (tb * static_cast<int>(blockDim.y) + static_cast<int>(threadIdx.y)) * steps;
  const int t1 = min(t0 + steps, a.len);
  if (t0 >= t1) return;
  float w[K][V], bias[V];
  conv_params<T, K, V>(a, c, w, bias);
  float win[K][V];  // win[j]: input at step t - K + 1 + j
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    Pack<T, V> p;
    row.load(p, t0 - (K - 1) + j);
#pragma unroll
    for (int v = 0; v < V; ++v) win[j + 1][v] = p.f(v);
  }
  T* y = static_cast<T*>(a.y) + (static_cast<long long>(b) * a.len + t0) * a.dim + c;
  for (int t = t0; t < t1; t += U) {
    Pack<T, V> in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) row.load(in[u], t + u);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Pack<T, V> out;
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) win[j][v] = win[j + 1][v];
        win[K - 1][v] = in[u].f(v);
        float s = bias[v];
#pragma unroll
        for (int j = 0; j < K; ++j) s = fmaf(w[j][v], win[j][v], s);
        out.set(v, t + u < len ? (a.silu ? siluf(s) : s) : 0.f);
      }
      if (t + u < t1) out.store(y + static_cast<long long>(t + u - t0) * a.dim, V, true);
    }
  }
}

// Work item i of a block's list is batch row i / tblocks, steps from
// (i % tblocks) * kConvBwdTy * steps on; the dw of all its items stay in registers.
template <class T, int K, int V>
__global__ void __launch_bounds__(kConvThreads)
    seq_conv_bwd_kernel(pt_conv_args a, float* part, int cblocks, int tblocks, int steps, int chunks) {
  __shared__ float red[kConvBwdTy][kConvBwdTx * V];
  const int tx = static_cast<int>(threadIdx.x), ty = static_cast<int>(threadIdx.y);
  const int cb = static_cast<int>(blockIdx.x) % cblocks, chunk = static_cast<int>(blockIdx.x) / cblocks;
  const int c = (cb * kConvBwdTx + tx) * V;
  const bool in = c < a.dim;
  float w[K][V], bias[V], dw[K][V], db[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    db[v] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) dw[j][v] = 0.f;
  }
  if (in) {
    conv_params<T, K, V>(a, c, w, bias);
    const long long items = static_cast<long long>(a.batch) * tblocks;
    for (long long item = chunk; item < items; item += chunks) {
      const int b = static_cast<int>(item / tblocks), tb = static_cast<int>(item % tblocks);
      const int len = row_length(a.lengths, b, a.len);
      const int t0 = (tb * kConvBwdTy + ty) * steps, t1 = min(t0 + steps, a.len);
      if (t0 >= t1 && !(t0 == 0)) continue;
      ConvRow<T, K, V> row{
          static_cast<const T*>(a.x) + b * a.x_batch + c,
          a.state_in ? static_cast<const T*>(a.state_in) + static_cast<long long>(b) * (K - 1) * a.dim + c : nullptr,
          a.x_step, a.dim, len};
      const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch + c;
      T* dx = a.dx ? static_cast<T*>(a.dx) + static_cast<long long>(b) * a.len * a.dim + c : nullptr;
      const T* dso = a.dstate_out
                         ? static_cast<const T*>(a.dstate_out) + static_cast<long long>(b) * (K - 1) * a.dim + c
                         : nullptr;
      T* dsi = a.dstate_in ? static_cast<T*>(a.dstate_in) + static_cast<long long>(b) * (K - 1) * a.dim + c : nullptr;
      float win[K][V], gw[K][V];  // gw[j]: g at step t - j
#pragma unroll
      for (int j = 0; j < K; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) gw[j][v] = 0.f;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        Pack<T, V> p;
        row.load(p, t0 - (K - 1) + j);
#pragma unroll
        for (int v = 0; v < V; ++v) win[j + 1][v] = p.f(v);
      }
      const int first = t0 == 0 ? -(K - 1) : t0;  // first position whose gradient this thread writes
      constexpr int U = 4;
      for (int tt = t0; tt < t1 + K - 1; tt += U) {
        Pack<T, V> xin[U], gin[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          row.load(xin[u], tt + u);
          if (tt + u < len)
            gin[u].load(dy + (tt + u) * a.dy_step, V, true);
          else
            gin[u].zero();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = tt + u, pos = t - (K - 1);
          Pack<T, V> out;
#pragma unroll
          for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < K - 1; ++j) win[j][v] = win[j + 1][v];
            win[K - 1][v] = xin[u].f(v);
            float g = gin[u].f(v);
            if (a.silu) {
              float pre = bias[v];
#pragma unroll
              for (int j = 0; j < K; ++j) pre = fmaf(w[j][v], win[j][v], pre);
              g *= silu_grad(pre, sigmoidf(pre));
            }
            // Steps behind the row's end have no output; their window may hold anything.
            g = t < len ? g : 0.f;
            if (t < t1 && t < len) {
#pragma unroll
              for (int j = 0; j < K; ++j) dw[j][v] = fmaf(g, win[j][v], dw[j][v]);
              db[v] += g;
            }
#pragma unroll
            for (int j = K - 1; j > 0; --j) gw[j][v] = gw[j - 1][v];
            gw[0][v] = g;
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j) s = fmaf(w[j][v], gw[j][v], s);
            if (dso && pos >= len - (K - 1) && pos < len)
              s += to_f<T>(dso[static_cast<long long>(pos - (len - (K - 1))) * a.dim + v]);
            out.set(v, s);
          }
          if (pos >= first && pos < t1) {
            if (pos >= 0) {
              if (dx) out.store(dx + static_cast<long long>(pos) * a.dim, V, true);
            } else if (dsi) {
              out.store(dsi + static_cast<long long>(pos + K - 1) * a.dim, V, true);
            }
          }
        }
      }
    }
  }
  // The block's sum, one tap after the other (K passes over a small array).
  float* mine = part + static_cast<long long>(chunk) * a.dim * (K + 1);
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) red[ty][tx * V + v] = j < K ? dw[j < K ? j : 0][v] : db[v];
    __syncthreads();
    for (int i = ty * kConvBwdTx + tx; i < kConvBwdTx * V; i += kConvThreads) {
      const int d = cb * kConvBwdTx * V + i;
      if (d < a.dim) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kConvBwdTy; ++r) s += red[r][i];
        mine[j < K ? static_cast<long long>(d) * K + j : static_cast<long long>(a.dim) * K + d] = s;
      }
    }
  }
}

template <class T, int K, int V>
__global__ void __launch_bounds__(kConvThreads) seq_conv_step_kernel(pt_conv_args a, int cblocks, unsigned* err) {
  const int cb = static_cast<int>(blockIdx.x) % cblocks, b = static_cast<int>(blockIdx.x) / cblocks;
  const int slot = a.slots ? slot_of(a.slots, b, a.cache_rows, err, static_cast<int>(threadIdx.x), kConvThreads) : b;
  const int c = (cb * kConvThreads + static_cast<int>(threadIdx.x)) * V;
  if (c >= a.dim) return;
  T* y = static_cast<T*>(a.y) + static_cast<long long>(b) * a.dim + c;
  Pack<T, V> out;
  if (slot < 0) {
    out.zero();
    out.store(y, V, true);
    return;
  }
  T* state = static_cast<T*>(a.state_out) + static_cast<long long>(slot) * a.state_row + c;
  Pack<T, V> in[K];
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const T* p = state + static_cast<long long>(j) * a.dim;
    // Plain loads: the cache is written below.
    if constexpr (V * sizeof(T) == 16) {
      *reinterpret_cast<uint4*>(in[j].v) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) in[j].v[v] = p[v];
    }
  }
  in[K - 1].load(static_cast<const T*>(a.x) + b * a.x_batch + c, V, true);
  float w[K][V], bias[V];
  conv_params<T, K, V>(a, c, w, bias);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s = bias[v];
#pragma unroll
    for (int j = 0; j < K; ++j) s = fmaf(w[j][v], in[j].f(v), s);
    out.set(v, a.silu ? siluf(s) : s);
  }
  out.store(y, V, true);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) in[j + 1].store(state + static_cast<long long>(j) * a.dim, V, true);
}

// ---------------------------------------------------------------- host side
// Whether every row that `ptr` leads to starts on a word of V elements.
inline bool conv_wide(const void* ptr, long long s0, long long s1, int v, size_t e) {
  return !ptr || (aligned(ptr, v * e) && s0 % v == 0 && s1 % v == 0);
}
inline int conv_width(const pt_conv_args& a, size_t e, int most) {
  for (int v = most; v > 1; v = v > 2 ? 2 : 1) {
    if (a.dim % v == 0 && conv_wide(a.x, a.x_batch, a.x_step, v, e) && conv_wide(a.dy, a.dy_batch, a.dy_step, v, e) &&
        conv_wide(a.state_in, 0, 0, v, e) && conv_wide(a.state_out, a.state_row, 0, v, e) && conv_wide(a.y, 0, 0, v, e) &&
        conv_wide(a.dx, 0, 0, v, e) && conv_wide(a.dstate_in, 0, 0, v, e))
      return v;
  }
  return 1;
}

// Calls fn(V as a constant, K as a constant).
template <int VMAX, class F>
cudaError_t by_width_taps(int v, int k, F&& fn) {
  auto taps = [&](auto vc) -> cudaError_t {
    switch (k) {
      case 1: return fn(vc, std::integral_constant<int, 1>());
      case 2: return fn(vc, std::integral_constant<int, 2>());
      case 3: return fn(vc, std::integral_constant<int, 3>());
      case 4: return fn(vc, std::integral_constant<int, 4>());
      case 5: return fn(vc, std::integral_constant<int, 5>());
      case 6: return fn(vc, std::integral_constant<int, 6>());
      case 7: return fn(vc, std::integral_constant<int, 7>());
      case 8: return fn(vc, std::integral_constant<int, 8>());
      default: return cudaErrorInvalidValue;
    }
  };
  if (v == 1) return taps(std::integral_constant<int, 1>());
  if (v == 2) return taps(std::integral_constant<int, 2>());
  return taps(std::integral_constant<int, VMAX>());
}

template <class T>
constexpr int conv_word = 16 / static_cast<int>(sizeof(T));  // forward: 16 bytes
template <class T>
constexpr int conv_bwd_word = sizeof(T) == 4 ? 4 : 4;  // backward: four channels (registers: five arrays of taps)

template <class T>
ConvBwdPlan conv_bwd_plan(const pt_conv_args& a, int sm_count) {
  ConvBwdPlan p;
  p.v = conv_width(a, sizeof(T), conv_bwd_word<T>);
  p.cblocks = static_cast<int>(cdiv(a.dim, kConvBwdTx * p.v));
  // As many steps per thread as leave eight blocks per SM, at least 8.
  p.steps = 64;
  while (p.steps > 8 && static_cast<long long>(p.cblocks) * a.batch * cdiv(a.len, p.steps * kConvBwdTy) < 8 * sm_count)
    p.steps /= 2;
  p.tblocks = static_cast<int>(cdiv(a.len > 0 ? a.len : 1, p.steps * kConvBwdTy));
  const long long items = static_cast<long long>(a.batch) * p.tblocks;
  const long long most = cdiv(8LL * sm_count, p.cblocks);
  p.chunks = static_cast<int>(items < most ? items : most);
  return p;
}

template <class T>
cudaError_t conv_fwd(const pt_conv_args& a, cudaStream_t stream) {
  const int v = conv_width(a, sizeof(T), conv_word<T>);
  const int groups = static_cast<int>(cdiv(a.dim, v));
  int tx = 32;
  while (tx < kConvThreads && tx < groups) tx *= 2;
  const int ty = kConvThreads / tx;
  const int cblocks = static_cast<int>(cdiv(groups, tx));
  int steps = 32;
  while (steps > 4 && static_cast<long long>(cblocks) * a.batch * cdiv(a.len, static_cast<long long>(steps) * ty) < 1184)
    steps /= 2;
  const int tblocks = static_cast<int>(cdiv(a.len > 0 ? a.len : 1, static_cast<long long>(steps) * ty));
  const long long grid = static_cast<long long>(cblocks) * tblocks * a.batch;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return by_width_taps<conv_word<T>>(v, a.taps, [&](auto vc, auto kc) {
    seq_conv_fwd_kernel<T, decltype(kc)::value, decltype(vc)::value>
        <<<static_cast<unsigned>(grid), dim3(tx, ty), 0, stream>>>(a, cblocks, tblocks, steps);
    return cudaGetLastError();
  });
}

template <class T>
cudaError_t conv_bwd(const pt_conv_args& a, float* ws, int sm_count, cudaStream_t stream) {
  const ConvBwdPlan p = conv_bwd_plan<T>(a, sm_count);
  cudaError_t e = by_width_taps<conv_bwd_word<T>>(p.v, a.taps, [&](auto vc, auto kc) {
    seq_conv_bwd_kernel<T, decltype(kc)::value, decltype(vc)::value>
        <<<static_cast<unsigned>(p.cblocks * p.chunks), dim3(kConvBwdTx, kConvBwdTy), 0, stream>>>(
            a, ws, p.cblocks, p.tblocks, p.steps, p.chunks);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  const int out = a.param_f32 ? PT_F32 : a.dtype;
  const long long m = static_cast<long long>(a.dim) * a.taps, all = m + a.dim;
  if (a.dw && (e = launch_reduce(ws, p.chunks, all, m, a.dw, out, stream)) != cudaSuccess) return e;
  if (a.dbias && (e = launch_reduce(ws + m, p.chunks, all, a.dim, a.dbias, out, stream)) != cudaSuccess) return e;
  return cudaSuccess;
}

template <class T>
cudaError_t conv_step(const pt_conv_args& a, unsigned* err, cudaStream_t stream) {
  const int v = conv_width(a, sizeof(T), conv_word<T>);
  const int cblocks = static_cast<int>(cdiv(a.dim, kConvThreads * v));
  const long long grid = static_cast<long long>(cblocks) * a.batch;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return by_width_taps<conv_word<T>>(v, a.taps, [&](auto vc, auto kc) {
    seq_conv_step_kernel<T, decltype(kc)::value, decltype(vc)::value>
        <<<static_cast<unsigned>(grid), kConvThreads, 0, stream>>>(a, cblocks, err);
    return cudaGetLastError();
  });
}

}  // namespace seq
}  // namespace pt
