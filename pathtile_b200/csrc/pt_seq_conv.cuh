// pt_seq_conv.cuh -- causal depthwise convolution of a few taps (1..8) over
// [batch, len, dim]: forward, backward and the single-token step.
//
// A thread owns V neighbouring channels and walks a stretch of steps; the last
// K inputs and the taps stay in registers, so every input is read once from
// memory (plus K-1 steps of overlap per stretch).  All rows' steps are laid end
// to end and cut into equal stretches, so that every thread has the same work
// whatever the batch; a stretch that crosses into the next row starts anew
// there.  V is a word of 16 bytes forward and 8 backward where every pointer,
// stride and row length allows it (and there are up to four taps), else two
// elements, else one.  The loads of the next U steps are
// under way while U steps are computed, in packed fp32 arithmetic.  The taps
// come through shared memory: read straight, a warp's taps lie V x K floats
// apart and cost more than the steps.
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

// Blocks per SM that the registers are kept down for, and steps whose loads are
// under way together.  One wave of long stretches beats several waves of short
// ones (8 x 2048 x 4096 bf16, 4 taps, before the loops were split: forward 60
// against 69 us with four waves; backward 129 us, 200 us at the 146 registers that
// it would take by itself).  Now 52 us (5.2 TB/s) and 100 us (4.0 TB/s).
// Narrow words (rows that are not aligned) need more threads and steps for the
// same bytes on their way.
template <int V>
constexpr int kConvFwdBlocks = V > 2 ? 4 : 8;
template <int V>
constexpr int kConvFwdAhead = V > 2 ? 4 : 8;
constexpr int kConvBwdBlocks = 4, kConvBwdAhead = 4;

__device__ __forceinline__ int row_length(const int* lengths, int b, int len) {
  if (!lengths) return len;
  const int n = __ldg(lengths + b);
  return n < 0 ? 0 : n > len ? len : n;
}

// V channels' values in packed pairs (V = 1: the second half is idle).
template <int V>
struct Packed {
  static constexpr int N = (V + 1) / 2;
  F2 p[N];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = 0;
  }
  template <class T>
  __device__ __forceinline__ void from(const Pack<T, V>& a) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = a.pair(i);
  }
  template <class T>
  __device__ __forceinline__ void to(Pack<T, V>& a) const {
#pragma unroll
    for (int i = 0; i < N; ++i) a.set_pair(i, p[i]);
  }
};

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
__device__ __forceinline__ ConvRow<T, K, V> conv_row(const pt_conv_args& a, int b, int c) {
  return ConvRow<T, K, V>{
      static_cast<const T*>(a.x) + b * a.x_batch + c,
      a.state_in ? static_cast<const T*>(a.state_in) + static_cast<long long>(b) * (K - 1) * a.dim + c : nullptr,
      a.x_step, a.dim, row_length(a.lengths, b, a.len)};
}

// Taps and bias of V channels.
template <int K, int V>
struct Taps {
  Packed<V> w[K], bias;
  __device__ __forceinline__ F2 pre(const Packed<V> (&win)[K], int i) const {
    F2 s = bias.p[i];
#pragma unroll
    for (int j = 0; j < K; ++j) s = fma2(w[j].p[i], win[j].p[i], s);
    return s;
  }
};

// The whole block loads the taps of its tx * V channels; buf: tx * (V * K + 1) floats.
template <class T, int K, int V>
__device__ __forceinline__ void load_taps(const pt_conv_args& a, int c0, float* buf, Taps<K, V>& taps) {
  const int tx = static_cast<int>(blockDim.x), me = static_cast<int>(threadIdx.x);
  const int n = min(tx * V, a.dim - c0) * K;
  for (int i = static_cast<int>(threadIdx.y) * tx + me; i < n; i += kConvThreads)
    buf[i / (V * K) * (V * K + 1) + i % (V * K)] = param<T>(a.w, static_cast<long long>(c0) * K + i, a.param_f32);
  __syncthreads();
  const bool in = c0 + me * V < a.dim;
  const float* mine = buf + me * (V * K + 1);
#pragma unroll
  for (int i = 0; i < Packed<V>::N; ++i) {
    const int v0 = 2 * i, v1 = 2 * i + 1 < V ? 2 * i + 1 : v0;
#pragma unroll
    for (int j = 0; j < K; ++j) taps.w[j].p[i] = in ? pack2(mine[v0 * K + j], v1 > v0 ? mine[v1 * K + j] : 0.f) : 0;
    const float b0 = in && a.bias ? param<T>(a.bias, c0 + me * V + v0, a.param_f32) : 0.f;
    const float b1 = in && a.bias && v1 > v0 ? param<T>(a.bias, c0 + me * V + v1, a.param_f32) : 0.f;
    taps.bias.p[i] = pack2(b0, b1);
  }
}

template <class T, int K, int V>
__global__ void __launch_bounds__(kConvThreads, kConvFwdBlocks<V>)
    seq_conv_fwd_kernel(pt_conv_args a, int cblocks, long long per) {
  constexpr int U = kConvFwdAhead<V>;
  extern __shared__ float tap_buf[];
  const int cb = static_cast<int>(blockIdx.x) % cblocks;
  const long long walker = static_cast<long long>(blockIdx.x / cblocks) * blockDim.y + threadIdx.y;
  const int c0 = cb * static_cast<int>(blockDim.x) * V, c = c0 + static_cast<int>(threadIdx.x) * V;
  Taps<K, V> taps;
  load_taps<T, K, V>(a, c0, tap_buf, taps);
  if (c >= a.dim) return;
  const long long walkers = static_cast<long long>(gridDim.x / cblocks) * blockDim.y;
  if (K > 1 && a.state_out) {
    for (long long b = walker; b < a.batch; b += walkers) {
      const ConvRow<T, K, V> row = conv_row<T, K, V>(a, static_cast<int>(b), c);
      T* out = static_cast<T*>(a.state_out) + b * (K - 1) * a.dim + c;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        Pack<T, V> p;
        row.load(p, row.len - (K - 1) + j);
        p.store(out + static_cast<long long>(j) * a.dim, V, true);
      }
    }
  }
  const long long all = static_cast<long long>(a.batch) * a.len;
  long long at = walker * per;
  const long long end = min(at + per, all);
  while (at < end) {
    const int b = static_cast<int>(at / a.len), t0 = static_cast<int>(at % a.len);
    const int t1 = static_cast<int>(min(static_cast<long long>(a.len), t0 + (end - at)));
    const ConvRow<T, K, V> row = conv_row<T, K, V>(a, b, c);
    Packed<V> win[K];  // win[j]: input at step t - K + 1 + j
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      Pack<T, V> p;
      row.load(p, t0 - (K - 1) + j);
      win[j + 1].from(p);
    }
    T* y = static_cast<T*>(a.y) + at * a.dim + c;
    const T* x = row.x + t0 * row.step;
    auto advance = [&](const Pack<T, V>& in) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) win[j] = win[j + 1];
      win[K - 1].from(in);
      Packed<V> s;
#pragma unroll
      for (int i = 0; i < Packed<V>::N; ++i) {
        s.p[i] = taps.pre(win, i);
        if (a.silu) s.p[i] = mul2(s.p[i], sigmoid2<T>(s.p[i]));
      }
      Pack<T, V> out;
      s.to(out);
      out.store(y, V, true);
      y += a.dim;
    };
    // U steps at a time, the next ones on their way; the rest one by one; zeros behind the row's end.
    int t = t0;
    const int valid = min(t1, row.len);
    Pack<T, V> next[U];
    auto fetch = [&]() {
#pragma unroll
      for (int u = 0; u < U; ++u, x += row.step) next[u].load(x, V, true);
    };
    if (t + U <= valid) fetch();
    for (; t + U <= valid; t += U) {
      Pack<T, V> in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) in[u] = next[u];
      if (t + 2 * U <= valid) fetch();
#pragma unroll
      for (int u = 0; u < U; ++u) advance(in[u]);
    }
    for (; t < valid; ++t, x += row.step) {
      Pack<T, V> in;
      in.load(x, V, true);
      advance(in);
    }
    for (; t < t1; ++t, y += a.dim) {
      Pack<T, V> out;
      out.zero();
      out.store(y, V, true);
    }
    at += t1 - t0;
  }
}

// Gradients of the steps [t0, t1) of row b: dx at those steps (at t0 = 0 the
// state's too), and what they add to the taps' and the bias' gradients.
template <class T, int K, int V>
__device__ __forceinline__ void conv_bwd_stretch(const pt_conv_args& a, const Taps<K, V>& taps, int b, int t0, int t1, int c,
                                                 Packed<V> (&dw)[K], Packed<V>& db) {
  constexpr int U = kConvBwdAhead;
  const ConvRow<T, K, V> row = conv_row<T, K, V>(a, b, c);
  const int len = row.len;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch + c;
  T* dx = a.dx ? static_cast<T*>(a.dx) + static_cast<long long>(b) * a.len * a.dim + c : nullptr;
  const long long s0 = static_cast<long long>(b) * (K - 1) * a.dim + c;
  const T* dso = a.dstate_out ? static_cast<const T*>(a.dstate_out) + s0 : nullptr;
  T* dsi = a.dstate_in ? static_cast<T*>(a.dstate_in) + s0 : nullptr;
  Packed<V> win[K], gw[K];  // win[j]: input at step t - K + 1 + j; gw[j]: g at step t - j
#pragma unroll
  for (int j = 0; j < K; ++j) gw[j].zero();
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    Pack<T, V> p;
    row.load(p, t0 - (K - 1) + j);
    win[j + 1].from(p);
  }
  const int first = t0 == 0 ? -(K - 1) : t0;  // first position whose gradient is written here
  const T* x = row.x + t0 * row.step;
  dy += t0 * a.dy_step;
  if (dx) dx += static_cast<long long>(t0 - (K - 1)) * a.dim;  // moves on with t, to position t - K + 1
  // Step t.  In the middle of a row (INNER) the step is valid and its position's gradient is this thread's to write;
  // elsewhere each of that is asked for.
  auto advance = [&](const Pack<T, V>& xin, const Pack<T, V>& gin, int t, auto inner) {
    constexpr bool INNER = decltype(inner)::value;
    const int pos = t - (K - 1);
    Packed<V> g, s;
    g.from(gin);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) win[j] = win[j + 1];
    win[K - 1].from(xin);
#pragma unroll
    for (int i = 0; i < Packed<V>::N; ++i) {
      if (a.silu) {
        const F2 pre = taps.pre(win, i), sig = sigmoid2<T>(pre);
        g.p[i] = mul2(g.p[i], silu_grad2(pre, sig));
      }
      // Steps behind the row's end have no output; their window may hold anything.
      if (!INNER && t >= len) g.p[i] = 0;
      if (INNER || (t < t1 && t < len)) {
#pragma unroll
        for (int j = 0; j < K; ++j) dw[j].p[i] = fma2(g.p[i], win[j].p[i], dw[j].p[i]);
        db.p[i] = add2(db.p[i], g.p[i]);
      }
#pragma unroll
      for (int j = K - 1; j > 0; --j) gw[j].p[i] = gw[j - 1].p[i];
      gw[0].p[i] = g.p[i];
      s.p[i] = 0;
#pragma unroll
      for (int j = 0; j < K; ++j) s.p[i] = fma2(taps.w[j].p[i], gw[j].p[i], s.p[i]);
    }
    if (INNER || (pos >= first && pos < t1)) {
      if (!INNER && dso && pos >= len - (K - 1) && pos < len) {
        Pack<T, V> more;
        more.load(dso + static_cast<long long>(pos - (len - (K - 1))) * a.dim, V, true);
#pragma unroll
        for (int i = 0; i < Packed<V>::N; ++i) s.p[i] = add2(s.p[i], more.pair(i));
      }
      Pack<T, V> out;
      s.to(out);
      if (INNER || pos >= 0) {
        if (dx) out.store(dx, V, true);
      } else if (dsi) {
        out.store(dsi + static_cast<long long>(pos + K - 1) * a.dim, V, true);
      }
    }
    if (dx) dx += a.dim;
  };
  auto edge = [&](int t) {
    Pack<T, V> xin, gin;
    if (t < len) {
      xin.load(x, V, true), gin.load(dy, V, true);
    } else {
      xin.zero(), gin.zero();
    }
    x += row.step, dy += a.dy_step;
    advance(xin, gin, t, std::integral_constant<bool, false>());
  };
  int t = t0;
  const int end = t1 + K - 1, valid = min(t1, len);
  for (; t < t0 + K - 1 && t < end; ++t) edge(t);
  Pack<T, V> xn[U], gn[U];
  auto fetch = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u, x += row.step, dy += a.dy_step) xn[u].load(x, V, true), gn[u].load(dy, V, true);
  };
  if (t + U <= valid) fetch();
  for (; t + U <= valid; t += U) {
    Pack<T, V> xin[U], gin[U];
#pragma unroll
    for (int u = 0; u < U; ++u) xin[u] = xn[u], gin[u] = gn[u];
    if (t + 2 * U <= valid) fetch();
#pragma unroll
    for (int u = 0; u < U; ++u) advance(xin[u], gin[u], t + u, std::integral_constant<bool, true>());
  }
  for (; t < end; ++t) edge(t);
}

template <class T, int K, int V>
__global__ void __launch_bounds__(kConvThreads, kConvBwdBlocks)
    seq_conv_bwd_kernel(pt_conv_args a, float* part, int cblocks, long long per) {
  extern __shared__ float tap_buf[];
  const int tx = static_cast<int>(blockDim.x), ty = static_cast<int>(blockDim.y);
  const int x = static_cast<int>(threadIdx.x), y = static_cast<int>(threadIdx.y);
  const int cb = static_cast<int>(blockIdx.x) % cblocks, chunk = static_cast<int>(blockIdx.x) / cblocks;
  const int c0 = cb * tx * V, c = c0 + x * V;
  Taps<K, V> taps;
  load_taps<T, K, V>(a, c0, tap_buf, taps);
  Packed<V> dw[K], db;
  db.zero();
#pragma unroll
  for (int j = 0; j < K; ++j) dw[j].zero();
  if (c < a.dim) {
    const long long walker = static_cast<long long>(chunk) * ty + y;
    if (a.len == 0) {
      // No steps: what the final state's gradient gives to the initial state.
      for (long long b = walker; b < a.batch; b += static_cast<long long>(gridDim.x / cblocks) * ty)
        conv_bwd_stretch<T, K, V>(a, taps, static_cast<int>(b), 0, 0, c, dw, db);
    } else {
      const long long all = static_cast<long long>(a.batch) * a.len;
      long long at = walker * per;
      const long long end = min(at + per, all);
      while (at < end) {
        const int b = static_cast<int>(at / a.len), t0 = static_cast<int>(at % a.len);
        const int t1 = static_cast<int>(min(static_cast<long long>(a.len), t0 + (end - at)));
        conv_bwd_stretch<T, K, V>(a, taps, b, t0, t1, c, dw, db);
        at += t1 - t0;
      }
    }
  }
  // The block's sum, one tap after the other (K passes over a small array).
  float* mine = part + static_cast<long long>(chunk) * a.dim * (K + 1);
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    const Packed<V>& from = j < K ? dw[j < K ? j : 0] : db;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) tap_buf[(y * tx + x) * V + v] = v & 1 ? hi2(from.p[v / 2]) : lo2(from.p[v / 2]);
    __syncthreads();
    for (int i = y * tx + x; i < tx * V; i += kConvThreads) {
      const int d = c0 + i;
      if (d < a.dim) {
        float s = 0.f;
        for (int r = 0; r < ty; ++r) s += tap_buf[r * tx * V + i];
        mine[j < K ? static_cast<long long>(d) * K + j : static_cast<long long>(a.dim) * K + d] = s;
      }
    }
  }
}

template <class T, int K, int V>
__global__ void __launch_bounds__(kConvThreads) seq_conv_step_kernel(pt_conv_args a, int cblocks, bool wide, unsigned* err) {
  const int cb = static_cast<int>(blockIdx.x) % cblocks, b = static_cast<int>(blockIdx.x) / cblocks;
  const int c = (cb * kConvThreads + static_cast<int>(threadIdx.x)) * V;
  const bool in = c < a.dim;
  const int tid = static_cast<int>(threadIdx.x);
  int slot = a.slots ? __ldg(a.slots + b) : b;
  if (slot >= a.cache_rows) {
    if (tid == 0) atomicOr(err, kSlotPastCache);
    slot = -1;
  }
  // Everything is on its way while the block looks whether an earlier row has the slot.
  T* state = static_cast<T*>(a.state_out) + slot * a.state_row + c;
  Pack<T, V> win[K];
  Pack<float, V * K> w;
  Pack<float, V> bias;
  if (in) {
    win[K - 1].load(static_cast<const T*>(a.x) + b * a.x_batch + c, V, true);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      // Plain loads, not the read-only ones: the cache is written below.
      const T* p = state + static_cast<long long>(j) * a.dim;
      if (slot < 0) {
        win[j].zero();
      } else if constexpr (V == 2 && sizeof(T) == 2) {
        *reinterpret_cast<unsigned*>(win[j].v) = *reinterpret_cast<const unsigned*>(p);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) win[j].v[v] = p[v];
      }
    }
    if (a.param_f32) {
      w.load(static_cast<const float*>(a.w) + static_cast<long long>(c) * K, V * K, wide);
    } else {
#pragma unroll
      for (int i = 0; i < V * K; ++i) w.v[i] = param<T>(a.w, static_cast<long long>(c) * K + i, false);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) bias.v[v] = a.bias ? param<T>(a.bias, c + v, a.param_f32) : 0.f;
  }
  if (a.slots && named_before(a.slots, b, slot, tid, kConvThreads)) {
    if (tid == 0) atomicOr(err, kSlotTwice);
    slot = -1;
  }
  if (!in) return;
  T* y = static_cast<T*>(a.y) + static_cast<long long>(b) * a.dim + c;
  Pack<T, V> out;
  if (slot < 0) {
    out.zero();
    out.store(y, V, true);
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s = bias.v[v];
#pragma unroll
    for (int j = 0; j < K; ++j) s = fmaf(w.v[v * K + j], win[j].f(v), s);
    out.set(v, a.silu ? s * lo2(sigmoid2<T>(pack2(s, s))) : s);
  }
  out.store(y, V, true);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) win[j + 1].store(state + static_cast<long long>(j) * a.dim, V, true);
}

// ---------------------------------------------------------------- host side
// Widest words; more than four taps leave registers for two channels only.
constexpr int kConvWideTaps = 4;

// Whether every row that `ptr` leads to starts on a word of V elements.
inline bool conv_wide(const void* ptr, long long s0, long long s1, int v, size_t e) {
  return !ptr || (aligned(ptr, v * e) && s0 % v == 0 && s1 % v == 0);
}
inline int conv_width(const pt_conv_args& a, size_t e, int most) {
  if (a.taps > kConvWideTaps && most > 2) most = 2;
  for (int v = most; v > 1; v = v > 2 ? 2 : 1) {
    if (a.dim % v == 0 && conv_wide(a.x, a.x_batch, a.x_step, v, e) && conv_wide(a.dy, a.dy_batch, a.dy_step, v, e) &&
        conv_wide(a.state_in, 0, 0, v, e) && conv_wide(a.state_out, a.state_row, 0, v, e) && conv_wide(a.y, 0, 0, v, e) &&
        conv_wide(a.dx, 0, 0, v, e) && conv_wide(a.dstate_in, 0, 0, v, e) &&
        conv_wide(a.dstate_out, 0, 0, v, e))
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
      default: break;
    }
    if constexpr (decltype(vc)::value <= 2) {
      switch (k) {
        case 5: return fn(vc, std::integral_constant<int, 5>());
        case 6: return fn(vc, std::integral_constant<int, 6>());
        case 7: return fn(vc, std::integral_constant<int, 7>());
        case 8: return fn(vc, std::integral_constant<int, 8>());
        default: break;
      }
    }
    return cudaErrorInvalidValue;
  };
  if (v == 1) return taps(std::integral_constant<int, 1>());
  if constexpr (VMAX > 2) {
    if (v > 2) return taps(std::integral_constant<int, VMAX>());
  }
  return taps(std::integral_constant<int, 2>());
}

template <class T>
constexpr int conv_word = 16 / static_cast<int>(sizeof(T));  // forward: 16 bytes
template <class T>
constexpr int conv_bwd_word = sizeof(T) == 4 ? 2 : 4;

// Threads along the channels (the rest of the block's 128 along the steps), and
// how many stretches of how many steps: `want` threads in all, at least `least`
// steps each, so that the overlap stays small.
struct ConvCut {
  int tx, ty, cblocks;
  long long per, walkers;
};
inline ConvCut conv_cut(const pt_conv_args& a, int v, long long want, int least) {
  ConvCut p;
  const long long groups = cdiv(a.dim, v), all = static_cast<long long>(a.batch) * a.len;
  p.tx = 32;
  while (p.tx < kConvThreads && p.tx < groups) p.tx *= 2;
  p.ty = kConvThreads / p.tx;
  p.cblocks = static_cast<int>(cdiv(groups, p.tx));
  const long long most = cdiv(want, static_cast<long long>(p.cblocks) * p.tx);
  p.per = cdiv(all > 0 ? all : 1, most);
  if (p.per < least) p.per = least;
  p.walkers = cdiv(all > 0 ? all : 1, p.per);
  return p;
}

template <class T>
ConvBwdPlan conv_bwd_plan(const pt_conv_args& a, int sm_count) {
  ConvBwdPlan p;
  p.v = conv_width(a, sizeof(T), conv_bwd_word<T>);
  const ConvCut c = conv_cut(a, p.v, kConvBwdBlocks * static_cast<long long>(kConvThreads) * sm_count, 24);
  p.tx = c.tx, p.cblocks = c.cblocks, p.per = c.per;
  p.chunks = static_cast<int>(cdiv(c.walkers, c.ty));
  return p;
}

template <class T>
cudaError_t conv_fwd(const pt_conv_args& a, int sm_count, cudaStream_t stream) {
  const int v = conv_width(a, sizeof(T), conv_word<T>);
  // One wave; with rows of different lengths four, whose stretches are dealt out as blocks finish.
  const int blocks = (v > 2 ? kConvFwdBlocks<4> : kConvFwdBlocks<2>) * (a.lengths ? 4 : 1);
  const ConvCut p = conv_cut(a, v, static_cast<long long>(blocks) * kConvThreads * sm_count, 8);
  const long long grid = p.cblocks * cdiv(p.walkers, p.ty);
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return by_width_taps<conv_word<T>>(v, a.taps, [&](auto vc, auto kc) {
    constexpr int V = decltype(vc)::value, K = decltype(kc)::value;
    seq_conv_fwd_kernel<T, K, V><<<static_cast<unsigned>(grid), dim3(p.tx, p.ty), sizeof(float) * p.tx * (V * K + 1), stream>>>(
        a, p.cblocks, p.per);
    return cudaGetLastError();
  });
}

template <class T>
cudaError_t conv_bwd(const pt_conv_args& a, float* ws, int sm_count, cudaStream_t stream) {
  const ConvBwdPlan p = conv_bwd_plan<T>(a, sm_count);
  const long long grid = static_cast<long long>(p.cblocks) * p.chunks;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaError_t e = by_width_taps<conv_bwd_word<T>>(p.v, a.taps, [&](auto vc, auto kc) {
    constexpr int V = decltype(vc)::value, K = decltype(kc)::value;
    const int floats = p.tx * (V * K + 1) > kConvThreads * V ? p.tx * (V * K + 1) : kConvThreads * V;
    seq_conv_bwd_kernel<T, K, V>
        <<<static_cast<unsigned>(grid), dim3(p.tx, kConvThreads / p.tx), sizeof(float) * floats, stream>>>(
            a, ws, p.cblocks, p.per);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return e;
  const int out = a.param_f32 ? PT_F32 : a.dtype;
  const long long m = static_cast<long long>(a.dim) * a.taps;
  return launch_reduce(ws, p.chunks, {{a.dw, m, out}, {a.dbias, a.dim, out}, {nullptr, 0, out}}, stream);
}

template <class T>
cudaError_t conv_step(const pt_conv_args& a, unsigned* err, cudaStream_t stream) {
  // Two channels per thread: a call is short, so many threads with little each.
  const int v = conv_width(a, sizeof(T), 2);
  const int cblocks = static_cast<int>(cdiv(a.dim, kConvThreads * v));
  const long long grid = static_cast<long long>(cblocks) * a.batch;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return by_width_taps<2>(v, a.taps, [&](auto vc, auto kc) {
    constexpr int V = decltype(vc)::value, K = decltype(kc)::value;
    const bool wide = aligned(a.w, Pack<float, V * K>::kWord);
    seq_conv_step_kernel<T, K, V><<<static_cast<unsigned>(grid), kConvThreads, 0, stream>>>(a, cblocks, wide, err);
    return cudaGetLastError();
  });
}

}  // namespace seq
}  // namespace pt
