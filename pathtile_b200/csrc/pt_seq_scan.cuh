// pt_seq_scan.cuh -- the selective state space scan
//   delta = dt + dt_bias (softplus of it);  h_t = exp(delta A) h_{t-1} + delta x B_t;
//   y_t = (C_t . h_t + D x) silu(z)
// over [batch, len, dim] activations: forward, backward, the single-token step.
//
// A thread owns 2 channels x 4 states and walks the steps in order, its states
// in registers; S lanes (2, 4, 8 or 16, for up to 8, 16, 32 or 64 states) share
// a channel pair, so a warp covers 64 / S channels.  A block of 4 warps stages
// tiles of 16 steps in shared memory (delta and delta x once per channel, B and
// C once for all channels of the group) and writes the outputs of a tile from
// shared memory in whole rows.  The sum over states crosses the S lanes by
// shuffles.
//
// Every (step, channel, state) costs an exponential: 16 per clock and SM, the
// bound for all but the shortest calls.
//
// Where batch x channels leave SMs idle, the length is cut into segments that
// run side by side: a first kernel scans each segment from a zero state and
// keeps its last state and the sum of its deltas, since a segment acts on the
// state before it as h -> exp(A sum delta) h + last.  The main kernel starts
// each segment from the states of the segments before it, joined in order.
//
// Backward: the states at every tile's start come from the forward pass
// (checkpoints); a tile is walked forward once more, keeping states and decays
// of 8 steps in registers, then backward:
//   dh_t = dy_t C_t + a_{t+1} dh_{t+1}
// dA, dD and ddt_bias stay with the channel; dB and dC sum over channels:
// across lanes by shuffles, across the block's warps in shared memory, across
// blocks through partial sums that a second kernel adds in a fixed order.
#pragma once

#include "pt_seq.h"
#include "pt_seq_common.cuh"

namespace pt {
namespace seq {

constexpr int kScanThreads = 128;
constexpr int kScanWarps = kScanThreads / 32;
constexpr int kTile = 16;      // steps per tile, and between checkpoints
constexpr int kHalf = kTile / 2;

template <int S>
struct ScanShape {
  static constexpr int kSlices = S;
  static constexpr int kStates = 4 * S;                      // padded number of states
  static constexpr int kWarpCh = 2 * (32 / S);               // channels per warp
  static constexpr int kCh = kScanWarps * kWarpCh;           // channels per block
  static constexpr int kRowThreads = kScanThreads / kTile;   // threads that stage one step: 8
  static constexpr int kE = kCh / kRowThreads;               // channels a thread stages
  static constexpr int kN = kStates / kRowThreads;           // states a thread stages (may be 1)
};

// Strides, sizes and flags as the kernels use them.
struct ScanDims {
  int cblocks, segs, seg_len, row_chunks;
  int wide;  // bit 0 x, 1 dt, 2 z, 3 dy, 4 contiguous outputs: rows may move in wide words
};

// Where a block works: its group, channels, segment.
template <int S>
struct ScanPlace {
  using P = ScanShape<S>;
  int g, c0, nch;  // group, first channel (of all), channels of this block
  __device__ __forceinline__ ScanPlace(const pt_scan_args& a, int cblocks, int cb) {
    const int per = a.dim / a.groups;
    g = cb / cblocks;
    const int first = (cb % cblocks) * P::kCh;
    c0 = g * per + first;
    nch = min(P::kCh, per - first);
  }
};

// Reads one step's states row (B or C) into shared memory.
template <class T, int S>
__device__ __forceinline__ void stage_states(const T* row, int n, bool live, float* dst) {
  using P = ScanShape<S>;
  const int k = static_cast<int>(threadIdx.x) & (P::kRowThreads - 1);
#pragma unroll
  for (int i = 0; i < P::kN; ++i) {
    const int j = k + i * P::kRowThreads;
    dst[j] = live && j < n ? to_f<T>(row[j]) : 0.f;
  }
}

__device__ __forceinline__ int scan_row_length(const pt_scan_args& a, int b) {
  if (!a.lengths) return a.len;
  const int n = __ldg(a.lengths + b);
  return n < 0 ? 0 : n > a.len ? a.len : n;
}

// This thread's decay rates times log2 e: exp(delta A) = 2^(delta A2).
template <int S>
__device__ __forceinline__ void load_rates(const pt_scan_args& a, int c, int nvalid_c, int s0, float (&A2)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      A2[i][j] = i < nvalid_c && s0 + j < a.state
                     ? __ldg(a.A + static_cast<long long>(c + i) * a.state + s0 + j) * kLog2e
                     : 0.f;
}

// A state array [rows, dim, state] (fp32): this thread's 2 x 4 values.
__device__ __forceinline__ void load_states(const float* p, const pt_scan_args& a, int c, int nvalid_c, int s0,
                                            float (&h)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      h[i][j] = i < nvalid_c && s0 + j < a.state ? p[static_cast<long long>(c + i) * a.state + s0 + j] : 0.f;
}
__device__ __forceinline__ void store_states(float* p, const pt_scan_args& a, int c, int nvalid_c, int s0,
                                             const float (&h)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i < nvalid_c && s0 + j < a.state) p[static_cast<long long>(c + i) * a.state + s0 + j] = h[i][j];
}

// Sum of v0 (for the pair's first channel) and v1 (second) over a channel's S
// lanes: an even lane gets the first channel's, an odd one the second's.
template <int S>
__device__ __forceinline__ float sum_slices(float v0, float v1, int slice) {
  const bool odd = slice & 1;
  float keep = odd ? v1 : v0;
  const float send = odd ? v0 : v1;
  keep += __shfl_xor_sync(0xffffffffu, send, 1);
#pragma unroll
  for (int m = 2; m < S; m *= 2) keep += __shfl_xor_sync(0xffffffffu, keep, m);
  return keep;
}

// ---------------------------------------------------------------- segments
// Forward (REV false): the state that a segment reaches from zero, and the sum
// of its deltas.  Backward: the gradient a_t dh_t that leaves the segment at
// its start when none enters at its end.
template <class T, int S, bool REV>
__global__ void __launch_bounds__(kScanThreads)
    seq_scan_segment_kernel(pt_scan_args a, ScanDims dm, float* seg_h, float* seg_d) {
  using P = ScanShape<S>;
  __shared__ float s_delta[kTile][P::kCh], s_in[kTile][P::kCh];
  __shared__ __align__(16) float s_B[kTile][P::kStates];
  const int nblk = dm.cblocks * a.groups;
  const int cb = static_cast<int>(blockIdx.x) % nblk;
  const int rest = static_cast<int>(blockIdx.x) / nblk;
  // The last segment (backward: the first) has none to hand its state to.
  const int seg = rest % (dm.segs - 1) + (REV ? 1 : 0);
  const int b = rest / (dm.segs - 1);
  const ScanPlace<S> at(a, dm.cblocks, cb);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int slice = lane & (S - 1), cl = warp * P::kWarpCh + 2 * (lane / S), s0 = 4 * slice;
  const int mine = max(0, min(2, at.nch - cl));
  float A2[2][4], h[2][4] = {}, dsum[2] = {0.f, 0.f};
  load_rates<S>(a, at.c0 + cl, mine, s0, A2);
  const int len = scan_row_length(a, b);
  const int t0 = seg * dm.seg_len, t1 = min(t0 + dm.seg_len, a.len);
  const int tiles = (t1 - t0 + kTile - 1) / kTile;
  const int tr = tid / P::kRowThreads, col = (tid % P::kRowThreads) * P::kE;
  const int ncol = max(0, min(P::kE, at.nch - col));
  float bias[P::kE];
#pragma unroll
  for (int i = 0; i < P::kE; ++i) bias[i] = i < ncol && a.dt_bias ? __ldg(a.dt_bias + at.c0 + col + i) : 0.f;
  for (int k = 0; k < tiles; ++k) {
    const int tile = t0 + (REV ? tiles - 1 - k : k) * kTile;
    const int t = tile + tr;
    const bool live = t < len && t < t1;
    Pack<T, P::kE> in, dt, z;
    if (live) {
      const long long c = at.c0 + col;
      dt.load(static_cast<const T*>(a.dt) + b * a.dt_batch + t * a.dt_step + c, ncol, dm.wide & 2);
      if (REV) {
        in.load(static_cast<const T*>(a.dy) + b * a.dy_batch + t * a.dy_step + c, ncol, dm.wide & 8);
        if (a.z) z.load(static_cast<const T*>(a.z) + b * a.z_batch + t * a.z_step + c, ncol, dm.wide & 4);
      } else {
        in.load(static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_step + c, ncol, dm.wide & 1);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P::kE; ++i) {
      float d = 0.f, v = 0.f;
      if (live && i < ncol) {
        d = dt.f(i) + bias[i];
        if (a.dt_softplus) d = softplusf(d);
        v = in.f(i);
        if (REV) {
          if (a.z) v *= siluf(z.f(i));
        } else {
          v *= d;
        }
      }
      s_delta[tr][col + i] = d;
      s_in[tr][col + i] = v;
    }
    const T* row = REV ? static_cast<const T*>(a.C) + b * a.C_batch + t * a.C_step + at.g * a.C_group
                       : static_cast<const T*>(a.B) + b * a.B_batch + t * a.B_step + at.g * a.B_group;
    stage_states<T, S>(row, a.state, live, s_B[tr]);
    __syncthreads();
#pragma unroll 4
    for (int q = 0; q < kTile; ++q) {
      const int i = REV ? kTile - 1 - q : q;
      const float4 Bv = *reinterpret_cast<const float4*>(&s_B[i][s0]);
      const float Bs[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float d = s_delta[i][cl + c], v = s_in[i][cl + c];
        dsum[c] += d;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = ex2(d * A2[c][j]);
          h[c][j] = REV ? e * fmaf(v, Bs[j], h[c][j]) : fmaf(e, h[c][j], v * Bs[j]);
        }
      }
    }
  }
  const long long row = static_cast<long long>(b) * dm.segs + seg;
  store_states(seg_h + row * a.dim * a.state, a, at.c0 + cl, mine, s0, h);
  if (slice == 0)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (c < mine) seg_d[row * a.dim + at.c0 + cl + c] = dsum[c];
}

// h <- exp(A sum delta of segment s) h + its own state.
__device__ __forceinline__ void join_segment(const pt_scan_args& a, const ScanDims& dm, const float* seg_h,
                                             const float* seg_d, int b, int s, int c, int mine, int s0,
                                             const float (&A2)[2][4], float (&h)[2][4]) {
  const long long row = static_cast<long long>(b) * dm.segs + s;
  float l[2][4];
  load_states(seg_h + row * a.dim * a.state, a, c, mine, s0, l);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float d = i < mine ? seg_d[row * a.dim + c + i] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[i][j] = fmaf(ex2(d * A2[i][j]), h[i][j], l[i][j]);
  }
}

// ---------------------------------------------------------------- forward
template <class T, int S, bool PAD>
__global__ void __launch_bounds__(kScanThreads)
    seq_scan_fwd_kernel(pt_scan_args a, ScanDims dm, const float* seg_h, const float* seg_d) {
  using P = ScanShape<S>;
  __shared__ float s_delta[kTile][P::kCh], s_in[kTile][P::kCh], s_y[kTile][P::kCh];
  __shared__ __align__(16) float s_B[kTile][P::kStates], s_C[kTile][P::kStates];
  const int nblk = dm.cblocks * a.groups;
  const int cb = static_cast<int>(blockIdx.x) % nblk;
  const int rest = static_cast<int>(blockIdx.x) / nblk;
  const int seg = rest % dm.segs, b = rest / dm.segs;
  const ScanPlace<S> at(a, dm.cblocks, cb);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int slice = lane & (S - 1), cl = warp * P::kWarpCh + 2 * (lane / S), s0 = 4 * slice;
  const int mine = max(0, min(2, at.nch - cl));
  float A2[2][4], h[2][4] = {};
  load_rates<S>(a, at.c0 + cl, mine, s0, A2);
  if (a.h0) load_states(a.h0 + static_cast<long long>(b) * a.dim * a.state, a, at.c0 + cl, mine, s0, h);
  for (int s = 0; s < seg; ++s) join_segment(a, dm, seg_h, seg_d, b, s, at.c0 + cl, mine, s0, A2, h);
  const int len = scan_row_length(a, b);
  const int t0 = seg * dm.seg_len, t1 = min(t0 + dm.seg_len, a.len);
  const int tr = tid / P::kRowThreads, col = (tid % P::kRowThreads) * P::kE;
  const int ncol = max(0, min(P::kE, at.nch - col));
  float bias[P::kE], Dv[P::kE];
#pragma unroll
  for (int i = 0; i < P::kE; ++i) {
    bias[i] = i < ncol && a.dt_bias ? __ldg(a.dt_bias + at.c0 + col + i) : 0.f;
    Dv[i] = i < ncol && a.D ? __ldg(a.D + at.c0 + col + i) : 0.f;
  }
  const long long ckpt_row = (static_cast<long long>(a.len) + kTile - 1) / kTile;
  for (int tile = t0; tile < t1; tile += kTile) {
    const int t = tile + tr;
    const bool live = t < len && t < t1;
    const long long c = at.c0 + col;
    Pack<T, P::kE> x, dt, z;
    if (live) {
      dt.load(static_cast<const T*>(a.dt) + b * a.dt_batch + t * a.dt_step + c, ncol, dm.wide & 2);
      x.load(static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_step + c, ncol, dm.wide & 1);
      if (a.z) z.load(static_cast<const T*>(a.z) + b * a.z_batch + t * a.z_step + c, ncol, dm.wide & 4);
    }
    if (a.checkpoints)
      store_states(a.checkpoints + (b * ckpt_row + tile / kTile) * a.dim * a.state, a, at.c0 + cl, mine, s0, h);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P::kE; ++i) {
      float d = 0.f, v = 0.f;
      if (live && i < ncol) {
        d = dt.f(i) + bias[i];
        if (a.dt_softplus) d = softplusf(d);
        v = d * x.f(i);
      }
      s_delta[tr][col + i] = d;
      s_in[tr][col + i] = v;
    }
    stage_states<T, S>(static_cast<const T*>(a.B) + b * a.B_batch + t * a.B_step + at.g * a.B_group, a.state, live,
                       s_B[tr]);
    stage_states<T, S>(static_cast<const T*>(a.C) + b * a.C_batch + t * a.C_step + at.g * a.C_group, a.state, live,
                       s_C[tr]);
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < kTile; ++i) {
      const float4 Bv = *reinterpret_cast<const float4*>(&s_B[i][s0]);
      const float4 Cv = *reinterpret_cast<const float4*>(&s_C[i][s0]);
      const float Bs[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, Cs[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
      float y[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float d = s_delta[i][cl + c], v = s_in[i][cl + c];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[c][j] = fmaf(ex2(d * A2[c][j]), h[c][j], v * Bs[j]);
          // States past the last one are not the operator's: 0 x inf must not reach y.
          s = PAD && s0 + j >= a.state ? s : fmaf(h[c][j], Cs[j], s);
        }
        y[c] = s;
      }
      const float sum = sum_slices<S>(y[0], y[1], slice);
      if (slice < 2) s_y[i][cl + slice] = sum;
    }
    __syncthreads();
    if (t < t1 && ncol > 0) {
      Pack<T, P::kE> out;
#pragma unroll
      for (int i = 0; i < P::kE; ++i) {
        float v = 0.f;
        if (live) {
          v = s_y[tr][col + i];
          if (a.D) v = fmaf(Dv[i], x.f(i), v);
          if (a.z) v *= siluf(z.f(i));
        }
        out.set(i, v);
      }
      out.store(static_cast<T*>(a.y) + (static_cast<long long>(b) * a.len + t) * a.dim + c, ncol, dm.wide & 16);
    }
  }
  if (a.hlast && seg == dm.segs - 1)
    store_states(a.hlast + static_cast<long long>(b) * a.dim * a.state, a, at.c0 + cl, mine, s0, h);
}

// ---------------------------------------------------------------- backward
// Eight values per lane (v[0..3] of dB, v[4..7] of dC for the slice's states),
// summed over the lanes that hold other channels; the lane's share of the sums
// is written to dst[0 .. 2 * states).
template <int S>
__device__ __forceinline__ void sum_channels(float (&v)[8], int lane, float* dst) {
  const int slice = lane & (S - 1), cg = lane / S;
  constexpr int L = 32 / S;  // lanes to sum over: 16, 8, 4 or 2
  int n = 8, first = 0;
#pragma unroll
  for (int m = L / 2; m >= 1; m /= 2) {
    if (n > 1) {
      const bool up = cg & m;
      n /= 2;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) {
          const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m * S);
        }
      first += up ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * S);
    }
  }
  // Value index i < 4: dB of state 4 slice + i; else dC of state 4 slice + i - 4.
  constexpr int kept = L >= 8 ? 1 : 8 / L;
  if (L <= 8 || (cg & (L / 8 - 1)) == 0) {
#pragma unroll
    for (int i = 0; i < kept; ++i) {
      const int k = first + i;
      dst[(k >> 2) * 4 * S + 4 * slice + (k & 3)] = v[i];
    }
  }
}

template <class T, int S, bool PAD>
__global__ void __launch_bounds__(kScanThreads)
    seq_scan_bwd_kernel(pt_scan_args a, ScanDims dm, const float* seg_h, const float* seg_d, float* part_bc,
                        float* part_a, float* part_d) {
  using P = ScanShape<S>;
  extern __shared__ __align__(16) float smem[];
  float(*s_delta)[P::kCh] = reinterpret_cast<float(*)[P::kCh]>(smem);
  float(*s_in)[P::kCh] = s_delta + kTile;   // delta x
  float(*s_dy)[P::kCh] = s_in + kTile;      // dout silu(z)
  float(*s_gB)[P::kCh] = s_dy + kTile;      // sum over states of dh B
  float(*s_gA)[P::kCh] = s_gB + kTile;      // sum over states of (d log a) A2
  float(*s_y)[P::kCh] = s_gA + kTile;       // sum over states of h C
  float(*s_accD)[P::kCh] = s_y + kTile;     // each staging thread's own sums of dD and ddt_bias
  float(*s_accb)[P::kCh] = s_accD + kTile;
  float(*s_B)[P::kStates] = reinterpret_cast<float(*)[P::kStates]>(s_accb + kTile);
  float(*s_C)[P::kStates] = s_B + kTile;
  float(*s_red)[kTile][2 * P::kStates] = reinterpret_cast<float(*)[kTile][2 * P::kStates]>(s_C + kTile);  // [warp]
  const int nblk = dm.cblocks * a.groups;
  const int cb = static_cast<int>(blockIdx.x) % nblk;
  const int rest = static_cast<int>(blockIdx.x) / nblk;
  const int seg = rest % dm.segs, chunk = rest / dm.segs;
  const ScanPlace<S> at(a, dm.cblocks, cb);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int slice = lane & (S - 1), cl = warp * P::kWarpCh + 2 * (lane / S), s0 = 4 * slice;
  const int mine = max(0, min(2, at.nch - cl));
  float A2[2][4], dA[2][4] = {};
  load_rates<S>(a, at.c0 + cl, mine, s0, A2);
  const int tr = tid / P::kRowThreads, col = (tid % P::kRowThreads) * P::kE;
  const int ncol = max(0, min(P::kE, at.nch - col));
#pragma unroll
  for (int i = 0; i < P::kE; ++i) s_accD[tr][col + i] = s_accb[tr][col + i] = 0.f;
  const int t0 = seg * dm.seg_len, t1 = min(t0 + dm.seg_len, a.len);
  const int tiles = max(0, (t1 - t0 + kTile - 1) / kTile);
  const long long ckpt_row = (static_cast<long long>(a.len) + kTile - 1) / kTile;
  const long long all = static_cast<long long>(a.dim) * a.state;
  for (int b = chunk; b < a.batch; b += dm.row_chunks) {
    const int len = scan_row_length(a, b);
    float g[2][4] = {};  // a_{t+1} dh_{t+1}
    if (a.dhlast) load_states(a.dhlast + b * all, a, at.c0 + cl, mine, s0, g);
    for (int s = dm.segs - 1; s > seg; --s) join_segment(a, dm, seg_h, seg_d, b, s, at.c0 + cl, mine, s0, A2, g);
    for (int k = tiles - 1; k >= 0; --k) {
      const int tile = t0 + k * kTile;
      const int t = tile + tr;
      const bool live = t < len && t < t1;
      const long long c = at.c0 + col;
      Pack<T, P::kE> x, dt, z, dy;
      x.zero(), dt.zero(), z.zero(), dy.zero();
      if (live) {
        dt.load(static_cast<const T*>(a.dt) + b * a.dt_batch + t * a.dt_step + c, ncol, dm.wide & 2);
        x.load(static_cast<const T*>(a.x) + b * a.x_batch + t * a.x_step + c, ncol, dm.wide & 1);
        dy.load(static_cast<const T*>(a.dy) + b * a.dy_batch + t * a.dy_step + c, ncol, dm.wide & 8);
        if (a.z) z.load(static_cast<const T*>(a.z) + b * a.z_batch + t * a.z_step + c, ncol, dm.wide & 4);
      }
      float h[2][4];
      load_states(a.checkpoints + (b * ckpt_row + tile / kTile) * all, a, at.c0 + cl, mine, s0, h);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < P::kE; ++i) {
        float d = 0.f, v = 0.f, w = 0.f;
        if (live && i < ncol) {
          d = dt.f(i) + (a.dt_bias ? __ldg(a.dt_bias + c + i) : 0.f);
          if (a.dt_softplus) d = softplusf(d);
          v = d * x.f(i);
          w = dy.f(i);
          if (a.z) w *= siluf(z.f(i));
        }
        s_delta[tr][col + i] = d;
        s_in[tr][col + i] = v;
        s_dy[tr][col + i] = w;
      }
      stage_states<T, S>(static_cast<const T*>(a.B) + b * a.B_batch + t * a.B_step + at.g * a.B_group, a.state, live,
                         s_B[tr]);
      stage_states<T, S>(static_cast<const T*>(a.C) + b * a.C_batch + t * a.C_step + at.g * a.C_group, a.state, live,
                         s_C[tr]);
      __syncthreads();
      // The state in the middle of the tile, then the later half, then the earlier one.
      float mid[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mid[i][j] = h[i][j];
#pragma unroll 2
      for (int i = 0; i < kHalf; ++i) {
        const float4 Bv = *reinterpret_cast<const float4*>(&s_B[i][s0]);
        const float Bs[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const float d = s_delta[i][cl + cc], v = s_in[i][cl + cc];
#pragma unroll
          for (int j = 0; j < 4; ++j) mid[cc][j] = fmaf(ex2(d * A2[cc][j]), mid[cc][j], v * Bs[j]);
        }
      }
#pragma unroll 1
      for (int half = 1; half >= 0; --half) {
        const int i0 = half * kHalf;
        float hs[kHalf + 1][2][4], as[kHalf][2][4];  // hs[i]: the state before step i0 + i
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
          for (int j = 0; j < 4; ++j) hs[0][cc][j] = half ? mid[cc][j] : h[cc][j];
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
          const float4 Bv = *reinterpret_cast<const float4*>(&s_B[i0 + i][s0]);
          const float Bs[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const float d = s_delta[i0 + i][cl + cc], v = s_in[i0 + i][cl + cc];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              as[i][cc][j] = ex2(d * A2[cc][j]);
              hs[i + 1][cc][j] = fmaf(as[i][cc][j], hs[i][cc][j], v * Bs[j]);
            }
          }
        }
#pragma unroll
        for (int i = kHalf - 1; i >= 0; --i) {
          const float4 Bv = *reinterpret_cast<const float4*>(&s_B[i0 + i][s0]);
          const float4 Cv = *reinterpret_cast<const float4*>(&s_C[i0 + i][s0]);
          const float Bs[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, Cs[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
          float bc[8] = {};
          float gB[2] = {}, gA[2] = {}, yy[2] = {};
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const float d = s_delta[i0 + i][cl + cc], v = s_in[i0 + i][cl + cc], w = s_dy[i0 + i][cl + cc];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bool real = !PAD || s0 + j < a.state;
              const float dh = fmaf(w, Cs[j], g[cc][j]);
              bc[j] = fmaf(dh, v, bc[j]);
              bc[4 + j] = fmaf(w, hs[i + 1][cc][j], bc[4 + j]);
              gB[cc] = real ? fmaf(dh, Bs[j], gB[cc]) : gB[cc];
              yy[cc] = real ? fmaf(hs[i + 1][cc][j], Cs[j], yy[cc]) : yy[cc];
              g[cc][j] = as[i][cc][j] * dh;
              const float dlog = g[cc][j] * hs[i][cc][j];
              gA[cc] = real ? fmaf(dlog, A2[cc][j], gA[cc]) : gA[cc];
              dA[cc][j] = fmaf(dlog, d, dA[cc][j]);
            }
          }
          sum_channels<S>(bc, lane, s_red[warp][i0 + i]);
          const float r0 = sum_slices<S>(gB[0], gB[1], slice);
          const float r1 = sum_slices<S>(gA[0], gA[1], slice);
          const float r2 = sum_slices<S>(yy[0], yy[1], slice);
          if (slice < 2) {
            s_gB[i0 + i][cl + slice] = r0;
            s_gA[i0 + i][cl + slice] = r1;
            s_y[i0 + i][cl + slice] = r2;
          }
        }
      }
      __syncthreads();
      if (t < t1 && ncol > 0) {
        Pack<T, P::kE> ox, odt, oz;
#pragma unroll
        for (int i = 0; i < P::kE; ++i) {
          float gx = 0.f, gd = 0.f, gz = 0.f;
          if (live && i < ncol) {
            const float xv = x.f(i), Dv = a.D ? __ldg(a.D + c + i) : 0.f, w = s_dy[tr][col + i];
            const float raw = dt.f(i) + (a.dt_bias ? __ldg(a.dt_bias + c + i) : 0.f);
            gx = s_gB[tr][col + i] * s_delta[tr][col + i];
            if (a.D) gx = fmaf(Dv, w, gx);
            gd = fmaf(s_gB[tr][col + i], xv, s_gA[tr][col + i] * kLn2);
            if (a.dt_softplus && raw <= 20.f) gd *= sigmoidf(raw);
            if (a.z) {
              const float zv = z.f(i);
              const float yv = a.D ? fmaf(Dv, xv, s_y[tr][col + i]) : s_y[tr][col + i];
              gz = dy.f(i) * yv * silu_grad(zv, sigmoidf(zv));
            }
            s_accD[tr][col + i] = fmaf(w, xv, s_accD[tr][col + i]);
            s_accb[tr][col + i] += gd;
          }
          ox.set(i, gx), odt.set(i, gd), oz.set(i, gz);
        }
        const long long o = (static_cast<long long>(b) * a.len + t) * a.dim + c;
        if (a.dx) ox.store(static_cast<T*>(a.dx) + o, ncol, dm.wide & 16);
        if (a.ddt) odt.store(static_cast<T*>(a.ddt) + o, ncol, dm.wide & 16);
        if (a.dz) oz.store(static_cast<T*>(a.dz) + o, ncol, dm.wide & 16);
      }
      if (part_bc) {
        // [block of the group's channels][batch][len][group][2 * states]
        const int steps = min(kTile, t1 - tile);
        for (int i = tid; i < steps * 2 * P::kStates; i += kScanThreads) {
          const int q = i / (2 * P::kStates), k2 = i % (2 * P::kStates);
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < kScanWarps; ++w) s += s_red[w][q][k2];
          part_bc[(((static_cast<long long>(cb % dm.cblocks) * a.batch + b) * a.len + tile + q) * a.groups + at.g) *
                      (2 * P::kStates) +
                  k2] = s;
        }
      }
    }
    if (a.dh0 && seg == 0) store_states(a.dh0 + b * all, a, at.c0 + cl, mine, s0, g);
  }
  const long long piece = static_cast<long long>(chunk) * dm.segs + seg;
  if (part_a) store_states(part_a + piece * all, a, at.c0 + cl, mine, s0, dA);
  __syncthreads();
  for (int i = tid; i < at.nch; i += kScanThreads) {
    float sD = 0.f, sb = 0.f;
#pragma unroll
    for (int q = 0; q < kTile; ++q) sD += s_accD[q][i], sb += s_accb[q][i];
    part_d[piece * 2 * a.dim + at.c0 + i] = sD;
    part_d[piece * 2 * a.dim + a.dim + at.c0 + i] = sb;
  }
}

template <int S>
constexpr int scan_bwd_smem() {
  using P = ScanShape<S>;
  return 4 * (8 * kTile * P::kCh + 2 * kTile * P::kStates + kScanWarps * kTile * 2 * P::kStates);
}

// dB and dC from the blocks' partial sums, in block order.
template <class T>
__global__ void seq_scan_bc_kernel(const float* part, int cblocks, long long rows, int states, int padded, T* dB,
                                   T* dC) {
  const long long n = rows * 2 * padded;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int k = 0; k < cblocks; ++k) s += part[k * n + i];
  const long long row = i / (2 * padded);
  const int k2 = static_cast<int>(i % (2 * padded));
  const int j = k2 < padded ? k2 : k2 - padded;
  T* out = k2 < padded ? dB : dC;
  if (out && j < states) out[row * states + j] = from_f<T>(s);
}

// ---------------------------------------------------------------- one token
// A lane holds four states of a channel, S lanes the channel.
template <class T, int S>
__global__ void __launch_bounds__(kScanThreads) seq_scan_step_kernel(pt_scan_args a, int cblocks, bool wide,
                                                                     unsigned* err) {
  constexpr int kCh = kScanThreads / S;
  const int cb = static_cast<int>(blockIdx.x) % cblocks, b = static_cast<int>(blockIdx.x) / cblocks;
  const int tid = static_cast<int>(threadIdx.x);
  const int slot = a.slots ? slot_of(a.slots, b, a.cache_rows, err, tid, kScanThreads) : b;
  const int slice = tid & (S - 1), s0 = 4 * slice;
  const int c = cb * kCh + tid / S;
  const bool in = c < a.dim;
  float y = 0.f;
  if (in && slot >= 0) {
    const int g = c / (a.dim / a.groups);
    float d = to_f<T>(static_cast<const T*>(a.dt)[b * a.dt_batch + c]) + (a.dt_bias ? __ldg(a.dt_bias + c) : 0.f);
    if (a.dt_softplus) d = softplusf(d);
    const float v = d * to_f<T>(static_cast<const T*>(a.x)[b * a.x_batch + c]);
    const T* Bp = static_cast<const T*>(a.B) + b * a.B_batch + g * a.B_group + s0;
    const T* Cp = static_cast<const T*>(a.C) + b * a.C_batch + g * a.C_group + s0;
    const float* Ap = a.A + static_cast<long long>(c) * a.state + s0;
    float* hp = a.hlast + slot * a.h_row + static_cast<long long>(c) * a.state + s0;
    if (wide && s0 + 4 <= a.state) {
      float4 h = *reinterpret_cast<const float4*>(hp);
      const float4 A = __ldg(reinterpret_cast<const float4*>(Ap));
      h.x = fmaf(ex2(d * (A.x * kLog2e)), h.x, v * to_f<T>(Bp[0]));
      h.y = fmaf(ex2(d * (A.y * kLog2e)), h.y, v * to_f<T>(Bp[1]));
      h.z = fmaf(ex2(d * (A.z * kLog2e)), h.z, v * to_f<T>(Bp[2]));
      h.w = fmaf(ex2(d * (A.w * kLog2e)), h.w, v * to_f<T>(Bp[3]));
      y = fmaf(h.x, to_f<T>(Cp[0]), fmaf(h.y, to_f<T>(Cp[1]), fmaf(h.z, to_f<T>(Cp[2]), h.w * to_f<T>(Cp[3]))));
      *reinterpret_cast<float4*>(hp) = h;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (s0 + j < a.state) {
          const float h = fmaf(ex2(d * (__ldg(Ap + j) * kLog2e)), hp[j], v * to_f<T>(Bp[j]));
          y = fmaf(h, to_f<T>(Cp[j]), y);
          hp[j] = h;
        }
      }
    }
  }
#pragma unroll
  for (int m = 1; m < S; m *= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
  if (in && slice == 0) {
    if (slot >= 0) {
      if (a.D) y = fmaf(__ldg(a.D + c), to_f<T>(static_cast<const T*>(a.x)[b * a.x_batch + c]), y);
      if (a.z) y *= siluf(to_f<T>(static_cast<const T*>(a.z)[b * a.z_batch + c]));
    }
    static_cast<T*>(a.y)[static_cast<long long>(b) * a.dim + c] = from_f<T>(y);
  }
}

// ---------------------------------------------------------------- host side
template <class F>
cudaError_t by_slices(int s, F&& fn) {
  switch (s) {
    case 2: return fn(std::integral_constant<int, 2>());
    case 4: return fn(std::integral_constant<int, 4>());
    case 8: return fn(std::integral_constant<int, 8>());
    case 16: return fn(std::integral_constant<int, 16>());
    default: return cudaErrorInvalidValue;
  }
}

template <class T, int S>
ScanDims scan_dims(const pt_scan_args& a, const ScanPlan& p) {
  using P = ScanShape<S>;
  constexpr int word = Pack<T, P::kE>::kWord, per = word / static_cast<int>(sizeof(T));
  const bool rows = (a.dim / a.groups) % per == 0;
  auto ok = [&](const void* q, long long s0, long long s1) {
    return rows && aligned(q, word) && s0 % per == 0 && s1 % per == 0;
  };
  ScanDims d{p.cblocks, p.segs, p.seg_len, p.row_chunks, 0};
  d.wide |= ok(a.x, a.x_batch, a.x_step) ? 1 : 0;
  d.wide |= ok(a.dt, a.dt_batch, a.dt_step) ? 2 : 0;
  d.wide |= ok(a.z, a.z_batch, a.z_step) ? 4 : 0;
  d.wide |= ok(a.dy, a.dy_batch, a.dy_step) ? 8 : 0;
  d.wide |= rows && aligned(a.y, word) && aligned(a.dx, word) && aligned(a.ddt, word) && aligned(a.dz, word) ? 16 : 0;
  return d;
}

// The segments' states and sums of deltas lie in the workspace's first floats.
inline size_t segment_floats(const pt_scan_args& a, const ScanPlan& p) {
  if (p.segs <= 1) return 0;
  const size_t n = static_cast<size_t>(a.batch) * p.segs * a.dim * (static_cast<size_t>(a.state) + 1);
  return (n + 3) / 4 * 4;
}

template <class T>
cudaError_t scan_fwd(const pt_scan_args& a, const ScanPlan& p, float* ws, cudaStream_t stream) {
  return by_slices(p.slices, [&](auto sc) -> cudaError_t {
    constexpr int S = decltype(sc)::value;
    const ScanDims dm = scan_dims<T, S>(a, p);
    float* seg_h = ws;
    float* seg_d = ws + static_cast<size_t>(a.batch) * p.segs * a.dim * a.state;
    const long long blocks = static_cast<long long>(p.cblocks) * a.groups * a.batch;
    if (blocks * p.segs > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (p.segs > 1) {
      seq_scan_segment_kernel<T, S, false>
          <<<static_cast<unsigned>(blocks * (p.segs - 1)), kScanThreads, 0, stream>>>(a, dm, seg_h, seg_d);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
    const unsigned grid = static_cast<unsigned>(blocks * p.segs);
    if (a.state == 4 * S)
      seq_scan_fwd_kernel<T, S, false><<<grid, kScanThreads, 0, stream>>>(a, dm, seg_h, seg_d);
    else
      seq_scan_fwd_kernel<T, S, true><<<grid, kScanThreads, 0, stream>>>(a, dm, seg_h, seg_d);
    return cudaGetLastError();
  });
}

template <class T>
cudaError_t scan_bwd(const pt_scan_args& a, const ScanPlan& p, float* ws, cudaStream_t stream) {
  return by_slices(p.slices, [&](auto sc) -> cudaError_t {
    constexpr int S = decltype(sc)::value;
    const ScanDims dm = scan_dims<T, S>(a, p);
    const long long pieces = static_cast<long long>(p.row_chunks) * p.segs;
    const long long all = static_cast<long long>(a.dim) * a.state;
    const long long rows = static_cast<long long>(a.batch) * a.len * a.groups;
    float* seg_h = ws;
    float* seg_d = ws + static_cast<size_t>(a.batch) * p.segs * a.dim * a.state;
    float* part_bc = ws + segment_floats(a, p);
    float* part_a = part_bc + p.cblocks * rows * 8 * S;
    float* part_d = part_a + pieces * all;
    const long long blocks = static_cast<long long>(p.cblocks) * a.groups;
    if (blocks * a.batch * p.segs > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    cudaError_t e;
    if (p.segs > 1) {
      seq_scan_segment_kernel<T, S, true>
          <<<static_cast<unsigned>(blocks * a.batch * (p.segs - 1)), kScanThreads, 0, stream>>>(a, dm, seg_h, seg_d);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    auto kernel = a.state == 4 * S ? seq_scan_bwd_kernel<T, S, false> : seq_scan_bwd_kernel<T, S, true>;
    constexpr int smem = scan_bwd_smem<S>();
    if (smem > 48 * 1024 &&
        (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess)
      return e;
    kernel<<<static_cast<unsigned>(blocks * pieces), kScanThreads, smem, stream>>>(
        a, dm, seg_h, seg_d, a.dB || a.dC ? part_bc : nullptr, a.dA ? part_a : nullptr, part_d);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if (a.dB || a.dC) {
      const long long n = rows * 8 * S;
      if (n > 0) {
        seq_scan_bc_kernel<T><<<static_cast<unsigned>(cdiv(n, 256)), 256, 0, stream>>>(
            part_bc, p.cblocks, rows, a.state, 4 * S, static_cast<T*>(a.dB), static_cast<T*>(a.dC));
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
      }
    }
    const int n = static_cast<int>(pieces);
    if (a.dA && (e = launch_reduce(part_a, n, all, all, a.dA, PT_F32, stream)) != cudaSuccess) return e;
    if (a.dD && (e = launch_reduce(part_d, n, 2LL * a.dim, a.dim, a.dD, PT_F32, stream)) != cudaSuccess) return e;
    if (a.ddt_bias &&
        (e = launch_reduce(part_d + a.dim, n, 2LL * a.dim, a.dim, a.ddt_bias, PT_F32, stream)) != cudaSuccess)
      return e;
    return cudaSuccess;
  });
}

template <class T>
cudaError_t scan_step(const pt_scan_args& a, int slices, unsigned* err, cudaStream_t stream) {
  return by_slices(slices, [&](auto sc) -> cudaError_t {
    constexpr int S = decltype(sc)::value;
    const int cblocks = static_cast<int>(cdiv(a.dim, kScanThreads / S));
    const long long grid = static_cast<long long>(cblocks) * a.batch;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    const bool wide = a.state % 4 == 0 && a.h_row % 4 == 0 && aligned(a.hlast, 16) && aligned(a.A, 16);
    seq_scan_step_kernel<T, S><<<static_cast<unsigned>(grid), kScanThreads, 0, stream>>>(a, cblocks, wide, err);
    return cudaGetLastError();
  });
}

}  // namespace seq
}  // namespace pt
