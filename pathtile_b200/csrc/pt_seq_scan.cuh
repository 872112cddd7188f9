// pt_seq_scan.cuh -- the selective state space scan
//   delta = dt + dt_bias (softplus of it);  h_t = exp(delta A) h_{t-1} + delta x B_t;
//   y_t = (C_t . h_t + D x) silu(z)
// over [batch, len, dim] activations: forward, backward, the single-token step.
//
// A scanning thread owns 2 channels x 4 states and walks the steps in order, its
// states in registers as packed pairs; S lanes (2, 4, 8 or 16, for up to 8, 16,
// 32 or 64 states) share a channel pair, so a warp covers 64 / S channels and a
// block's four scanning warps 256 / S.  Tiles of 16 steps lie in shared memory:
// delta and delta x once per channel, B and C once for all of the block's
// channels.  Other warps of the block convert the next tile from memory (softplus,
// products, gates) and write the last one's outputs in whole rows, while the
// scanners work on this one; the block meets once per tile.  The sum over states
// crosses the S lanes by shuffles, two steps of two channels together.
//
// Every (step, channel, state) costs an exponential: 16 per clock and SM, the
// bound for all but the shortest calls (8 x 2048 x 2048 channels with 16 states:
// 115 us; forward in bf16 with checkpoints 240 us, of which 14 % are places that
// 256 blocks leave empty on 148 SMs; the exponentials' pipe is busy 69 % of the
// time where two blocks sit on an SM).
//
// Where batch x channels leave SMs idle, the length is cut into segments that
// run side by side: a first kernel scans each segment from a zero state and
// keeps its last state and the sum of its deltas, since a segment acts on the
// state before it as h -> exp(A sum delta) h + last.  The main kernel starts
// each segment from the states of the segments before it, joined in order
// (1 x 16384 x 2048 in 9 segments: 173 + 217 us).
//
// Backward: the states at every tile's start come from the forward pass
// (checkpoints); a tile is walked forward once more, keeping states and decays
// of 4 steps in registers, then backward:
//   dh_t = dy_t C_t + a_{t+1} dh_{t+1}
// dA, dD and ddt_bias stay with the channel; dB and dC sum over channels:
// across lanes by shuffles, across the block's warps in shared memory, across
// blocks through partial sums that a second kernel adds in a fixed order.
// 763 us for the shape above: an instruction of a scanning warp every five
// cycles or so, and registers for two such warps per scheduler.
#pragma once

#include "pt_seq.h"
#include "pt_seq_common.cuh"

namespace pt {
namespace seq {

constexpr int kTile = 16;  // steps per tile, and between checkpoints
constexpr int kSub = 4;    // backward: steps whose states and decays are in registers together

// A block: 4 warps that scan, and some that stage.  Two blocks per SM are launched
// with the registers that leaves for each thread; the stagers give up what the
// scanners need.
constexpr int kScanners = 128, kScanWarps = kScanners / 32;
template <int STAGERS, int SCANNER_REGS, int STAGER_REGS>
struct ScanTeam {
  static constexpr int kStagers = STAGERS, kBlock = kScanners + STAGERS;
  static constexpr int kScannerRegs = SCANNER_REGS, kStagerRegs = STAGER_REGS;
  static constexpr int kLaunchRegs = 65536 / 2 / kBlock / 8 * 8;
  static_assert(kScanners * SCANNER_REGS + STAGERS * STAGER_REGS <= kBlock * kLaunchRegs, "more registers than launched with");
};
// Forward, eight staging warps with little each keep up with the scanners (238 us
// for 8 x 2048 x 2048 channels with 16 states in bf16; with four 243).  Backward,
// four are enough and leave the scanners more registers (762 us; with eight, which
// spill, 827).
// fp32 rows on their way take twice the registers (2048 x 48 x 256: 215 us, 283 us
// with the other split; 8 more with the exponentials of fp32 calls).
template <class T>
using ForwardTeam = ScanTeam<256, sizeof(T) == 4 ? 80 : 112, sizeof(T) == 4 ? 80 : 64>;
using BackwardTeam = ScanTeam<128, 136, 120>;

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int S, class TEAM>
struct ScanShape {
  static constexpr int kStates = 4 * S;                     // padded number of states
  static constexpr int kWarpCh = 2 * (32 / S);              // channels per scanning warp
  static constexpr int kCh = kScanWarps * kWarpCh;          // channels per block
  static constexpr int kRowThreads = TEAM::kStagers / kTile;  // threads that stage one step
  static constexpr int kE = kCh / kRowThreads;              // neighbouring channels a thread stages
  static constexpr int kN = (kStates + kRowThreads - 1) / kRowThreads;  // states a thread stages
};

// The whole block meets; scanners and stagers call it from their own code.
template <class TEAM>
__device__ __forceinline__ void meet() {
  asm volatile("barrier.sync 1, %0;" ::"n"(TEAM::kBlock) : "memory");
}

// Strides, sizes and flags as the kernels use them.
struct ScanDims {
  int cblocks, segs, seg_len, row_chunks;
  int wide;  // bit 0 x, 1 dt, 2 z, 3 dy, 4 outputs: rows may move in wide words
};

// A scanning thread's place: 2 channels, 4 states.
template <int S, class TEAM>
struct Scanner {
  using P = ScanShape<S, TEAM>;
  int lane, warp, slice, cl, s0, c, mine;  // cl: channel pair in the block, c: of all channels, mine: of the pair that exist
  __device__ __forceinline__ Scanner(int tid, int c0, int nch) {
    lane = tid & 31, warp = tid >> 5, slice = lane & (S - 1);
    cl = warp * P::kWarpCh + 2 * (lane / S), s0 = 4 * slice;
    c = c0 + cl;
    mine = max(0, min(2, nch - cl));
  }
};

// A staging thread's place: one step of the tile, kE channels.
template <int S, class TEAM>
struct Stager {
  using P = ScanShape<S, TEAM>;
  static constexpr int kPairs = (P::kE + 1) / 2;
  int tr, pr, col, c, n;  // tr: step, pr: place in the row, col: first channel in the block, c: of all, n: channels that exist
  __device__ __forceinline__ Stager(int tid, int c0, int nch) {
    tr = tid / P::kRowThreads, pr = tid % P::kRowThreads;
    col = pr * P::kE;
    c = c0 + col;
    n = max(0, min(P::kE, nch - col));
  }
  __device__ __forceinline__ void params(const float* p, F2 (&out)[kPairs]) const {
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      out[i] = pack2(p && 2 * i < n ? __ldg(p + c + 2 * i) : 0.f, p && 2 * i + 1 < n ? __ldg(p + c + 2 * i + 1) : 0.f);
  }
};

// A tensor's rows as a staging thread meets them, one tile after the other: the
// address moves on by a constant, instead of being made anew from strides.
template <class T>
struct Walk {
  const T* p;
  long long by;
  __device__ __forceinline__ Walk(const void* base, long long first, long long step, int tiles) {
    p = static_cast<const T*>(base) + first;
    by = step * (tiles * kTile);
  }
  __device__ __forceinline__ void on() { p += by; }
};

// One step's B or C row on its way to shared memory.
template <class T, int S, class TEAM>
struct StateRow {
  using P = ScanShape<S, TEAM>;
  T v[P::kN];
  __device__ __forceinline__ void load(const T* row, int n, bool live, int k) {
#pragma unroll
    for (int i = 0; i < P::kN; ++i) {
      const int j = k + i * P::kRowThreads;
      v[i] = live && j < n ? __ldg(row + j) : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(float* dst, int k) const {
#pragma unroll
    for (int i = 0; i < P::kN; ++i) {
      const int j = k + i * P::kRowThreads;
      if (P::kStates % P::kRowThreads == 0 || j < P::kStates) dst[j] = to_f<T>(v[i]);
    }
  }
};

__device__ __forceinline__ int scan_row_length(const pt_scan_args& a, int b) {
  if (!a.lengths) return a.len;
  const int n = __ldg(a.lengths + b);
  return n < 0 ? 0 : n > a.len ? a.len : n;
}

// A thread's values of [2 channels][4 states] are two packed pairs per channel.
using Quad = F2[2][2];

// A state array [dim, state] in global memory (fp32): this thread's values.
template <int S, class TEAM>
__device__ __forceinline__ void load_states(const float* p, const pt_scan_args& a, const Scanner<S, TEAM>& me, Quad& h) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* q = p + static_cast<long long>(me.c + i) * a.state + me.s0;
    if (i < me.mine && (a.state & 3) == 0 && me.s0 < a.state && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const float4 v = *reinterpret_cast<const float4*>(q);
      h[i][0] = pack2(v.x, v.y), h[i][1] = pack2(v.z, v.w);
    } else {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = i < me.mine && me.s0 + j < a.state ? q[j] : 0.f;
      h[i][0] = pack2(v[0], v[1]), h[i][1] = pack2(v[2], v[3]);
    }
  }
}
template <int S, class TEAM>
__device__ __forceinline__ void store_states(float* p, const pt_scan_args& a, const Scanner<S, TEAM>& me, const Quad& h) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float* q = p + static_cast<long long>(me.c + i) * a.state + me.s0;
    const float v[4] = {lo2(h[i][0]), hi2(h[i][0]), lo2(h[i][1]), hi2(h[i][1])};
    if (i < me.mine && (a.state & 3) == 0 && me.s0 < a.state && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i < me.mine && me.s0 + j < a.state) q[j] = v[j];
    }
  }
}

// Decay rates times log2 e: exp(delta A) = 2^(delta A2).
template <int S, class TEAM>
__device__ __forceinline__ void load_rates(const pt_scan_args& a, const Scanner<S, TEAM>& me, Quad& A2) {
  load_states(a.A, a, me, A2);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int p = 0; p < 2; ++p) A2[i][p] = mul2(A2[i][p], pack2(kLog2e, kLog2e));
}

// exp(delta A) = 2^(delta A2).  A state that forgets slowly multiplies hundreds of
// these, so what counts is their mean error: the hardware's 2^x lies 2e-8 low on
// the average between -0.25 and -0.001 (measured; a float's half step below 1 is
// 3e-8).  Raising the exponent by 2e-8 costs nothing and leaves a few 1e-9; 2^0
// stays 1, so a step of no duration leaves a state as it is.
constexpr float kCentre = 2e-8f;
__device__ __forceinline__ F2 decay(F2 delta, F2 A2) { return ex2x2(fma2(delta, A2, same2(kCentre))); }

// A channel pair's values of one step, each twice: ready for packed arithmetic over states.
struct Both {
  F2 v[2];
  __device__ __forceinline__ Both() {}
  __device__ __forceinline__ explicit Both(const float* p) {
    const float2 f = *reinterpret_cast<const float2*>(p);
    v[0] = pack2(f.x, f.x), v[1] = pack2(f.y, f.y);
  }
};
// Four states' values of one step, in packed pairs.
struct Four {
  F2 v[2];
  __device__ __forceinline__ Four() {}
  __device__ __forceinline__ explicit Four(const float* p) {
    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(p);
    v[0] = f.x, v[1] = f.y;
  }
};

// Sums over a channel's S lanes of the values of two steps and two channels
// (v[step][channel]).  Lane 0 gets step 0 channel 0, lane 1 step 0 channel 1,
// lanes 2 and 3 step 1; with two lanes each gets its channel's both steps.
template <int S>
__device__ __forceinline__ void sum_slices(float (&v)[2][2], int slice, float& first, float& second) {
  const bool odd = slice & 1;
  if constexpr (S == 2) {
    first = (odd ? v[0][1] : v[0][0]) + __shfl_xor_sync(0xffffffffu, odd ? v[0][0] : v[0][1], 1);
    second = (odd ? v[1][1] : v[1][0]) + __shfl_xor_sync(0xffffffffu, odd ? v[1][0] : v[1][1], 1);
  } else {
    const bool up = slice & 2;
    const float a0 = (up ? v[1][0] : v[0][0]) + __shfl_xor_sync(0xffffffffu, up ? v[0][0] : v[1][0], 2);
    const float a1 = (up ? v[1][1] : v[0][1]) + __shfl_xor_sync(0xffffffffu, up ? v[0][1] : v[1][1], 2);
    first = (odd ? a1 : a0) + __shfl_xor_sync(0xffffffffu, odd ? a0 : a1, 1);
#pragma unroll
    for (int m = 4; m < S; m *= 2) first += __shfl_xor_sync(0xffffffffu, first, m);
    second = 0.f;
  }
}
// Writes what sum_slices left, to rows i and i + 1 of dst.
template <int S>
__device__ __forceinline__ void put_sums(float (*dst)[64 / S * kScanWarps], int i, int cl, int slice, float first,
                                         float second) {
  if constexpr (S == 2) {
    dst[i][cl + slice] = first;
    dst[i + 1][cl + slice] = second;
  } else {
    if (slice < 4) dst[i + (slice >> 1)][cl + (slice & 1)] = first;
  }
}

// How the states fill their lanes' fours: all do, some lanes have none, or one
// lane has some.  What padded states hold must not reach a sum (0 x inf): a lane
// without states gives 0, a lane with some leaves the others out one by one.
enum Fill { kFull, kLanes, kPartial };
inline Fill fill_of(int states, int slices) {
  return states == 4 * slices ? kFull : states % 4 == 0 ? kLanes : kPartial;
}

// s + h . c over the pair's states that exist.
__device__ __forceinline__ float dot2(F2 h, F2 c, float s, int first, int states) {
  if (first < states) s = fmaf(lo2(h), lo2(c), s);
  if (first + 1 < states) s = fmaf(hi2(h), hi2(c), s);
  return s;
}

// Where a block works.
template <int S, class TEAM>
struct ScanBlock {
  int cb, rest, g, c0, nch;  // block of channels, index of the rest of the grid, group, first channel, channels
  __device__ __forceinline__ ScanBlock(const pt_scan_args& a, int cblocks) {
    const int nblk = cblocks * a.groups;
    cb = static_cast<int>(blockIdx.x) % nblk;
    rest = static_cast<int>(blockIdx.x) / nblk;
    const int per = a.dim / a.groups, first = (cb % cblocks) * 64 / S * kScanWarps;
    g = cb / cblocks;
    c0 = g * per + first;
    nch = min(64 / S * kScanWarps, per - first);
  }
};

// ---------------------------------------------------------------- segments
// Forward (REV false): the state that a segment reaches from zero, and the sum
// of its deltas.  Backward: the gradient a_t dh_t that leaves the segment at
// its start when none enters at its end.
template <int S, class TEAM>
struct SegmentSmem {
  using P = ScanShape<S, TEAM>;
  float d[2][kTile][P::kCh], v[2][kTile][P::kCh];  // delta; delta x or dout silu(z)
  float B[2][kTile][P::kStates];
};

template <class T, int S, bool REV>
__global__ void __launch_bounds__(ForwardTeam<T>::kBlock, 2)
    seq_scan_segment_kernel(pt_scan_args a, ScanDims dm, float* seg_h, float* seg_d) {
  using TEAM = ForwardTeam<T>;
  using P = ScanShape<S, TEAM>;
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sm = *reinterpret_cast<SegmentSmem<S, TEAM>*>(smem);
  const ScanBlock<S, TEAM> at(a, dm.cblocks);
  // The last segment (backward: the first) has none to hand its state to.
  const int seg = at.rest % (dm.segs - 1) + (REV ? 1 : 0), b = at.rest / (dm.segs - 1);
  const int len = scan_row_length(a, b);
  const int t0 = seg * dm.seg_len, t1 = min(t0 + dm.seg_len, a.len);
  const int tiles = (t1 - t0 + kTile - 1) / kTile;
  auto tile_of = [&](int k) { return t0 + (REV ? tiles - 1 - k : k) * kTile; };
  const int tid = static_cast<int>(threadIdx.x);
  if (tid >= kScanners) {
    fewer_registers<TEAM::kStagerRegs>();
    const Stager<S, TEAM> me(tid - kScanners, at.c0, at.nch);
    F2 bias[me.kPairs];
    me.params(a.dt_bias, bias);
    Pack<T, P::kE> dt, in, z;
    StateRow<T, S, TEAM> row;
    const int end = min(len, t1), way = REV ? -1 : 1;
    int t = tile_of(0) + me.tr, t_in = t;  // of the tile to load, of the one loaded last
    const void* in_base = REV ? a.dy : a.x;
    const long long in_batch = REV ? a.dy_batch : a.x_batch, in_step = REV ? a.dy_step : a.x_step;
    Walk<T> wdt(a.dt, b * a.dt_batch + t * a.dt_step + me.c, a.dt_step, way);
    Walk<T> win(in_base, b * in_batch + t * in_step + me.c, in_step, way);
    Walk<T> wz(a.z, a.z ? b * a.z_batch + t * a.z_step + me.c : 0, a.z_step, way);
    Walk<T> wrow(REV ? a.C : a.B,
                 REV ? b * a.C_batch + t * a.C_step + at.g * a.C_group : b * a.B_batch + t * a.B_step + at.g * a.B_group,
                 REV ? a.C_step : a.B_step, way);
    const bool gated = REV && a.z;
    auto load = [&]() {
      const bool live = t < end;
      if (live) {
        dt.load(wdt.p, me.n, dm.wide & 2);
        in.load(win.p, me.n, dm.wide & (REV ? 8 : 1));
        if (gated) z.load(wz.p, me.n, dm.wide & 4);
      }
      row.load(wrow.p, a.state, live, me.pr);
      t_in = t;
      t += way * kTile;
      wdt.on(), win.on(), wz.on(), wrow.on();
    };
    auto convert = [&](int k) {
      F2 d[me.kPairs] = {}, v[me.kPairs] = {};
      if (t_in < end) {
#pragma unroll
        for (int i = 0; i < me.kPairs; ++i) {
          d[i] = add2(dt.pair(i), bias[i]);
          if (a.dt_softplus) d[i] = softplus2<T>(d[i]);
          v[i] = in.pair(i);
          if constexpr (REV) {
            if (gated) {
              const F2 zi = z.pair(i);
              v[i] = mul2(v[i], mul2(zi, sigmoid2<T>(zi)));
            }
          } else {
            v[i] = mul2(v[i], d[i]);
          }
        }
      }
      put_pairs<P::kE>(&sm.d[k & 1][me.tr][me.col], d);
      put_pairs<P::kE>(&sm.v[k & 1][me.tr][me.col], v);
      row.store(sm.B[k & 1][me.tr], me.pr);
    };
    if (tiles > 0) {
      load();
      convert(0);
      if (tiles > 1) load();
    }
    meet<TEAM>();
    for (int k = 0; k < tiles; ++k) {
      if (k + 1 < tiles) convert(k + 1);
      if (k + 2 < tiles) load();
      meet<TEAM>();
    }
    return;
  }
  more_registers<TEAM::kScannerRegs>();
  const Scanner<S, TEAM> me(tid, at.c0, at.nch);
  Quad A2, h = {};
  float dsum[2] = {0.f, 0.f};
  load_rates(a, me, A2);
  meet<TEAM>();
  for (int k = 0; k < tiles; ++k) {
    const int st = k & 1;
    if (tile_of(k) >= len) {  // behind the row's end nothing moves
      meet<TEAM>();
      continue;
    }
#pragma unroll 8
    for (int q = 0; q < kTile; ++q) {
      const int i = REV ? kTile - 1 - q : q;
      const Both d(&sm.d[st][i][me.cl]), v(&sm.v[st][i][me.cl]);
      const Four B(&sm.B[st][i][me.s0]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        dsum[c] += lo2(d.v[c]);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const F2 e = decay(d.v[c], A2[c][p]);
          h[c][p] = REV ? mul2(e, fma2(v.v[c], B.v[p], h[c][p])) : fma2(e, h[c][p], mul2(v.v[c], B.v[p]));
        }
      }
    }
    meet<TEAM>();
  }
  const long long out = static_cast<long long>(b) * dm.segs + seg;
  store_states(seg_h + out * a.dim * a.state, a, me, h);
  if (me.slice == 0)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (c < me.mine) seg_d[out * a.dim + me.c + c] = dsum[c];
}

// exp(delta A) h.  Of a whole segment the factor may be past the largest float where the product is not, so it
// is applied as two square roots; a state of zero stays zero whatever the factor.
__device__ __forceinline__ F2 carry(F2 delta, F2 A2, F2 h) {
  const F2 root = ex2x2(mul2(fma2(delta, A2, same2(kCentre)), same2(0.5f)));
  const F2 p = mul2(mul2(root, h), root);
  return pack2(lo2(h) == 0.f ? 0.f : lo2(p), hi2(h) == 0.f ? 0.f : hi2(p));
}

// h <- exp(A sum delta of segment s) h + its own state.
template <int S, class TEAM>
__device__ __forceinline__ void join_segment(const pt_scan_args& a, const ScanDims& dm, const float* seg_h,
                                             const float* seg_d, int b, int s, const Scanner<S, TEAM>& me, const Quad& A2,
                                             Quad& h) {
  const long long row = static_cast<long long>(b) * dm.segs + s;
  Quad l;
  load_states(seg_h + row * a.dim * a.state, a, me, l);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float d = i < me.mine ? seg_d[row * a.dim + me.c + i] : 0.f;
#pragma unroll
    for (int p = 0; p < 2; ++p) h[i][p] = add2(carry(pack2(d, d), A2[i][p], h[i][p]), l[i][p]);
  }
}

// ---------------------------------------------------------------- forward
template <int S, class TEAM>
struct ForwardSmem {
  using P = ScanShape<S, TEAM>;
  float d[2][kTile][P::kCh], v[2][kTile][P::kCh], y[2][kTile][P::kCh];  // delta, delta x, sums over states of h C
  float B[2][kTile][P::kStates], C[2][kTile][P::kStates];
};

template <class T, int S, Fill FILL>
__global__ void __launch_bounds__(ForwardTeam<T>::kBlock, 2)
    seq_scan_fwd_kernel(pt_scan_args a, ScanDims dm, const float* seg_h, const float* seg_d) {
  using TEAM = ForwardTeam<T>;
  using P = ScanShape<S, TEAM>;
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sm = *reinterpret_cast<ForwardSmem<S, TEAM>*>(smem);
  const ScanBlock<S, TEAM> at(a, dm.cblocks);
  const int seg = at.rest % dm.segs, b = at.rest / dm.segs;
  const int len = scan_row_length(a, b);
  const int t0 = seg * dm.seg_len, t1 = min(t0 + dm.seg_len, a.len);
  const int tiles = max(0, (t1 - t0 + kTile - 1) / kTile);
  const int tid = static_cast<int>(threadIdx.x);
  if (tid >= kScanners) {
    fewer_registers<TEAM::kStagerRegs>();
    const Stager<S, TEAM> me(tid - kScanners, at.c0, at.nch);
    F2 bias[me.kPairs], Dv[me.kPairs];
    me.params(a.dt_bias, bias);
    me.params(a.D, Dv);
    // x and z of three tiles: the one whose outputs are next, the one being scanned, the next one.
    Pack<T, P::kE> dt, x[3], z[3];
    StateRow<T, S, TEAM> rowB, rowC;
    const int end = min(len, t1);
    int t = t0 + me.tr;  // of the tile to load; t_in of the one to convert, t_out of the one to write
    int t_in = t, t_out = t;
    Walk<T> wdt(a.dt, b * a.dt_batch + t * a.dt_step + me.c, a.dt_step, 1);
    Walk<T> wx(a.x, b * a.x_batch + t * a.x_step + me.c, a.x_step, 1);
    Walk<T> wz(a.z, a.z ? b * a.z_batch + t * a.z_step + me.c : 0, a.z_step, 1);
    Walk<T> wB(a.B, b * a.B_batch + t * a.B_step + at.g * a.B_group, a.B_step, 1);
    Walk<T> wC(a.C, b * a.C_batch + t * a.C_step + at.g * a.C_group, a.C_step, 1);
    T* y_out = static_cast<T*>(a.y) + (static_cast<long long>(b) * a.len + t) * a.dim + me.c;
    auto load = [&]() {
      const bool live = t < end;
      if (live) {
        dt.load(wdt.p, me.n, dm.wide & 2);
        x[2].load(wx.p, me.n, dm.wide & 1);
        if (a.z) z[2].load(wz.p, me.n, dm.wide & 4);
      }
      rowB.load(wB.p, a.state, live, me.pr);
      rowC.load(wC.p, a.state, live, me.pr);
      t += kTile;
      wdt.on(), wx.on(), wz.on(), wB.on(), wC.on();
    };
    auto convert = [&](int k) {
      x[0] = x[1], z[0] = z[1], x[1] = x[2], z[1] = z[2];
      F2 d[me.kPairs] = {}, v[me.kPairs] = {};
      if (t_in < end) {
#pragma unroll
        for (int i = 0; i < me.kPairs; ++i) {
          d[i] = add2(dt.pair(i), bias[i]);
          if (a.dt_softplus) d[i] = softplus2<T>(d[i]);
          v[i] = mul2(d[i], x[1].pair(i));
        }
      }
      put_pairs<P::kE>(&sm.d[k & 1][me.tr][me.col], d);
      put_pairs<P::kE>(&sm.v[k & 1][me.tr][me.col], v);
      rowB.store(sm.B[k & 1][me.tr], me.pr);
      rowC.store(sm.C[k & 1][me.tr], me.pr);
      t_in += kTile;
    };
    auto finish = [&](int k) {
      if (t_out < t1) {
        Pack<T, P::kE> out;
        out.zero();
        if (t_out < len) {
          F2 y[me.kPairs];
          get_pairs<P::kE>(&sm.y[k & 1][me.tr][me.col], y);
#pragma unroll
          for (int i = 0; i < me.kPairs; ++i) {
            if (a.D) y[i] = fma2(Dv[i], x[0].pair(i), y[i]);
            if (a.z) {
              const F2 zi = z[0].pair(i);
              y[i] = mul2(y[i], mul2(zi, sigmoid2<T>(zi)));
            }
            out.set_pair(i, y[i]);
          }
        }
        out.store(y_out, me.n, dm.wide & 16);
      }
      t_out += kTile;
      y_out += static_cast<long long>(kTile) * a.dim;
    };
    if (tiles > 0) {
      load();
      convert(0);
      if (tiles > 1) load();
    }
    meet<TEAM>();
    for (int k = 0; k < tiles; ++k) {
      if (k > 0) finish(k - 1);
      if (k + 1 < tiles) {
        convert(k + 1);
        if (k + 2 < tiles) load();
      } else {
        x[0] = x[1], z[0] = z[1];
      }
      meet<TEAM>();
    }
    if (tiles > 0) finish(tiles - 1);
    return;
  }
  more_registers<TEAM::kScannerRegs>();
  const Scanner<S, TEAM> me(tid, at.c0, at.nch);
  Quad A2, h = {};
  load_rates(a, me, A2);
  if (a.h0) load_states(a.h0 + static_cast<long long>(b) * a.dim * a.state, a, me, h);
  for (int s = 0; s < seg; ++s) join_segment(a, dm, seg_h, seg_d, b, s, me, A2, h);
  const long long ckpt_row = (static_cast<long long>(a.len) + kTile - 1) / kTile;
  meet<TEAM>();
  for (int k = 0; k < tiles; ++k) {
    const int st = k & 1;
    if (t0 + k * kTile < len) {  // behind the row's end nothing moves
      if (a.checkpoints)
        store_states(a.checkpoints + (b * ckpt_row + t0 / kTile + k) * a.dim * a.state, a, me, h);
      // Decays of the next pair of steps are computed while this pair is scanned, and its sums cross the lanes one
      // pair later: no instruction waits for the one before it.
      F2 e[2][2][2];
      Four Bn[2] = {Four(&sm.B[st][0][me.s0]), Four(&sm.B[st][1][me.s0])};
      Both vn[2] = {Both(&sm.v[st][0][me.cl]), Both(&sm.v[st][1][me.cl])};
      Both dn[2] = {Both(&sm.d[st][0][me.cl]), Both(&sm.d[st][1][me.cl])};
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int p = 0; p < 2; ++p) e[q][c][p] = decay(dn[q].v[c], A2[c][p]);
      dn[0] = Both(&sm.d[st][2][me.cl]), dn[1] = Both(&sm.d[st][3][me.cl]);
      float last[2][2];
#pragma unroll
      for (int i = 0; i < kTile; i += 2) {
        F2 en[2][2][2];
        Both v[2] = {vn[0], vn[1]};
        Four B[2] = {Bn[0], Bn[1]};
        const Four C[2] = {Four(&sm.C[st][i][me.s0]), Four(&sm.C[st][i + 1][me.s0])};
        if (i + 2 < kTile) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int p = 0; p < 2; ++p) en[q][c][p] = decay(dn[q].v[c], A2[c][p]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            vn[q] = Both(&sm.v[st][i + 2 + q][me.cl]);
            Bn[q] = Four(&sm.B[st][i + 2 + q][me.s0]);
            if (i + 4 < kTile) dn[q] = Both(&sm.d[st][i + 4 + q][me.cl]);
          }
        }
        float y[2][2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int p = 0; p < 2; ++p) h[c][p] = fma2(e[q][c][p], h[c][p], mul2(v[q].v[c], B[q].v[p]));
            if constexpr (FILL == kPartial) {
              y[q][c] = dot2(h[c][1], C[q].v[1], dot2(h[c][0], C[q].v[0], 0.f, me.s0, a.state), me.s0 + 2, a.state);
            } else {
              const F2 s = fma2(h[c][1], C[q].v[1], mul2(h[c][0], C[q].v[0]));
              y[q][c] = lo2(s) + hi2(s);
              if (FILL == kLanes && me.s0 >= a.state) y[q][c] = 0.f;
            }
          }
        if (i > 0) {
          float first, second;
          sum_slices<S>(last, me.slice, first, second);
          put_sums<S>(sm.y[st], i - 2, me.cl, me.slice, first, second);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            last[q][c] = y[q][c];
#pragma unroll
            for (int p = 0; p < 2; ++p) e[q][c][p] = en[q][c][p];
          }
      }
      float first, second;
      sum_slices<S>(last, me.slice, first, second);
      put_sums<S>(sm.y[st], kTile - 2, me.cl, me.slice, first, second);
    }
    meet<TEAM>();
  }
  if (a.hlast && seg == dm.segs - 1)
    store_states(a.hlast + static_cast<long long>(b) * a.dim * a.state, a, me, h);
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

template <int S, class TEAM>
struct BackwardSmem {
  using P = ScanShape<S, TEAM>;
  float d[2][kTile][P::kCh];                          // delta
  float v[2][kTile][P::kCh], w[2][kTile][P::kCh];     // delta x, dout silu(z); then the sums over states of dh B, h C
  float gA[2][kTile][P::kCh];                         // sums over states of (d log a) A2
  float B[2][kTile][P::kStates], C[2][kTile][P::kStates];
  float red[2][kScanWarps][kTile][2 * P::kStates];    // the warps' sums over channels, of dB and dC
  float4 ck[2][kScanners];                            // the next tile's checkpoint; each thread's own
  float4 start[kTile / kSub - 1][2][kScanners];       // states at the later parts of the tile
  float4 accA[2][kScanners];                          // dA
  float accD[kTile][P::kCh], accb[kTile][P::kCh];     // dD and ddt_bias at the end
};

template <class T, int S, Fill FILL>
__global__ void __launch_bounds__(BackwardTeam::kBlock, 2)
    seq_scan_bwd_kernel(pt_scan_args a, ScanDims dm, const float* seg_h, const float* seg_d, float* part_bc,
                        float* part_p) {
  using TEAM = BackwardTeam;
  using P = ScanShape<S, TEAM>;
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sm = *reinterpret_cast<BackwardSmem<S, TEAM>*>(smem);
  const ScanBlock<S, TEAM> at(a, dm.cblocks);
  const int seg = at.rest % dm.segs, chunk = at.rest / dm.segs;
  const int t0 = seg * dm.seg_len, t1 = min(t0 + dm.seg_len, a.len);
  const int tiles = max(0, (t1 - t0 + kTile - 1) / kTile);
  const long long ckpt_row = (static_cast<long long>(a.len) + kTile - 1) / kTile;
  const long long all = static_cast<long long>(a.dim) * a.state;
  // This block's partial sums of dA [dim, state], dD [dim], ddt_bias [dim].
  float* mine = part_p + (static_cast<long long>(chunk) * dm.segs + seg) * (all + 2 * a.dim);
  const int tid = static_cast<int>(threadIdx.x);
  // Tiles are taken from the last to the first; k counts them in that order.
  auto tile_of = [&](int k) { return t0 + (tiles - 1 - k) * kTile; };

  if (tid >= kScanners) {
    fewer_registers<TEAM::kStagerRegs>();
    const Stager<S, TEAM> me(tid - kScanners, at.c0, at.nch);
    F2 bias[me.kPairs], Dv[me.kPairs], accD[me.kPairs] = {}, accb[me.kPairs] = {};
    me.params(a.dt_bias, bias);
    me.params(a.D, Dv);
    for (int b = chunk; b < a.batch; b += dm.row_chunks) {
      const int len = scan_row_length(a, b), end = min(len, t1);
      // A tile takes the scanners far longer than a trip to memory, so nothing is fetched ahead and few registers do.
      Pack<T, P::kE> dt, x, z, dy;
      int t_in = tile_of(0) + me.tr, t_out = t_in;  // of the tile to convert, of the one whose gradients are next
      Walk<T> wdt(a.dt, b * a.dt_batch + t_in * a.dt_step + me.c, a.dt_step, -1);
      Walk<T> wx(a.x, b * a.x_batch + t_in * a.x_step + me.c, a.x_step, -1);
      Walk<T> wdy(a.dy, b * a.dy_batch + t_in * a.dy_step + me.c, a.dy_step, -1);
      Walk<T> wz(a.z, a.z ? b * a.z_batch + t_in * a.z_step + me.c : 0, a.z_step, -1);
      Walk<T> wB(a.B, b * a.B_batch + t_in * a.B_step + at.g * a.B_group, a.B_step, -1);
      Walk<T> wC(a.C, b * a.C_batch + t_in * a.C_step + at.g * a.C_group, a.C_step, -1);
      long long o = (static_cast<long long>(b) * a.len + t_out) * a.dim + me.c;  // gradients of t_out
      // The inputs of a tile, `back` tiles behind the walk.
      auto load = [&](int back) {
        dt.load(wdt.p - back * wdt.by, me.n, dm.wide & 2);
        x.load(wx.p - back * wx.by, me.n, dm.wide & 1);
        dy.load(wdy.p - back * wdy.by, me.n, dm.wide & 8);
        if (a.z) z.load(wz.p - back * wz.by, me.n, dm.wide & 4);
      };
      auto convert = [&](int k) {
        const bool live = t_in < end;
        StateRow<T, S, TEAM> rowB, rowC;
        rowB.load(wB.p, a.state, live, me.pr);
        rowC.load(wC.p, a.state, live, me.pr);
        F2 d[me.kPairs] = {}, v[me.kPairs] = {}, w[me.kPairs] = {};
        if (live) {
          load(0);
#pragma unroll
          for (int i = 0; i < me.kPairs; ++i) {
            d[i] = add2(dt.pair(i), bias[i]);
            if (a.dt_softplus) d[i] = softplus2<T>(d[i]);
            v[i] = mul2(d[i], x.pair(i));
            w[i] = dy.pair(i);
            if (a.z) {
              const F2 zi = z.pair(i);
              w[i] = mul2(w[i], mul2(zi, sigmoid2<T>(zi)));
            }
          }
        }
        put_pairs<P::kE>(&sm.d[k & 1][me.tr][me.col], d);
        put_pairs<P::kE>(&sm.v[k & 1][me.tr][me.col], v);
        put_pairs<P::kE>(&sm.w[k & 1][me.tr][me.col], w);
        rowB.store(sm.B[k & 1][me.tr], me.pr);
        rowC.store(sm.C[k & 1][me.tr], me.pr);
        t_in -= kTile;
        wdt.on(), wx.on(), wdy.on(), wz.on(), wB.on(), wC.on();
      };
      auto finish = [&](int k, int back) {
        const int st = k & 1;
        if (t_out < t1) {
          Pack<T, P::kE> ox, odt, oz;
          ox.zero(), odt.zero(), oz.zero();
          if (t_out < len) {
            load(back);
            F2 d[me.kPairs], gB[me.kPairs], gA[me.kPairs], y[me.kPairs];
            get_pairs<P::kE>(&sm.d[st][me.tr][me.col], d);
            get_pairs<P::kE>(&sm.v[st][me.tr][me.col], gB);
            get_pairs<P::kE>(&sm.gA[st][me.tr][me.col], gA);
            get_pairs<P::kE>(&sm.w[st][me.tr][me.col], y);
#pragma unroll
            for (int i = 0; i < me.kPairs; ++i) {
              const F2 xv = x.pair(i), dyv = dy.pair(i);
              F2 w = dyv;
              if (a.z) {
                const F2 zv = z.pair(i), s = sigmoid2<T>(zv);
                w = mul2(w, mul2(zv, s));
                const F2 yv = a.D ? fma2(Dv[i], xv, y[i]) : y[i];
                oz.set_pair(i, mul2(mul2(dyv, yv), silu_grad2(zv, s)));
              }
              F2 gd = fma2(gB[i], xv, mul2(gA[i], same2(kLn2)));
              if (a.dt_softplus) gd = mul2(gd, sigmoid2<T>(add2(dt.pair(i), bias[i])));
              F2 gx = mul2(gB[i], d[i]);
              if (a.D) gx = fma2(Dv[i], w, gx);
              ox.set_pair(i, gx);
              odt.set_pair(i, gd);
              accD[i] = fma2(w, xv, accD[i]);
              accb[i] = add2(accb[i], gd);
            }
          }
          const bool wide = dm.wide & 16;
          if (a.dx) ox.store(static_cast<T*>(a.dx) + o, me.n, wide);
          if (a.ddt) odt.store(static_cast<T*>(a.ddt) + o, me.n, wide);
          if (a.dz) oz.store(static_cast<T*>(a.dz) + o, me.n, wide);
        }
        if (part_bc) {
          // [block of the group's channels][batch][len][group][2 * states]
          constexpr int kRow = 2 * P::kStates, kEach = 4;
          const int tile = t_out - me.tr, rows = min(kTile, t1 - tile), valid = len - tile;
          const long long row = (static_cast<long long>(at.cb % dm.cblocks) * a.batch + b) * a.len + tile;
#pragma unroll 1
          for (int i = (tid - kScanners) * kEach; i < rows * kRow; i += TEAM::kStagers * kEach) {
            const int q = i / kRow, k2 = i % kRow;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            if (q < valid) {
              s = *reinterpret_cast<const float4*>(&sm.red[st][0][q][k2]);
#pragma unroll
              for (int w = 1; w < kScanWarps; ++w) {
                const float4 m = *reinterpret_cast<const float4*>(&sm.red[st][w][q][k2]);
                s.x += m.x, s.y += m.y, s.z += m.z, s.w += m.w;
              }
            }
            *reinterpret_cast<float4*>(part_bc + ((row + q) * a.groups + at.g) * kRow + k2) = s;
          }
        }
        t_out -= kTile;
        o -= static_cast<long long>(kTile) * a.dim;
      };
      if (tiles > 0) convert(0);
      meet<TEAM>();
      for (int k = 0; k < tiles; ++k) {
        if (k > 0) finish(k - 1, 2);  // the walk is at tile k + 1
        if (k + 1 < tiles) convert(k + 1);
        meet<TEAM>();
      }
      if (tiles > 0) finish(tiles - 1, 1);
      meet<TEAM>();
    }
    put_pairs<P::kE>(&sm.accD[me.tr][me.col], accD);
    put_pairs<P::kE>(&sm.accb[me.tr][me.col], accb);
    meet<TEAM>();
    for (int c = tid - kScanners; c < at.nch; c += TEAM::kStagers) {
      float sD = 0.f, sb = 0.f;
#pragma unroll
      for (int q = 0; q < kTile; ++q) sD += sm.accD[q][c], sb += sm.accb[q][c];
      mine[all + at.c0 + c] = sD;
      mine[all + a.dim + at.c0 + c] = sb;
    }
    return;
  }

  more_registers<TEAM::kScannerRegs>();
  const Scanner<S, TEAM> me(tid, at.c0, at.nch);
  Quad A2;
  load_rates(a, me, A2);
  sm.accA[0][tid] = sm.accA[1][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool quads = (a.state & 3) == 0 && (reinterpret_cast<uintptr_t>(a.checkpoints) & 15) == 0;
  for (int b = chunk; b < a.batch; b += dm.row_chunks) {
    const int len = scan_row_length(a, b);
    auto fetch = [&](int k) {
      const float* ck = a.checkpoints + (b * ckpt_row + tile_of(k) / kTile) * all;
      if (quads) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i < me.mine && me.s0 < a.state)
            copy_async<16>(&sm.ck[i][tid], ck + static_cast<long long>(me.c + i) * a.state + me.s0);
          else
            sm.ck[i][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      } else {
        Quad h;
        load_states(ck, a, me, h);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          sm.ck[i][tid] = make_float4(lo2(h[i][0]), hi2(h[i][0]), lo2(h[i][1]), hi2(h[i][1]));
      }
      copy_commit();
    };
    if (tiles > 0) fetch(0);
    Quad g = {};  // a_{t+1} dh_{t+1}
    if (a.dhlast) load_states(a.dhlast + b * all, a, me, g);
    for (int s = dm.segs - 1; s > seg; --s) join_segment(a, dm, seg_h, seg_d, b, s, me, A2, g);
    meet<TEAM>();
    for (int k = 0; k < tiles; ++k) {
      const int st = k & 1;
      Quad first, h;  // the state at the tile's start, and walking on from it
      copy_wait<0>();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.ck[c][tid]);
        first[c][0] = h[c][0] = v.x, first[c][1] = h[c][1] = v.y;
      }
      if (k + 1 < tiles) fetch(k + 1);
      if (tile_of(k) >= len) {  // behind the row's end: no gradients, and no checkpoint was kept
        meet<TEAM>();
        continue;
      }
      // The states at the later parts' starts.
#pragma unroll 1
      for (int sub = 0; sub < kTile / kSub - 1; ++sub) {
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          const int t = sub * kSub + i;
          const Both d(&sm.d[st][t][me.cl]), v(&sm.v[st][t][me.cl]);
          const Four B(&sm.B[st][t][me.s0]);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              h[c][p] = fma2(decay(d.v[c], A2[c][p]), h[c][p], mul2(v.v[c], B.v[p]));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<ulonglong2*>(&sm.start[sub][c][tid]) = make_ulonglong2(h[c][0], h[c][1]);
      }
      Quad dA = {};
#pragma unroll 2
      for (int sub = kTile / kSub - 1; sub >= 0; --sub) {
        const int i0 = sub * kSub;
        F2 hs[kSub + 1][2][2], as[kSub][2][2];  // hs[i]: the state before step i0 + i
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (sub > 0) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.start[sub - 1][c][tid]);
            hs[0][c][0] = v.x, hs[0][c][1] = v.y;
          } else {
            hs[0][c][0] = first[c][0], hs[0][c][1] = first[c][1];
          }
        }
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          const Both d(&sm.d[st][i0 + i][me.cl]), v(&sm.v[st][i0 + i][me.cl]);
          const Four B(&sm.B[st][i0 + i][me.s0]);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              as[i][c][p] = decay(d.v[c], A2[c][p]);
              hs[i + 1][c][p] = fma2(as[i][c][p], hs[i][c][p], mul2(v.v[c], B.v[p]));
            }
        }
        float gB[2][2], gA[2][2], yy[2][2];
#pragma unroll
        for (int i = kSub - 1; i >= 0; --i) {
          const Both d(&sm.d[st][i0 + i][me.cl]), v(&sm.v[st][i0 + i][me.cl]), w(&sm.w[st][i0 + i][me.cl]);
          const Four B(&sm.B[st][i0 + i][me.s0]), C(&sm.C[st][i0 + i][me.s0]);
          F2 bB[2], bC[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            F2 sB = 0, sA = 0, sy = 0;  // two zeros each
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              const F2 dh = fma2(w.v[c], C.v[p], g[c][p]);
              bB[p] = c ? fma2(dh, v.v[c], bB[p]) : mul2(dh, v.v[c]);
              bC[p] = c ? fma2(w.v[c], hs[i + 1][c][p], bC[p]) : mul2(w.v[c], hs[i + 1][c][p]);
              g[c][p] = mul2(as[i][c][p], dh);
              const F2 dlog = mul2(g[c][p], hs[i][c][p]);
              dA[c][p] = fma2(dlog, d.v[c], dA[c][p]);
              if constexpr (FILL == kPartial) {
                const int f = me.s0 + 2 * p;
                sB = pack2(dot2(dh, B.v[p], lo2(sB), f, a.state), 0.f);
                sA = pack2(dot2(dlog, A2[c][p], lo2(sA), f, a.state), 0.f);
                sy = pack2(dot2(hs[i + 1][c][p], C.v[p], lo2(sy), f, a.state), 0.f);
              } else {
                sB = p ? fma2(dh, B.v[p], sB) : mul2(dh, B.v[p]);
                sA = p ? fma2(dlog, A2[c][p], sA) : mul2(dlog, A2[c][p]);
                sy = p ? fma2(hs[i + 1][c][p], C.v[p], sy) : mul2(hs[i + 1][c][p], C.v[p]);
              }
            }
            gB[i & 1][c] = lo2(sB) + hi2(sB);
            gA[i & 1][c] = lo2(sA) + hi2(sA);
            yy[i & 1][c] = lo2(sy) + hi2(sy);
            if (FILL == kLanes && me.s0 >= a.state) gB[i & 1][c] = gA[i & 1][c] = yy[i & 1][c] = 0.f;
          }
          float bc[8] = {lo2(bB[0]), hi2(bB[0]), lo2(bB[1]), hi2(bB[1]), lo2(bC[0]), hi2(bC[0]), lo2(bC[1]), hi2(bC[1])};
          sum_channels<S>(bc, me.lane, sm.red[st][me.warp][i0 + i]);
          if ((i & 1) == 0) {
            float f0, f1, f2, s0, s1, s2;
            sum_slices<S>(gB, me.slice, f0, s0);
            sum_slices<S>(gA, me.slice, f1, s1);
            sum_slices<S>(yy, me.slice, f2, s2);
            __syncwarp();  // v and w of these steps have been read by the channel's other lanes
            put_sums<S>(sm.v[st], i0 + i, me.cl, me.slice, f0, s0);
            put_sums<S>(sm.gA[st], i0 + i, me.cl, me.slice, f1, s1);
            put_sums<S>(sm.w[st], i0 + i, me.cl, me.slice, f2, s2);
          }
        }
      }
      // Tile by tile, so that a long row's sum is not one chain of additions.
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float4 s = sm.accA[c][tid];
        s.x += lo2(dA[c][0]), s.y += hi2(dA[c][0]), s.z += lo2(dA[c][1]), s.w += hi2(dA[c][1]);
        sm.accA[c][tid] = s;
      }
      meet<TEAM>();
    }
    if (a.dh0 && seg == 0) store_states(a.dh0 + b * all, a, me, g);
    meet<TEAM>();  // the next row's tiles overwrite what this row's last gradients are made from
  }
  if (a.dA) {
    Quad dA;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float4 s = sm.accA[c][tid];
      dA[c][0] = pack2(s.x, s.y), dA[c][1] = pack2(s.z, s.w);
    }
    store_states(mine, a, me, dA);
  }
  meet<TEAM>();
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
// S lanes hold N neighbouring channels, each lane four states of every one.  The
// first N lanes also take one channel each: its delta, its gate, its output;
// what the others need of it crosses by shuffles, so nothing is computed twice.
// Bound by reading and writing the states: those, and all else, are on their way
// while the block looks whether an earlier row has the slot.  256 rows of 4096
// channels with 16 states: 31 us (4.6 TB/s; 53 us with every lane computing its
// channel's delta and gate itself); one row of 2048: 2.6 us.
template <int S>
constexpr int kStepChannels = S == 2 ? 2 : 4;

// FOURS: the states are a multiple of four, so a lane has four or none and packed
// arithmetic does (256 rows of 4096 channels: 31.1 us, 32.1 state by state).
template <class T, int S, bool FOURS>
__global__ void __launch_bounds__(128) seq_scan_step_kernel(pt_scan_args a, int cblocks, int wide, unsigned* err) {
  constexpr int N = kStepChannels<S>;
  const int cb = static_cast<int>(blockIdx.x) % cblocks, b = static_cast<int>(blockIdx.x) / cblocks;
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
  const int slice = tid & (S - 1), s0 = 4 * slice, left = a.state - s0;  // left: states of this lane that exist
  int slot = a.slots ? __ldg(a.slots + b) : b;
  if (slot >= a.cache_rows) {
    if (tid == 0) atomicOr(err, kSlotPastCache);
    slot = -1;
  }
  const int c0 = (cb * (threads / S) + tid / S) * N;  // the lanes' first channel
  const int n = min(N, a.dim - c0);                   // channels that exist
  // B and C of the first channel's group; a group that begins within the N channels is rare.
  int g = 0, next = a.dim;
  if (a.groups > 1) {
    const int per = a.dim / a.groups;
    g = min(c0 / per, a.groups - 1), next = (g + 1) * per;
  }
  Pack<T, 4> B, C;
  auto load_group = [&]() {
    B.load(static_cast<const T*>(a.B) + b * a.B_batch + g * a.B_group + s0, left, wide & 2);
    C.load(static_cast<const T*>(a.C) + b * a.C_batch + g * a.C_group + s0, left, wide & 2);
  };
  load_group();
  float* hp = a.hlast + slot * a.h_row + static_cast<long long>(c0) * a.state + s0;
  const float* Ap = a.A + static_cast<long long>(c0) * a.state + s0;
  float h[N][4], A[N][4];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((wide & 1) && i < n && left > 0) {
      const float4 Av = __ldg(reinterpret_cast<const float4*>(Ap + i * a.state));
      A[i][0] = Av.x, A[i][1] = Av.y, A[i][2] = Av.z, A[i][3] = Av.w;
      const float4 hv = slot >= 0 ? *reinterpret_cast<const float4*>(hp + i * a.state) : make_float4(0.f, 0.f, 0.f, 0.f);
      h[i][0] = hv.x, h[i][1] = hv.y, h[i][2] = hv.z, h[i][3] = hv.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        A[i][j] = i < n && j < left ? __ldg(Ap + i * a.state + j) : 0.f;
        h[i][j] = i < n && j < left && slot >= 0 ? hp[i * a.state + j] : 0.f;
      }
    }
  }
  // This lane's own channel.
  const int c = c0 + slice;
  const bool own = slice < n;
  float delta = 0.f, v = 0.f, x = 0.f, z = 0.f, D = 0.f;
  if (own) {
    delta = to_f<T>(static_cast<const T*>(a.dt)[b * a.dt_batch + c]) + (a.dt_bias ? __ldg(a.dt_bias + c) : 0.f);
    x = to_f<T>(static_cast<const T*>(a.x)[b * a.x_batch + c]);
    if (a.z) z = to_f<T>(static_cast<const T*>(a.z)[b * a.z_batch + c]);
    if (a.D) D = __ldg(a.D + c);
    if (a.dt_softplus) delta = softplusf<T>(delta);
    v = delta * x;
  }
  if (a.slots && named_before(a.slots, b, slot, tid, threads)) {
    if (tid == 0) atomicOr(err, kSlotTwice);
    slot = -1;
  }
  F2 Bp[2], Cp[2];
  auto pairs = [&]() {
#pragma unroll
    for (int p = 0; p < 2; ++p) Bp[p] = B.pair(p), Cp[p] = C.pair(p);
  };
  pairs();
  float y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = __shfl_sync(0xffffffffu, delta, i, S) * kLog2e, u = __shfl_sync(0xffffffffu, v, i, S);
    if (c0 + i >= next && i < n) {
      ++g, next += a.dim / a.groups;
      load_group();
      pairs();
    }
    float s = 0.f;
    if constexpr (FOURS) {
      F2 sum = 0;  // two zeros
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const F2 e = decay(same2(d), pack2(A[i][2 * p], A[i][2 * p + 1]));
        const F2 hn = fma2(e, pack2(h[i][2 * p], h[i][2 * p + 1]), mul2(same2(u), Bp[p]));
        h[i][2 * p] = lo2(hn), h[i][2 * p + 1] = hi2(hn);
        sum = p ? fma2(hn, Cp[p], sum) : mul2(hn, Cp[p]);
      }
      s = left > 0 ? sum2(sum) : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) {
          h[i][j] = fmaf(ex2(fmaf(d, A[i][j], kCentre)), h[i][j], u * B.f(j));
          s = fmaf(h[i][j], C.f(j), s);
        }
    }
    y[i] = s;
    if (i < n && slot >= 0) {
      if ((wide & 1) && left > 0) {
        *reinterpret_cast<float4*>(hp + i * a.state) = make_float4(h[i][0], h[i][1], h[i][2], h[i][3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) hp[i * a.state + j] = h[i][j];
      }
    }
  }
  // Sums over the lanes; lane i < N ends with channel i's.
  const bool odd = slice & 1;
  if constexpr (N == 4) {
    const bool up = slice & 2;
    const float p = (up ? y[2] : y[0]) + __shfl_xor_sync(0xffffffffu, up ? y[0] : y[2], 2);
    const float q = (up ? y[3] : y[1]) + __shfl_xor_sync(0xffffffffu, up ? y[1] : y[3], 2);
    y[0] = p, y[1] = q;
  }
  float sum = (odd ? y[1] : y[0]) + __shfl_xor_sync(0xffffffffu, odd ? y[0] : y[1], 1);
#pragma unroll
  for (int m = 4; m < S; m *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (own) {
    if (slot >= 0) {
      if (a.D) sum = fmaf(D, x, sum);
      if (a.z) sum *= siluf<T>(z);
    } else {
      sum = 0.f;
    }
    static_cast<T*>(a.y)[static_cast<long long>(b) * a.dim + c] = from_f<T>(sum);
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

template <class T, int S, class TEAM>
ScanDims scan_dims(const pt_scan_args& a, const ScanPlan& p) {
  using P = ScanShape<S, TEAM>;
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
  d.wide |= ok(a.y, 0, 0) && ok(a.dx, 0, 0) && ok(a.ddt, 0, 0) && ok(a.dz, 0, 0) ? 16 : 0;
  return d;
}

// The segments' states and sums of deltas lie in the workspace's first floats.
inline size_t segment_floats(const pt_scan_args& a, const ScanPlan& p) {
  if (p.segs <= 1) return 0;
  const size_t n = static_cast<size_t>(a.batch) * p.segs * a.dim * (static_cast<size_t>(a.state) + 1);
  return (n + 3) / 4 * 4;
}

// Launches a kernel whose shared memory is one Smem.
template <class TEAM, class Smem, class K, class... A>
cudaError_t launch_with(K kernel, long long grid, cudaStream_t stream, A... args) {
  constexpr int bytes = static_cast<int>(sizeof(Smem));
  // The scanners wait for the registers that the split promises them: without those, no launch.
  cudaFuncAttributes attr;
  const cudaError_t known = cudaFuncGetAttributes(&attr, kernel);
  if (known != cudaSuccess) return known;
  if (attr.numRegs < TEAM::kLaunchRegs) return cudaErrorLaunchOutOfResources;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  kernel<<<static_cast<unsigned>(grid), TEAM::kBlock, bytes, stream>>>(args...);
  return cudaGetLastError();
}

template <class T>
cudaError_t scan_fwd(const pt_scan_args& a, const ScanPlan& p, float* ws, cudaStream_t stream) {
  return by_slices(p.slices, [&](auto sc) -> cudaError_t {
    constexpr int S = decltype(sc)::value;
    const ScanDims dm = scan_dims<T, S, ForwardTeam<T>>(a, p);
    float* seg_h = ws;
    float* seg_d = ws + static_cast<size_t>(a.batch) * p.segs * a.dim * a.state;
    const long long blocks = static_cast<long long>(p.cblocks) * a.groups * a.batch;
    if (blocks * p.segs > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (p.segs > 1) {
      const cudaError_t e = launch_with<ForwardTeam<T>, SegmentSmem<S, ForwardTeam<T>>>(
          seq_scan_segment_kernel<T, S, false>, blocks * (p.segs - 1), stream, a, dm, seg_h, seg_d);
      if (e != cudaSuccess) return e;
    }
    const Fill fill = fill_of(a.state, S);
    auto kernel = fill == kFull    ? seq_scan_fwd_kernel<T, S, kFull>
                  : fill == kLanes ? seq_scan_fwd_kernel<T, S, kLanes>
                                   : seq_scan_fwd_kernel<T, S, kPartial>;
    return launch_with<ForwardTeam<T>, ForwardSmem<S, ForwardTeam<T>>>(kernel, blocks * p.segs, stream, a, dm, seg_h, seg_d);
  });
}

template <class T>
cudaError_t scan_bwd(const pt_scan_args& a, const ScanPlan& p, float* ws, cudaStream_t stream) {
  return by_slices(p.slices, [&](auto sc) -> cudaError_t {
    constexpr int S = decltype(sc)::value;
    const ScanDims dm = scan_dims<T, S, BackwardTeam>(a, p);
    const long long pieces = static_cast<long long>(p.row_chunks) * p.segs;
    const long long all = static_cast<long long>(a.dim) * a.state;
    const long long rows = static_cast<long long>(a.batch) * a.len * a.groups;
    float* seg_h = ws;
    float* seg_d = ws + static_cast<size_t>(a.batch) * p.segs * a.dim * a.state;
    float* part_bc = ws + segment_floats(a, p);
    float* part_p = part_bc + bc_floats(a, p);
    const long long blocks = static_cast<long long>(p.cblocks) * a.groups;
    if (blocks * a.batch * p.segs > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    cudaError_t e;
    if (p.segs > 1) {
      const ScanDims dm = scan_dims<T, S, ForwardTeam<T>>(a, p);
      e = launch_with<ForwardTeam<T>, SegmentSmem<S, ForwardTeam<T>>>(seq_scan_segment_kernel<T, S, true>, blocks * a.batch * (p.segs - 1),
                                               stream, a, dm, seg_h, seg_d);
      if (e != cudaSuccess) return e;
    }
    const Fill fill = fill_of(a.state, S);
    auto kernel = fill == kFull    ? seq_scan_bwd_kernel<T, S, kFull>
                  : fill == kLanes ? seq_scan_bwd_kernel<T, S, kLanes>
                                   : seq_scan_bwd_kernel<T, S, kPartial>;
    e = launch_with<BackwardTeam, BackwardSmem<S, BackwardTeam>>(kernel, blocks * pieces, stream, a, dm, seg_h, seg_d,
                                        a.dB || a.dC ? part_bc : nullptr, part_p);
    if (e != cudaSuccess) return e;
    if (a.dB || a.dC) {
      const long long n = rows * 8 * S;
      if (n > 0) {
        seq_scan_bc_kernel<T><<<static_cast<unsigned>(cdiv(n, 256)), 256, 0, stream>>>(
            part_bc, p.cblocks, rows, a.state, 4 * S, static_cast<T*>(a.dB), static_cast<T*>(a.dC));
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
      }
    }
    return launch_reduce(part_p, pieces, {{a.dA, all, PT_F32}, {a.dD, a.dim, PT_F32}, {a.ddt_bias, a.dim, PT_F32}},
                         stream);
  });
}

template <class T>
cudaError_t scan_step(const pt_scan_args& a, int slices, int sm_count, unsigned* err, cudaStream_t stream) {
  return by_slices(slices, [&](auto sc) -> cudaError_t {
    constexpr int S = decltype(sc)::value;
    const long long lanes = cdiv(a.dim, kStepChannels<S>) * S;
    // A call that does not fill the SMs is spread over small blocks.
    const int threads = lanes * a.batch < 512LL * sm_count ? 32 : 128;
    const int cblocks = static_cast<int>(cdiv(lanes, threads));
    const long long grid = static_cast<long long>(cblocks) * a.batch;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    // Bit 0: states and rates, bit 1: B and C move four at a time.
    const size_t four = 4 * sizeof(T);
    int wide = a.state % 4 == 0 && a.h_row % 4 == 0 && aligned(a.hlast, 16) && aligned(a.A, 16);
    wide |= a.state % 4 == 0 && aligned(a.B, four) && aligned(a.C, four) && a.B_batch % 4 == 0 && a.B_group % 4 == 0 &&
                    a.C_batch % 4 == 0 && a.C_group % 4 == 0
                ? 2
                : 0;
    auto kernel = a.state % 4 == 0 ? seq_scan_step_kernel<T, S, true> : seq_scan_step_kernel<T, S, false>;
    kernel<<<static_cast<unsigned>(grid), threads, 0, stream>>>(a, cblocks, wide, err);
    return cudaGetLastError();
  });
}

}  // namespace seq
}  // namespace pt
