// pt_seq_api.cu -- C entry points of the sequence operators: argument checks,
// the scan's plan and dispatch by type.
#include <climits>
#include <type_traits>

#include "pt_seq.h"
#include "pt_seq_common.cuh"

namespace pt {
namespace seq {

// Defined and instantiated per activation type in pt_seq_conv_*.cu and pt_seq_scan_*.cu.
template <class T>
cudaError_t conv_fwd(const pt_conv_args&, int, cudaStream_t);
template <class T>
cudaError_t conv_bwd(const pt_conv_args&, float*, int, cudaStream_t);
template <class T>
cudaError_t conv_step(const pt_conv_args&, unsigned*, cudaStream_t);
template <class T>
ConvBwdPlan conv_bwd_plan(const pt_conv_args&, int);
template <class T>
cudaError_t scan_fwd(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template <class T>
cudaError_t scan_bwd(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template <class T>
cudaError_t scan_step(const pt_scan_args&, int, int, unsigned*, cudaStream_t);

namespace {

constexpr int kTileSteps = 16;  // kTile of pt_seq_scan.cuh

int status(cudaError_t e) { return e == cudaSuccess ? PT_OK : seq_cuda_fail(e); }
// The kernels count a little past a row's end in 32 bits.
bool length_ok(int len) { return len <= INT_MAX - 4096; }
bool type_ok(int t) { return t == PT_F32 || t == PT_BF16 || t == PT_F16; }

int check(const pt_conv_args* a) {
  if (!a || !type_ok(a->dtype)) return PT_ERR_ARGS;
  if (a->batch < 0 || a->len < 0 || a->dim < 1 || a->taps < 1) return PT_ERR_ARGS;
  if (a->taps > PT_CONV_MAX_TAPS || !length_ok(a->len)) return PT_ERR_UNSUPPORTED;
  if (a->batch > 0 && (!a->w || (a->len > 0 && !a->x))) return PT_ERR_ARGS;
  return PT_OK;
}

int check_sizes(const pt_scan_args* a) {
  if (!a || !type_ok(a->dtype)) return PT_ERR_ARGS;
  if (a->batch < 0 || a->len < 0 || a->dim < 1 || a->state < 1 || a->groups < 1 || a->dim % a->groups) return PT_ERR_ARGS;
  return a->state > PT_SCAN_MAX_STATE || !length_ok(a->len) ? PT_ERR_UNSUPPORTED : PT_OK;
}

int check(const pt_scan_args* a) {
  const int rc = check_sizes(a);
  if (rc != PT_OK) return rc;
  if (a->batch > 0 && (!a->A || (a->len > 0 && (!a->x || !a->dt || !a->B || !a->C)))) return PT_ERR_ARGS;
  return PT_OK;
}

int check(const pt_norm_args* a) {
  if (!a || !type_ok(a->dtype)) return PT_ERR_ARGS;
  if (a->rows < 0 || a->dim < 1 || a->groups < 1 || a->dim % a->groups) return PT_ERR_ARGS;
  if (a->dim / a->groups > PT_NORM_MAX_WIDTH) return PT_ERR_UNSUPPORTED;
  if (a->rows > 0 && (!a->x || !a->weight || (a->residual && !a->r))) return PT_ERR_ARGS;
  return PT_OK;
}

}  // namespace

ScanPlan scan_plan(const pt_scan_args& a, int sm_count, bool backward) {
  ScanPlan p;
  p.slices = a.state <= 8 ? 2 : a.state <= 16 ? 4 : a.state <= 32 ? 8 : 16;
  p.ch = 256 / p.slices;
  p.cblocks = static_cast<int>(cdiv(a.dim / a.groups, p.ch));
  const long long blocks = static_cast<long long>(p.cblocks) * a.groups * a.batch;
  // Two blocks fill an SM.  A segment costs its exponentials twice, so the length is cut only where whole rows leave
  // half of those places empty or more (as many segments as fill them); at least 64 steps keep the join of the states
  // before it short.
  long long segs = blocks > 0 ? 2LL * sm_count / blocks : 1;
  const long long most = cdiv(a.len, 64);
  segs = segs < most ? segs : most;
  segs = segs > 1 ? segs : 1;
  p.seg_len = static_cast<int>(cdiv(cdiv(a.len > 0 ? a.len : 1, segs), kTileSteps)) * kTileSteps;
  p.segs = static_cast<int>(cdiv(a.len > 0 ? a.len : 1, p.seg_len));
  p.row_chunks = a.batch;
  if (backward) {
    // Blocks that walk several rows write fewer partial sums of dA.
    const long long want = cdiv(8LL * sm_count, static_cast<long long>(p.cblocks) * a.groups * p.segs);
    if (p.row_chunks > want) p.row_chunks = static_cast<int>(want);
  }
  return p;
}

namespace {
size_t segment_bytes(const pt_scan_args& a, const ScanPlan& p) {
  if (p.segs <= 1) return 0;
  const size_t n = static_cast<size_t>(a.batch) * p.segs * a.dim * (static_cast<size_t>(a.state) + 1);
  return sizeof(float) * ((n + 3) / 4 * 4);
}
}  // namespace

size_t scan_fwd_workspace(const pt_scan_args& a, int sm_count) { return segment_bytes(a, scan_plan(a, sm_count, false)); }
size_t scan_bwd_workspace(const pt_scan_args& a, int sm_count) {
  const ScanPlan p = scan_plan(a, sm_count, true);
  const size_t pieces = static_cast<size_t>(p.row_chunks) * p.segs;
  return segment_bytes(a, p) + sizeof(float) * (bc_floats(a, p) + pieces * a.dim * a.state + pieces * 2 * a.dim);
}

// Partial sums of dB and dC: one of all (padded) states for every step and block of channels, so 2 bytes per step and
// channel up to 16 states, 8 up to 32 and 32 up to 64.
size_t bc_floats(const pt_scan_args& a, const ScanPlan& p) {
  if (!a.dB && !a.dC) return 0;
  return static_cast<size_t>(p.cblocks) * a.batch * a.len * a.groups * 8 * p.slices;
}

}  // namespace seq
}  // namespace pt

using namespace pt;
using namespace pt::seq;

#define PT_TRY(call)                 \
  do {                               \
    const int rc_ = (call);          \
    if (rc_ != PT_OK) return rc_;    \
  } while (0)

extern "C" {

int pt_causal_conv(const pt_conv_args* a, void* stream) {
  PT_TRY(check(a));
  if (a->batch > 0 && a->len > 0 && !a->y) return PT_ERR_ARGS;
  if (a->batch == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  return status(by_type(a->dtype, [&](auto t) { return conv_fwd<decltype(t)>(*a, sms, static_cast<cudaStream_t>(stream)); }));
}

size_t pt_causal_conv_bwd_workspace_bytes(const pt_conv_args* a) {
  int sms;
  unsigned* err;
  if (check(a) != PT_OK || a->batch == 0 || seq_device(&sms, &err) != PT_OK) return 0;
  size_t chunks = 0;
  by_type(a->dtype, [&](auto t) {
    chunks = static_cast<size_t>(conv_bwd_plan<decltype(t)>(*a, sms).chunks);
    return cudaSuccess;
  });
  return sizeof(float) * chunks * a->dim * (a->taps + 1);
}

int pt_causal_conv_bwd(const pt_conv_args* a, void* ws, size_t ws_bytes, void* stream) {
  PT_TRY(check(a));
  if (a->batch > 0 && a->len > 0 && !a->dy) return PT_ERR_ARGS;
  if (a->batch == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  if (!ws || ws_bytes < pt_causal_conv_bwd_workspace_bytes(a)) return PT_ERR_WORKSPACE;
  if (!aligned(ws, 16)) return PT_ERR_ALIGN;
  return status(by_type(a->dtype, [&](auto t) {
    return conv_bwd<decltype(t)>(*a, static_cast<float*>(ws), sms, static_cast<cudaStream_t>(stream));
  }));
}

int pt_causal_conv_step(const pt_conv_args* a, void* stream) {
  PT_TRY(check(a));
  if (a->len != 1 || a->cache_rows < 0) return PT_ERR_ARGS;
  if (a->batch > 0 && (!a->y || (a->taps > 1 && a->cache_rows > 0 && !a->state_out))) return PT_ERR_ARGS;
  if (!a->slots && a->cache_rows < a->batch) return PT_ERR_ARGS;
  if (a->batch == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  return status(by_type(a->dtype, [&](auto t) { return conv_step<decltype(t)>(*a, err, static_cast<cudaStream_t>(stream)); }));
}

size_t pt_scan_checkpoint_bytes(const pt_scan_args* a) {
  if (check_sizes(a) != PT_OK) return 0;
  return sizeof(float) * static_cast<size_t>(a->batch) * cdiv(a->len, kTileSteps) * a->dim * a->state;
}

size_t pt_scan_workspace_bytes(const pt_scan_args* a) {
  int sms;
  unsigned* err;
  if (check(a) != PT_OK || a->batch == 0 || seq_device(&sms, &err) != PT_OK) return 0;
  return scan_fwd_workspace(*a, sms);
}

int pt_scan(const pt_scan_args* a, void* ws, size_t ws_bytes, void* stream) {
  PT_TRY(check(a));
  if (a->batch > 0 && a->len > 0 && !a->y) return PT_ERR_ARGS;
  if (a->batch == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  const ScanPlan p = scan_plan(*a, sms, false);
  const size_t need = segment_bytes(*a, p);
  if (need && (!ws || ws_bytes < need)) return PT_ERR_WORKSPACE;
  if (need && !aligned(ws, 16)) return PT_ERR_ALIGN;
  return status(by_type(a->dtype, [&](auto t) {
    return scan_fwd<decltype(t)>(*a, p, static_cast<float*>(ws), static_cast<cudaStream_t>(stream));
  }));
}

size_t pt_scan_bwd_workspace_bytes(const pt_scan_args* a) {
  int sms;
  unsigned* err;
  if (check(a) != PT_OK || a->batch == 0 || seq_device(&sms, &err) != PT_OK) return 0;
  return scan_bwd_workspace(*a, sms);
}

int pt_scan_bwd(const pt_scan_args* a, void* ws, size_t ws_bytes, void* stream) {
  PT_TRY(check(a));
  if (a->batch > 0 && a->len > 0 && (!a->dy || !a->checkpoints)) return PT_ERR_ARGS;
  if (a->batch == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  if (!ws || ws_bytes < scan_bwd_workspace(*a, sms)) return PT_ERR_WORKSPACE;
  if (!aligned(ws, 16)) return PT_ERR_ALIGN;
  const ScanPlan p = scan_plan(*a, sms, true);
  return status(by_type(a->dtype, [&](auto t) {
    return scan_bwd<decltype(t)>(*a, p, static_cast<float*>(ws), static_cast<cudaStream_t>(stream));
  }));
}

int pt_scan_step(const pt_scan_args* a, void* stream) {
  PT_TRY(check(a));
  if (a->len != 1 || a->cache_rows < 0) return PT_ERR_ARGS;
  if (a->batch > 0 && (!a->y || (a->cache_rows > 0 && !a->hlast))) return PT_ERR_ARGS;
  if (!a->slots && a->cache_rows < a->batch) return PT_ERR_ARGS;
  if (a->batch == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  const int slices = scan_plan(*a, sms, false).slices;
  return status(by_type(a->dtype, [&](auto t) {
    return scan_step<decltype(t)>(*a, slices, sms, err, static_cast<cudaStream_t>(stream));
  }));
}

int pt_fused_norm(const pt_norm_args* a, void* stream) {
  PT_TRY(check(a));
  if (a->rows > 0 && !a->y) return PT_ERR_ARGS;
  if (a->rows == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  return status(launch_norm_fwd(*a, sms, static_cast<cudaStream_t>(stream)));
}

size_t pt_fused_norm_bwd_workspace_bytes(const pt_norm_args* a) {
  int sms;
  unsigned* err;
  if (check(a) != PT_OK || a->rows == 0 || seq_device(&sms, &err) != PT_OK) return 0;
  return norm_bwd_workspace(*a, sms);
}

int pt_fused_norm_bwd(const pt_norm_args* a, void* ws, size_t ws_bytes, void* stream) {
  PT_TRY(check(a));
  if (a->rows > 0 && !a->dy) return PT_ERR_ARGS;
  if (a->rows == 0) return PT_OK;
  int sms;
  unsigned* err;
  PT_TRY(seq_device(&sms, &err));
  if (!ws || ws_bytes < norm_bwd_workspace(*a, sms)) return PT_ERR_WORKSPACE;
  if (!aligned(ws, 16)) return PT_ERR_ALIGN;
  return status(launch_norm_bwd(*a, static_cast<float*>(ws), sms, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
