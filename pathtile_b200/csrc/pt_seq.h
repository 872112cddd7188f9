// pt_seq.h -- host launchers of the sequence operators (causal convolution,
// selective scan, fused norm).  Layouts and semantics: include/pathtile_b200.h.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

#include "pathtile_b200.h"

namespace pt {

// Current device (pt_api.cu): PT_OK and its SM count and error word, or a status.
int seq_device(int* sm_count, unsigned** err);
int seq_cuda_fail(cudaError_t e);

namespace seq {

// Sums of partial results: with p running over chunks, part[p * stride + i], i
// counting through the outputs' elements one output after the other.  In a fixed
// order, in fp32, rounded once to each output's type; outputs may be null.
struct ReduceOut {
  void* out;
  long long m;  // elements
  int dtype;
};
cudaError_t launch_reduce(const float* part, long long chunks, const ReduceOut (&outs)[3], cudaStream_t stream);

// How the convolution's backward pass is cut (pt_seq_conv.cuh).
struct ConvBwdPlan {
  int v, tx, cblocks, chunks;
  long long per;
};

// How a scan is cut: `segs` pieces of `seg_len` steps run side by side.
struct ScanPlan {
  int slices;    // lanes that share a channel, four states each
  int ch;        // channels per block
  int cblocks;   // blocks per group of channels
  int segs, seg_len;
  int row_chunks;  // backward only: blocks along the batch, each looping over rows
};
ScanPlan scan_plan(const pt_scan_args& a, int sm_count, bool backward);
// Floats of the partial sums of dB and dC in the backward workspace, behind the segments'.
size_t bc_floats(const pt_scan_args& a, const ScanPlan& p);

cudaError_t launch_norm_fwd(const pt_norm_args& a, int sm_count, cudaStream_t stream);
cudaError_t launch_norm_bwd(const pt_norm_args& a, float* ws, int sm_count, cudaStream_t stream);
size_t norm_bwd_workspace(const pt_norm_args& a, int sm_count);

}  // namespace seq
}  // namespace pt
