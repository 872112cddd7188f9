// pt_seq_conv_f32.cu -- the causal convolution's kernels for f32 activations.
#include "pt_seq_conv.cuh"

namespace pt {
namespace seq {
template cudaError_t conv_fwd<float>(const pt_conv_args&, int, cudaStream_t);
template cudaError_t conv_bwd<float>(const pt_conv_args&, float*, int, cudaStream_t);
template cudaError_t conv_step<float>(const pt_conv_args&, unsigned*, cudaStream_t);
template ConvBwdPlan conv_bwd_plan<float>(const pt_conv_args&, int);
}  // namespace seq
}  // namespace pt
