// pt_seq_conv_bf16.cu -- the causal convolution's kernels for bf16 activations.
#include "pt_seq_conv.cuh"

namespace pt {
namespace seq {
template cudaError_t conv_fwd<__nv_bfloat16>(const pt_conv_args&, int, cudaStream_t);
template cudaError_t conv_bwd<__nv_bfloat16>(const pt_conv_args&, float*, int, cudaStream_t);
template cudaError_t conv_step<__nv_bfloat16>(const pt_conv_args&, unsigned*, cudaStream_t);
template ConvBwdPlan conv_bwd_plan<__nv_bfloat16>(const pt_conv_args&, int);
}  // namespace seq
}  // namespace pt
