// pt_seq_conv_f16.cu -- the causal convolution's kernels for f16 activations.
#include "pt_seq_conv.cuh"

namespace pt {
namespace seq {
template cudaError_t conv_fwd<__half>(const pt_conv_args&, int, cudaStream_t);
template cudaError_t conv_bwd<__half>(const pt_conv_args&, float*, int, cudaStream_t);
template cudaError_t conv_step<__half>(const pt_conv_args&, unsigned*, cudaStream_t);
template ConvBwdPlan conv_bwd_plan<__half>(const pt_conv_args&, int);
}  // namespace seq
}  // namespace pt
