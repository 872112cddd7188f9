// pt_seq_scan_bf16.cu -- the selective scan's kernels for bf16 activations.
#include "pt_seq_scan.cuh"

namespace pt {
namespace seq {
template cudaError_t scan_fwd<__nv_bfloat16>(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template cudaError_t scan_bwd<__nv_bfloat16>(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template cudaError_t scan_step<__nv_bfloat16>(const pt_scan_args&, int, int, unsigned*, cudaStream_t);
}  // namespace seq
}  // namespace pt
