// pt_seq_scan_f16.cu -- the selective scan's kernels for f16 activations.
#include "pt_seq_scan.cuh"

namespace pt {
namespace seq {
template cudaError_t scan_fwd<__half>(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template cudaError_t scan_bwd<__half>(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template cudaError_t scan_step<__half>(const pt_scan_args&, int, int, unsigned*, cudaStream_t);
}  // namespace seq
}  // namespace pt
