// pt_seq_scan_f32.cu -- the selective scan's kernels for f32 activations.
#include "pt_seq_scan.cuh"

namespace pt {
namespace seq {
template cudaError_t scan_fwd<float>(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template cudaError_t scan_bwd<float>(const pt_scan_args&, const ScanPlan&, float*, cudaStream_t);
template cudaError_t scan_step<float>(const pt_scan_args&, int, int, unsigned*, cudaStream_t);
}  // namespace seq
}  // namespace pt
