// Selective scan backward, bf16 instantiations.
#include "ssm_scan_bwd_launch.cuh"

namespace greta {
namespace ssm {
cudaError_t scan_bwd_bf16(const ScanParams& p, const ScanGrads& g, cudaStream_t st) { return scan_bwd<__nv_bfloat16>(p, g, st); }
}  // namespace ssm
}  // namespace greta
