// Selective scan backward, f32 instantiations.
#include "ssm_scan_bwd_launch.cuh"

namespace greta {
namespace ssm {
cudaError_t scan_bwd_f32(const ScanParams& p, const ScanGrads& g, cudaStream_t st) { return scan_bwd<float>(p, g, st); }
}  // namespace ssm
}  // namespace greta
