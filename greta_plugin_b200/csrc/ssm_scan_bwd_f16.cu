// Selective scan backward, f16 instantiations.
#include "ssm_scan_bwd_launch.cuh"

namespace greta {
namespace ssm {
cudaError_t scan_bwd_f16(const ScanParams& p, const ScanGrads& g, cudaStream_t st) { return scan_bwd<__half>(p, g, st); }
}  // namespace ssm
}  // namespace greta
