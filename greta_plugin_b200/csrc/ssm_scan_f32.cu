// Selective scan, f32 instantiations.
#include "ssm_scan_launch.cuh"

namespace greta {
namespace ssm {
cudaError_t scan_fwd_f32(const ScanParams& p, cudaStream_t st) { return scan_fwd<float>(p, st); }
cudaError_t scan_decode_f32(const ScanParams& p, cudaStream_t st) { return scan_decode<float>(p, st); }
}  // namespace ssm
}  // namespace greta
