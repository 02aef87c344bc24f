// Selective scan, f16 instantiations.
#include "ssm_scan_launch.cuh"

namespace greta {
namespace ssm {
cudaError_t scan_fwd_f16(const ScanParams& p, cudaStream_t st) { return scan_fwd<__half>(p, st); }
cudaError_t scan_decode_f16(const ScanParams& p, cudaStream_t st) { return scan_decode<__half>(p, st); }
}  // namespace ssm
}  // namespace greta
