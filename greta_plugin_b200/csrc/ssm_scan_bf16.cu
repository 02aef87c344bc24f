// Selective scan, bf16 instantiations.
#include "ssm_scan_launch.cuh"

namespace greta {
namespace ssm {
cudaError_t scan_fwd_bf16(const ScanParams& p, cudaStream_t st) { return scan_fwd<__nv_bfloat16>(p, st); }
cudaError_t scan_decode_bf16(const ScanParams& p, cudaStream_t st) { return scan_decode<__nv_bfloat16>(p, st); }
}  // namespace ssm
}  // namespace greta
