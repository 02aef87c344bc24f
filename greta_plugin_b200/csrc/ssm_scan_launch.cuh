// Dispatch from the number of states to an instantiation, one element type per
// translation unit (ssm_scan_<dtype>.cu, ssm_scan_bwd_<dtype>.cu).
#pragma once

#include "ssm_launch.cuh"
#include "ssm_scan.cuh"

namespace greta {
namespace ssm {

// Lanes per channel: N / 4 rounded up to 4, 8, 16 or 32.
inline int lanes_of(int64_t N) { return N <= 16 ? 4 : N <= 32 ? 8 : N <= 64 ? 16 : 32; }

// Channel slices (one warp each) per group of the forward and carry kernels and
// of the backward kernel.
inline int fwd_slices_per_group(int64_t D, int64_t N, int64_t F) {
  return (int)cdiv(D / F, 32 / lanes_of(N) * 4);
}
inline int bwd_slices_per_group(int64_t D, int64_t N, int64_t F) {
  return (int)cdiv(D / F, 32 / lanes_of(N) * 2);
}

template <typename F>
auto with_lanes(int N, F f) {
  switch (lanes_of(N)) {
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    default: return f(std::integral_constant<int, 32>());
  }
}

// Warps per CTA: the slices of a group are dealt to CTAs of up to kScanWarps.
inline dim3 slices_grid(const ScanParams& p, int y) {
  return dim3((unsigned)cdiv((int64_t)p.F * p.spg, kScanWarps), (unsigned)y);
}

template <typename T>
cudaError_t scan_fwd(const ScanParams& p, cudaStream_t st) {
  return with_lanes(p.N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    const size_t smem = (size_t)kScanWarps * FwdSmem<T, LN, kFwdChans>::kWarp;
    const dim3 grid = slices_grid(p, p.R), block(kScanWarps * 32);
    if (p.R > 1) {
      auto k = ssm_scan_fwd_kernel<T, LN, kPhaseCarry>;
      cudaError_t e = allow_smem(k, smem);
      if (e == cudaSuccess) e = launch(k, grid, block, smem, st, p);
      if (e != cudaSuccess) return e;
    }
    auto k = ssm_scan_fwd_kernel<T, LN, kPhaseMain>;
    cudaError_t e = allow_smem(k, smem);
    if (e != cudaSuccess) return e;
    return launch(k, grid, block, smem, st, p);
  });
}

template <typename T>
cudaError_t scan_decode(const ScanParams& p, cudaStream_t st) {
  return with_lanes(p.N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    const dim3 grid = slices_grid(p, (int)cdiv(p.q.nseq, p.L)), block(kScanWarps * 32);
    const size_t smem = (size_t)kScanWarps * DecodeSmem<T, LN>::kWarp;
    auto k = ssm_scan_decode_kernel<T, LN>;
    cudaError_t e = allow_smem(k, smem);
    if (e != cudaSuccess) return e;
    return launch(k, grid, block, smem, st, p);
  });
}

// dA, dskip, ddbias and dB, dC: null where there is no such gradient. blocks: those
// of the main kernel that one launch takes, and acc: the groups' sums between
// launches.
struct ScanGrads {
  float *dA, *dskip, *dbias;
  void *dB, *dC;
  int blocks;
  float* acc;
};

cudaError_t scan_fwd_f32(const ScanParams&, cudaStream_t);
cudaError_t scan_fwd_f16(const ScanParams&, cudaStream_t);
cudaError_t scan_fwd_bf16(const ScanParams&, cudaStream_t);
cudaError_t scan_decode_f32(const ScanParams&, cudaStream_t);
cudaError_t scan_decode_f16(const ScanParams&, cudaStream_t);
cudaError_t scan_decode_bf16(const ScanParams&, cudaStream_t);
cudaError_t scan_bwd_f32(const ScanParams&, const ScanGrads&, cudaStream_t);
cudaError_t scan_bwd_f16(const ScanParams&, const ScanGrads&, cudaStream_t);
cudaError_t scan_bwd_bf16(const ScanParams&, const ScanGrads&, cudaStream_t);

}  // namespace ssm
}  // namespace greta
