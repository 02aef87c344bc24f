// The backward's launches for one element type (ssm_scan_bwd_<dtype>.cu).
#pragma once

#include "ssm_scan_bwd.cuh"
#include "ssm_scan_launch.cuh"

namespace greta {
namespace ssm {

template <typename T>
cudaError_t scan_bwd(const ScanParams& p, const ScanGrads& g, cudaStream_t st) {
  if (p.R > 1) {
    const cudaError_t e = with_lanes(p.N, [&](auto ln) {
      constexpr int LN = decltype(ln)::value;
      auto k = ssm_scan_bwd_carry_kernel<T, LN>;
      const size_t smem = (size_t)kScanWarps * FwdSmem<T, LN, kFwdChans>::kWarp;
      cudaError_t e = allow_smem(k, smem);
      if (e != cudaSuccess) return e;
      return launch(k, slices_grid(p, p.R), dim3(kScanWarps * 32), smem, st, p);
    });
    if (e != cudaSuccess) return e;
  }
  // the main kernel's slices: half as many channels as the carry kernel's
  ScanParams m = p;
  m.spg = bwd_slices_per_group(p.D, p.N, p.F);
  const int bpg = (int)cdiv(m.spg, kScanWarps), blocks = p.F * bpg;
  for (int lo = 0; lo < blocks; lo += g.blocks) {
    const int hi = blocks - lo < g.blocks ? blocks : lo + g.blocks;
    m.b0 = lo;
    cudaError_t e = with_lanes(p.N, [&](auto ln) {
      constexpr int LN = decltype(ln)::value;
      auto k = ssm_scan_bwd_kernel<T, LN>;
      const size_t smem = BwdSmem<T, LN>::kTotal;
      static_assert(BwdSmem<T, LN>::kTotal <= 227 * 1024, "shared memory of a CTA");
      cudaError_t e = allow_smem(k, smem);
      if (e != cudaSuccess) return e;
      return launch(k, dim3((unsigned)(hi - lo), (unsigned)p.R), dim3(kScanWarps * 32), smem, st, m);
    });
    if (e != cudaSuccess) return e;
    // the groups that have blocks in [lo, hi), as many at a time as a grid's y dimension holds
    const int kRow = 65535, f1 = (hi - 1) / bpg + 1;
    for (int f0 = lo / bpg; f0 < f1; f0 += kRow) {
      const unsigned groups = f1 - f0 < kRow ? f1 - f0 : kRow;
      e = launch(ssm_scan_reduce_bc_kernel<T>, dim3((unsigned)cdiv((int64_t)p.q.T * 2 * p.N, 256), groups), dim3(256),
                 0, st, (const float*)p.part_bc, g.acc, (T*)g.dB, (T*)g.dC, bpg, lo, hi, p.q.T, p.N, p.F, f0);
      if (e != cudaSuccess) return e;
    }
  }
  return launch(ssm_scan_reduce_a_kernel<4>, dim3((unsigned)cdiv((int64_t)p.D * (p.N + 2), 256)), dim3(256), 0, st,
                (const float*)p.part_a, (const float*)p.part_d, g.dA, g.dskip, g.dbias, p.R, p.D, p.N);
}

}  // namespace ssm
}  // namespace greta
