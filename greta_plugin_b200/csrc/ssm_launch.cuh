// Host side shared by the state-space operators' launches.
#pragma once

#include <climits>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "greta_ssm.h"
#include "ssm_common.cuh"

namespace greta {
namespace ssm {

inline int esize(int dtype) { return dtype == GRETA_DT_F32 ? 4 : dtype == GRETA_DT_F16 || dtype == GRETA_DT_BF16 ? 2 : 0; }
inline bool aligned(const void* p, int64_t a) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % a == 0; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Multiprocessors of the current device.
int sm_count();

// Programmatic stream serialization, as the convolution's launches: the kernel
// may start while the one ahead finishes and waits for it (pdl_wait).
template <typename... P, typename... A>
cudaError_t launch(void (*k)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, static_cast<P>(a)...);
}

// Lets a kernel's launches have `smem` bytes: the same value in every call of that
// kernel, since a smaller one would lower the limit under another host thread.
template <typename K>
cudaError_t allow_smem(K kernel, size_t smem) {
  if (smem <= 48 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
}

// GRETA_SSM_LONGEST and the truth value that it was added to.
inline int64_t longest_of(int flags) { return flags >> 8; }
inline int truth_of(int flags) { return (flags & 0xff) != 0; }

inline int finish(cudaError_t e) { return e == cudaSuccess ? GRETA_OK : GRETA_ERR_LAUNCH; }

// Layout of a [slots, D, H] state from its strides for vectors of nv elements.
inline int state_layout(const void* state, int64_t s_slot, int64_t s_d, int64_t s_h, int64_t H, int nv, int es) {
  if (!aligned(state, (int64_t)nv * es) || s_slot % nv != 0) return kStGeneric;
  if (s_h == 1 && s_d == H) return kStDS;
  if (s_d == 1 && s_h % nv == 0) return kStSD;
  return kStGeneric;
}

}  // namespace ssm
}  // namespace greta
