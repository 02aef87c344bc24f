// C ABI of the short causal convolution: checks, launch shapes, dispatch.
#include "ssm_conv.cuh"
#include "ssm_launch.cuh"

namespace greta {
namespace ssm {

int sm_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cache[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cache[dev] = n;
  }
  return cache[dev];
}

namespace {

constexpr int kRuns = 4;  // runs per block (one warp each)

int check(int dtype, const void* x, int64_t ldx, const void* w, const void* y, const void* cu, int64_t num_seqs,
          int64_t T, int64_t D, int64_t W) {
  if (esize(dtype) == 0) return GRETA_ERR_UNSUPPORTED;
  if (T < 0 || D <= 0 || W <= 0 || num_seqs < 0) return GRETA_ERR_INVALID_ARG;
  if (T >= INT_MAX - 1024 || D > INT_MAX / 64 || num_seqs >= INT_MAX - 64) return GRETA_ERR_INVALID_ARG;
  if (W > kMaxWGeneric) return GRETA_ERR_UNSUPPORTED;
  if (T == 0) return GRETA_OK;
  if (x == nullptr || w == nullptr || y == nullptr) return GRETA_ERR_INVALID_ARG;
  if (ldx < D) return GRETA_ERR_INVALID_ARG;
  if (cu == nullptr && num_seqs != 0) return GRETA_ERR_INVALID_ARG;
  return GRETA_OK;
}

// Tokens beyond one per request up to which a batch is a decode batch: its
// longest request then has at most kDecodeExtra + 1 tokens, walked one after
// another, or more beside empty ones, whose lengths the host does not know unless
// it is told the longest. 4, 32 and 256 requests of 4096 channels and 8 tokens
// more, all of one request: decode kernel 6.6, 6.1, 7.9 us, runs 5.3, 5.4, 9.2;
// spread: 4.7, 4.4, 8.1 and 5.8, 5.6, 9.2. 16 more of one request: 9.6, 9.1, 10.3
// and 5.3, 5.4, 9.3. One request of 256 tokens beside 255 empty ones: 121 us in a
// graph, runs 14 (256 of one token: 16).
constexpr int64_t kDecodeExtra = 8;

// Tokens per run, whole groups of four: as few as fill every SM with the CTAs it
// has registers for, rounded up so that none is left over, or fill it several
// times where a run would be longer than kMaxRun. Backward of 16288 x 4096 x 4
// taps, bf16: runs of 56 tokens (four fills) 115 us, 112 104, 228 100; 220, with
// 16 CTAs left over, 129.
constexpr int64_t kCtasPerSm = 4;
constexpr int64_t kMaxRun = 256;
int run_tokens(int64_t T, int64_t ctas_per_row, int lo) {
  const int64_t wave = (int64_t)sm_count() * kCtasPerSm;
  int64_t L = T;
  for (int64_t k = cdiv(T * ctas_per_row, wave * kRuns * kMaxRun); ; ++k) {
    const int64_t rows = wave * k / ctas_per_row;
    if (rows < 1) continue;
    L = cdiv(T, rows * kRuns);
    if (L <= kMaxRun) break;
  }
  if (L > kGroup) L = cdiv(L, kGroup) * kGroup;
  return (int)(L < lo ? lo : L);
}

// Elements of a thread's vector for a kernel of WT taps: 16 bytes for the small
// kernels, half and a quarter of it for the wide ones, whose windows and
// filters take W registers a channel each.
template <typename T, int WT>
constexpr int vec_of() {
  constexpr int bytes = WT > 0 ? 16 : WT == -8 ? 8 : 4;
  return bytes / (int)sizeof(T);
}

// The kernel's template value for W taps.
template <typename F>
int with_taps(int W, F f) {
  switch (W) {
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, 4>());
  }
  return W <= 8 ? f(std::integral_constant<int, -8>()) : f(std::integral_constant<int, -kMaxWGeneric>());
}

template <typename T, int NV, int WT, bool PACKED>
int fwd_one(ConvParams p, int64_t longest, cudaStream_t st) {
  p.vec_w = p.sw_d == 1 && p.sw_k % NV == 0 && aligned(p.w, NV * sizeof(T));
  if (p.state != nullptr) p.st_layout = state_layout(p.state, p.s_slot, p.s_d, p.s_h, p.W - 1, NV, sizeof(T));
  const int64_t cw = cdiv(cdiv(p.D, NV), 32);
  p.nblk = (int)cw;
  if (PACKED && p.q.nseq > 0 && p.q.T <= p.q.nseq + kDecodeExtra && longest <= kDecodeExtra + 1) {
    const int64_t blocks = cdiv(p.q.nseq, kRuns) * cw;
    if (blocks > INT_MAX) return GRETA_ERR_INVALID_ARG;
    return finish(launch(ssm_conv_decode_kernel<T, NV, WT>, dim3((unsigned)blocks), dim3(32, kRuns), 0, st, p));
  }
  p.L = run_tokens(p.q.T, cw, 1);
  const int64_t blocks = cdiv(cdiv(p.q.T, p.L), kRuns) * cw;
  if (blocks > INT_MAX) return GRETA_ERR_INVALID_ARG;
  const size_t smem = NV > 1 ? (size_t)kRuns * ConvRing<T, NV>::kBytes : 0;
  return finish(launch(ssm_conv_fwd_kernel<T, NV, WT, PACKED>, dim3((unsigned)blocks), dim3(32, kRuns), smem, st, p));
}

// Whole vectors where every row starts on one; else single elements.
template <typename T, bool PACKED>
int fwd_type(const ConvParams& p, int64_t longest, cudaStream_t st) {
  return with_taps(p.W, [&](auto taps) {
    constexpr int WT = decltype(taps)::value, NV = vec_of<T, WT>();
    const bool vec = p.D % NV == 0 && p.ldx % NV == 0 && aligned(p.x, NV * sizeof(T)) && aligned(p.y, NV * sizeof(T));
    return vec ? fwd_one<T, NV, WT, PACKED>(p, longest, st) : fwd_one<T, 1, WT, PACKED>(p, longest, st);
  });
}

// longest: the most tokens of a request, 0 when it is not known
template <bool PACKED>
int fwd(int dtype, const ConvParams& p, int64_t longest, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case GRETA_DT_F32: return fwd_type<float, PACKED>(p, longest, st);
    case GRETA_DT_F16: return fwd_type<__half, PACKED>(p, longest, st);
    default: return fwd_type<__nv_bfloat16, PACKED>(p, longest, st);
  }
}

constexpr int kBwdMinRun = 8;

// Rows of partial sums of the backward, for vectors of NV channels; the most of
// them over the vectors that bwd_type takes (the workspace is asked for by the
// sizes alone).
int64_t bwd_rows(int64_t T, int L) { return cdiv(cdiv(T, L), kRuns); }
int64_t bwd_rows_most(int64_t T, int64_t D) {
  int64_t most = 0;
  for (int nv = 1; nv <= 4; nv *= 2) {
    const int64_t r = bwd_rows(T, run_tokens(T, cdiv(cdiv(D, nv), 32), kBwdMinRun));
    if (r > most) most = r;
  }
  return most;
}

// The gradients of the filters and the bias.
struct ParamGrads {
  void *dw, *dbias;
  bool f32;  // fp32 arrays, else of the element type
};

template <typename T>
int reduce(const ConvParams& p, int64_t rows, const ParamGrads& g, cudaStream_t st) {
  const int64_t cols = cdiv((int64_t)(p.W + 1) * p.D, 32);
  return finish(launch(ssm_conv_reduce_kernel<T>, dim3((unsigned)cols), dim3(32, 8), 0, st, (const float*)p.part,
                       reinterpret_cast<T*>(g.dw), reinterpret_cast<T*>(g.dbias), (long long)rows, p.D, p.W));
}

template <typename T, int NV, int WT>
int bwd_one(ConvParams p, const ParamGrads& g, cudaStream_t st) {
  static_assert(NV == 1 || NV == 2 || NV == 4, "counted by bwd_rows_most");
  p.vec_w = p.sw_d == 1 && p.sw_k % NV == 0 && aligned(p.w, NV * sizeof(T));
  const int64_t cw = cdiv(cdiv(p.D, NV), 32);
  p.L = run_tokens(p.q.T, cw, kBwdMinRun);
  p.nblk = (int)cw;
  const int64_t rows = bwd_rows(p.q.T, p.L);
  if (rows * cw > INT_MAX) return GRETA_ERR_INVALID_ARG;
  const size_t sums = (size_t)kRuns * (p.W + 1) * 32 * NV * sizeof(float);
  const size_t rings = NV > 1 ? (size_t)kRuns * 2 * ConvRing<T, NV>::kBytes : 0;
  const size_t smem = sums > rings ? sums : rings;
  auto k = ssm_conv_bwd_kernel<T, NV, WT>;
  cudaError_t e = allow_smem(k, smem);
  if (e == cudaSuccess) e = launch(k, dim3((unsigned)(rows * cw)), dim3(32, kRuns), smem, st, p);
  if (e != cudaSuccess) return GRETA_ERR_LAUNCH;
  return g.f32 ? reduce<float>(p, rows, g, st) : reduce<T>(p, rows, g, st);
}

// Vectors of half the forward's: with the filters and the window in fp32, as they
// are here, a thread has 4 W - 1 registers a channel, 2 W of them sums.
template <typename T>
int bwd_type(const ConvParams& p, const ParamGrads& g, cudaStream_t st) {
  return with_taps(p.W, [&](auto taps) {
    constexpr int WT = decltype(taps)::value, NV = vec_of<T, WT>() >= 4 ? vec_of<T, WT>() / 2 : vec_of<T, WT>();
    const bool vec = p.D % NV == 0 && p.ldx % NV == 0 && aligned(p.x, NV * sizeof(T)) &&
                     aligned(p.dout, NV * sizeof(T)) && aligned(p.dx, NV * sizeof(T));
    return vec ? bwd_one<T, NV, WT>(p, g, st) : bwd_one<T, 1, WT>(p, g, st);
  });
}

ConvParams base(const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d, const void* bias,
                const void* cu, int cu64, int64_t num_seqs, int64_t T, int64_t D, int64_t W, int silu) {
  ConvParams p{};
  p.x = x; p.w = w; p.bias = bias;
  p.q = Seqs{cu, cu64, cu == nullptr ? 1 : (int)num_seqs, (int)T};
  p.ldx = ldx; p.sw_k = sw_k; p.sw_d = sw_d;
  p.D = (int)D; p.W = (int)W;
  p.silu = silu != 0;
  return p;
}

}  // namespace
}  // namespace ssm
}  // namespace greta

using namespace greta;
using namespace greta::ssm;

extern "C" {

int greta_ssm_conv_fwd(int dtype, const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d,
                       const void* bias, void* y, const void* cu_seqlens, int cu_int64, int64_t num_seqs, int64_t T,
                       int64_t D, int64_t W, int silu, void* stream) {
  const int c = check(dtype, x, ldx, w, y, cu_seqlens, num_seqs, T, D, W);
  if (c != GRETA_OK || T == 0) return c;
  ConvParams p = base(x, ldx, w, sw_k, sw_d, bias, cu_seqlens, cu_int64, num_seqs, T, D, W, silu);
  p.y = y;
  p.zero_rest = 1;
  return fwd<false>(dtype, p, 0, stream);
}

int64_t greta_ssm_conv_bwd_workspace(int64_t T, int64_t D, int64_t W) {
  if (T <= 0 || D <= 0 || W <= 0) return 0;
  return bwd_rows_most(T, D) * (W + 1) * D * (int64_t)sizeof(float);
}

int greta_ssm_conv_bwd(int dtype, const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d,
                       const void* bias, const void* dout, void* dx, void* dw, void* dbias, const void* cu_seqlens,
                       int cu_int64, int64_t num_seqs, int64_t T, int64_t D, int64_t W, int silu, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  const int c = check(dtype, x, ldx, w, dx, cu_seqlens, num_seqs, T, D, W);
  if (c != GRETA_OK) return c;
  if (dw == nullptr || (bias == nullptr) != (dbias == nullptr)) return GRETA_ERR_INVALID_ARG;
  if (T > 0 && dout == nullptr) return GRETA_ERR_INVALID_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const ParamGrads g{dw, dbias, (silu & GRETA_SSM_GRADS_F32) != 0};
  silu &= ~GRETA_SSM_GRADS_F32;
  if (T == 0) {  // sums over no tokens
    const int es = g.f32 ? 4 : esize(dtype);
    cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)(W * D) * es, st);
    if (e == cudaSuccess && dbias != nullptr) e = cudaMemsetAsync(dbias, 0, (size_t)D * es, st);
    return finish(e);
  }
  if (workspace == nullptr || workspace_bytes < greta_ssm_conv_bwd_workspace(T, D, W)) return GRETA_ERR_INVALID_ARG;
  if (!aligned(workspace, 16)) return GRETA_ERR_ALIGNMENT;
  ConvParams p = base(x, ldx, w, sw_k, sw_d, bias, cu_seqlens, cu_int64, num_seqs, T, D, W, silu);
  p.dout = dout;
  p.dx = dx;
  p.part = reinterpret_cast<float*>(workspace);
  switch (dtype) {
    case GRETA_DT_F32: return bwd_type<float>(p, g, st);
    case GRETA_DT_F16: return bwd_type<__half>(p, g, st);
    default: return bwd_type<__nv_bfloat16>(p, g, st);
  }
}

int greta_ssm_conv_packed(int dtype, const void* x, int64_t ldx, const void* w, int64_t sw_k, int64_t sw_d,
                          const void* bias, void* y, void* state, int64_t num_slots, int64_t s_slot, int64_t s_d,
                          int64_t s_h, const int32_t* starts, const int32_t* slots, const int8_t* has_initial,
                          int64_t num_reqs, int64_t T, int64_t D, int64_t W, int silu, int zero_rest,
                          int32_t* error_flags, void* stream) {
  const int c = check(dtype, x, ldx, w, y, starts, num_reqs, T, D, W);
  if (c != GRETA_OK || T == 0) return c;
  if (starts == nullptr || num_slots < 0) return GRETA_ERR_INVALID_ARG;
  if (num_reqs > 0 && (slots == nullptr || has_initial == nullptr)) return GRETA_ERR_INVALID_ARG;
  if (W > 1 && num_slots > 0 && state == nullptr) return GRETA_ERR_INVALID_ARG;
  ConvParams p = base(x, ldx, w, sw_k, sw_d, bias, starts, 0, num_reqs, T, D, W, silu);
  p.y = y;
  if (W > 1 && num_slots > 0) {
    p.state = state;
    p.s_slot = s_slot; p.s_d = s_d; p.s_h = s_h;
  }
  p.num_slots = num_slots;
  p.slots = slots;
  p.initial = reinterpret_cast<const signed char*>(has_initial);
  p.err = error_flags;
  p.zero_rest = truth_of(zero_rest);
  return fwd<true>(dtype, p, longest_of(zero_rest), stream);
}

}  // extern "C"
