// C ABI of the selective scan: checks, ranges and workspaces, dispatch.

#include "ssm_scan_launch.cuh"

namespace greta {
namespace ssm {
namespace {

constexpr int64_t kMaxStates = 128;
constexpr int kMaxRanges = 64;
constexpr int kMinRange = 32;  // tokens

int64_t slices(int64_t D, int64_t N, int64_t F) { return F * fwd_slices_per_group(D, N, F); }

// Ranges the stream is cut into, none shorter than kMinRange tokens. The
// forward: two waves of the CTAs that run at once, so that SMs that are done
// early find more (4096 x 4096 x 16: one wave 281 us with the carries, two 253;
// 2048 tokens 152, 146), or one where two would be shorter than kTwoWaves tokens
// (898 tokens: 60 us, 62). The backward: four waves (one 957 us, two 764, four
// 597), or two where four are too short (2000 x 1024 x 16: 94 us, 111 for ranges
// of kMinRange). Twice as many where they are longer than kLongRange (30000 tokens: two
// waves 1640 us, four 1544; backward four 4078, eight 3903). R is rounded down:
// one CTA in 38 left over cost 965 us instead of 794.
// Returns the tokens per range (a multiple of kTile) and sets R.
constexpr int kFwdCtasPerSm = 4, kBwdCtasPerSm = 3;
constexpr int64_t kTwoWaves = 48, kLongRange = 512;
int64_t plan_ranges(int64_t T, int64_t D, int64_t N, int64_t F, int asked, bool backward, int& R) {
  int64_t r = asked;
  if (asked <= 0) {
    const int64_t ctas = cdiv(slices(D, N, F), kScanWarps);  // of a range (forward)
    const int64_t wave = (int64_t)sm_count() * (backward ? kBwdCtasPerSm : kFwdCtasPerSm);
    r = 2 * wave / ctas;  // four waves in the backward, which has twice the CTAs a range
    if (backward ? T < r * kMinRange : T < r * kTwoWaves) r = wave / ctas;
    if (r < 1) r = 1;
    if (T > r * kLongRange) r *= 2;
  }
  if (r > kMaxRanges) r = kMaxRanges;
  const int64_t least = asked > 0 ? kTile : kMinRange;
  int64_t L = cdiv(cdiv(T, r), kTile) * kTile;
  if (L < least) L = least;
  R = (int)cdiv(T, L);
  return L;
}

// The longest sequence with which ranges take whole sequences (Ranges): kWholeShare of
// the tokens that each scheduler has to walk in all (four an SM). Measured at
// 4096 x 16, forward and backward: 16 sequences of 128 tokens (0.29) 106 + 298 us
// split, 73 + 263 whole; 12 of 1365 (0.39) 715 + 2038, 681 + 1882; 8 of 256 (0.58)
// 116 + 297, 108 + 322; 8 of 2048 (0.58) 749 + 2039, 1014 + 2320. With more states
// the same lengths are a smaller share: 4096 x 64, 3 of 683 tokens (0.39) 409 + 1315, 392 + 1241; 4096 x 128, 2 of 1024 (0.29) 767 +
// 2516, 643 + 2585, 9 of 227 (0.06) 732 + 2445, 605 + 2375. (Rows that no sequence
// holds count like one: 8192 rows of four sequences of 100 tokens and no others,
// 4096 x 16, forward: 1014 us whole, 111 split.)
constexpr double kWholeShare = 0.4;
int whole_limit(int64_t T, int64_t D, int64_t N, int64_t F, int asked) {
  if (asked > 0) return 0;
  const double walk = kWholeShare * (double)T * slices(D, N, F) / (4.0 * sm_count());
  return (int)(walk > T ? T : walk);
}

int64_t a16(int64_t v) { return (v + 15) / 16 * 16; }

struct Workspace {
  int64_t carry, hinit, dsum, reset, total;
  Workspace(int64_t R, int64_t D, int64_t N) {
    const int64_t states = R > 1 ? a16(R * D * N * 4) : 0;
    carry = 0;
    hinit = states;
    dsum = 2 * states;
    reset = dsum + (R > 1 ? a16(R * D * 4) : 0);
    total = reset + (R > 1 ? a16(R * 4) : 0);
  }
};

int check(int dtype, const ScanParams& p, const void* cu, int64_t num_seqs, int64_t T, int64_t D, int64_t N,
          int64_t F, int ranges) {
  if (esize(dtype) == 0) return GRETA_ERR_UNSUPPORTED;
  if (T < 0 || D <= 0 || N <= 0 || F <= 0 || num_seqs < 0 || ranges < 0) return GRETA_ERR_INVALID_ARG;
  if (T >= INT_MAX - 1024 || D > INT_MAX / 256 || num_seqs >= INT_MAX - 64) return GRETA_ERR_INVALID_ARG;
  if (D % F != 0) return GRETA_ERR_INVALID_ARG;
  if (N > kMaxStates) return GRETA_ERR_UNSUPPORTED;
  if (T == 0) return GRETA_OK;
  if (p.u == nullptr || p.delta == nullptr || p.A == nullptr || p.B == nullptr || p.C == nullptr)
    return GRETA_ERR_INVALID_ARG;
  if (p.ldu < D || p.ldd < D || (p.gate != nullptr && p.ldg < D) || p.ldb < F * N || p.ldc < F * N)
    return GRETA_ERR_INVALID_ARG;
  if (cu == nullptr && num_seqs != 0) return GRETA_ERR_INVALID_ARG;
  if (!aligned(p.A, 16)) return GRETA_ERR_ALIGNMENT;
  return GRETA_OK;
}

// Vector paths: a lane's loads of V channels and of 4 states start on whole
// aligned vectors in every row and group.
void plan_vectors(ScanParams& p, int es, int chans, std::initializer_list<const void*> rows) {
  const int CHW = 32 / lanes_of(p.N) * chans;
  const int V = CHW < 4 ? CHW : kTile * CHW >= 256 ? 8 : 4;  // TileVecs::V
  const int64_t a = (int64_t)V * es < 16 ? (int64_t)V * es : 16;
  bool ok = p.Dg % V == 0 && p.D % V == 0 && p.ldu % V == 0 && p.ldd % V == 0 &&
            (p.gate == nullptr || p.ldg % V == 0);
  for (const void* q : rows) ok = ok && aligned(q, a);
  p.vec = ok;
  p.vec_bc = p.N % 4 == 0 && p.ldb % 4 == 0 && p.ldc % 4 == 0 && aligned(p.B, 4 * es) && aligned(p.C, 4 * es);
}

ScanParams base(const void* u, int64_t ldu, const void* delta, int64_t ldd, const void* gate, int64_t ldg,
                const void* B, int64_t ldb, const void* C, int64_t ldc, const float* A, const float* skip,
                const float* dbias, void* out, const void* cu, int cu64, int64_t num_seqs, int64_t T, int64_t D,
                int64_t N, int64_t F, int softplus) {
  ScanParams p{};
  p.u = u; p.delta = delta; p.gate = gate; p.B = B; p.C = C;
  p.A = A; p.skip = skip; p.dbias = dbias;
  p.out = out;
  p.ldu = ldu; p.ldd = ldd; p.ldg = gate == nullptr ? 0 : ldg; p.ldb = ldb; p.ldc = ldc;
  p.q = Seqs{cu, cu64, cu == nullptr ? 1 : (int)num_seqs, (int)T};
  p.D = (int)D; p.N = (int)N; p.F = (int)F;
  if (D > 0 && F > 0 && N > 0) {
    p.Dg = (int)(D / F);
    p.spg = fwd_slices_per_group(D, N, F);
  }
  p.softplus = softplus != 0;
  return p;
}

int set_workspace(ScanParams& p, void* ws, int64_t bytes) {
  const Workspace w(p.R, p.D, p.N);
  if (w.total == 0) return GRETA_OK;
  if (ws == nullptr || bytes < w.total) return GRETA_ERR_INVALID_ARG;
  if (!aligned(ws, 16)) return GRETA_ERR_ALIGNMENT;
  char* b = reinterpret_cast<char*>(ws);
  p.carry = reinterpret_cast<float*>(b + w.carry);
  p.hinit = reinterpret_cast<float*>(b + w.hinit);
  p.dsum = reinterpret_cast<float*>(b + w.dsum);
  p.reset = reinterpret_cast<int*>(b + w.reset);
  return GRETA_OK;
}

int run_fwd(int dtype, const ScanParams& p, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case GRETA_DT_F32: return finish(scan_fwd_f32(p, st));
    case GRETA_DT_F16: return finish(scan_fwd_f16(p, st));
    default: return finish(scan_fwd_bf16(p, st));
  }
}

int run_decode(int dtype, const ScanParams& p, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case GRETA_DT_F32: return finish(scan_decode_f32(p, st));
    case GRETA_DT_F16: return finish(scan_decode_f16(p, st));
    default: return finish(scan_decode_bf16(p, st));
  }
}

// Blocks of the backward's main kernel that one launch takes. Each leaves a row of
// 2 N sums for every token, and a block has 64 channels for up to 16 states but 8
// for 128, so the rows of all of them grow with T D N: 8.6 GB for 16384 x 4096 x
// 128. Where that is more than kPartBytes, as many blocks as keep to it, in whole
// waves of CTAs, or one wave: 1.3 GB, in seven launches (backward 19.6 ms, 19.1 in one).
constexpr int64_t kPartBytes = int64_t(2) << 30;
int64_t bwd_blocks(int64_t blocks, int64_t R, int64_t T, int64_t N) {
  int64_t most = kPartBytes / (T * 2 * N * 4);
  if (blocks <= most) return blocks;
  int64_t wave = (int64_t)sm_count() * kBwdCtasPerSm / R;
  if (wave < 1) wave = 1;
  most = most < wave ? wave : most / wave * wave;
  return most < blocks ? most : blocks;
}

// The backward's workspace: the carries', then the parts of the sums.
struct BwdWorkspace {
  int64_t blocks, bc, acc, a, d, total;
  BwdWorkspace(int64_t R, int64_t T, int64_t D, int64_t N, int64_t F) {
    const int64_t per_group = cdiv(bwd_slices_per_group(D, N, F), kScanWarps), all = F * per_group;
    blocks = bwd_blocks(all, R, T, N);
    bc = a16(Workspace(R, D, N).total);
    acc = bc + a16(blocks * T * 2 * N * 4);
    a = acc + (blocks < all && per_group > 1 ? a16(F * T * 2 * N * 4) : 0);
    d = a + a16(R * D * N * 4);
    total = d + a16(R * 2 * D * 4);
  }
};

int run_bwd(int dtype, const ScanParams& p, const ScanGrads& g, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case GRETA_DT_F32: return finish(scan_bwd_f32(p, g, st));
    case GRETA_DT_F16: return finish(scan_bwd_f16(p, g, st));
    default: return finish(scan_bwd_bf16(p, g, st));
  }
}

// Tokens beyond one per request up to which a batch is a decode batch: its
// longest request then has at most kDecodeExtra + 1 tokens, walked one after
// another, or more beside empty ones, whose lengths the host does not know unless
// it is told the longest. 4, 32 and 256 requests of 4096 x 16 and 32 tokens more,
// all of one request: decode kernel 25, 27, 50 us, ranges 25, 38, 75; spread: 9, 8,
// 37 and 23, 32, 55. 16 more: 14, 17, 38 and 12, 37, 55. One request of 256 tokens
// beside 255 empty ones: 266 us in a graph, ranges 35 (256 of one token: 33). Rows
// copied ahead in that walk made it 150 us, and 29.0 us of a decode step 29.4.
constexpr int64_t kDecodeExtra = 32;
// (the grid has a row per chunk of up to 32 requests)
bool is_decode(int64_t num_reqs, int64_t T, int ranges, int64_t longest) {
  return ranges == 0 && num_reqs > 0 && T <= num_reqs + kDecodeExtra && longest <= kDecodeExtra + 1 &&
         num_reqs <= 65535;
}
constexpr int kDecodeWarps = 16;  // per SM (20: 29.0 us instead of 27.8 at 256 requests of 4096 x 16)

}  // namespace
}  // namespace ssm
}  // namespace greta

using namespace greta;
using namespace greta::ssm;

extern "C" {

int64_t greta_ssm_scan_workspace(int packed, int64_t num_seqs, int64_t T, int64_t D, int64_t N, int64_t F,
                                 int ranges) {
  if (T <= 0 || D <= 0 || N <= 0 || F <= 0 || D % F != 0 || N > kMaxStates || ranges < 0) return 0;
  if (truth_of(packed) && is_decode(num_seqs, T, ranges, longest_of(packed))) return 0;
  int R = 1;
  plan_ranges(T, D, N, F, ranges, false, R);
  return Workspace(R, D, N).total;
}

int greta_ssm_scan_fwd(int dtype, const void* u, int64_t ldu, const void* delta, int64_t ldd, const void* gate,
                       int64_t ldg, const void* B, int64_t ldb, const void* C, int64_t ldc, const float* A,
                       const float* skip, const float* delta_bias, void* out, float* saved, const void* cu_seqlens,
                       int cu_int64, int64_t num_seqs, int64_t T, int64_t D, int64_t N, int64_t F, int softplus,
                       int ranges, void* workspace, int64_t workspace_bytes, void* stream) {
  ScanParams p = base(u, ldu, delta, ldd, gate, ldg, B, ldb, C, ldc, A, skip, delta_bias, out, cu_seqlens, cu_int64,
                      num_seqs, T, D, N, F, softplus);
  int c = check(dtype, p, cu_seqlens, num_seqs, T, D, N, F, ranges);
  if (c != GRETA_OK || T == 0) return c;
  if (out == nullptr) return GRETA_ERR_INVALID_ARG;
  if (!aligned(saved, 16)) return GRETA_ERR_ALIGNMENT;
  p.ckpt = saved;
  p.zero_rest = 1;
  plan_vectors(p, esize(dtype), kFwdChans, {u, delta, gate, out});
  p.L = (int)plan_ranges(T, D, N, F, ranges, false, p.R);
  p.whole_limit = whole_limit(T, D, N, F, ranges);
  c = set_workspace(p, workspace, workspace_bytes);
  if (c != GRETA_OK) return c;
  return run_fwd(dtype, p, stream);
}

int greta_ssm_scan_packed(int dtype, const void* u, int64_t ldu, const void* delta, int64_t ldd, const void* gate,
                          int64_t ldg, const void* B, int64_t ldb, const void* C, int64_t ldc, const float* A,
                          const float* skip, const float* delta_bias, void* out, float* state, int64_t num_slots,
                          int64_t s_slot, int64_t s_d, int64_t s_n, const int32_t* starts, const int32_t* slots,
                          const int8_t* has_initial, int64_t num_reqs, int64_t T, int64_t D, int64_t N, int64_t F,
                          int softplus, int zero_rest, int ranges, int32_t* error_flags, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  ScanParams p = base(u, ldu, delta, ldd, gate, ldg, B, ldb, C, ldc, A, skip, delta_bias, out, starts, 0, num_reqs,
                      T, D, N, F, softplus);
  int c = check(dtype, p, starts, num_reqs, T, D, N, F, ranges);
  if (c != GRETA_OK || T == 0) return c;
  if (out == nullptr || starts == nullptr || num_slots < 0) return GRETA_ERR_INVALID_ARG;
  if (num_reqs > 0 && (slots == nullptr || has_initial == nullptr)) return GRETA_ERR_INVALID_ARG;
  if (num_slots > 0 && state == nullptr) return GRETA_ERR_INVALID_ARG;
  p.zero_rest = truth_of(zero_rest);
  if (num_slots > 0) {
    p.state = state;
    p.s_slot = s_slot; p.s_d = s_d; p.s_n = s_n; p.num_slots = num_slots;
    p.st_vec = s_n == 1 && s_d % 4 == 0 && s_slot % 4 == 0 && N % 4 == 0 && aligned(state, 16);
  } else if (error_flags != nullptr) {
    // no slot is in range, so nothing is read there, but the kernels look at the
    // slots (a test of its own for this in slot_of: training's forward 466 us, not 459)
    p.state = const_cast<float*>(A);
  }
  p.slots = slots;
  p.initial = reinterpret_cast<const signed char*>(has_initial);
  p.err = error_flags;
  plan_vectors(p, esize(dtype), kFwdChans, {u, delta, gate, out});
  if (is_decode(num_reqs, T, ranges, longest_of(zero_rest))) {
    // chunks of requests that leave every SM kDecodeWarps warps
    const int64_t chunks = (int64_t)sm_count() * kDecodeWarps / slices(D, N, F);
    int64_t per = cdiv(num_reqs, chunks < 1 ? 1 : chunks);
    p.L = (int)(per > 32 ? 32 : per);
    return run_decode(dtype, p, stream);
  }
  p.L = (int)plan_ranges(T, D, N, F, ranges, false, p.R);
  p.whole_limit = whole_limit(T, D, N, F, ranges);
  c = set_workspace(p, workspace, workspace_bytes);
  if (c != GRETA_OK) return c;
  return run_fwd(dtype, p, stream);
}

int64_t greta_ssm_scan_bwd_workspace(int64_t num_seqs, int64_t T, int64_t D, int64_t N, int64_t F, int ranges) {
  (void)num_seqs;
  if (T <= 0 || D <= 0 || N <= 0 || F <= 0 || D % F != 0 || N > kMaxStates || ranges < 0) return 0;
  int R = 1;
  plan_ranges(T, D, N, F, ranges, true, R);
  return BwdWorkspace(R, T, D, N, F).total;
}

int greta_ssm_scan_bwd(int dtype, const void* u, int64_t ldu, const void* delta, int64_t ldd, const void* gate,
                       int64_t ldg, const void* B, int64_t ldb, const void* C, int64_t ldc, const float* A,
                       const float* skip, const float* delta_bias, const float* saved, const void* dout, void* du,
                       void* ddelta, void* dgate, void* dB, void* dC, float* dA, float* dskip, float* ddelta_bias,
                       const void* cu_seqlens, int cu_int64, int64_t num_seqs, int64_t T, int64_t D, int64_t N,
                       int64_t F, int softplus, int ranges, void* workspace, int64_t workspace_bytes, void* stream) {
  ScanParams p = base(u, ldu, delta, ldd, gate, ldg, B, ldb, C, ldc, A, skip, delta_bias, nullptr, cu_seqlens,
                      cu_int64, num_seqs, T, D, N, F, softplus);
  int c = check(dtype, p, cu_seqlens, num_seqs, T, D, N, F, ranges);
  if (c != GRETA_OK) return c;
  if (dA == nullptr || (skip != nullptr && dskip == nullptr) || (delta_bias != nullptr && ddelta_bias == nullptr))
    return GRETA_ERR_INVALID_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (T == 0) {  // sums over no tokens
    cudaError_t e = cudaMemsetAsync(dA, 0, (size_t)(D * N) * 4, st);
    if (e == cudaSuccess && dskip != nullptr) e = cudaMemsetAsync(dskip, 0, (size_t)D * 4, st);
    if (e == cudaSuccess && ddelta_bias != nullptr) e = cudaMemsetAsync(ddelta_bias, 0, (size_t)D * 4, st);
    return finish(e);
  }
  if (saved == nullptr || dout == nullptr || du == nullptr || ddelta == nullptr || dB == nullptr || dC == nullptr ||
      (gate != nullptr && dgate == nullptr))
    return GRETA_ERR_INVALID_ARG;
  if (!aligned(saved, 16)) return GRETA_ERR_ALIGNMENT;
  p.ckpt = const_cast<float*>(saved);
  p.dout = dout;
  p.du = du; p.ddelta = ddelta; p.dgate = dgate;
  plan_vectors(p, esize(dtype), kFwdChans, {u, delta, gate, dout, du, ddelta, dgate});
  p.L = (int)plan_ranges(T, D, N, F, ranges, true, p.R);
  p.whole_limit = whole_limit(T, D, N, F, ranges);
  const BwdWorkspace w(p.R, T, D, N, F);
  if (workspace == nullptr || workspace_bytes < w.total) return GRETA_ERR_INVALID_ARG;
  if (!aligned(workspace, 16)) return GRETA_ERR_ALIGNMENT;
  c = set_workspace(p, workspace, workspace_bytes);
  if (c != GRETA_OK) return c;
  char* b = reinterpret_cast<char*>(workspace);
  p.part_bc = reinterpret_cast<float*>(b + w.bc);
  p.part_a = reinterpret_cast<float*>(b + w.a);
  p.part_d = reinterpret_cast<float*>(b + w.d);
  return run_bwd(dtype, p,
                 ScanGrads{dA, dskip, ddelta_bias, dB, dC, (int)w.blocks, reinterpret_cast<float*>(b + w.acc)}, stream);
}

}  // extern "C"
