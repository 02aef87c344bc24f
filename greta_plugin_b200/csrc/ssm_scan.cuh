// Selective state-space scan. Per token t, channel d and state n, with the
// channel's group f = d / (D / F):
//
//   dt       = softplus(delta[t, d] + delta_bias[d])      (softplus and bias optional)
//   h[n]     = exp(dt A[d, n]) h[n] + dt u[t, d] B[t, f, n]
//   y        = sum_n C[t, f, n] h[n] + skip[d] u[t, d]
//   out[t,d] = y SiLU(gate[t, d])                          (skip, gate optional)
//
// What bounds it: one exponential per (token, channel, state). The SM's
// special-function unit takes 16 a clock, so T D N / (148 * 16) clocks, three
// times what the reads and writes need at N = 16. The other work per state
// (two multiplications, two fused additions) is half of that on the fp32 pipe,
// issued for two channels an instruction.
//
// Split. A warp works alone: LN lanes a channel with four states each (LN =
// N / 4 rounded up to a power of two from 4 on) and KD channels a lane, so a
// lane keeps 4 KD states and their decay rates in registers, a token's B and C
// are read once for KD channels, and sums over n take log2(LN) shuffles for KD
// channels together. The packed stream is cut into ranges by position
// (ssm_common.cuh); a warp walks its range in tiles of 8 tokens, whose rows are
// copied to shared memory as vectors while the tile before is computed (the
// copies hold no registers: loads that did were moved behind the computation,
// and a third of the time was spent waiting for them); (dt, dt u) are computed
// once per token and channel, the recurrence runs from shared memory, and skip
// and gate are applied to the tile's y, again as vectors. Two channels of a
// lane share an instruction, so dt, dt u, states and y are register pairs as
// they come, and only B and C are doubled when they are widened.
//
// A range that begins inside a sequence needs the state at its first token.
// The first kernel (kPhaseCarry) runs the recurrence of each range that such a
// range follows, from the last sequence start in it, and leaves the end state
// S and the sum of dt; the second adds them up over the ranges back to the
// sequence's start: h = S_j + exp(A sum dt_j) h. So the exponentials of split
// sequences are paid twice, and the host cuts no finer than it takes to fill
// the GPU; where the longest sequence allows it, ranges take whole sequences
// instead (Ranges).
// 16288 tokens of nine sequences, 4096 x 16, bf16: carries 330 us (71 % of the
// exponentials' rate), outputs and saved states 465 us (50 %; 168 instructions a
// warp and token, six in ten issue slots). 8000 x 2048 x 64, fp16: 327 + 431 us.
#pragma once

#include "ssm_common.cuh"

namespace greta {

constexpr int kTile = 8;         // tokens per tile, and per saved state
constexpr int kLaneStates = 4;   // states per lane
constexpr int kFwdChans = 4;     // channels per lane of the forward kernels
constexpr int kScanWarps = 4;    // warps per CTA

struct ScanParams {
  const void *u, *delta, *gate, *B, *C;
  const float *A, *skip, *dbias;  // [D, N], [D] or null, [D] or null
  void* out;                      // [T, D]
  long long ldu, ldd, ldg, ldb, ldc;
  Seqs q;
  int D, N, F, Dg;  // Dg = D / F channels per group
  int spg;          // channel slices per group
  int R, L;         // ranges, tokens per range
  int whole_limit;  // longest sequence with which ranges take whole sequences
  int softplus;
  int zero_rest;    // rows outside every sequence: zeros (else left alone)
  int vec;          // rows of u, delta, gate, out (and the backward's) are whole aligned vectors
  int vec_bc;       // rows of B and C too
  // carries between ranges: end states [R][D][N], sums of dt [R][D], whether
  // the carry holds a sequence start [R], copies of initial states [R][D][N]
  float *carry, *dsum, *hinit;
  int* reset;
  float* ckpt;  // [T / 8 + 1][D][N]: state ahead of every 8th token, or null
  // cache-slot state (packed batches)
  float* state;
  long long s_slot, s_d, s_n, num_slots;
  int st_vec;  // states of a channel are whole aligned float4
  const int* slots;
  const signed char* initial;
  int* err;
  // backward
  const void* dout;
  void *du, *ddelta, *dgate;
  int b0;          // first of the launch's D blocks
  float *part_bc;  // [the launch's D blocks][T][2][N]
  float *part_a;   // [R][D][N]
  float *part_d;   // [R][2][D]: dskip, d(delta_bias)
};

// Which channels and states a lane has.
template <int LN, int KD_ = kFwdChans>
struct Lanes {
  static constexpr int KD = KD_;
  static constexpr int CHW = 32 / LN * KD;  // channels per warp
  static constexpr int NP = LN * kLaneStates;
  int lane, dg, nq;  // the lane's KD channels and its four states
  int f, c0, nch;    // group, first channel, channels of the slice
  __device__ __forceinline__ Lanes(const ScanParams& p, int slice, int lane_) {
    lane = lane_;
    dg = lane / LN;
    nq = lane % LN;
    f = slice / p.spg;
    c0 = f * p.Dg + (slice % p.spg) * CHW;
    nch = min(CHW, (f + 1) * p.Dg - c0);
  }
  __device__ __forceinline__ int ch(int j) const { return dg * KD + j; }
  __device__ __forceinline__ int n0() const { return nq * kLaneStates; }
};

// Values of a lane: [pair of channels][state]
template <int KD>
using LaneStates = f2[KD / 2][kLaneStates];

__device__ __forceinline__ void pack_pair(const float4& a, const float4& b, f2 (&h)[4]) {
  h[0] = pack2(a.x, b.x);
  h[1] = pack2(a.y, b.y);
  h[2] = pack2(a.z, b.z);
  h[3] = pack2(a.w, b.w);
}
__device__ __forceinline__ void unpack_pair(const f2 (&h)[4], float4& a, float4& b) {
  unpack2(h[0], a.x, b.x);
  unpack2(h[1], a.y, b.y);
  unpack2(h[2], a.z, b.z);
  unpack2(h[3], a.w, b.w);
}

// Up to four states (n of them, s apart; vec: one aligned float4), else zeros.
__device__ __forceinline__ float4 load_four(const float* r, long long s, int n, bool vec) {
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec) {
    if (n > 0) x = *reinterpret_cast<const float4*>(r);
  } else {
    if (n > 0) x.x = r[0];
    if (n > 1) x.y = r[s];
    if (n > 2) x.z = r[2 * s];
    if (n > 3) x.w = r[3 * s];
  }
  return x;
}
__device__ __forceinline__ void store_four(float* r, long long s, int n, bool vec, const float4& x) {
  if (vec) {
    if (n > 0) *reinterpret_cast<float4*>(r) = x;
  } else {
    if (n > 0) r[0] = x.x;
    if (n > 1) r[s] = x.y;
    if (n > 2) r[2 * s] = x.z;
    if (n > 3) r[3 * s] = x.w;
  }
}

// The lane's part of an fp32 [D, N] array with element strides (s_d, s_n).
template <int LN, int KD>
__device__ __forceinline__ void load_states(const float* p, const Lanes<LN, KD>& l, int N, long long s_d,
                                            long long s_n, bool vec, LaneStates<KD>& h) {
#pragma unroll
  for (int j = 0; j < KD; j += 2) {
    float4 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      x[i] = load_four(p + (l.c0 + l.ch(j + i)) * s_d + l.n0() * s_n, s_n, l.ch(j + i) < l.nch ? N - l.n0() : 0, vec);
    pack_pair(x[0], x[1], h[j / 2]);
  }
}
template <int LN, int KD>
__device__ __forceinline__ void store_states(float* p, const Lanes<LN, KD>& l, int N, long long s_d, long long s_n,
                                             bool vec, const LaneStates<KD>& h) {
#pragma unroll
  for (int j = 0; j < KD; j += 2) {
    float4 x[2];
    unpack_pair(h[j / 2], x[0], x[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      store_four(p + (l.c0 + l.ch(j + i)) * s_d + l.n0() * s_n, s_n, l.ch(j + i) < l.nch ? N - l.n0() : 0, vec, x[i]);
  }
}
// ... contiguous, on 16-byte boundaries where N % 4 == 0.
template <int LN, int KD>
__device__ __forceinline__ void load_states(const float* p, const Lanes<LN, KD>& l, int N, LaneStates<KD>& h) {
  load_states(p, l, N, N, 1, N % 4 == 0, h);
}
template <int LN, int KD>
__device__ __forceinline__ void store_states(float* p, const Lanes<LN, KD>& l, int N, const LaneStates<KD>& h) {
  store_states(p, l, N, N, 1, N % 4 == 0, h);
}

template <int KD>
__device__ __forceinline__ void zero_states(LaneStates<KD>& h) {
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) h[j][0] = h[j][1] = h[j][2] = h[j][3] = 0ull;
}

// A slot's states of this lane, through the cache's strides.
template <int LN, int KD>
__device__ __forceinline__ void load_slot(const ScanParams& p, int slot, const Lanes<LN, KD>& l, LaneStates<KD>& h) {
  load_states(p.state + slot * p.s_slot, l, p.N, p.s_d, p.s_n, p.st_vec, h);
}
template <int LN, int KD>
__device__ __forceinline__ void store_slot(const ScanParams& p, int slot, const Lanes<LN, KD>& l,
                                           const LaneStates<KD>& h) {
  store_states(p.state + slot * p.s_slot, l, p.N, p.s_d, p.s_n, p.st_vec, h);
}

// The request's slot, or -1 for none (negative or out of range, which is
// flagged once).
__device__ __forceinline__ int slot_of(const ScanParams& p, int s, bool flag) {
  if (p.state == nullptr) return -1;
  const int raw = p.slots[s];
  if (raw >= p.num_slots && p.err != nullptr && flag) atomicOr(p.err, 1);
  return raw >= 0 && raw < p.num_slots ? raw : -1;
}

// A tile's rows of channels as vectors: V channels of a token, NVEC of them per
// lane.
template <int CHW>
struct TileVecs {
  static constexpr int V = CHW < 4 ? CHW : (kTile * CHW >= 256 ? 8 : 4);
  static constexpr int VPR = CHW / V;  // vectors per row
  static constexpr int COUNT = kTile * VPR;
  static constexpr int NVEC = (COUNT + 31) / 32;
  // vector k of a lane: its row and first channel
  static __device__ __forceinline__ bool has(int k, int lane) { return COUNT % 32 == 0 || k * 32 + lane < COUNT; }
  static __device__ __forceinline__ int row(int k, int lane) { return (k * 32 + lane) / VPR; }
  static __device__ __forceinline__ int chan(int lane) { return lane % VPR * V; }
};

// Rows [ta, tb) of a tile of a [T, D] operand into shared memory ([token][CHW]);
// zeros elsewhere. A lane copies the vectors that it reads itself.
template <typename T, int LN, int KD>
__device__ __forceinline__ void copy_tile(const void* base, long long ld, bool vec, const Lanes<LN, KD>& l, int tile0,
                                          int ta, int tb, T* s) {
  constexpr int CHW = Lanes<LN, KD>::CHW;
  using TV = TileVecs<CHW>;
  const T* b = reinterpret_cast<const T*>(base);
#pragma unroll
  for (int k = 0; k < TV::NVEC; ++k) {
    if (!TV::has(k, l.lane)) continue;
    const int r = TV::row(k, l.lane), t = tile0 + r, c = TV::chan(l.lane);
    const int n = t >= ta && t < tb ? l.nch - c : 0;
    copy_part<T, TV::V>(s + r * CHW + c, b + t * ld + l.c0 + c, b, n, vec && (n >= TV::V || n <= 0));
  }
}

// A slice whose every vector is whole: its whole tiles are copied without a
// test (most of what a tile takes beside the recurrence was such tests).
template <int LN, int KD>
__device__ __forceinline__ bool regular(const ScanParams& p, const Lanes<LN, KD>& l) {
  return p.vec && p.vec_bc && l.nch == Lanes<LN, KD>::CHW;
}

// The lane's vector of row 0 of a [T, D] operand; a whole tile of it.
template <typename T, int LN, int KD>
__device__ __forceinline__ const T* lane_row(const void* base, long long ld, const Lanes<LN, KD>& l) {
  using TV = TileVecs<Lanes<LN, KD>::CHW>;
  return reinterpret_cast<const T*>(base) + TV::row(0, l.lane) * ld + l.c0 + TV::chan(l.lane);
}
template <typename T, int LN, int KD>
__device__ __forceinline__ void copy_whole(const T* row0, long long ld, const Lanes<LN, KD>& l, int tile0, T* s) {
  constexpr int CHW = Lanes<LN, KD>::CHW;
  using TV = TileVecs<CHW>;
  static_assert(TV::NVEC == 1, "a vector of a tile per lane");
  if (TV::has(0, l.lane))
    copy_vec<T, TV::V>(s + TV::row(0, l.lane) * CHW + TV::chan(l.lane), row0 + tile0 * ld);
}
// B and C of a whole tile (lane `at` of `lanes`); states past N stay as they are.
template <typename T, int LN, int KD>
__device__ __forceinline__ void copy_whole_bc(const ScanParams& p, const Lanes<LN, KD>& l, int tile0, T* s, int at,
                                              int lanes) {
#pragma unroll
  for (int i0 = 0; i0 < kTile * 2 * LN; i0 += lanes) {
    const int i = i0 + at, n = i % LN * 4;
    if (kTile * 2 * LN % lanes != 0 && i >= kTile * 2 * LN) break;
    const bool b = i / LN % 2 == 0;
    if (n < p.N)
      copy_vec<T, 4>(s + i * 4, reinterpret_cast<const T*>(b ? p.B : p.C) +
                                    (tile0 + i / (2 * LN)) * (b ? p.ldb : p.ldc) + (long long)l.f * p.N + n);
  }
}

// A lane's vector k of a tile in shared memory.
template <typename T, int CHW>
__device__ __forceinline__ Pack<T, TileVecs<CHW>::V> tile_vec(const T* s, int k, int lane) {
  using TV = TileVecs<CHW>;
  return load_part<T, TV::V>(s + TV::row(k, lane) * CHW + TV::chan(lane), TV::V, true);
}

// B and C of a tile into shared memory, [token][B | C][states], by `lanes`
// lanes of which this is number `at`.
template <typename T, int LN, int KD>
__device__ __forceinline__ void copy_bc(const ScanParams& p, const Lanes<LN, KD>& l, int tile0, int ta, int tb, T* s,
                                        int at, int lanes) {
  const T* bg = reinterpret_cast<const T*>(p.B);
  const T* cg = reinterpret_cast<const T*>(p.C);
#pragma unroll
  for (int i = at; i < kTile * 2 * LN; i += lanes) {
    const int n = i % LN * 4, t = tile0 + i / (2 * LN);
    const bool b = i / LN % 2 == 0;
    const T* base = b ? bg : cg;
    copy_part<T, 4>(s + i * 4, base + t * (b ? p.ldb : p.ldc) + (long long)l.f * p.N + n, base,
                    t >= ta && t < tb ? p.N - n : 0, p.vec_bc);
  }
}

// Four states of B or C (as they lie in shared memory), and in fp32, each twice
// (for two channels).
template <typename T>
__device__ __forceinline__ Pack<T, 4> read_four(const T* s) {
  return load_part<T, 4>(s, 4, true);
}
template <typename T>
__device__ __forceinline__ void twice(const Pack<T, 4>& r, f2 (&o)[4]) {
  const float4 v = widen4(r);
  o[0] = pack2(v.x, v.x);
  o[1] = pack2(v.y, v.y);
  o[2] = pack2(v.z, v.z);
  o[3] = pack2(v.w, v.w);
}

__device__ __forceinline__ f2 step_sizes(const ScanParams& p, float x0, float x1) {
  f2 e;
  return p.softplus ? softplus2(x0, x1, e) : pack2(x0, x1);
}

// One token of the recurrence for the lane's states, dl = (dt, dt u) of its
// pairs of channels; y: the lane's part of sum_n C h.
template <bool WITH_Y, int KD>
__device__ __forceinline__ void scan_step(LaneStates<KD>& h, const LaneStates<KD>& A2, const ulonglong2 (&dl)[KD / 2],
                                          const f2 (&b)[4], const f2 (&c)[4], f2 (&y)[KD / 2]) {
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f2 a = f2_decay(dl[j].x, A2[j][i]);
      h[j][i] = f2_fma(a, h[j][i], f2_mul(dl[j].y, b[i]));
      if (WITH_Y) y[j] = i == 0 ? f2_mul(c[i], h[j][i]) : f2_fma(c[i], h[j][i], y[j]);
    }
  }
}

// v (pairs of channels) summed over the LN lanes of the channels: the first
// exchanges give each lane one channel, sum_channel, the rest add it up. Lanes
// with nq < KD hold the sums.
template <int LN>
__device__ __forceinline__ float sum_over_states(const f2 (&v)[2], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
  float k0, k1, s0, s1;
  unpack2(b0 ? v[1] : v[0], k0, k1);
  unpack2(b0 ? v[0] : v[1], s0, s1);
  k0 += __shfl_xor_sync(0xffffffffu, s0, 1);
  k1 += __shfl_xor_sync(0xffffffffu, s1, 1);
  float s = (b1 ? k1 : k0) + __shfl_xor_sync(0xffffffffu, b1 ? k0 : k1, 2);
#pragma unroll
  for (int o = 4; o < LN; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
template <int LN>
__device__ __forceinline__ float sum_over_states(const f2 (&v)[1], int lane) {
  const bool b0 = lane & 1;
  float v0, v1;
  unpack2(v[0], v0, v1);
  float s = (b0 ? v1 : v0) + __shfl_xor_sync(0xffffffffu, b0 ? v0 : v1, 1);
#pragma unroll
  for (int o = 2; o < LN; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
template <int KD>
__device__ __forceinline__ int sum_channel(int lane) {
  return KD == 4 ? (lane & 1) * 2 + ((lane >> 1) & 1) : lane & 1;
}

// Factors of a state: of one that is zero, 0 (a range's growth may be past what fp32
// holds where no token's is, and inf times 0 would be NaN).
__device__ __forceinline__ f2 f2_keep(f2 a, f2 h) {
  float a0, a1, h0, h1;
  unpack2(a, a0, a1);
  unpack2(h, h0, h1);
  return pack2(h0 == 0.f ? 0.f : a0, h1 == 0.f ? 0.f : a1);
}

// A state (or adjoint) brought through the ranges `from`, .., `to` (in that
// direction): the first one's carry, then carry + exp(A sum dt) times what came.
template <int LN, int KD>
__device__ __forceinline__ void carry_through(const ScanParams& p, const Lanes<LN, KD>& l, int from, int to, int step,
                                              const LaneStates<KD>& A2, LaneStates<KD>& h) {
  const long long DN = (long long)p.D * p.N;
  zero_states<KD>(h);
#pragma unroll 2
  for (int j = from; j != to + step; j += step) {
    LaneStates<KD> s;
    load_states(p.carry + j * DN, l, p.N, s);
#pragma unroll
    for (int c = 0; c < KD / 2; ++c) {
      float d[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ch = l.ch(2 * c + i);
        d[i] = ch < l.nch ? p.dsum[(long long)j * p.D + l.c0 + ch] : 0.f;
      }
      const f2 d2 = pack2(d[0], d[1]);
#pragma unroll
      for (int k = 0; k < 4; ++k) h[c][k] = f2_fma(f2_keep(f2_decay(d2, A2[c][k]), h[c][k]), h[c][k], s[c][k]);
    }
  }
}

// The state at the start of range i, which lies inside a sequence: from the
// last range before whose carry holds that sequence's start.
template <int LN, int KD>
__device__ __forceinline__ void carry_in(const ScanParams& p, const Lanes<LN, KD>& l, int i, const LaneStates<KD>& A2,
                                         LaneStates<KD>& h) {
  int j0 = 0;
  for (int hi = i - 1; hi >= 0; hi -= 32) {
    const int k = hi - l.lane;
    const unsigned m = __ballot_sync(0xffffffffu, k >= 0 && p.reset[k] != 0);
    if (m != 0) {
      j0 = hi - (__ffs(m) - 1);
      break;
    }
  }
  carry_through(p, l, j0, i - 1, 1, A2, h);
}

// A log2(e): decays are 2^(dt A2).
template <int LN, int KD>
__device__ __forceinline__ void load_rates(const ScanParams& p, const Lanes<LN, KD>& l, LaneStates<KD>& A2) {
  load_states(p.A, l, p.N, A2);
  const f2 e = pack2(kLog2e, kLog2e);
#pragma unroll
  for (int j = 0; j < KD / 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[j][i] = f2_mul(A2[j][i], e);
}

// A per-channel operand for the lane's vector column (zeros without one).
template <int V>
__device__ __forceinline__ void load_column(const float* v, int c0, int n, float (&o)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = v != nullptr && e < n ? v[c0 + e] : 0.f;
}

// Bits of the tile's rows [ta, tb).
__device__ __forceinline__ unsigned tile_rows(int tile0, int ta, int tb) {
  return ((1u << (tb - ta)) - 1) << (ta - tile0);
}

// The step sizes of a tile in shared memory: [token][pair of channels] (dt0, dt1,
// dt0 u0, dt1 u1). Lanes write four channels each, two float4: the pairs of a
// row's upper half are swapped two by two so that the eight lanes of a row
// write to different banks.
__device__ __forceinline__ int step_slot(int pair) { return pair ^ ((pair >> 3) & 1); }

// How the steps of a tile are dealt to the lanes: four channels a time (CHW of
// a narrow slice).
template <int CHW>
struct StepVecs {
  static constexpr int V = CHW < 4 ? CHW : 4;
  static constexpr int VPR = CHW / V;
  static constexpr int COUNT = kTile * VPR;
  static constexpr int NVEC = (COUNT + 31) / 32;
  static __device__ __forceinline__ bool has(int k, int lane) { return COUNT % 32 == 0 || k * 32 + lane < COUNT; }
  static __device__ __forceinline__ int row(int k, int lane) { return (k * 32 + lane) / VPR; }
  static __device__ __forceinline__ int chan(int lane) { return lane % VPR * V; }
};

// All rows and channels of the tile: those that are not there were copied as
// zeros, have no input and are not stored (a step that no recurrence takes).
// The rows were copied by other lanes: a barrier lies ahead.
template <typename T, int LN, int KD>
__device__ __forceinline__ void stage_steps(const ScanParams& p, const Lanes<LN, KD>& l, const T* u, const T* d,
                                            const float (&bias)[StepVecs<Lanes<LN, KD>::CHW>::V], float4* dl) {
  constexpr int CHW = Lanes<LN, KD>::CHW;
  using SV = StepVecs<CHW>;
  constexpr int V = SV::V;
#pragma unroll
  for (int k = 0; k < SV::NVEC; ++k) {
    if (!SV::has(k, l.lane)) continue;
    const int at = SV::row(k, l.lane) * CHW + SV::chan(l.lane);
    const Pack<T, V> uv = load_part<T, V>(u + at, V, true), dv = load_part<T, V>(d + at, V, true);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const f2 s = step_sizes(p, to_f(dv.v[e]) + bias[e], to_f(dv.v[e + 1]) + bias[e + 1]);
      const f2 x = f2_mul(s, pack2(to_f(uv.v[e]), to_f(uv.v[e + 1])));
      float4 o;
      unpack2(s, o.x, o.y);
      unpack2(x, o.z, o.w);
      dl[step_slot((at + e) / 2)] = o;
    }
  }
}

// The steps of the lane's channels at `at` = token * CHW + channel.
template <int KD>
__device__ __forceinline__ void read_steps(const float4* dl, int at, ulonglong2 (&v)[KD / 2]) {
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) v[j] = *reinterpret_cast<const ulonglong2*>(dl + step_slot(at / 2 + j));
}

// The sums of dt of a range.
template <int LN, int KD>
__device__ __forceinline__ void store_sums(const ScanParams& p, const Lanes<LN, KD>& l, int range,
                                           const f2 (&dsum)[KD / 2]) {
#pragma unroll
  for (int j = 0; j < KD; ++j) {
    float v[2];
    unpack2(dsum[j / 2], v[0], v[1]);
    if (l.ch(j) < l.nch) p.dsum[(long long)range * p.D + l.c0 + l.ch(j)] = v[j % 2];
  }
}

// Shared memory of a warp of the forward, in bytes.
template <typename T, int LN, int KD>
struct FwdSmem {
  static constexpr int CHW = Lanes<LN, KD>::CHW;
  static constexpr int kDl = kTile * CHW * 8;  // (dt, dt u)
  static constexpr int kY = kTile * CHW * 4;
  static constexpr int kRow = kTile * CHW * (int)sizeof(T);        // a tile of an operand
  static constexpr int kBC = kTile * 2 * LN * 4 * (int)sizeof(T);  // [token][B | C]
  static constexpr int kStage = 3 * kRow + kBC;                    // u, delta, gate; B, C
  static constexpr int kWarp = kDl + kY + 2 * kStage;
};

// kPhaseCarry: the end state and sum of dt of a range that a range inside the
// same sequence follows. kPhaseMain: outputs, saved states, slots.
enum ScanPhase { kPhaseCarry = 0, kPhaseMain = 1 };

template <typename T, int LN, int PHASE>
__global__ void __launch_bounds__(kScanWarps * 32, 4) ssm_scan_fwd_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  constexpr int KD = kFwdChans;
  using L = Lanes<LN, KD>;
  using S = FwdSmem<T, LN, KD>;
  constexpr int CHW = L::CHW, NP = L::NP;
  using TV = TileVecs<CHW>;
  constexpr int V = TV::V;
  constexpr bool kMain = PHASE == kPhaseMain;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* mine = reinterpret_cast<char*>(smem4) + warp * S::kWarp;
  float4* dl = reinterpret_cast<float4*>(mine);
  float* ys = reinterpret_cast<float*>(mine + S::kDl);
  auto stage = [&](int s, int part) {  // part: u, delta, gate, (B, C)
    return reinterpret_cast<T*>(mine + S::kDl + S::kY + s * S::kStage + part * S::kRow);
  };
  pdl_wait();
  pdl_trigger();
  const int slice = blockIdx.x * (blockDim.x >> 5) + warp;
  if (slice >= p.F * p.spg) return;
  const L l(p, slice, lane);
  const int ri = blockIdx.y;
  const SeqView sv(p.q, lane);
  const Ranges ranges(sv, p.L, p.whole_limit);
  if (!kMain && ranges.whole) return;  // no range needs a carry
  int t0 = ranges.begin(sv, ri);
  const int t1 = ri + 1 < p.R ? ranges.begin(sv, ri + 1) : p.q.T;
  if (t0 >= t1) return;

  LaneStates<KD> A2, h;
  const long long DN = (long long)p.D * p.N;
  Seg g;
  int slot = -1;
  if (!kMain) {
    if (t1 >= p.q.T) return;
    g = sv.at(t1);
    if (!g.in || g.b >= t1) return;  // the next range begins with a sequence, or outside
    load_rates(p, l, A2);
    zero_states<KD>(h);
    const bool reset = g.b >= t0;
    if (slice == 0 && lane == 0) p.reset[ri] = reset;
    if (reset) {
      t0 = g.b;
      slot = slot_of(p, g.s, false);
      if (slot >= 0 && p.initial[g.s] != 0) {
        load_slot(p, slot, l, h);
        store_states(p.hinit + ri * DN, l, p.N, h);
      }
    }
  } else {
    g = sv.at(t0);
    load_rates(p, l, A2);
    zero_states<KD>(h);
    if (g.in && g.b < t0) {
      carry_in(p, l, ri, A2, h);
      slot = slot_of(p, g.s, false);
    }
  }
  using SV = StepVecs<CHW>;
  float bias[SV::V], skip[V];
  load_column<SV::V>(p.dbias, l.c0 + SV::chan(lane), l.nch - SV::chan(lane), bias);
  if (kMain) load_column<V>(p.skip, l.c0 + TV::chan(lane), l.nch - TV::chan(lane), skip);
  f2 dsum[KD / 2];
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) dsum[j] = 0ull;

  int cur = 0;
  const T* bc;
  const bool reg = regular(p, l);
  const T* u0 = lane_row<T>(p.u, p.ldu, l);
  const T* d0 = lane_row<T>(p.delta, p.ldd, l);
  const T* z0 = lane_row<T>(p.gate, p.ldg, l);
  auto fetch = [&](int tile0, int s) {
    if (reg && tile0 >= t0 && tile0 + kTile <= t1) {
      copy_whole(u0, p.ldu, l, tile0, stage(s, 0));
      copy_whole(d0, p.ldd, l, tile0, stage(s, 1));
      if (kMain && p.gate != nullptr) copy_whole(z0, p.ldg, l, tile0, stage(s, 2));
      copy_whole_bc<T>(p, l, tile0, stage(s, 3), lane, 32);
    } else {
      const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
      copy_tile<T>(p.u, p.ldu, p.vec, l, tile0, ta, tb, stage(s, 0));
      copy_tile<T>(p.delta, p.ldd, p.vec, l, tile0, ta, tb, stage(s, 1));
      if (kMain && p.gate != nullptr) copy_tile<T>(p.gate, p.ldg, p.vec, l, tile0, ta, tb, stage(s, 2));
      copy_bc<T>(p, l, tile0, ta, tb, stage(s, 3), lane, 32);
    }
    copy_commit();
  };
  // states past N: B and C of both stages zero for good
  if (p.N < NP) {
    for (int i = lane; i < kTile * 2 * NP; i += 32) stage(0, 3)[i] = stage(1, 3)[i] = from_f<T>(0.f);
    __syncwarp();
  }
  // What token r of the tile needs from shared memory; its recurrence; its sum.
  // Whole tiles read a token ahead and sum a token behind, so that neither the
  // reads nor the shuffles of a sum stand between two tokens' recurrences.
  struct Operands {
    ulonglong2 dl[KD / 2];
    Pack<T, 4> b, c;
  };
  auto read = [&](int r, Operands& o) {
    read_steps<KD>(dl, r * CHW + l.ch(0), o.dl);
    o.b = read_four(bc + r * 2 * NP + l.n0());
    if (kMain) o.c = read_four(bc + (r * 2 + 1) * NP + l.n0());
  };
  auto step = [&](const Operands& o, f2 (&y)[KD / 2]) {
    f2 b[4], c[4];
    twice(o.b, b);
    if (kMain) twice(o.c, c);
    scan_step<kMain, KD>(h, A2, o.dl, b, c, y);
    if (!kMain) {
#pragma unroll
      for (int j = 0; j < KD / 2; ++j) dsum[j] = f2_add(dsum[j], o.dl[j].x);
    }
  };
  auto sum = [&](int r, const f2 (&y)[KD / 2]) {
    if (kMain) {
      const float s = sum_over_states<LN>(y, lane);
      if (l.nq < KD) ys[r * CHW + l.ch(sum_channel<KD>(lane))] = s;
    }
  };

  // (a carry, and a range of whole sequences, may begin inside a tile)
  const int tile_first = t0 / kTile * kTile;
  fetch(tile_first, 0);
  for (int tile0 = tile_first; tile0 < t1; tile0 += kTile, cur ^= 1) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    copy_wait();
    __syncwarp();
    bc = stage(cur, 3);
    stage_steps<T>(p, l, stage(cur, 0), stage(cur, 1), bias, dl);
    __syncwarp();
    // (the other stage's B and C were last read ahead of the barrier before)
    if (tile0 + kTile < t1) fetch(tile0 + kTile, cur ^ 1);
    if (kMain && p.ckpt != nullptr && ta == tile0) store_states(p.ckpt + (tile0 / kTile) * DN, l, p.N, h);
    // out of the tile's sums, for the lane's vector
    auto output = [&](int tt, bool in, int n, bool vec) {
      const int r = TV::row(0, lane), c = TV::chan(lane);
      const Pack<T, V> u = tile_vec<T, CHW>(stage(cur, 0), 0, lane);
      const Pack<float, V> y = load_part<float, V>(ys + r * CHW + c, V, true);
      Pack<T, V> z, o;
      if (p.gate != nullptr) z = tile_vec<T, CHW>(stage(cur, 2), 0, lane);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = fmaf(skip[e], to_f(u.v[e]), y.v[e]);
        if (p.gate != nullptr) v *= to_f(z.v[e]) * sigmoid_t<T>(to_f(z.v[e]));
        o.v[e] = from_f<T>(in ? v : 0.f);
      }
      store_part<T, V>(reinterpret_cast<T*>(p.out) + (long long)tt * p.D + l.c0 + c, o, n, vec);
    };
    if (reg && g.in && g.b < ta && g.e > tb && tb - ta == kTile) {
      // a whole tile inside a sequence
      Operands o[2];
      f2 y[2][KD / 2];
      read(0, o[0]);
#pragma unroll
      for (int r = 0; r < kTile; ++r) {
        if (r + 1 < kTile) read(r + 1, o[(r + 1) % 2]);
        step(o[r % 2], y[r % 2]);
        if (r > 0) sum(r - 1, y[(r + 1) % 2]);
      }
      sum(kTile - 1, y[(kTile - 1) % 2]);
      __syncwarp();
      if (kMain && TV::has(0, lane)) output(tile0 + TV::row(0, lane), true, V, true);
      continue;
    }
    unsigned live = 0;  // tokens of the tile that a sequence holds
    int t = ta;
    while (t < tb) {
      const int stop = min(g.e, tb);
      if (g.in) {
        if (kMain && t == g.b) {
          zero_states<KD>(h);
          slot = slot_of(p, g.s, slice == 0 && lane == 0);
          if (slot >= 0 && p.initial[g.s] != 0) {
            // a sequence that goes on in a later range: its last range may have
            // written the slot by now, so the copy of the first kernel
            if (g.e > t1)
              load_states(p.hinit + ri * DN, l, p.N, h);
            else
              load_slot(p, slot, l, h);
          }
        }
#pragma unroll 1
        for (int r = t - tile0; r < stop - tile0; ++r) {
          Operands o;
          f2 y[KD / 2];
          read(r, o);
          step(o, y);
          sum(r, y);
        }
        live |= tile_rows(tile0, t, stop);
        if (kMain && stop == g.e && slot >= 0) store_slot(p, slot, l, h);
      }
      t = stop;
      if (t == g.e && t < t1) g = sv.next(g);
    }
    __syncwarp();
    if (kMain && TV::has(0, lane)) {
      const int r = TV::row(0, lane), tt = tile0 + r, n = l.nch - TV::chan(lane);
      const bool in = (live >> r) & 1;
      if (tt >= ta && tt < tb && n > 0 && (in || p.zero_rest)) output(tt, in, n, p.vec && n >= V);
    }
  }
  if (!kMain) {
    store_states(p.carry + ri * DN, l, p.N, h);
    if (l.nq == 0) store_sums(p, l, ri, dsum);
  }
}

// Batches of (nearly) one token per request: bound by the states' read and
// write, 8 D N bytes a request. A warp has the channels and states of Lanes for
// a chunk of up to 32 requests, whose metadata its lanes hold and whose decay
// rates it reads once; states and first rows of the next kAhead requests are
// on their way in asynchronous copies while one is computed. (A warp per
// request or two, with loads into registers, spent its time on one chain of
// latencies after the other: 44 us for 256 requests of 4096 x 16; now 27 us,
// 4.8 TB/s.) Requests of
// more tokens (few, by the host's rule) are walked token by token.
constexpr int kAhead = 3;

template <typename T, int LN>
struct DecodeSmem {
  static constexpr int CHW = Lanes<LN>::CHW, NP = Lanes<LN>::NP;
  static constexpr int kStates = 32 * kFwdChans * 16;                      // [channel][lane] float4
  static constexpr int kRows = (3 * CHW + 2 * NP) * (int)sizeof(T);        // u, delta, gate, B, C of a token
  static constexpr int kStage = kStates + (kRows + 15) / 16 * 16;
  static constexpr int kWarp = (kAhead + 1) * kStage;
};

template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32, 4) ssm_scan_decode_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  constexpr int KD = kFwdChans;
  using L = Lanes<LN, KD>;
  using S = DecodeSmem<T, LN>;
  constexpr int CHW = L::CHW, NP = L::NP;
  constexpr int V = CHW < 4 ? CHW : 4;  // elements a copy
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.x * (blockDim.x >> 5) + warp;
  if (slice >= p.F * p.spg) return;
  const L l(p, slice, lane);
  char* mine = reinterpret_cast<char*>(smem4) + warp * S::kWarp;
  auto states = [&](int q) { return reinterpret_cast<float4*>(mine + q % (kAhead + 1) * S::kStage) + lane; };
  auto rows = [&](int q) { return reinterpret_cast<T*>(mine + q % (kAhead + 1) * S::kStage + S::kStates); };
  // the channel whose step and output this lane computes
  const int cj = l.ch(sum_channel<KD>(lane));
  const bool own = l.nq < KD && cj < l.nch;
  const int c = l.c0 + cj;
  pdl_wait();
  pdl_trigger();
  const int r0 = blockIdx.y * p.L, count = min(p.L, p.q.nseq - r0);  // (L: requests per chunk, at most 32)
  int mb = 0, me = 0, mslot = -1, minit = 0;
  if (lane < count) {
    mb = seq_start(p.q, r0 + lane);
    me = seq_start(p.q, r0 + lane + 1);
    if (p.state != nullptr) {
      const int raw = p.slots[r0 + lane];
      minit = p.initial[r0 + lane];
      if (mb < me && raw >= p.num_slots && p.err != nullptr && slice == 0) atomicOr(p.err, 1);
      mslot = mb < me && raw >= 0 && raw < p.num_slots ? raw : -1;
    }
  }
  LaneStates<KD> A2;
  load_rates(p, l, A2);
  const float bias = p.dbias != nullptr && own ? p.dbias[c] : 0.f;
  const float skip = p.skip != nullptr && own ? p.skip[c] : 0.f;

  // token t's rows: u, delta, gate of the channels, B and C of the states
  auto copy_rows = [&](int q, int t) {
    constexpr int ROW = CHW / V, ALL = 3 * ROW + 2 * LN;
    T* s = rows(q);
#pragma unroll
    for (int i0 = 0; i0 < ALL; i0 += 32) {
      const int i = i0 + lane;
      if (i < 3 * ROW) {
        const int op = i / ROW, at = i % ROW * V, n = l.nch - at;
        const T* g = reinterpret_cast<const T*>(op == 0 ? p.u : op == 1 ? p.delta : p.gate);
        const long long ld = op == 0 ? p.ldu : op == 1 ? p.ldd : p.ldg;
        if (g != nullptr)
          copy_part<T, V>(s + op * CHW + at, g + t * ld + l.c0 + at, g, n, p.vec && (n >= V || n <= 0));
      } else if (i < ALL) {
        const int k = i - 3 * ROW, op = k / LN, at = k % LN * 4;
        const T* g = reinterpret_cast<const T*>(op == 0 ? p.B : p.C);
        copy_part<T, 4>(s + 3 * CHW + op * NP + at, g + t * (op == 0 ? p.ldb : p.ldc) + (long long)l.f * p.N + at, g,
                        p.N - at, p.vec_bc);
      }
    }
  };
  auto issue = [&](int q) {
    if (q < count) {
      const int b = __shfl_sync(0xffffffffu, mb, q), e = __shfl_sync(0xffffffffu, me, q);
      const int slot = __shfl_sync(0xffffffffu, mslot, q), initial = __shfl_sync(0xffffffffu, minit, q);
      if (b < e) {
        copy_rows(q, b);
        const bool from = slot >= 0 && initial != 0;
        if (p.st_vec || !from) {
          const float* s = p.state + (from ? slot * p.s_slot : 0);
#pragma unroll
          for (int j = 0; j < KD; ++j) {
            const bool ok = from && l.ch(j) < l.nch && l.n0() < p.N;
            copy_async<16>(states(q) + j * 32, ok ? s + (l.c0 + l.ch(j)) * p.s_d + l.n0() : p.A, ok);
          }
        } else {
#pragma unroll
          for (int j = 0; j < KD; ++j)
            states(q)[j * 32] = load_four(p.state + slot * p.s_slot + (l.c0 + l.ch(j)) * p.s_d + l.n0() * p.s_n, p.s_n,
                                          l.ch(j) < l.nch ? p.N - l.n0() : 0, false);
        }
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int q = 0; q < kAhead; ++q) issue(q);
#pragma unroll 1
  for (int q = 0; q < count; ++q) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    __syncwarp();
    issue(q + kAhead);
    const int b = __shfl_sync(0xffffffffu, mb, q), e = __shfl_sync(0xffffffffu, me, q);
    const int slot = __shfl_sync(0xffffffffu, mslot, q);
    if (b >= e) continue;
    LaneStates<KD> h;
#pragma unroll
    for (int j = 0; j < KD; j += 2) pack_pair(states(q)[j * 32], states(q)[(j + 1) * 32], h[j / 2]);
    for (int t = b; t < e; ++t) {
      if (t > b) {
        __syncwarp();
        copy_rows(q, t);
        copy_commit();
        copy_wait();
        __syncwarp();
      }
      const T* s = rows(q);
      const float u = own ? to_f(s[cj]) : 0.f;
      float dt = 0.f, other;
      if (own) unpack2(step_sizes(p, to_f(s[CHW + cj]) + bias, 0.f), dt, other);
      ulonglong2 d[KD / 2];
#pragma unroll
      for (int j = 0; j < KD / 2; ++j) {
        float x[2], y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // that channel's lane: sum_channel is its own inverse
          const int src = l.dg * LN + sum_channel<KD>(2 * j + i);
          x[i] = __shfl_sync(0xffffffffu, dt, src);
          y[i] = __shfl_sync(0xffffffffu, dt * u, src);
        }
        d[j].x = pack2(x[0], x[1]);
        d[j].y = pack2(y[0], y[1]);
      }
      f2 b2[4], c2[4], y[KD / 2];
      twice(read_four(s + 3 * CHW + l.n0()), b2);
      twice(read_four(s + 3 * CHW + NP + l.n0()), c2);
      scan_step<true, KD>(h, A2, d, b2, c2, y);
      float o = sum_over_states<LN>(y, lane);
      if (own) {
        o = fmaf(skip, u, o);
        if (p.gate != nullptr) o *= to_f(s[2 * CHW + cj]) * sigmoid_t<T>(to_f(s[2 * CHW + cj]));
        reinterpret_cast<T*>(p.out)[(long long)t * p.D + c] = from_f<T>(o);
      }
    }
    if (slot >= 0) store_slot(p, slot, l, h);
  }
  if (p.zero_rest && own) {
    T* og = reinterpret_cast<T*>(p.out) + c;
    const T z = from_f<T>(0.f);
    if (blockIdx.y == 0)
      for (int t = 0; t < seq_start(p.q, 0); ++t) og[(long long)t * p.D] = z;
    if (blockIdx.y == gridDim.y - 1)
      for (int t = seq_start(p.q, p.q.nseq); t < p.q.T; ++t) og[(long long)t * p.D] = z;
  }
}

}  // namespace greta
