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
// (three multiplications, two fused additions) is half of that on the fp32
// pipe, issued two states an instruction.
//
// Split. A warp works alone: CHW = 128 / LN channels of one group and all
// their states, LN lanes a channel and four states a lane (LN = N / 4 rounded
// up to a power of two from 4 on), four channels a lane. So a lane keeps 16
// states and their 16 decay rates in registers, a token's B and C are read by
// four channels at a time, and sums over n take log2(LN) shuffles for four
// channels together. The packed stream is cut into ranges by position
// (ssm_common.cuh); a warp walks its range in tiles of 16 tokens: it loads the
// tile's rows as vectors, computes (dt, dt u) once per token and channel into
// shared memory, runs the recurrence from there, and applies skip and gate to
// the tile's y, again as vectors.
//
// A range that begins inside a sequence needs the state at its first token.
// The first kernel (kPhaseCarry) runs the recurrence of each range that such a
// range follows, from the last sequence start in it, and leaves the end state
// S and the sum of dt; the second adds them up over the ranges back to the
// sequence's start: h = S_j + exp(A sum dt_j) h. So the exponentials of split
// sequences are paid twice, and the host cuts no finer than it takes to fill
// the GPU.
#pragma once

#include "ssm_common.cuh"

namespace greta {

constexpr int kTile = 16;        // tokens per tile, and per saved state
constexpr int kLaneStates = 4;   // states per lane
constexpr int kLaneChans = 4;    // channels per lane
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
  int softplus;
  int zero_rest;    // rows outside every sequence: zeros (else left alone)
  int vec;          // rows of u, delta, gate, out (and the backward's) are whole aligned vectors
  int vec_bc;       // rows of B and C too
  // carries between ranges: end states [R][D][N], sums of dt [R][D], whether
  // the carry holds a sequence start [R], copies of initial states [R][D][N]
  float *carry, *dsum, *hinit;
  int* reset;
  float* ckpt;  // [T / 16 + 1][D][N]: state ahead of every 16th token, or null
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
  float *part_bc;  // [D blocks][T][2][N]
  float *part_a;   // [R][D][N]
  float *part_d;   // [R][2][D]: dskip, d(delta_bias)
};

// Which channels and states a lane has.
template <int LN>
struct Lanes {
  static constexpr int CHW = 128 / LN;  // channels per warp
  static constexpr int NP = LN * kLaneStates;
  int lane, dg, nq;  // channel group of four and states' quarter
  int f, c0, nch;    // group, first channel, channels of the slice
  __device__ __forceinline__ Lanes(const ScanParams& p, int slice, int lane_) {
    lane = lane_;
    dg = lane / LN;
    nq = lane % LN;
    f = slice / p.spg;
    c0 = f * p.Dg + (slice % p.spg) * CHW;
    nch = min(CHW, (f + 1) * p.Dg - c0);
  }
  __device__ __forceinline__ int ch(int j) const { return dg * kLaneChans + j; }
  __device__ __forceinline__ int n0() const { return nq * kLaneStates; }
};

// Values of a lane: [channel][pair of states]
using LaneStates = f2[kLaneChans][kLaneStates / 2];

// p[(c0 + ch) * N + n] of this lane (rows of N floats), zeros where there is
// no such channel or state.
template <int LN>
__device__ __forceinline__ void load_states(const float* p, const Lanes<LN>& l, int N, float (&v)[4][4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool okc = l.ch(j) < l.nch;
    const float* r = p + (long long)(l.c0 + l.ch(j)) * N + l.n0();
    if (okc && N % 4 == 0 && l.n0() < N) {
      const float4 x = *reinterpret_cast<const float4*>(r);
      v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = okc && l.n0() + i < N ? r[i] : 0.f;
    }
  }
}

template <int LN>
__device__ __forceinline__ void store_states(float* p, const Lanes<LN>& l, int N, const LaneStates& h) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (l.ch(j) >= l.nch) continue;
    float* r = p + (long long)(l.c0 + l.ch(j)) * N + l.n0();
    float4 x;
    unpack2(h[j][0], x.x, x.y);
    unpack2(h[j][1], x.z, x.w);
    if (N % 4 == 0) {
      if (l.n0() < N) *reinterpret_cast<float4*>(r) = x;
    } else {
      const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (l.n0() + i < N) r[i] = v[i];
    }
  }
}

__device__ __forceinline__ void pack_states(const float (&v)[4][4], LaneStates& h) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j][0] = pack2(v[j][0], v[j][1]);
    h[j][1] = pack2(v[j][2], v[j][3]);
  }
}

__device__ __forceinline__ void zero_states(LaneStates& h) {
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j][0] = h[j][1] = 0ull;
}

// A slot's states of this lane, through the cache's strides.
template <int LN>
__device__ __forceinline__ void load_slot(const ScanParams& p, int slot, const Lanes<LN>& l, LaneStates& h) {
  const float* b = p.state + slot * p.s_slot;
  float v[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool okc = l.ch(j) < l.nch;
    const float* r = b + (l.c0 + l.ch(j)) * p.s_d + l.n0() * p.s_n;
    if (p.st_vec && okc && l.n0() < p.N) {
      const float4 x = *reinterpret_cast<const float4*>(r);
      v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = okc && l.n0() + i < p.N ? r[i * p.s_n] : 0.f;
    }
  }
  pack_states(v, h);
}

template <int LN>
__device__ __forceinline__ void store_slot(const ScanParams& p, int slot, const Lanes<LN>& l, const LaneStates& h) {
  float* b = p.state + slot * p.s_slot;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (l.ch(j) >= l.nch) continue;
    float* r = b + (l.c0 + l.ch(j)) * p.s_d + l.n0() * p.s_n;
    float4 x;
    unpack2(h[j][0], x.x, x.y);
    unpack2(h[j][1], x.z, x.w);
    if (p.st_vec) {
      if (l.n0() < p.N) *reinterpret_cast<float4*>(r) = x;
    } else {
      const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (l.n0() + i < p.N) r[i * p.s_n] = v[i];
    }
  }
}

// The request's slot, or -1 for none (negative or out of range, which is
// flagged once).
__device__ __forceinline__ int slot_of(const ScanParams& p, int s, bool flag) {
  if (p.state == nullptr) return -1;
  const int raw = p.slots[s];
  if (raw >= p.num_slots && p.err != nullptr && flag) atomicOr(p.err, 1);
  return raw >= 0 && raw < p.num_slots ? raw : -1;
}

// Vectors of a tile: V channels of a token's row, NVEC of them per lane.
template <int LN>
struct TileVecs {
  static constexpr int CHW = Lanes<LN>::CHW;
  static constexpr int V = CHW < 8 ? CHW : 8;
  static constexpr int VPR = CHW / V;  // vectors per row
  static constexpr int COUNT = kTile * VPR;
  static constexpr int NVEC = (COUNT + 31) / 32;
};

// Shared memory of a warp, in floats.
template <int LN>
struct FwdSmem {
  static constexpr int kDl = kTile * Lanes<LN>::CHW * 2;  // (dt, dt u)
  static constexpr int kY = kTile * Lanes<LN>::CHW;
  static constexpr int kBC = kTile * Lanes<LN>::NP * 2;   // [token][B | C]
  static constexpr int kWarp = kDl + kY + kBC;
};

template <typename T, int LN>
__device__ __forceinline__ void stage_bc(const ScanParams& p, const Lanes<LN>& l, int tile0, int ta, int tb,
                                         float* bc, bool with_c) {
  constexpr int NP = Lanes<LN>::NP;
  const T* bg = reinterpret_cast<const T*>(p.B) + (long long)l.f * p.N;
  const T* cg = reinterpret_cast<const T*>(p.C) + (long long)l.f * p.N;
  // four states at a time
  for (int i = l.lane; i < kTile * LN * 2; i += 32) {
    const int which = i / (kTile * LN);
    const int r = (i / LN) % kTile, n = (i % LN) * 4, t = tile0 + r;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t >= ta && t < tb && (which == 0 || with_c)) {
      const T* s = (which == 0 ? bg + (long long)t * p.ldb : cg + (long long)t * p.ldc) + n;
      const Pack<T, 4> v = load_part<T, 4>(s, p.N - n, p.vec_bc && n < p.N);
      o = make_float4(to_f(v.v[0]), to_f(v.v[1]), to_f(v.v[2]), to_f(v.v[3]));
    }
    *reinterpret_cast<float4*>(bc + (r * 2 + which) * NP + n) = o;
  }
}

__device__ __forceinline__ float step_size(const ScanParams& p, float raw) { return p.softplus ? softplusf_(raw) : raw; }

// One token of the recurrence for the lane's states; y[j] += the lane's part
// of sum_n C h.
template <bool WITH_Y>
__device__ __forceinline__ void scan_step(LaneStates& h, const LaneStates& A2, const float2 (&dl)[4], float4 b,
                                          float4 c, float (&y)[4]) {
  const f2 b2[2] = {pack2(b.x, b.y), pack2(b.z, b.w)};
  const f2 c2[2] = {pack2(c.x, c.y), pack2(c.z, c.w)};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f2 d = pack2(dl[j].x, dl[j].x), du = pack2(dl[j].y, dl[j].y);
    const f2 a0 = f2_ex2(f2_mul(d, A2[j][0])), a1 = f2_ex2(f2_mul(d, A2[j][1]));
    h[j][0] = f2_fma(a0, h[j][0], f2_mul(du, b2[0]));
    h[j][1] = f2_fma(a1, h[j][1], f2_mul(du, b2[1]));
    if (WITH_Y) y[j] = f2_sum(f2_fma(c2[0], h[j][0], f2_mul(c2[1], h[j][1])));
  }
}

// y[j] summed over the LN lanes of the channels; lane nq of the group keeps
// channel (bit 0 of nq) * 2 + (bit 1 of nq).
template <int LN>
__device__ __forceinline__ float sum_over_states(const float (&y)[4], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
  const float s0 = (b0 ? y[2] : y[0]) + __shfl_xor_sync(0xffffffffu, b0 ? y[0] : y[2], 1);
  const float s1 = (b0 ? y[3] : y[1]) + __shfl_xor_sync(0xffffffffu, b0 ? y[1] : y[3], 1);
  float s = (b1 ? s1 : s0) + __shfl_xor_sync(0xffffffffu, b1 ? s0 : s1, 2);
#pragma unroll
  for (int o = 4; o < LN; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ int sum_channel(int lane) { return (lane & 1) * 2 + ((lane >> 1) & 1); }

// The state at the start of range i, which lies inside a sequence that began
// in range j0 < i (j0: the last range whose carry holds a sequence start).
template <int LN>
__device__ __forceinline__ void carry_in(const ScanParams& p, const Lanes<LN>& l, int i, const LaneStates& A2,
                                         LaneStates& h) {
  int j0 = i - 1;
  for (int hi = i - 1; hi >= 0; hi -= 32) {
    const int k = hi - l.lane;
    const unsigned m = __ballot_sync(0xffffffffu, k >= 0 && p.reset[k] != 0);
    if (m != 0) {
      j0 = hi - (__ffs(m) - 1);
      break;
    }
    j0 = max(0, hi - 31);
  }
  const long long DN = (long long)p.D * p.N;
  zero_states(h);
  for (int j = j0; j < i; ++j) {
    float s[4][4];
    load_states(p.carry + j * DN, l, p.N, s);
    LaneStates s2;
    pack_states(s, s2);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float d = l.ch(c) < l.nch && j > j0 ? p.dsum[(long long)j * p.D + l.c0 + l.ch(c)] : 0.f;
      const f2 d2 = pack2(d, d);
#pragma unroll
      for (int k = 0; k < 2; ++k) h[c][k] = f2_fma(f2_ex2(f2_mul(d2, A2[c][k])), h[c][k], s2[c][k]);
    }
  }
}

template <int LN>
__device__ __forceinline__ void load_rates(const ScanParams& p, const Lanes<LN>& l, LaneStates& A2) {
  float v[4][4];
  load_states(p.A, l, p.N, v);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] *= kLog2e;
  pack_states(v, A2);
}

// (dt, dt u) of a tile into shared memory; rows outside [ta, tb) and channels
// that are not there get zeros (a decay of 1 and no input).
template <typename T, int LN>
__device__ __forceinline__ void stage_steps(const ScanParams& p, const Lanes<LN>& l, int tile0, int ta, int tb,
                                            float* dl, Pack<T, TileVecs<LN>::V> (&u)[TileVecs<LN>::NVEC]) {
  using TV = TileVecs<LN>;
  constexpr int V = TV::V, CHW = TV::CHW;
#pragma unroll
  for (int k = 0; k < TV::NVEC; ++k) {
    const int i = k * 32 + l.lane;
    if (TV::COUNT % 32 != 0 && i >= TV::COUNT) continue;
    const int r = i / TV::VPR, c = (i % TV::VPR) * V, t = tile0 + r;
    const int n = l.nch - c;
    zero(u[k]);
    float2 o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = make_float2(0.f, 0.f);
    if (t >= ta && t < tb && n > 0) {
      const bool vec = p.vec && n >= V;
      u[k] = load_part<T, V>(reinterpret_cast<const T*>(p.u) + t * p.ldu + l.c0 + c, n, vec);
      const Pack<T, V> d = load_part<T, V>(reinterpret_cast<const T*>(p.delta) + t * p.ldd + l.c0 + c, n, vec);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (e < n) {
          const float bias = p.dbias != nullptr ? p.dbias[l.c0 + c + e] : 0.f;
          const float s = step_size(p, to_f(d.v[e]) + bias);
          o[e] = make_float2(s, s * to_f(u[k].v[e]));
        }
      }
    }
    float4* w = reinterpret_cast<float4*>(dl + (r * CHW + c) * 2);
#pragma unroll
    for (int e = 0; e < V; e += 2) w[e / 2] = make_float4(o[e].x, o[e].y, o[e + 1].x, o[e + 1].y);
  }
}

template <int LN>
__device__ __forceinline__ void read_steps(const float* dl, const Lanes<LN>& l, int r, float2 (&v)[4]) {
  const float4* s = reinterpret_cast<const float4*>(dl + (r * Lanes<LN>::CHW + l.ch(0)) * 2);
  const float4 a = s[0], b = s[1];
  v[0] = make_float2(a.x, a.y);
  v[1] = make_float2(a.z, a.w);
  v[2] = make_float2(b.x, b.y);
  v[3] = make_float2(b.z, b.w);
}

// kPhaseCarry: the end state and sum of dt of a range that a range inside the
// same sequence follows. kPhaseMain: outputs, saved states, slots.
enum ScanPhase { kPhaseCarry = 0, kPhaseMain = 1 };

template <typename T, int LN, int PHASE>
__global__ void __launch_bounds__(kScanWarps * 32) ssm_scan_fwd_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  using TV = TileVecs<LN>;
  constexpr int CHW = TV::CHW, V = TV::V, NP = Lanes<LN>::NP;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* dl = reinterpret_cast<float*>(smem4) + warp * FwdSmem<LN>::kWarp;
  float* ys = dl + FwdSmem<LN>::kDl;
  float* bc = ys + FwdSmem<LN>::kY;
  pdl_wait();
  pdl_trigger();
  const int slice = blockIdx.x * (blockDim.x >> 5) + warp;
  if (slice >= p.F * p.spg) return;
  const Lanes<LN> l(p, slice, lane);
  const int ri = blockIdx.y;
  int t0 = range_begin(p.q, ri, p.R, p.L, lane);
  const int t1 = range_begin(p.q, ri + 1, p.R, p.L, lane);
  if (t0 >= t1 && PHASE == kPhaseMain) return;

  LaneStates A2, h;
  load_rates(p, l, A2);
  zero_states(h);
  const long long DN = (long long)p.D * p.N;
  float dsum[4] = {0.f, 0.f, 0.f, 0.f};
  Seg g;
  if (PHASE == kPhaseCarry) {
    if (ri + 1 >= p.R || t1 >= p.q.T) return;
    g = seg_at(p.q, t1, lane);
    if (!g.in || g.b >= t1) return;  // the next range begins with a sequence, or outside
    const bool reset = g.b >= t0;
    if (slice == 0 && lane == 0) p.reset[ri] = reset;
    if (reset) {
      t0 = g.b;
      const int slot = slot_of(p, g.s, false);
      if (slot >= 0 && p.initial[g.s] != 0) {
        load_slot(p, slot, l, h);
        store_states(p.hinit + ri * DN, l, p.N, h);
      }
    }
  } else {
    g = seg_at(p.q, t0, lane);
    if (g.in && g.b < t0) carry_in(p, l, ri, A2, h);
  }
  int slot = -1;
  if (PHASE == kPhaseMain && g.in && g.b < t0) slot = slot_of(p, g.s, false);

  for (int tile0 = t0 / kTile * kTile; tile0 < t1; tile0 += kTile) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    Pack<T, V> u[TV::NVEC];
    stage_steps<T, LN>(p, l, tile0, ta, tb, dl, u);
    stage_bc<T, LN>(p, l, tile0, ta, tb, bc, PHASE == kPhaseMain);
    __syncwarp();
    if (PHASE == kPhaseMain && p.ckpt != nullptr && ta == tile0)
      store_states(p.ckpt + (tile0 / kTile) * DN, l, p.N, h);
    unsigned live = 0;  // tokens of the tile that a sequence holds
    int t = ta;
    while (t < tb) {
      const int stop = min(g.e, tb);
      if (g.in) {
        if (PHASE == kPhaseMain && t == g.b) {
          zero_states(h);
          slot = slot_of(p, g.s, slice == 0 && lane == 0);
          if (slot >= 0 && p.initial[g.s] != 0) {
            // a sequence that goes on in a later range: its last range may have
            // written the slot by now, so the copy of the first kernel
            if (g.e > t1) {
              float v[4][4];
              load_states(p.hinit + ri * DN, l, p.N, v);
              pack_states(v, h);
            } else {
              load_slot(p, slot, l, h);
            }
          }
        }
#pragma unroll 2
        for (int r = t - tile0; r < stop - tile0; ++r) {
          float2 d[4];
          read_steps(dl, l, r, d);
          const float4 b = *reinterpret_cast<const float4*>(bc + (r * 2) * NP + l.n0());
          float y[4];
          if (PHASE == kPhaseMain) {
            const float4 c = *reinterpret_cast<const float4*>(bc + (r * 2 + 1) * NP + l.n0());
            scan_step<true>(h, A2, d, b, c, y);
            const float s = sum_over_states<LN>(y, lane);
            if (l.nq < 4) ys[r * CHW + l.ch(sum_channel(lane))] = s;
          } else {
            scan_step<false>(h, A2, d, b, b, y);
#pragma unroll
            for (int j = 0; j < 4; ++j) dsum[j] += d[j].x;
          }
        }
        live |= (0xffffu >> (kTile - (stop - t))) << (t - tile0);
        if (PHASE == kPhaseMain && stop == g.e && slot >= 0) store_slot(p, slot, l, h);
      }
      t = stop;
      if (t == g.e && t < t1) g = seg_next(p.q, g);
    }
    __syncwarp();
    if (PHASE == kPhaseMain) {
#pragma unroll
      for (int k = 0; k < TV::NVEC; ++k) {
        const int i = k * 32 + lane;
        if (TV::COUNT % 32 != 0 && i >= TV::COUNT) continue;
        const int r = i / TV::VPR, c = (i % TV::VPR) * V, tt = tile0 + r;
        const int n = l.nch - c;
        if (tt < ta || tt >= tb || n <= 0) continue;
        const bool in = (live >> r) & 1;
        if (!in && !p.zero_rest) continue;
        const bool vec = p.vec && n >= V;
        Pack<T, V> o;
        zero(o);
        if (in) {
          Pack<T, V> z;
          if (p.gate != nullptr)
            z = load_part<T, V>(reinterpret_cast<const T*>(p.gate) + tt * p.ldg + l.c0 + c, n, vec);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (e < n) {
              float y = ys[r * CHW + c + e];
              if (p.skip != nullptr) y = fmaf(p.skip[l.c0 + c + e], to_f(u[k].v[e]), y);
              if (p.gate != nullptr) y *= to_f(z.v[e]) * sigmoid_exact(to_f(z.v[e]));
              o.v[e] = from_f<T>(y);
            }
          }
        }
        store_part<T, V>(reinterpret_cast<T*>(p.out) + (long long)tt * p.D + l.c0 + c, o, n, vec);
      }
    }
  }
  if (PHASE == kPhaseCarry) {
    store_states(p.carry + ri * DN, l, p.N, h);
    if (l.nq == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (l.ch(j) < l.nch) p.dsum[(long long)ri * p.D + l.c0 + l.ch(j)] = dsum[j];
    }
  }
}

// Batches of (nearly) one token per request: bound by the states' read and
// write, 8 D N bytes a request. A warp has the channels and states of Lanes for
// RQ requests, all of whose states, rows and metadata it asks for before it
// computes, with the decay rates read once; requests of more tokens (few, by
// the host's rule) are walked token by token.
template <typename T, int LN, int RQ>
__global__ void __launch_bounds__(kScanWarps * 32) ssm_scan_decode_kernel(const ScanParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.x * (blockDim.x >> 5) + warp;
  if (slice >= p.F * p.spg) return;
  const Lanes<LN> l(p, slice, lane);
  // the channel whose step and output this lane computes
  const int cj = l.ch(sum_channel(lane));
  const bool mine = l.nq < 4 && cj < l.nch;
  const int c = l.c0 + cj;
  const T* ug = reinterpret_cast<const T*>(p.u);
  const T* dg = reinterpret_cast<const T*>(p.delta);
  const T* zg = reinterpret_cast<const T*>(p.gate);
  const T* bg = reinterpret_cast<const T*>(p.B) + (long long)l.f * p.N + l.n0();
  const T* cg = reinterpret_cast<const T*>(p.C) + (long long)l.f * p.N + l.n0();
  T* og = reinterpret_cast<T*>(p.out);
  pdl_wait();
  pdl_trigger();
  LaneStates A2;
  load_rates(p, l, A2);
  const float bias = p.dbias != nullptr && mine ? p.dbias[c] : 0.f;
  const float skip = p.skip != nullptr && mine ? p.skip[c] : 0.f;
  LaneStates h[RQ];
  int tb[RQ], te[RQ], slot[RQ];
  struct Row {
    T u, d, z;
    Pack<T, 4> b, c;
  } row[RQ];
  auto load_row = [&](int t, Row& r) {
    if (mine) {
      r.u = ug[t * p.ldu + c];
      r.d = dg[t * p.ldd + c];
      if (zg != nullptr) r.z = zg[t * p.ldg + c];
    }
    const bool v = p.vec_bc && l.n0() < p.N;
    r.b = load_part<T, 4>(bg + t * p.ldb, p.N - l.n0(), v);
    r.c = load_part<T, 4>(cg + t * p.ldc, p.N - l.n0(), v);
  };
#pragma unroll
  for (int q = 0; q < RQ; ++q) {
    const int r = blockIdx.y * RQ + q;
    const bool ok = r < p.q.nseq;
    tb[q] = ok ? seq_start(p.q, r) : 0;
    te[q] = ok ? seq_start(p.q, r + 1) : 0;
    slot[q] = tb[q] < te[q] ? slot_of(p, r, slice == 0 && lane == 0) : -1;
    zero_states(h[q]);
    if (slot[q] >= 0 && p.initial[r] != 0) load_slot(p, slot[q], l, h[q]);
    if (tb[q] < te[q]) load_row(tb[q], row[q]);
  }
#pragma unroll
  for (int q = 0; q < RQ; ++q) {
    for (int t = tb[q]; t < te[q]; ++t) {
      if (t > tb[q]) load_row(t, row[q]);
      float2 own = make_float2(0.f, 0.f);
      const float u = mine ? to_f(row[q].u) : 0.f;
      if (mine) {
        own.x = step_size(p, to_f(row[q].d) + bias);
        own.y = own.x * u;
      }
      float2 d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // channel j's lane: sum_channel is its own inverse on two bits
        const int src = l.dg * LN + sum_channel(j);
        d[j].x = __shfl_sync(0xffffffffu, own.x, src);
        d[j].y = __shfl_sync(0xffffffffu, own.y, src);
      }
      const Pack<T, 4>&b = row[q].b, &cc = row[q].c;
      float y[4];
      scan_step<true>(h[q], A2, d, make_float4(to_f(b.v[0]), to_f(b.v[1]), to_f(b.v[2]), to_f(b.v[3])),
                      make_float4(to_f(cc.v[0]), to_f(cc.v[1]), to_f(cc.v[2]), to_f(cc.v[3])), y);
      float o = sum_over_states<LN>(y, lane);
      if (mine) {
        o = fmaf(skip, u, o);
        if (zg != nullptr) o *= to_f(row[q].z) * sigmoid_exact(to_f(row[q].z));
        og[(long long)t * p.D + c] = from_f<T>(o);
      }
    }
    if (slot[q] >= 0) store_slot(p, slot[q], l, h[q]);
  }
  if (p.zero_rest && mine) {
    const T z = from_f<T>(0.f);
    if (blockIdx.y == 0)
      for (int t = 0; t < seq_start(p.q, 0); ++t) og[(long long)t * p.D + c] = z;
    if (blockIdx.y == gridDim.y - 1)
      for (int t = seq_start(p.q, p.q.nseq); t < p.q.T; ++t) og[(long long)t * p.D + c] = z;
  }
}

}  // namespace greta
