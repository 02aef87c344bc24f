// Backward of the selective scan (ssm_scan.cuh). With a = exp(dt A), and all
// products over one sequence:
//
//   dy[t]   = dout[t] SiLU(gate[t]),   dgate = dout y SiLU'(gate)
//   g[t, n] = C[t, n] dy[t] + a[t+1, n] g[t+1, n]        (adjoint of h[t, n])
//   dC[t,n] = sum_d dy h[t],           dB[t, n] = sum_d g dt u
//   du      = skip dy + dt sum_n g B
//   d(dt)   = sum_n g a h[t-1] A + u sum_n g B           (times softplus' = sigmoid)
//   dA      = sum_t g a h[t-1] dt,     dskip = sum_t dy u,  d(delta_bias) = sum_t d(delta)
//
// The forward left the states ahead of every 8th token. The main kernel walks
// its range's tiles of 8 tokens from the last to the first: it runs a tile's
// recurrence again from the saved state with the tile's states in registers,
// and goes back through them with g. So two exponentials and some thirteen fp32
// operations per (token, channel, state), 16 and 13 clocks a warp. A lane has
// two channels of four states: 8 x 8 states, and their rates, adjoints and
// sums, are what its registers hold (with four channels the saved states would
// be ahead of every 4th token). What bounds it is the issue of instructions and
// the shared memory beside them, so: two states of a channel share an
// instruction here (doubling dt, dt u and dy takes fewer moves than doubling B
// and C, and the sums over channels need no adding of halves), and the lanes'
// parts of dB and dC are not exchanged but stored, two vectors a token, and
// added for all of the CTA's channels at once. The CTA's warps take
// neighbouring channels of one group; its dB and dC go, one row per token, to
// `part_bc`; dA, dskip and d(delta_bias) of the range stay with the lane,
// added tile by tile to keep long sums short. Small kernels add the parts in a
// fixed order, so the same call gives the same bits.
//
// A range that ends inside a sequence needs a g of the next token: the carry
// kernel runs g alone over the part of each range up to the first sequence end
// in it, as the forward's does for h.
// 16288 tokens of nine sequences, 4096 x 16, bf16: carries 338 us, 1592 us, sums
// over CTAs and ranges 38 us. The main kernel has the shared memory 64 % busy
// (74 rows of 128 bytes a warp and token) and issues in 50 % of the slots, at
// three warps a scheduler: its registers leave room for no more.
#pragma once

#include "ssm_scan.cuh"

namespace greta {

constexpr int kBwdChans = 2;  // channels per lane of the backward kernel

// The sequences of a tile's tokens [ta, tb): bit r of `first`: token tile0 + r
// is the first of its sequence; of `live`: a sequence holds it. g: the segment
// of ta on return (its own on entry, when it reaches that far).
struct TileSeqs {
  unsigned first, live;
};
__device__ __forceinline__ TileSeqs tile_seqs(const SeqView& sv, int tile0, int ta, int tb, Seg& g) {
  TileSeqs s{0u, 0u};
  if (!(g.in && g.b <= ta && g.e >= tb)) g = sv.at(ta);
  Seg w = g;
  int t = ta;
  while (true) {
    const int stop = min(w.e, tb);
    if (w.in) {
      if (w.b == t) s.first |= 1u << (t - tile0);
      s.live |= tile_rows(tile0, t, stop);
    }
    t = stop;
    if (t >= tb) return s;
    w = sv.next(w);
  }
}

// The adjoint's carry at the end of range i, inside a sequence that goes on:
// a[t] g[t] of the next range's first token t, from the first range behind
// whose carry holds the sequence's end.
template <int LN, int KD>
__device__ __forceinline__ void carry_back(const ScanParams& p, const Lanes<LN, KD>& l, int i, const LaneStates<KD>& A2,
                                           LaneStates<KD>& r) {
  int j1 = p.R - 1;
  for (int lo = i + 1; lo < p.R; lo += 32) {
    const int k = lo + l.lane;
    const unsigned m = __ballot_sync(0xffffffffu, k < p.R && p.reset[k] != 0);
    if (m != 0) {
      j1 = lo + __ffs(m) - 1;
      break;
    }
  }
  carry_through(p, l, j1, i + 1, -1, A2, r);
}

// dy of a tile into shared memory.
template <typename T, int LN, int KD>
__device__ __forceinline__ void stage_dy(const ScanParams& p, const Lanes<LN, KD>& l, const T* g, const T* z,
                                         float* dy) {
  constexpr int CHW = Lanes<LN, KD>::CHW;
  using SV = StepVecs<CHW>;
  constexpr int V = SV::V;
#pragma unroll
  for (int k = 0; k < SV::NVEC; ++k) {
    if (!SV::has(k, l.lane)) continue;
    const int at = SV::row(k, l.lane) * CHW + SV::chan(l.lane);
    const Pack<T, V> gv = load_part<T, V>(g + at, V, true);
    Pack<T, V> zv;
    if (p.gate != nullptr) zv = load_part<T, V>(z + at, V, true);
    Pack<float, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      o.v[e] = to_f(gv.v[e]);
      if (p.gate != nullptr) o.v[e] *= to_f(zv.v[e]) * sigmoid_t<T>(to_f(zv.v[e]));
    }
    store_part<float, V>(dy + at, o, V, true);
  }
}

// KD channels' dy as pairs.
template <int KD>
__device__ __forceinline__ void read_dy(const float* dy, f2 (&o)[KD / 2]) {
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) o[j] = reinterpret_cast<const f2*>(dy)[j];
}

// g alone over the head of each range that begins inside a sequence.
template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32, 4) ssm_scan_bwd_carry_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  constexpr int KD = kFwdChans;
  using L = Lanes<LN, KD>;
  using S = FwdSmem<T, LN, KD>;  // the forward's parts: (dt, -), dy; dout, delta, gate, (B, C)
  constexpr int CHW = L::CHW, NP = L::NP;
  using TV = TileVecs<CHW>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* mine = reinterpret_cast<char*>(smem4) + warp * S::kWarp;
  float4* dl = reinterpret_cast<float4*>(mine);
  float* dy = reinterpret_cast<float*>(mine + S::kDl);
  auto stage = [&](int s, int part) {
    return reinterpret_cast<T*>(mine + S::kDl + S::kY + s * S::kStage + part * S::kRow);
  };
  pdl_wait();
  pdl_trigger();
  const int slice = blockIdx.x * (blockDim.x >> 5) + warp;
  if (slice >= p.F * p.spg) return;
  const L l(p, slice, lane);
  const int ri = blockIdx.y;
  if (ri == 0) return;
  const SeqView sv(p.q, lane);
  const Ranges ranges(sv, p.L, p.whole_limit);
  if (ranges.whole) return;  // no range needs a carry
  const int t0 = ranges.begin(sv, ri);
  int t1 = ranges.begin(sv, ri + 1);
  if (t0 >= t1) return;
  const Seg g = sv.at(t0);
  if (!g.in || g.b >= t0) return;
  const bool reset = g.e <= t1;
  if (slice == 0 && lane == 0) p.reset[ri] = reset;
  t1 = min(t1, g.e);
  LaneStates<KD> A2, r;
  load_rates(p, l, A2);
  zero_states<KD>(r);
  using SV = StepVecs<CHW>;
  float bias[SV::V];
  load_column<SV::V>(p.dbias, l.c0 + SV::chan(lane), l.nch - SV::chan(lane), bias);
  f2 dsum[KD / 2];
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) dsum[j] = 0ull;
  int cur = 0;
  const T* bc;
  const bool reg = regular(p, l);
  const T* g0 = lane_row<T>(p.dout, p.D, l);
  const T* d0 = lane_row<T>(p.delta, p.ldd, l);
  const T* z0 = lane_row<T>(p.gate, p.ldg, l);
  auto fetch = [&](int tile0, int s) {
    if (reg && tile0 >= t0 && tile0 + kTile <= t1) {
      copy_whole(g0, p.D, l, tile0, stage(s, 0));
      copy_whole(d0, p.ldd, l, tile0, stage(s, 1));
      if (p.gate != nullptr) copy_whole(z0, p.ldg, l, tile0, stage(s, 2));
      copy_whole_bc<T>(p, l, tile0, stage(s, 3), lane, 32);
    } else {
      const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
      copy_tile<T>(p.dout, p.D, p.vec, l, tile0, ta, tb, stage(s, 0));
      copy_tile<T>(p.delta, p.ldd, p.vec, l, tile0, ta, tb, stage(s, 1));
      if (p.gate != nullptr) copy_tile<T>(p.gate, p.ldg, p.vec, l, tile0, ta, tb, stage(s, 2));
      copy_bc<T>(p, l, tile0, ta, tb, stage(s, 3), lane, 32);
    }
    copy_commit();
  };
  if (p.N < NP) {  // states past N: B and C of both stages zero for good
    for (int i = lane; i < kTile * 2 * NP; i += 32) stage(0, 3)[i] = stage(1, 3)[i] = from_f<T>(0.f);
    __syncwarp();
  }
  auto step = [&](int i) {
    ulonglong2 d[KD / 2];
    f2 c[4], y[KD / 2];
    read_steps<KD>(dl, i * CHW + l.ch(0), d);
    twice(read_four(bc + (i * 2 + 1) * NP + l.n0()), c);
    read_dy<KD>(dy + i * CHW + l.ch(0), y);
#pragma unroll
    for (int j = 0; j < KD / 2; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r[j][k] = f2_mul(f2_decay(d[j].x, A2[j][k]), f2_fma(c[k], y[j], r[j][k]));
      dsum[j] = f2_add(dsum[j], d[j].x);
    }
  };
  const int last = (t1 - 1) / kTile * kTile;
  fetch(last, 0);
  for (int tile0 = last; tile0 + kTile > t0; tile0 -= kTile, cur ^= 1) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    copy_wait();
    __syncwarp();
    bc = stage(cur, 3);
    stage_steps<T>(p, l, stage(cur, 0), stage(cur, 1), bias, dl);
    stage_dy<T>(p, l, stage(cur, 0), stage(cur, 2), dy);
    __syncwarp();
    if (tile0 > t0) fetch(tile0 - kTile, cur ^ 1);
    if (tb - ta == kTile) {
#pragma unroll
      for (int i = kTile - 1; i >= 0; --i) step(i);
    } else {
      for (int i = tb - 1 - tile0; i >= ta - tile0; --i) step(i);
    }
    __syncwarp();
  }
  store_states(p.carry + ri * (long long)p.D * p.N, l, p.N, r);
  if (l.nq == 0) store_sums(p, l, ri, dsum);
}

// Shared memory of the backward, in bytes: of a warp, and what the CTA shares.
template <typename T, int LN>
struct BwdSmem {
  static constexpr int CHW = Lanes<LN, kBwdChans>::CHW, NP = Lanes<LN, kBwdChans>::NP, V = TileVecs<CHW>::V;
  static constexpr int kRow = kTile * CHW * (int)sizeof(T);  // a tile of an operand
  static constexpr int kRowF = kTile * CHW * 4;
  // fp32: dy, slopes and dout SiLU' take the places of dout, delta and gate, whose
  // values they are made of (with places of their own a third CTA had no room)
  static constexpr bool kInPlace = sizeof(T) == 4;
  static constexpr int kDl = 0;                       // (dt, dt u)
  static constexpr int kDy = kDl + 2 * kRowF;         // dy
  static constexpr int kSlope = kDy + (kInPlace ? 0 : kRowF);  // d(dt) / d(raw step)
  static constexpr int kGk = kSlope + (kInPlace ? 0 : kRowF);  // dout SiLU'(gate)
  static constexpr int kY = kGk + (kInPlace ? 0 : kRowF);      // sum C h
  static constexpr int kPair = kY + kRowF;            // (sum kept A2, sum g B)
  static constexpr int kCols = kPair + 2 * kRowF;     // [bias | skip][CHW]; 16-bit types: a copy per lane (1606 us, not 1623)
  static constexpr int kColBytes = kInPlace ? (CHW * 4 + 15) / 16 * 16 : 32 * V * 4;
  static constexpr int kSum = kCols + 2 * kColBytes;  // [dskip | d(delta_bias)][lane] V floats
  static constexpr int kPart = kSum + 2 * 32 * V * 4;  // [token][dB | dC][lane] float4
  static constexpr int kStage0 = kPart + kTile * 2 * 32 * 16;
  static constexpr int kStage = 4 * kRow + 32 * kBwdChans * 16;  // u, delta, gate, dout; saved states
  static constexpr int kWarp = kStage0 + 2 * kStage;
  static constexpr int kBC = kTile * 2 * NP * (int)sizeof(T);
  static constexpr int kWide = sizeof(T) == 4 ? 0 : kTile * 2 * NP * 4;  // B and C in fp32
  static constexpr int kTotal = kScanWarps * kWarp + 2 * kBC + kWide;
};

// Four states of B or C, as pairs of states.
__device__ __forceinline__ void read_pairs(const float* s, f2 (&o)[2]) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(s);
  o[0] = v.x;
  o[1] = v.y;
}

// Pairs of channels to pairs of states.
__device__ __forceinline__ void by_states(const f2 (&h)[4], f2 (&o)[2][2]) {
  float4 a, b;
  unpack_pair(h, a, b);
  o[0][0] = pack2(a.x, a.y);
  o[0][1] = pack2(a.z, a.w);
  o[1][0] = pack2(b.x, b.y);
  o[1][1] = pack2(b.z, b.w);
}

template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32, 3) ssm_scan_bwd_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  constexpr int KD = kBwdChans;
  using L = Lanes<LN, KD>;
  using S = BwdSmem<T, LN>;
  constexpr int CHW = L::CHW, NP = L::NP;
  using TV = TileVecs<CHW>;
  constexpr int V = TV::V;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  char* base = reinterpret_cast<char*>(smem4);
  char* mine = base + 2 * S::kBC + warp * S::kWarp;
  float4* dl = reinterpret_cast<float4*>(mine + S::kDl);
  float* ys = reinterpret_cast<float*>(mine + S::kY);
  float2* pair = reinterpret_cast<float2*>(mine + S::kPair);
  float* cols = reinterpret_cast<float*>(mine + S::kCols) + (S::kInPlace ? TV::chan(lane) : lane * V);
  float* sums = reinterpret_cast<float*>(mine + S::kSum) + lane * V;
  float4* part = reinterpret_cast<float4*>(mine + S::kPart) + lane;
  auto stage = [&](int s, int op) {  // u, delta, gate, dout
    return reinterpret_cast<T*>(mine + S::kStage0 + s * S::kStage + op * S::kRow);
  };
  auto saved = [&](int s) {  // [channel][lane]
    return reinterpret_cast<float4*>(mine + S::kStage0 + s * S::kStage + 4 * S::kRow) + lane;
  };
  pdl_wait();
  pdl_trigger();
  const int bpg = (p.spg + kScanWarps - 1) / kScanWarps;  // CTAs per group
  const int block = p.b0 + blockIdx.x;
  const int f = block / bpg, in_group = block % bpg * kScanWarps + warp;
  const bool have = in_group < p.spg;  // else a warp without channels, which only keeps the CTA's steps
  L l(p, f * p.spg + (have ? in_group : 0), lane);
  if (!have) l.nch = 0;
  const int ri = blockIdx.y;
  const SeqView sv(p.q, lane);
  const Ranges ranges(sv, p.L, p.whole_limit);
  const int t0 = ranges.begin(sv, ri);
  const int t1 = ri + 1 < p.R ? ranges.begin(sv, ri + 1) : p.q.T;
  const long long DN = (long long)p.D * p.N;
  f2 A2[KD][2], dA[KD][2], rr[KD][2];
  {
    LaneStates<KD> a, r;
    load_rates(p, l, a);
    zero_states<KD>(r);
    if (t0 < t1 && t1 < p.q.T) {
      const Seg g = sv.at(t1);
      if (g.in && g.b < t1) carry_back(p, l, ri, a, r);
    }
    by_states(a[0], A2);
    by_states(r[0], rr);
  }
#pragma unroll
  for (int j = 0; j < KD; ++j) dA[j][0] = dA[j][1] = 0ull;
  {
    float v[V];
    load_column<V>(p.dbias, l.c0 + TV::chan(lane), l.nch - TV::chan(lane), v);
#pragma unroll
    for (int e = 0; e < V; ++e) cols[e] = v[e];
    load_column<V>(p.skip, l.c0 + TV::chan(lane), l.nch - TV::chan(lane), v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      cols[S::kColBytes / 4 + e] = v[e];
      sums[e] = sums[32 * V + e] = 0.f;
    }
  }
  Seg g{-1, 0, 0, false};

  const bool reg = regular(p, l) && p.N % 4 == 0;
  const T* u0 = lane_row<T>(p.u, p.ldu, l);
  const T* d0 = lane_row<T>(p.delta, p.ldd, l);
  const T* z0 = lane_row<T>(p.gate, p.ldg, l);
  const T* g0 = lane_row<T>(p.dout, p.D, l);
  const float* h0 = p.ckpt + (long long)(l.c0 + l.ch(0)) * p.N + l.n0();
  auto fetch = [&](int tile0, int s) {
    T* bcs = reinterpret_cast<T*>(base + s * S::kBC);
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    // (a range that begins inside a tile begins there with a sequence, or
    // outside, and does not use the states saved ahead of the tile)
    if (reg && tb - ta == kTile) {
      copy_whole(u0, p.ldu, l, tile0, stage(s, 0));
      copy_whole(d0, p.ldd, l, tile0, stage(s, 1));
      if (p.gate != nullptr) copy_whole(z0, p.ldg, l, tile0, stage(s, 2));
      copy_whole(g0, p.D, l, tile0, stage(s, 3));
      if (l.n0() < p.N) {
        const float* c = h0 + (tile0 / kTile) * DN;
#pragma unroll
        for (int j = 0; j < KD; ++j) copy_async<16>(saved(s) + j * 32, c + j * p.N, true);
      }
    } else {
      copy_tile<T>(p.u, p.ldu, p.vec, l, tile0, ta, tb, stage(s, 0));
      copy_tile<T>(p.delta, p.ldd, p.vec, l, tile0, ta, tb, stage(s, 1));
      if (p.gate != nullptr) copy_tile<T>(p.gate, p.ldg, p.vec, l, tile0, ta, tb, stage(s, 2));
      copy_tile<T>(p.dout, p.D, p.vec, l, tile0, ta, tb, stage(s, 3));
      const float* c = p.ckpt + (tile0 / kTile) * DN;
#pragma unroll
      for (int j = 0; j < KD; ++j)
        copy_part<float, 4>(reinterpret_cast<float*>(saved(s) + j * 32),
                            c + (long long)(l.c0 + l.ch(j)) * p.N + l.n0(), p.ckpt,
                            l.ch(j) < l.nch ? p.N - l.n0() : 0, p.N % 4 == 0);
    }
    if (p.vec_bc && tb - ta == kTile)
      copy_whole_bc<T>(p, l, tile0, bcs, threadIdx.x, kScanWarps * 32);
    else
      copy_bc<T>(p, l, tile0, ta, tb, bcs, threadIdx.x, kScanWarps * 32);
    copy_commit();
  };
  if (p.N < NP) {  // states past N: B, C and saved states of both stages zero for good
    for (int i = threadIdx.x; i < 2 * kTile * 2 * NP; i += kScanWarps * 32) reinterpret_cast<T*>(base)[i] = from_f<T>(0.f);
#pragma unroll
    for (int j = 0; j < 2 * KD; ++j) saved(j / KD)[j % KD * 32] = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
  }
  const int last = t1 > t0 ? (t1 - 1) / kTile * kTile : -kTile;
  if (last >= 0) fetch(last, 0);
  int cur = 0;
  for (int tile0 = last; tile0 + kTile > t0 && tile0 >= 0; tile0 -= kTile, cur ^= 1) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    const TileSeqs q = tile_seqs(sv, tile0, ta, tb, g);
    copy_wait();
    float* dys = S::kInPlace ? reinterpret_cast<float*>(stage(cur, 3)) : reinterpret_cast<float*>(mine + S::kDy);
    float* slope = S::kInPlace ? reinterpret_cast<float*>(stage(cur, 1)) : reinterpret_cast<float*>(mine + S::kSlope);
    float* gk = S::kInPlace ? reinterpret_cast<float*>(stage(cur, 2)) : reinterpret_cast<float*>(mine + S::kGk);
    // B and C widened once for the CTA (each thread what it copied itself)
    const float* bc = reinterpret_cast<const float*>(base + cur * S::kBC);
    if (sizeof(T) != 4) {
      float* wide = reinterpret_cast<float*>(base + 2 * S::kBC + kScanWarps * S::kWarp);
      const T* bcs = reinterpret_cast<const T*>(base + cur * S::kBC);
#pragma unroll
      for (int i = threadIdx.x; i < kTile * 2 * LN; i += kScanWarps * 32)
        *reinterpret_cast<float4*>(wide + i * 4) = widen4(read_four(bcs + i * 4));
      bc = wide;
    }
    f2 hs[kTile + 1][KD][2];
#pragma unroll
    for (int j = 0; j < KD; ++j) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(saved(cur) + j * 32);
      hs[0][j][0] = v.x;
      hs[0][j][1] = v.y;
    }
    // per token and channel: (dt, dt u), the step's slope, dy and dout SiLU'
#pragma unroll
    for (int k = 0; k < TV::NVEC; ++k) {
      if (!TV::has(k, lane)) continue;
      const int r = TV::row(k, lane), c = TV::chan(lane), at = r * CHW + c;
      const bool in = (q.live >> r) & 1;
      const Pack<T, V> u = tile_vec<T, CHW>(stage(cur, 0), k, lane), d = tile_vec<T, CHW>(stage(cur, 1), k, lane),
                       go = tile_vec<T, CHW>(stage(cur, 3), k, lane);
      const Pack<float, V> bias = load_part<float, V>(cols, V, true);
      Pack<float, V> sl, dy, gs;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float x0 = to_f(d.v[e]) + bias.v[e], x1 = to_f(d.v[e + 1]) + bias.v[e + 1];
        f2 s = pack2(x0, x1), ex;
        sl.v[e] = sl.v[e + 1] = 1.f;
        if (p.softplus) {
          s = softplus2(x0, x1, ex);
          float e0, e1;
          unpack2(ex, e0, e1);
          sl.v[e] = softplus_slope(x0, e0);
          sl.v[e + 1] = softplus_slope(x1, e1);
        }
        const f2 su = f2_mul(s, pack2(to_f(u.v[e]), to_f(u.v[e + 1])));
        float4 o;
        unpack2(s, o.x, o.y);
        unpack2(su, o.z, o.w);
        if (!in) o = make_float4(0.f, 0.f, 0.f, 0.f);
        dl[step_slot((at + e) / 2)] = o;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) dy.v[e] = to_f(go.v[e]);
      if (p.gate != nullptr) {
        const Pack<T, V> z = tile_vec<T, CHW>(stage(cur, 2), k, lane);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float zv = to_f(z.v[e]), sg = sigmoid_t<T>(zv), gsg = dy.v[e] * sg;
          gs.v[e] = gsg * fmaf(zv, 1.f - sg, 1.f);
          dy.v[e] = gsg * zv;
        }
        store_part<float, V>(gk + at, gs, V, true);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) dy.v[e] = in ? dy.v[e] : 0.f;
      store_part<float, V>(slope + at, sl, V, true);
      store_part<float, V>(dys + at, dy, V, true);
    }
    __syncthreads();
    if (tile0 > t0) fetch(tile0 - kTile, cur ^ 1);

    // The tile's states, as the forward computed them; rows that no sequence of
    // the range holds (dt = dy = 0) pass states and adjoints on, and what they
    // give is not used. `general`: the tile has such rows, or first tokens.
    auto forward = [&](auto general) {
#pragma unroll
      for (int r = 0; r < kTile; ++r) {
        const float4 dv = dl[step_slot((r * CHW + l.ch(0)) / 2)];
        const float dt[KD] = {dv.x, dv.y}, du[KD] = {dv.z, dv.w};
        f2 b[2], c[2];
        float y[KD];
        read_pairs(bc + r * 2 * NP + l.n0(), b);
        if (p.gate != nullptr) read_pairs(bc + (r * 2 + 1) * NP + l.n0(), c);
        const bool first = decltype(general)::value && ((q.first >> r) & 1);
#pragma unroll
        for (int j = 0; j < KD; ++j) {
          const f2 d2 = pack2(dt[j], dt[j]), du2 = pack2(du[j], du[j]);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            hs[r + 1][j][k] = f2_fma(f2_decay(d2, A2[j][k]), first ? 0ull : hs[r][j][k], f2_mul(du2, b[k]));
          if (p.gate != nullptr) y[j] = f2_sum(f2_fma(c[1], hs[r + 1][j][1], f2_mul(c[0], hs[r + 1][j][0])));
        }
        if (p.gate != nullptr) {
          const f2 yp[1] = {pack2(y[0], y[1])};
          const float s = sum_over_states<LN>(yp, lane);
          if (l.nq < KD) ys[r * CHW + l.ch(sum_channel<KD>(lane))] = s;
        }
      }
    };
    // the exponentials are taken again: kept from the first pass they would need
    // 64 more registers
    auto again = [&] {
#pragma unroll
      for (int j = 0; j < KD; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) asm volatile("" : "+l"(A2[j][k])::"memory");
    };
    // back through them
    f2 dAt[KD][2];
#pragma unroll
    for (int j = 0; j < KD; ++j) dAt[j][0] = dAt[j][1] = 0ull;
    auto backward = [&](auto general) {
#pragma unroll
      for (int r = kTile - 1; r >= 0; --r) {
        const bool first = decltype(general)::value && ((q.first >> r) & 1);
        const bool none = decltype(general)::value && !((q.live >> r) & 1);
        const float4 dv = dl[step_slot((r * CHW + l.ch(0)) / 2)];
        const float2 dyv = *reinterpret_cast<const float2*>(dys + r * CHW + l.ch(0));
        const float dt[KD] = {dv.x, dv.y}, du[KD] = {dv.z, dv.w}, dy[KD] = {dyv.x, dyv.y};
        f2 b[2], c[2], dB[2], dC[2];
        float sa[KD], gb[KD];
        read_pairs(bc + r * 2 * NP + l.n0(), b);
        read_pairs(bc + (r * 2 + 1) * NP + l.n0(), c);
#pragma unroll
        for (int j = 0; j < KD; ++j) {
          const f2 d2 = pack2(dt[j], dt[j]), du2 = pack2(du[j], du[j]), y2 = pack2(dy[j], dy[j]);
          f2 s2 = 0ull, g2 = 0ull;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const f2 a = f2_decay(d2, A2[j][k]);
            const f2 gg = f2_fma(c[k], y2, rr[j][k]);
            const f2 ag = first ? 0ull : f2_mul(a, gg);
            // (what is ahead of a first token is another sequence's, maybe NaN)
            const f2 kept = none ? 0ull : f2_mul(ag, first ? 0ull : hs[r][j][k]);
            s2 = k == 0 ? f2_mul(kept, A2[j][k]) : f2_fma(kept, A2[j][k], s2);
            g2 = k == 0 ? f2_mul(gg, b[k]) : f2_fma(gg, b[k], g2);
            dAt[j][k] = f2_fma(kept, d2, dAt[j][k]);
            dB[k] = j == 0 ? f2_mul(gg, du2) : f2_fma(gg, du2, dB[k]);
            dC[k] = j == 0 ? f2_mul(y2, hs[r + 1][j][k]) : f2_fma(y2, hs[r + 1][j][k], dC[k]);
            rr[j][k] = none ? rr[j][k] : ag;
          }
          sa[j] = f2_sum(s2);
          gb[j] = f2_sum(g2);
        }
        const f2 sp[1] = {pack2(sa[0], sa[1])}, gp[1] = {pack2(gb[0], gb[1])};
        const float2 s = make_float2(sum_over_states<LN>(sp, lane), sum_over_states<LN>(gp, lane));
        if (l.nq < KD) pair[r * CHW + l.ch(sum_channel<KD>(lane))] = s;
        reinterpret_cast<ulonglong2*>(part)[(r * 2) * 32] = make_ulonglong2(dB[0], dB[1]);
        reinterpret_cast<ulonglong2*>(part)[(r * 2 + 1) * 32] = make_ulonglong2(dC[0], dC[1]);
      }
    };
    if (q.first == 0 && q.live == (1u << kTile) - 1) {
      forward(std::false_type());
      again();
      backward(std::false_type());
    } else {
      forward(std::true_type());
      again();
      backward(std::true_type());
    }
#pragma unroll
    for (int j = 0; j < KD; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) dA[j][k] = f2_add(dA[j][k], dAt[j][k]);
    __syncthreads();
    // the tile's gradients by token and channel
#pragma unroll
    for (int k = 0; k < TV::NVEC; ++k) {
      const int r = TV::row(k, lane), c = TV::chan(lane), t = tile0 + r, n = l.nch - c, at = r * CHW + c;
      if (!TV::has(k, lane) || t < ta || t >= tb || n <= 0) continue;
      const bool vec = p.vec && n >= V, in = (q.live >> r) & 1;
      const Pack<T, V> u = tile_vec<T, CHW>(stage(cur, 0), k, lane);
      const Pack<float, V> sl = load_part<float, V>(slope + at, V, true), dy = load_part<float, V>(dys + at, V, true),
                           skip = load_part<float, V>(cols + S::kColBytes / 4, V, true);
      const Pack<float, 2 * V> sp = load_part<float, 2 * V>(reinterpret_cast<const float*>(pair + at), 2 * V, true);
      Pack<float, V> s0 = load_part<float, V>(sums, V, true), s1 = load_part<float, V>(sums + 32 * V, V, true);
      Pack<T, V> du, dd, dz;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float4 st = dl[step_slot((at + e) / 2)];
        const float uv = to_f(u.v[e]), dt = e % 2 == 0 ? st.x : st.y, sa = sp.v[2 * e], gb = sp.v[2 * e + 1];
        const float ddt = fmaf(kLn2, sa, uv * gb) * sl.v[e];
        du.v[e] = from_f<T>(in ? fmaf(dt, gb, skip.v[e] * dy.v[e]) : 0.f);
        dd.v[e] = from_f<T>(in ? ddt : 0.f);
        s0.v[e] = in ? fmaf(dy.v[e], uv, s0.v[e]) : s0.v[e];
        s1.v[e] = in ? s1.v[e] + ddt : s1.v[e];
      }
      store_part<float, V>(sums, s0, V, true);
      store_part<float, V>(sums + 32 * V, s1, V, true);
      const long long o = (long long)t * p.D + l.c0 + c;
      store_part<T, V>(reinterpret_cast<T*>(p.du) + o, du, n, vec);
      store_part<T, V>(reinterpret_cast<T*>(p.ddelta) + o, dd, n, vec);
      if (p.gate != nullptr) {
        const Pack<float, V> y = load_part<float, V>(ys + at, V, true), gs = load_part<float, V>(gk + at, V, true);
#pragma unroll
        for (int e = 0; e < V; ++e)
          dz.v[e] = from_f<T>(in ? gs.v[e] * fmaf(skip.v[e], to_f(u.v[e]), y.v[e]) : 0.f);
        store_part<T, V>(reinterpret_cast<T*>(p.dgate) + o, dz, n, vec);
      }
    }
    // dB and dC of the CTA's channels: four states of a token's dB or dC per
    // item, `PER` threads for one, each adding every PER-th channel group of all
    // warps (the next tile's parts are written behind its own barrier; a warp
    // without channels has zeros)
    constexpr int ITEMS = kTile * 2 * LN;
    constexpr int PER = ITEMS >= kScanWarps * 32 ? 1 : kScanWarps * 32 / ITEMS;
    constexpr int GROUPS = 32 / LN;
    static_assert(PER <= 2 && GROUPS % PER == 0, "a thread pair per item at most");
    float* out = p.part_bc + ((long long)blockIdx.x * p.q.T + tile0) * 2 * p.N;
#pragma unroll
    for (int i0 = 0; i0 < ITEMS * PER; i0 += kScanWarps * 32) {
      const int i = i0 + threadIdx.x, nq = i % LN, sub = i / LN % PER, item = i / (LN * PER), r = item / 2, k = item % 2;
      f2 s0 = 0ull, s1 = 0ull;
#pragma unroll
      for (int w = 0; w < kScanWarps; ++w) {
        const ulonglong2* b = reinterpret_cast<const ulonglong2*>(base + 2 * S::kBC + w * S::kWarp + S::kPart);
#pragma unroll
        for (int dg = 0; dg < GROUPS; dg += PER) {
          const ulonglong2 v = b[(r * 2 + k) * 32 + (dg + sub) * LN + nq];
          s0 = f2_add(s0, v.x);
          s1 = f2_add(s1, v.y);
        }
      }
      if (PER == 2) {
        s0 = f2_add(s0, __shfl_xor_sync(0xffffffffu, s0, LN));
        s1 = f2_add(s1, __shfl_xor_sync(0xffffffffu, s1, LN));
      }
      float4 v;
      unpack2(s0, v.x, v.y);
      unpack2(s1, v.z, v.w);
      if (!((q.live >> r) & 1)) v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (sub == 0 && r >= ta - tile0 && r < tb - tile0)
        store_four(out + (r * 2 + k) * p.N + nq * 4, 1, p.N - nq * 4, p.N % 4 == 0, v);
    }
  }
  if (!have) return;
#pragma unroll
  for (int j = 0; j < KD; ++j) {
    float4 v;
    unpack2(dA[j][0], v.x, v.y);
    unpack2(dA[j][1], v.z, v.w);
    store_four(p.part_a + ri * DN + (long long)(l.c0 + l.ch(j)) * p.N + l.n0(), 1, l.ch(j) < l.nch ? p.N - l.n0() : 0,
               p.N % 4 == 0, v);
  }
  // lanes of one vector column: the same lane % VPR
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float2 s = make_float2(sums[e], sums[32 * V + e]);
#pragma unroll
    for (int o = TV::VPR; o < 32; o <<= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    const int c = TV::chan(lane) + e;
    if (lane < TV::VPR && c < l.nch) {
      p.part_d[(long long)ri * 2 * p.D + l.c0 + c] = s.x;
      p.part_d[(long long)ri * 2 * p.D + p.D + l.c0 + c] = s.y;
    }
  }
}

// dB[t, f, n], dC[t, f, n] = sums over the CTAs of group f, of which a launch of the
// main kernel left blocks [lo, hi); a group's sums over the launches before are
// in `acc` [F][T][2][N]. One addition after the other, so the launches make no
// difference to the bits. (A loop over the groups in here takes 57 us instead of
// 27 with one of them.)
template <typename T>
__global__ void __launch_bounds__(256) ssm_scan_reduce_bc_kernel(const float* part, float* acc, T* dB, T* dC, int bpg,
                                                                 int lo, int hi, int T_, int N, int F, int f0) {
  pdl_wait();
  pdl_trigger();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x, per = (long long)T_ * 2 * N;
  const int f = f0 + blockIdx.y;
  if (i >= per) return;
  const int b0 = max(lo - f * bpg, 0), b1 = min(hi - f * bpg, bpg);
  const float* s = part + ((long long)f * bpg - lo) * per + i;
  float v = b0 > 0 ? acc[f * per + i] : 0.f;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) v += s[b * per];
  if (b1 < bpg) {
    acc[f * per + i] = v;
    return;
  }
  const long long t = i / (2 * N);
  const int k = (int)(i / N % 2), n = (int)(i % N);
  (k == 0 ? dB : dC)[(t * F + f) * N + n] = from_f<T>(v);
}

// dA, dskip, d(delta_bias) = sums over the ranges (fp32).
template <int V>
__global__ void __launch_bounds__(256) ssm_scan_reduce_a_kernel(const float* part_a, const float* part_d, float* dA,
                                                                float* dskip, float* dbias, int R, int D, int N) {
  pdl_wait();
  pdl_trigger();
  const long long DN = (long long)D * N, i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= DN + 2 * D) return;
  const float* s = i < DN ? part_a + i : part_d + (i - DN);
  const long long step = i < DN ? DN : 2 * D;
  float v = 0.f;
#pragma unroll V
  for (int r = 0; r < R; ++r) v += s[r * step];
  if (i < DN)
    dA[i] = v;
  else if (i < DN + D) {
    if (dskip != nullptr) dskip[i - DN] = v;
  } else if (dbias != nullptr)
    dbias[i - DN - D] = v;
}

}  // namespace greta
