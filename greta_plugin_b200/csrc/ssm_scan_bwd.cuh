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
// operations per (token, channel, state): 16 and 14 clocks a warp, both pipes
// about equally full, and as many issue slots again for the sums over states
// and channels. A lane has two channels of four states: 8 x 8 states, and
// their rates, adjoints and sums, are what its registers hold (with four
// channels the saved states would be ahead of every 4th token). The
// CTA's warps take neighbouring channels of one group; their parts of dB
// and dC are added in shared memory and go, one row per token and CTA, to
// `part_bc`; dA, dskip and d(delta_bias) of the range stay with the lane,
// added tile by tile to keep long sums short. Small kernels add the parts in a
// fixed order, so the same call gives the same bits.
//
// A range that ends inside a sequence needs a g of the next token: the carry
// kernel runs g alone over the part of each range up to the first sequence end
// in it, as the forward's does for h.
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
__device__ __forceinline__ TileSeqs tile_seqs(const Seqs& q, int tile0, int ta, int tb, int lane, Seg& g) {
  TileSeqs s{0u, 0u};
  if (!(g.in && g.b <= ta && g.e >= tb)) g = seg_at(q, ta, lane);
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
    w = seg_next(q, w);
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

// dy of a tile into shared memory (zeros in rows without their bit).
template <typename T, int LN, int KD>
__device__ __forceinline__ void stage_dy(const ScanParams& p, const Lanes<LN, KD>& l, const T* g, const T* z,
                                         unsigned rows, float* dy) {
  constexpr int CHW = Lanes<LN, KD>::CHW;
  using TV = TileVecs<CHW>;
  constexpr int V = TV::V;
#pragma unroll
  for (int k = 0; k < TV::NVEC; ++k) {
    if (!TV::has(k, l.lane)) continue;
    const int r = TV::row(k, l.lane);
    const Pack<T, V> gv = tile_vec<T, CHW>(g, k, l.lane);
    Pack<T, V> zv;
    if (p.gate != nullptr) zv = tile_vec<T, CHW>(z, k, l.lane);
    Pack<float, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v = to_f(gv.v[e]);
      if (p.gate != nullptr) v *= to_f(zv.v[e]) * sigmoid_t<T>(to_f(zv.v[e]));
      o.v[e] = (rows >> r) & 1 ? v : 0.f;
    }
    store_part<float, V>(dy + r * CHW + TV::chan(l.lane), o, V, true);
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
  const int t0 = range_begin(p.q, ri, p.R, p.L, lane);
  int t1 = range_begin(p.q, ri + 1, p.R, p.L, lane);
  if (t0 >= t1) return;
  const Seg g = seg_at(p.q, t0, lane);
  if (!g.in || g.b >= t0) return;
  const bool reset = g.e <= t1;
  if (slice == 0 && lane == 0) p.reset[ri] = reset;
  t1 = min(t1, g.e);
  LaneStates<KD> A2, r;
  load_rates(p, l, A2);
  zero_states<KD>(r);
  float bias[TV::V];
  load_column<TV::V>(p.dbias, l.c0 + TV::chan(lane), l.nch - TV::chan(lane), bias);
  f2 dsum[KD / 2];
#pragma unroll
  for (int j = 0; j < KD / 2; ++j) dsum[j] = 0ull;
  int cur = 0;
  const T* bc;
  auto fetch = [&](int tile0, int s) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    copy_tile<T>(p.dout, p.D, p.vec, l, tile0, ta, tb, stage(s, 0));
    copy_tile<T>(p.delta, p.ldd, p.vec, l, tile0, ta, tb, stage(s, 1));
    if (p.gate != nullptr) copy_tile<T>(p.gate, p.ldg, p.vec, l, tile0, ta, tb, stage(s, 2));
    copy_bc<T>(p, l, tile0, ta, tb, stage(s, 3), lane, 32);
    copy_commit();
  };
  auto step = [&](int i) {
    ulonglong2 d[KD / 2];
    f2 c[4], y[KD / 2];
    read_steps<KD>(dl, i * CHW + l.ch(0), d);
    read_four(bc + (i * 2 + 1) * NP + l.n0(), c);
    read_dy<KD>(dy + i * CHW + l.ch(0), y);
#pragma unroll
    for (int j = 0; j < KD / 2; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r[j][k] = f2_mul(f2_ex2(f2_mul(d[j].x, A2[j][k])), f2_fma(c[k], y[j], r[j][k]));
      dsum[j] = f2_add(dsum[j], d[j].x);
    }
  };
  const int last = (t1 - 1) / kTile * kTile;
  fetch(last, 0);
  for (int tile0 = last; tile0 + kTile > t0; tile0 -= kTile, cur ^= 1) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    copy_wait();
    bc = stage(cur, 3);
    const unsigned rows = tile_rows(tile0, ta, tb);
    stage_steps<T>(p, l, rows, stage(cur, 0), stage(cur, 1), bias, dl);
    stage_dy<T>(p, l, stage(cur, 0), stage(cur, 2), rows, dy);
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

// The eight values of a lane summed over the channel groups of the warp (lane
// bits LN, 2 LN, .. 16): halves are exchanged while there are some, so that
// M = LN / 4 values, from index `base`, stay with a lane.
template <int LN>
__device__ __forceinline__ void sum_over_channels(float (&v)[8], int lane, int& base) {
  base = 0;
  int m = 8;
#pragma unroll
  for (int o = LN; o < 32; o <<= 1) {
    const bool hi = lane & o;
    m >>= 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < m) {
        const float send = hi ? v[i] : v[m + i], keep = hi ? v[m + i] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
    }
    if (hi) base += m;
  }
}

// Shared memory of the backward, in bytes: of a warp, and what the CTA shares.
template <typename T, int LN>
struct BwdSmem {
  static constexpr int CHW = Lanes<LN, kBwdChans>::CHW, NP = Lanes<LN, kBwdChans>::NP;
  static constexpr int kDl = kTile * CHW * 8;    // (dt, dt u)
  static constexpr int kDy = kTile * CHW * 4;
  static constexpr int kY = kTile * CHW * 4;
  static constexpr int kPair = kTile * CHW * 8;  // (sum kept A2, sum g B)
  static constexpr int kSum = 32 * TileVecs<CHW>::V * 8;     // dskip, d(delta_bias) of the lanes
  static constexpr int kPart = kTile * 2 * NP * 4;           // dB, dC of the warp's channels
  static constexpr int kRow = kTile * CHW * (int)sizeof(T);  // a tile of an operand
  static constexpr int kH = 32 * kBwdChans * 16;             // saved states
  static constexpr int kStage = 4 * kRow + kH;               // u, delta, gate, dout; states
  static constexpr int kWarp = kDl + kDy + kY + kPair + kSum + kPart + 2 * kStage;
  static constexpr int kBC = kTile * 2 * NP * (int)sizeof(T);
  static constexpr int kTotal = kScanWarps * kWarp + 2 * kBC;
};

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
  float4* dl = reinterpret_cast<float4*>(mine);
  float* dys = reinterpret_cast<float*>(mine + S::kDl);
  float* ys = reinterpret_cast<float*>(mine + S::kDl + S::kDy);
  float2* pair = reinterpret_cast<float2*>(mine + S::kDl + S::kDy + S::kY);
  float2* sums = reinterpret_cast<float2*>(mine + S::kDl + S::kDy + S::kY + S::kPair) + lane;  // [V][32]
  constexpr int kPartAt = S::kDl + S::kDy + S::kY + S::kPair + S::kSum;
  float* part = reinterpret_cast<float*>(mine + kPartAt);
  auto stage = [&](int s, int op) {  // u, delta, gate, dout, (states)
    return reinterpret_cast<T*>(mine + kPartAt + S::kPart + s * S::kStage + op * S::kRow);
  };
  auto saved = [&](int s) {  // [channel][lane]
    return reinterpret_cast<float4*>(mine + kPartAt + S::kPart + s * S::kStage + 4 * S::kRow) + lane;
  };
  pdl_wait();
  pdl_trigger();
  const int bpg = (p.spg + kScanWarps - 1) / kScanWarps;  // CTAs per group
  const int f = blockIdx.x / bpg, in_group = blockIdx.x % bpg * kScanWarps + warp;
  const bool have = in_group < p.spg;  // else a warp without channels, which only keeps the CTA's steps
  L l(p, f * p.spg + (have ? in_group : 0), lane);
  if (!have) l.nch = 0;
  const int ri = blockIdx.y;
  const int t0 = range_begin(p.q, ri, p.R, p.L, lane);
  const int t1 = range_begin(p.q, ri + 1, p.R, p.L, lane);
  const long long DN = (long long)p.D * p.N;
  LaneStates<KD> A2, dA, rr;
  load_rates(p, l, A2);
  zero_states<KD>(dA);
  zero_states<KD>(rr);
  float bias[V], skip[V];
  load_column<V>(p.dbias, l.c0 + TV::chan(lane), l.nch - TV::chan(lane), bias);
  load_column<V>(p.skip, l.c0 + TV::chan(lane), l.nch - TV::chan(lane), skip);
#pragma unroll
  for (int e = 0; e < V; ++e) sums[e * 32] = make_float2(0.f, 0.f);
  Seg g{-1, 0, 0, false};
  if (t0 < t1 && t1 < p.q.T) {
    g = seg_at(p.q, t1, lane);
    if (g.in && g.b < t1) carry_back(p, l, ri, A2, rr);
  }

  auto fetch = [&](int tile0, int s) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    copy_tile<T>(p.u, p.ldu, p.vec, l, tile0, ta, tb, stage(s, 0));
    copy_tile<T>(p.delta, p.ldd, p.vec, l, tile0, ta, tb, stage(s, 1));
    if (p.gate != nullptr) copy_tile<T>(p.gate, p.ldg, p.vec, l, tile0, ta, tb, stage(s, 2));
    copy_tile<T>(p.dout, p.D, p.vec, l, tile0, ta, tb, stage(s, 3));
    copy_bc<T>(p, l, tile0, ta, tb, reinterpret_cast<T*>(base + s * S::kBC), threadIdx.x, kScanWarps * 32);
    // a range that begins inside a tile begins there with a sequence, or outside
    const float* c = p.ckpt + (tile0 / kTile) * DN;
#pragma unroll
    for (int j = 0; j < KD; ++j)
      copy_part<float, 4>(reinterpret_cast<float*>(saved(s) + j * 32),
                          c + (long long)(l.c0 + l.ch(j)) * p.N + l.n0(), p.ckpt,
                          ta == tile0 && l.ch(j) < l.nch ? p.N - l.n0() : 0, p.N % 4 == 0);
    copy_commit();
  };
  const int last = t1 > t0 ? (t1 - 1) / kTile * kTile : -kTile;
  if (last >= 0) fetch(last, 0);
  int cur = 0;
  for (int tile0 = last; tile0 + kTile > t0 && tile0 >= 0; tile0 -= kTile, cur ^= 1) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    const TileSeqs q = tile_seqs(p.q, tile0, ta, tb, lane, g);
    copy_wait();
    const T* bc = reinterpret_cast<T*>(base + cur * S::kBC);
    f2 hs[kTile + 1][4];
    pack_pair(saved(cur)[0], saved(cur)[32], hs[0]);
    stage_steps<T>(p, l, q.live, stage(cur, 0), stage(cur, 1), bias, dl);
    stage_dy<T>(p, l, stage(cur, 3), stage(cur, 2), q.live, dys);
    __syncthreads();
    if (tile0 > t0) fetch(tile0 - kTile, cur ^ 1);

    // The tile's states, as the forward computed them; rows that no sequence of
    // the range holds (dt = dy = 0) pass states and adjoints on, and what they
    // give is not used. `general`: the tile has such rows, or first tokens.
    auto forward = [&](auto general) {
#pragma unroll
      for (int r = 0; r < kTile; ++r) {
        ulonglong2 dv[1];
        f2 b[4], c[4], y[1];
        read_steps<KD>(dl, r * CHW + l.ch(0), dv);
        read_four(bc + r * 2 * NP + l.n0(), b);
        if (p.gate != nullptr) read_four(bc + (r * 2 + 1) * NP + l.n0(), c);
        LaneStates<KD> h;
        const bool first = decltype(general)::value && ((q.first >> r) & 1);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[0][k] = first ? 0ull : hs[r][k];
        if (p.gate != nullptr) {
          scan_step<true, KD>(h, A2, dv, b, c, y);
          const float s = sum_over_states<LN>(y, lane);
          if (l.nq < KD) ys[r * CHW + l.ch(sum_channel<KD>(lane))] = s;
        } else {
          scan_step<false, KD>(h, A2, dv, b, c, y);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) hs[r + 1][k] = h[0][k];
      }
    };
    // the exponentials are taken again: kept from the first pass they would need
    // 64 more registers
    auto again = [&] {
#pragma unroll
      for (int k = 0; k < 4; ++k) asm volatile("" : "+l"(A2[0][k])::"memory");
    };
    // back through them
    f2 dAt[4] = {0ull, 0ull, 0ull, 0ull};
    auto backward = [&](auto general) {
#pragma unroll
      for (int r = kTile - 1; r >= 0; --r) {
        const bool first = decltype(general)::value && ((q.first >> r) & 1);
        const bool none = decltype(general)::value && !((q.live >> r) & 1);
        ulonglong2 dv[1];
        f2 b[4], c[4], y[1], s2[1], g2[1];
        read_steps<KD>(dl, r * CHW + l.ch(0), dv);
        read_dy<KD>(dys + r * CHW + l.ch(0), y);
        read_four(bc + r * 2 * NP + l.n0(), b);
        read_four(bc + (r * 2 + 1) * NP + l.n0(), c);
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f2 a = f2_ex2(f2_mul(dv[0].x, A2[0][k]));
          const f2 gg = f2_fma(c[k], y[0], rr[0][k]);
          const f2 ag = first ? 0ull : f2_mul(a, gg);
          // (what is ahead of a first token is another sequence's, maybe NaN)
          const f2 kept = none ? 0ull : f2_mul(ag, first ? 0ull : hs[r][k]);
          s2[0] = k == 0 ? f2_mul(kept, A2[0][k]) : f2_fma(kept, A2[0][k], s2[0]);
          g2[0] = k == 0 ? f2_mul(gg, b[k]) : f2_fma(gg, b[k], g2[0]);
          dAt[k] = f2_fma(kept, dv[0].x, dAt[k]);
          v[k] = f2_sum(f2_mul(gg, dv[0].y));
          v[4 + k] = f2_sum(f2_mul(y[0], hs[r + 1][k]));
          rr[0][k] = none ? rr[0][k] : ag;
        }
        const float2 s = make_float2(sum_over_states<LN>(s2, lane), sum_over_states<LN>(g2, lane));
        if (l.nq < KD) pair[r * CHW + l.ch(sum_channel<KD>(lane))] = s;
        int vb;
        sum_over_channels<LN>(v, lane, vb);
#pragma unroll
        for (int i = 0; i < LN / 4; ++i) {
          const int k = vb + i;  // 0..3: dB, 4..7: dC of states n0 + k % 4
          part[(r * 2 + k / 4) * NP + l.n0() + k % 4] = v[i];
        }
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
    for (int k = 0; k < 4; ++k) dA[0][k] = f2_add(dA[0][k], dAt[k]);
    __syncwarp();
    // the tile's gradients by token and channel
#pragma unroll
    for (int k = 0; k < TV::NVEC; ++k) {
      const int r = TV::row(k, lane), c = TV::chan(lane), t = tile0 + r, n = l.nch - c;
      if (!TV::has(k, lane) || t < ta || t >= tb || n <= 0) continue;
      const bool vec = p.vec && n >= V, in = (q.live >> r) & 1;
      const Pack<T, V> u = tile_vec<T, CHW>(stage(cur, 0), k, lane), d = tile_vec<T, CHW>(stage(cur, 1), k, lane);
      Pack<T, V> z, go, du, dd, dz;
      if (p.gate != nullptr) {
        z = tile_vec<T, CHW>(stage(cur, 2), k, lane);
        go = tile_vec<T, CHW>(stage(cur, 3), k, lane);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int at = r * CHW + c + e;
        const float uv = to_f(u.v[e]), dt = reinterpret_cast<const float*>(dl)[at / 2 * 4 + e % 2], dy = dys[at];
        const float2 s = pair[at];
        du.v[e] = from_f<T>(in ? fmaf(dt, s.y, skip[e] * dy) : 0.f);
        float ddt = fmaf(kLn2, s.x, uv * s.y);
        if (p.softplus) ddt *= sigmoid_exact(to_f(d.v[e]) + bias[e]);
        dd.v[e] = from_f<T>(in ? ddt : 0.f);
        if (in) {
          const float2 o = sums[e * 32];
          sums[e * 32] = make_float2(fmaf(dy, uv, o.x), o.y + ddt);
        }
        if (p.gate != nullptr) {
          const float zv = to_f(z.v[e]), sg = sigmoid_t<T>(zv);
          const float y = fmaf(skip[e], uv, ys[at]);
          dz.v[e] = from_f<T>(in ? to_f(go.v[e]) * y * sg * (1.f + zv * (1.f - sg)) : 0.f);
        }
      }
      const long long o = (long long)t * p.D + l.c0 + c;
      store_part<T, V>(reinterpret_cast<T*>(p.du) + o, du, n, vec);
      store_part<T, V>(reinterpret_cast<T*>(p.ddelta) + o, dd, n, vec);
      if (p.gate != nullptr) store_part<T, V>(reinterpret_cast<T*>(p.dgate) + o, dz, n, vec);
    }
    __syncthreads();
    // dB and dC of the CTA's channels, the warps' parts in order (the next
    // tile's parts are written behind its own barrier)
    const int warps = min(kScanWarps, p.spg - blockIdx.x % bpg * kScanWarps);
    float* out = p.part_bc + ((long long)blockIdx.x * p.q.T + tile0) * 2 * p.N;
    for (int i = threadIdx.x; i < kTile * 2 * NP; i += blockDim.x) {
      const int r = i / (2 * NP), k = i / NP % 2, n = i % NP;
      if (r < ta - tile0 || r >= tb - tile0 || n >= p.N) continue;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kScanWarps; ++w)
        if (w < warps) s += reinterpret_cast<float*>(base + 2 * S::kBC + w * S::kWarp + kPartAt)[i];
      out[(r * 2 + k) * p.N + n] = (q.live >> r) & 1 ? s : 0.f;
    }
  }
  if (!have) return;
  store_states(p.part_a + ri * DN, l, p.N, dA);
  // lanes of one vector column: the same lane % VPR
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float2 s = sums[e * 32];
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

// dB[t, f, n], dC[t, f, n] = sums over the CTAs of group f.
template <typename T>
__global__ void __launch_bounds__(256) ssm_scan_reduce_bc_kernel(const float* part, T* dB, T* dC, int bpg, int T_,
                                                                 int N, int F) {
  pdl_wait();
  pdl_trigger();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x, per = (long long)T_ * 2 * N;
  const int f = blockIdx.y;
  if (i >= per) return;
  const float* s = part + (long long)f * bpg * per + i;
  float v = 0.f;
#pragma unroll 8
  for (int b = 0; b < bpg; ++b) v += s[b * per];
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
