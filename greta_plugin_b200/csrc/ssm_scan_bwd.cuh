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
// The forward left the states ahead of every 16th token (4 bytes a token and
// channel at N = 16, as much as two 16-bit tensors: less than a third pass of
// exponentials would take). The main kernel walks its range's tiles from the
// last to the first: it runs a tile's recurrence again from the saved state,
// leaves the 16 states of every lane in shared memory, and then goes back
// through them with g in registers. So two exponentials and some fourteen fp32
// operations per (token, channel, state): both pipes are about equally full.
// The CTA's warps take neighbouring channels of one group; their parts of dB
// and dC are added in shared memory and go, one row per token and CTA, to
// `part_bc`; dA, dskip and d(delta_bias) of the range stay in registers. Small
// kernels add the parts in a fixed order, so the same call gives the same bits.
//
// A range that ends inside a sequence needs a g of the next token: the carry
// kernel runs g alone over the part of each range up to the first sequence end
// in it, as the forward's does for h.
#pragma once

#include "ssm_scan.cuh"

namespace greta {

// Shared memory in floats: of a warp, and what the CTA shares.
template <int LN>
struct BwdSmem {
  static constexpr int CHW = Lanes<LN>::CHW, NP = Lanes<LN>::NP;
  static constexpr int kH = (kTile + 1) * 4 * 32 * 4;  // states: [token + 1][channel][lane] float4
  static constexpr int kDl = kTile * CHW * 2;          // (dt, dt u)
  static constexpr int kDy = kTile * CHW;
  static constexpr int kY = kTile * CHW;
  static constexpr int kPair = kTile * CHW * 2;        // (sum kept A2, sum g B)
  static constexpr int kPart = kTile * 2 * NP;         // dB, dC of the warp's channels
  static constexpr int kWarp = kH + kDl + kDy + kY + kPair + kPart;
  static constexpr int kBC = kTile * 2 * NP;
  static constexpr int kTotal = kScanWarps * kWarp + kBC;
};

// (dt, dt u) and dy of a tile; the raw rows stay with the lane for the tile's
// outputs.
template <typename T, int LN>
struct TileRows {
  Pack<T, TileVecs<LN>::V> u[TileVecs<LN>::NVEC], d[TileVecs<LN>::NVEC], z[TileVecs<LN>::NVEC],
      g[TileVecs<LN>::NVEC];
};

template <typename T, int LN, bool WITH_U>
__device__ __forceinline__ void stage_bwd(const ScanParams& p, const Lanes<LN>& l, int tile0, int ta, int tb,
                                          float* dl, float* dy, TileRows<T, LN>& rows) {
  using TV = TileVecs<LN>;
  constexpr int V = TV::V, CHW = TV::CHW;
#pragma unroll
  for (int k = 0; k < TV::NVEC; ++k) {
    const int i = k * 32 + l.lane;
    if (TV::COUNT % 32 != 0 && i >= TV::COUNT) continue;
    const int r = i / TV::VPR, c = (i % TV::VPR) * V, t = tile0 + r;
    const int n = l.nch - c;
    zero(rows.u[k]);
    zero(rows.d[k]);
    zero(rows.z[k]);
    zero(rows.g[k]);
    if (t >= ta && t < tb && n > 0) {
      const bool vec = p.vec && n >= V;
      if (WITH_U) rows.u[k] = load_part<T, V>(reinterpret_cast<const T*>(p.u) + t * p.ldu + l.c0 + c, n, vec);
      rows.d[k] = load_part<T, V>(reinterpret_cast<const T*>(p.delta) + t * p.ldd + l.c0 + c, n, vec);
      if (p.gate != nullptr)
        rows.z[k] = load_part<T, V>(reinterpret_cast<const T*>(p.gate) + t * p.ldg + l.c0 + c, n, vec);
      rows.g[k] =
          load_part<T, V>(reinterpret_cast<const T*>(p.dout) + (long long)t * p.D + l.c0 + c, n, vec);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s = 0.f, g = 0.f;
      if (t >= ta && t < tb && e < n) {
        const float bias = p.dbias != nullptr ? p.dbias[l.c0 + c + e] : 0.f;
        s = step_size(p, to_f(rows.d[k].v[e]) + bias);
        g = to_f(rows.g[k].v[e]);
        if (p.gate != nullptr) {
          const float z = to_f(rows.z[k].v[e]);
          g *= z * sigmoid_exact(z);
        }
      }
      dl[(r * CHW + c + e) * 2] = s;
      dl[(r * CHW + c + e) * 2 + 1] = s * to_f(rows.u[k].v[e]);
      dy[r * CHW + c + e] = g;
    }
  }
}

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
      s.live |= (0xffffu >> (kTile - (stop - t))) << (t - tile0);
    }
    t = stop;
    if (t >= tb) return s;
    w = seg_next(q, w);
  }
}

// The adjoint's carry at the end of range i, inside a sequence that goes on:
// r = a[t] g[t] of the next range's first token t.
template <int LN>
__device__ __forceinline__ void carry_back(const ScanParams& p, const Lanes<LN>& l, int i, const LaneStates& A2,
                                           LaneStates& r) {
  int j1 = i + 1;
  for (int lo = i + 1; lo < p.R; lo += 32) {
    const int k = lo + l.lane;
    const unsigned m = __ballot_sync(0xffffffffu, k < p.R && p.reset[k] != 0);
    if (m != 0) {
      j1 = lo + __ffs(m) - 1;
      break;
    }
    j1 = min(p.R - 1, lo + 31);
  }
  const long long DN = (long long)p.D * p.N;
  zero_states(r);
  for (int j = j1; j > i; --j) {
    float s[4][4];
    load_states(p.carry + j * DN, l, p.N, s);
    LaneStates s2;
    pack_states(s, s2);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float d = l.ch(c) < l.nch && j < j1 ? p.dsum[(long long)j * p.D + l.c0 + l.ch(c)] : 0.f;
      const f2 d2 = pack2(d, d);
#pragma unroll
      for (int k = 0; k < 2; ++k) r[c][k] = f2_fma(f2_ex2(f2_mul(d2, A2[c][k])), r[c][k], s2[c][k]);
    }
  }
}

// g alone over the head of each range that begins inside a sequence.
template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32) ssm_scan_bwd_carry_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  using S = FwdSmem<LN>;  // same layout: (dt, -), dy, (-, C)
  constexpr int CHW = Lanes<LN>::CHW, NP = Lanes<LN>::NP;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* dl = reinterpret_cast<float*>(smem4) + warp * S::kWarp;
  float* dy = dl + S::kDl;
  float* bc = dy + S::kY;
  pdl_wait();
  pdl_trigger();
  const int slice = blockIdx.x * (blockDim.x >> 5) + warp;
  if (slice >= p.F * p.spg) return;
  const Lanes<LN> l(p, slice, lane);
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
  LaneStates A2, r;
  load_rates(p, l, A2);
  zero_states(r);
  float dsum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int tile0 = (t1 - 1) / kTile * kTile; tile0 + kTile > t0; tile0 -= kTile) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    TileRows<T, LN> rows;
    __syncwarp();
    stage_bwd<T, LN, false>(p, l, tile0, ta, tb, dl, dy, rows);
    stage_bc<T, LN>(p, l, tile0, ta, tb, bc, true);
    __syncwarp();
#pragma unroll 2
    for (int i = tb - 1 - tile0; i >= ta - tile0; --i) {
      float2 d[4];
      read_steps(dl, l, i, d);
      const float4 y = *reinterpret_cast<const float4*>(dy + i * CHW + l.ch(0));
      const float4 c = *reinterpret_cast<const float4*>(bc + (i * 2 + 1) * NP + l.n0());
      const f2 c2[2] = {pack2(c.x, c.y), pack2(c.z, c.w)};
      const float yv[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f2 d2 = pack2(d[j].x, d[j].x), y2 = pack2(yv[j], yv[j]);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          r[j][k] = f2_mul(f2_ex2(f2_mul(d2, A2[j][k])), f2_fma(c2[k], y2, r[j][k]));
        dsum[j] += d[j].x;
      }
    }
  }
  store_states(p.carry + ri * (long long)p.D * p.N, l, p.N, r);
  if (l.nq == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (l.ch(j) < l.nch) p.dsum[(long long)ri * p.D + l.c0 + l.ch(j)] = dsum[j];
  }
}

// v0, v1 summed over the LN lanes of each of four channels; lane nq < 4 keeps
// channel sum_channel(lane)'s.
template <int LN>
__device__ __forceinline__ float2 sum_pair(const float (&a)[4], const float (&b)[4], int lane) {
  return make_float2(sum_over_states<LN>(a, lane), sum_over_states<LN>(b, lane));
}

// The eight values of a lane summed over the channel groups of the warp (lane
// bits LN, 2 LN, .. 16): halves are exchanged while there are some, so that
// M = max(1, 8 LN / 32) values, from index `base`, stay with a lane.
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

template <typename T, int LN>
__global__ void __launch_bounds__(kScanWarps * 32, 1) ssm_scan_bwd_kernel(const ScanParams p) {
  extern __shared__ float4 smem4[];
  using S = BwdSmem<LN>;
  using TV = TileVecs<LN>;
  constexpr int CHW = TV::CHW, V = TV::V, NP = Lanes<LN>::NP;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* base = reinterpret_cast<float*>(smem4);
  float* bc = base;
  float* mine = base + S::kBC + warp * S::kWarp;
  float4* hs = reinterpret_cast<float4*>(mine) + lane;  // [token + 1][channel]: stride 32
  float* dl = mine + S::kH;
  float* dys = dl + S::kDl;
  float* ys = dys + S::kDy;
  float* pair = ys + S::kY;
  float* part = pair + S::kPair;
  pdl_wait();
  pdl_trigger();
  const int bpg = (p.spg + kScanWarps - 1) / kScanWarps;  // CTAs per group
  const int f = blockIdx.x / bpg, in_group = blockIdx.x % bpg * kScanWarps + warp;
  const bool have = in_group < p.spg;  // else a warp without channels, which only keeps the CTA's steps
  const Lanes<LN> l(p, f * p.spg + (have ? in_group : 0), lane);
  const int ri = blockIdx.y;
  const int t0 = range_begin(p.q, ri, p.R, p.L, lane);
  const int t1 = range_begin(p.q, ri + 1, p.R, p.L, lane);
  const long long DN = (long long)p.D * p.N;
  LaneStates A2, dA, rr, hc;
  load_rates(p, l, A2);
  zero_states(dA);
  zero_states(rr);
  float dskip[V], dbias[V];
#pragma unroll
  for (int e = 0; e < V; ++e) dskip[e] = dbias[e] = 0.f;
  Seg g{-1, 0, 0, false};
  if (t0 < t1 && t1 < p.q.T) {
    g = seg_at(p.q, t1, lane);
    if (g.in && g.b < t1) carry_back(p, l, ri, A2, rr);
  }

  for (int tile0 = t1 > t0 ? (t1 - 1) / kTile * kTile : -kTile; tile0 + kTile > t0 && tile0 >= 0; tile0 -= kTile) {
    const int ta = max(t0, tile0), tb = min(t1, tile0 + kTile);
    const TileSeqs q = tile_seqs(p.q, tile0, ta, tb, lane, g);
    TileRows<T, LN> rows;
    if (have) {
      stage_bwd<T, LN, true>(p, l, tile0, ta, tb, dl, dys, rows);
      if (warp == 0) stage_bc<T, LN>(p, l, tile0, ta, tb, bc, true);
      float v[4][4];
      if (ta == tile0) {
        load_states(p.ckpt + (tile0 / kTile) * DN, l, p.N, v);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = 0.f;
      }
      pack_states(v, hc);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        hs[((ta - tile0) * 4 + j) * 32] = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
    }
    __syncthreads();
    if (have) {
      // the tile's states, as the forward computed them
      for (int r = ta - tile0; r < tb - tile0; ++r) {
        if ((q.first >> r) & 1) zero_states(hc);
        float2 d[4];
        read_steps(dl, l, r, d);
        const float4 b = *reinterpret_cast<const float4*>(bc + (r * 2) * NP + l.n0());
        const float4 c = *reinterpret_cast<const float4*>(bc + (r * 2 + 1) * NP + l.n0());
        float y[4];
        scan_step<true>(hc, A2, d, b, c, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float4 o;
          unpack2(hc[j][0], o.x, o.y);
          unpack2(hc[j][1], o.z, o.w);
          hs[((r + 1) * 4 + j) * 32] = o;
        }
        if (p.gate != nullptr) {
          const float s = sum_over_states<LN>(y, lane);
          if (l.nq < 4) ys[r * CHW + l.ch(sum_channel(lane))] = s;
        }
      }
      // back through them
      for (int r = tb - 1 - tile0; r >= ta - tile0; --r) {
        float v[8];
        float sa[4], gb[4];
        if ((q.live >> r) & 1) {
          const bool first = (q.first >> r) & 1;
          float2 d[4];
          read_steps(dl, l, r, d);
          const float4 dy4 = *reinterpret_cast<const float4*>(dys + r * CHW + l.ch(0));
          const float dyv[4] = {dy4.x, dy4.y, dy4.z, dy4.w};
          const float4 b = *reinterpret_cast<const float4*>(bc + (r * 2) * NP + l.n0());
          const float4 c = *reinterpret_cast<const float4*>(bc + (r * 2 + 1) * NP + l.n0());
          const f2 b2[2] = {pack2(b.x, b.y), pack2(b.z, b.w)};
          const f2 c2[2] = {pack2(c.x, c.y), pack2(c.z, c.w)};
          f2 dB[2] = {0ull, 0ull}, dC[2] = {0ull, 0ull};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 hp = hs[(r * 4 + j) * 32];
            const f2 prev[2] = {pack2(hp.x, hp.y), pack2(hp.z, hp.w)};
            const f2 d2 = pack2(d[j].x, d[j].x), du2 = pack2(d[j].y, d[j].y), y2 = pack2(dyv[j], dyv[j]);
            f2 s2 = 0ull, g2 = 0ull;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const f2 a = f2_ex2(f2_mul(d2, A2[j][k]));
              const f2 gg = f2_fma(c2[k], y2, rr[j][k]);
              const f2 ag = first ? 0ull : f2_mul(a, gg);
              // (what is ahead of a first token is another sequence's, maybe NaN)
              const f2 kept = f2_mul(ag, first ? 0ull : prev[k]);
              s2 = f2_fma(kept, A2[j][k], s2);
              dA[j][k] = f2_fma(kept, d2, dA[j][k]);
              g2 = f2_fma(gg, b2[k], g2);
              dB[k] = f2_fma(gg, du2, dB[k]);
              dC[k] = f2_fma(y2, hc[j][k], dC[k]);
              rr[j][k] = ag;
              hc[j][k] = prev[k];
            }
            sa[j] = f2_sum(s2);
            gb[j] = f2_sum(g2);
          }
          unpack2(dB[0], v[0], v[1]);
          unpack2(dB[1], v[2], v[3]);
          unpack2(dC[0], v[4], v[5]);
          unpack2(dC[1], v[6], v[7]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sa[j] = gb[j] = 0.f;
            const float4 hp = hs[(r * 4 + j) * 32];
            hc[j][0] = pack2(hp.x, hp.y);
            hc[j][1] = pack2(hp.z, hp.w);
          }
          zero_states(rr);
        }
        const float2 s = sum_pair<LN>(sa, gb, lane);
        if (l.nq < 4) reinterpret_cast<float2*>(pair)[r * CHW + l.ch(sum_channel(lane))] = s;
        int vb;
        sum_over_channels<LN>(v, lane, vb);
        constexpr int M = LN >= 4 ? LN / 4 : 1;  // values left of a lane
#pragma unroll
        for (int i = 0; i < M; ++i) {
          const int k = vb + i;  // 0..3: dB, 4..7: dC of states n0 + k % 4
          part[(r * 2 + k / 4) * NP + l.n0() + k % 4] = v[i];
        }
      }
      __syncwarp();
      // the tile's gradients by token and channel
#pragma unroll
      for (int k = 0; k < TV::NVEC; ++k) {
        const int i = k * 32 + lane;
        if (TV::COUNT % 32 != 0 && i >= TV::COUNT) continue;
        const int r = i / TV::VPR, c = (i % TV::VPR) * V, t = tile0 + r;
        const int n = l.nch - c;
        if (t < ta || t >= tb || n <= 0) continue;
        const bool vec = p.vec && n >= V, in = (q.live >> r) & 1;
        Pack<T, V> du, dd, dz;
        zero(du);
        zero(dd);
        zero(dz);
        if (in) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (e >= n) continue;
            const int at = r * CHW + c + e;
            const float u = to_f(rows.u[k].v[e]), dt = dl[at * 2], dy = dys[at];
            const float2 s = reinterpret_cast<const float2*>(pair)[at];
            const float sk = p.skip != nullptr ? p.skip[l.c0 + c + e] : 0.f;
            du.v[e] = from_f<T>(fmaf(dt, s.y, sk * dy));
            float ddt = fmaf(kLn2, s.x, u * s.y);
            if (p.softplus) {
              const float bias = p.dbias != nullptr ? p.dbias[l.c0 + c + e] : 0.f;
              ddt *= sigmoid_exact(to_f(rows.d[k].v[e]) + bias);
            }
            dd.v[e] = from_f<T>(ddt);
            dbias[e] += ddt;
            dskip[e] = fmaf(dy, u, dskip[e]);
            if (p.gate != nullptr) {
              const float z = to_f(rows.z[k].v[e]), sg = sigmoid_exact(z);
              const float y = fmaf(sk, u, ys[at]);
              dz.v[e] = from_f<T>(to_f(rows.g[k].v[e]) * y * sg * (1.f + z * (1.f - sg)));
            }
          }
        }
        const long long o = (long long)t * p.D + l.c0 + c;
        store_part<T, V>(reinterpret_cast<T*>(p.du) + o, du, n, vec);
        store_part<T, V>(reinterpret_cast<T*>(p.ddelta) + o, dd, n, vec);
        if (p.gate != nullptr) store_part<T, V>(reinterpret_cast<T*>(p.dgate) + o, dz, n, vec);
      }
    }
    __syncthreads();
    // dB and dC of the CTA's channels, the warps' parts in order
    const int warps = min(kScanWarps, p.spg - blockIdx.x % bpg * kScanWarps);
    float* out = p.part_bc + ((long long)blockIdx.x * p.q.T + tile0) * 2 * p.N;
    for (int i = threadIdx.x; i < (tb - ta) * 2 * p.N; i += blockDim.x) {
      const int r = ta - tile0 + i / (2 * p.N), k = i / p.N % 2, n = i % p.N;
      float s = 0.f;
      for (int w = 0; w < warps; ++w)
        s += base[S::kBC + w * S::kWarp + (S::kWarp - S::kPart) + (r * 2 + k) * NP + n];
      out[(long long)r * 2 * p.N + k * p.N + n] = s;
    }
    __syncthreads();
  }
  if (!have) return;
  store_states(p.part_a + ri * DN, l, p.N, dA);
  // lanes of one vector column: the same l.lane % VPR
#pragma unroll
  for (int e = 0; e < V; ++e) {
#pragma unroll
    for (int o = TV::VPR; o < 32; o <<= 1) {
      dskip[e] += __shfl_xor_sync(0xffffffffu, dskip[e], o);
      dbias[e] += __shfl_xor_sync(0xffffffffu, dbias[e], o);
    }
    const int c = lane * V + e;
    if (lane < TV::VPR && c < l.nch) {
      p.part_d[(long long)ri * 2 * p.D + l.c0 + c] = dskip[e];
      p.part_d[(long long)ri * 2 * p.D + p.D + l.c0 + c] = dbias[e];
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
