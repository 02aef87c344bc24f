// Short causal depthwise convolution with static filters:
//
//   pre[t, d] = bias[d] + sum_k w[k, d] x[t + k - W + 1, d]   (tap W-1 = current token)
//   out[t, d] = pre or SiLU(pre)
//
// Bound by HBM: 2 W + 4 operations per element read and written. A thread owns
// NV channels (16 bytes of a row for the kernel sizes in use) of a run of L
// consecutive tokens of the packed stream and keeps the last W-1 inputs in
// registers, so a row is read once, plus W-1 rows ahead of each run from L2.
// Runs are cut by position, so ragged batches are balanced; a run's warp
// follows the sequence borders in it (ssm_common.cuh). Rows come four at a time
// through a ring in shared memory, three such groups ahead, in asynchronous
// copies of which a lane reads only its own (no barrier, and no registers for
// what is on its way: with loads into registers the compiler kept two to four
// rows in flight, half of what HBM needs). Four tokens that lie inside one
// sequence are computed without a test between them, so that the window moves
// by renaming registers.
// W is a template parameter for 2, 3 and 4 (the kernel sizes in use); WT = -8
// and -16 take any W up to that, with narrower vectors for their windows:
// filters and window are aligned to the current token's end (index MW-1 and
// MW-2), so that no register index depends on W.
#pragma once

#include "ssm_common.cuh"

namespace greta {

struct ConvParams {
  const void* x;     // [T, D], rows ldx apart
  const void* w;     // w[k * sw_k + d * sw_d]
  const void* bias;  // [D] or null
  void* y;           // [T, D]
  Seqs q;
  long long ldx, sw_k, sw_d;
  int D, W, L, nblk;  // blockIdx.x = run block * nblk + channel block
  int silu;
  int zero_rest;  // rows outside every sequence: zeros (else left alone)
  int vec_w;      // the filters' rows are whole aligned vectors (sw_d == 1)
  // cache-slot state (packed batches)
  void* state;
  long long s_slot, s_d, s_h, num_slots;
  int st_layout;  // StateLayout
  const int* slots;
  const signed char* initial;
  int* err;
  // backward
  const void* dout;  // [T, D]
  void* dx;          // [T, D]
  float* part;       // [run blocks][W + 1][D]: sums of the block's runs for w and bias
};

constexpr int kGroup = 4;   // tokens at a time
constexpr int kStages = 4;  // groups in the ring

// A lane's part of the ring for one operand: [stage][token][lane] vectors.
// Single elements (rows that are not whole vectors) are loaded when the group
// is due.
template <typename T, int NV>
struct ConvRing {
  static constexpr int kBytes = kStages * kGroup * 32 * NV * (int)sizeof(T);  // of a warp
  Pack<T, NV>* mine;
  const T* g;  // the lane's first channel of row 0
  long long ld;
  int n;

  // Rows t .. t + 3 that are below `end`.
  __device__ __forceinline__ void fetch(int group, int t, int end) const {
    if (NV > 1) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
        if (t + i < end && n == NV)
          copy_async<NV * (int)sizeof(T)>(mine + (group % kStages * kGroup + i) * 32, g + (long long)(t + i) * ld, true);
      copy_commit();
    }
  }
  // Row t + i of the group that begins at t.
  __device__ __forceinline__ Pack<T, NV> row(int group, int t, int i) const {
    if (NV > 1) return load_part<T, NV>(reinterpret_cast<const T*>(mine + (group % kStages * kGroup + i) * 32), NV, true);
    return load_part<T, NV>(g + (long long)(t + i) * ld, n, false);
  }
};
// The copies of all but the last kStages - 1 groups have landed.
__device__ __forceinline__ void ring_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory"); }

// NV channels as fp32 pairs (the last one's second half is idle when NV is 1).
template <int NV>
using Chans = f2[(NV + 1) / 2];

template <typename T, int NV>
__device__ __forceinline__ void widen(const Pack<T, NV>& r, Chans<NV>& o) {
#pragma unroll
  for (int c = 0; c < NV; c += 2) o[c / 2] = pack2(to_f(r.v[c]), c + 1 < NV ? to_f(r.v[c + 1 < NV ? c + 1 : c]) : 0.f);
}
template <typename T, int NV>
__device__ __forceinline__ Pack<T, NV> narrow(const Chans<NV>& v) {
  Pack<T, NV> o;
#pragma unroll
  for (int c = 0; c < NV; c += 2) {
    float a, b;
    unpack2(v[c / 2], a, b);
    o.v[c] = from_f<T>(a);
    if (c + 1 < NV) o.v[c + 1 < NV ? c + 1 : c] = from_f<T>(b);
  }
  return o;
}

// The filters (tap k at index MW - W + k) and the bias of this thread's channels.
template <typename T, int NV, int MW>
__device__ __forceinline__ void conv_weights(const ConvParams& p, int c0, int n, int W, Chans<NV> (&w)[MW],
                                             Chans<NV>& bias) {
  const T* wg = reinterpret_cast<const T*>(p.w);
#pragma unroll
  for (int k = 0; k < MW; ++k) {
    Pack<T, NV> r;
    zero(r);
    const int tap = k - (MW - W);
    if (tap >= 0) {
      if (p.vec_w) {
        r = load_part<T, NV>(wg + (long long)tap * p.sw_k + c0, n, n == NV);
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c)
          if (c < n) r.v[c] = wg[(long long)tap * p.sw_k + (long long)(c0 + c) * p.sw_d];
      }
    }
    widen<T, NV>(r, w[k]);
  }
  Pack<T, NV> r;
#pragma unroll
  for (int c = 0; c < NV; ++c)
    r.v[c] = p.bias != nullptr && c < n ? reinterpret_cast<const T*>(p.bias)[c0 + c] : from_f<T>(0.f);
  widen<T, NV>(r, bias);
}

// The slot's H = W-1 inputs of this thread's channels, oldest first, at the end
// of the window's MH places.
template <typename T, int NV, int MH>
__device__ __forceinline__ void conv_load_state(const ConvParams& p, int slot, int c0, int n, int H,
                                                Pack<T, NV> (&win)[MH], bool exact) {
  const T* base = reinterpret_cast<const T*>(p.state) + slot * p.s_slot;
  if (exact && p.st_layout == kStDS && n == NV) {
    // [D, H] contiguous: H vectors hold NV channels of H inputs
    const T* b = base + (long long)c0 * MH;
    Pack<T, NV> r[MH];
#pragma unroll
    for (int i = 0; i < MH; ++i) r[i] = load_part<T, NV>(b + i * NV, NV, true);
#pragma unroll
    for (int h = 0; h < MH; ++h)
#pragma unroll
      for (int c = 0; c < NV; ++c) win[h].v[c] = r[(c * MH + h) / NV].v[(c * MH + h) % NV];
  } else if (p.st_layout == kStSD && n == NV) {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h >= MH - H) win[h] = load_part<T, NV>(base + (long long)(h - (MH - H)) * p.s_h + c0, NV, true);
  } else {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h >= MH - H) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
          win[h].v[c] =
              c < n ? base[(long long)(c0 + c) * p.s_d + (long long)(h - (MH - H)) * p.s_h] : from_f<T>(0.f);
      }
  }
}

template <typename T, int NV, int MH>
__device__ __forceinline__ void conv_store_state(const ConvParams& p, int slot, int c0, int n, int H,
                                                 const Pack<T, NV> (&win)[MH], bool exact) {
  T* base = reinterpret_cast<T*>(p.state) + slot * p.s_slot;
  if (exact && p.st_layout == kStDS && n == NV) {
    T* b = base + (long long)c0 * MH;
    Pack<T, NV> r[MH];
#pragma unroll
    for (int h = 0; h < MH; ++h)
#pragma unroll
      for (int c = 0; c < NV; ++c) r[(c * MH + h) / NV].v[(c * MH + h) % NV] = win[h].v[c];
#pragma unroll
    for (int i = 0; i < MH; ++i) store_part<T, NV>(b + i * NV, r[i], NV, true);
  } else if (p.st_layout == kStSD && n == NV) {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h >= MH - H) store_part<T, NV>(base + (long long)(h - (MH - H)) * p.s_h + c0, win[h], NV, true);
  } else {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h >= MH - H) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
          if (c < n) base[(long long)(c0 + c) * p.s_d + (long long)(h - (MH - H)) * p.s_h] = win[h].v[c];
      }
  }
}

// Pre-activation of one token: taps oldest first, the window under the first
// W-1 and the token itself under the last.
template <int NV, int MW, int MH>
__device__ __forceinline__ void conv_pre(const Chans<NV> (&w)[MW], const Chans<NV>& bias, const Chans<NV> (&win)[MH],
                                         const Chans<NV>& x, int W, Chans<NV>& pre) {
#pragma unroll
  for (int c = 0; c < (NV + 1) / 2; ++c) {
    f2 s = bias[c];
#pragma unroll
    for (int k = 0; k < MW; ++k) {
      if (k == MW - 1)
        s = f2_fma(w[k][c], x[c], s);
      else if (k >= MW - W)
        s = f2_fma(w[k][c], win[k < MH ? k : 0][c], s);
    }
    pre[c] = s;
  }
}

template <int NV, int MH>
__device__ __forceinline__ void conv_push(Chans<NV> (&win)[MH], const Chans<NV>& x) {
#pragma unroll
  for (int h = 0; h < MH; ++h)
#pragma unroll
    for (int c = 0; c < (NV + 1) / 2; ++c) win[h][c] = h + 1 < MH ? win[h + 1 < MH ? h + 1 : h][c] : x[c];
}

template <int NV, int MH>
__device__ __forceinline__ void conv_zero(Chans<NV> (&win)[MH]) {
#pragma unroll
  for (int h = 0; h < MH; ++h)
#pragma unroll
    for (int c = 0; c < (NV + 1) / 2; ++c) win[h][c] = 0ull;
}

template <typename T, int NV>
__device__ __forceinline__ void conv_silu(Chans<NV>& v) {
#pragma unroll
  for (int c = 0; c < (NV + 1) / 2; ++c) {
    float a, b;
    unpack2(v[c], a, b);
    v[c] = pack2(a * sigmoid_t<T>(a), NV > 1 ? b * sigmoid_t<T>(b) : 0.f);
  }
}

// PACKED: history from and to the requests' cache slots; else zero history.
template <typename T, int NV, int WT, bool PACKED>
__global__ void __launch_bounds__(128) ssm_conv_fwd_kernel(const ConvParams p) {
  constexpr int MW = WT > 0 ? WT : -WT;
  constexpr int MH = MW > 1 ? MW - 1 : 1;
  constexpr bool kVec = NV > 1;  // every row is whole aligned vectors (the host's choice)
  const int W = WT > 0 ? WT : p.W;
  const int H = W - 1;
  const int lane = threadIdx.x & 31;
  const int c0 = ((int)(blockIdx.x % p.nblk) * 32 + lane) * NV;
  const int n = max(0, min(NV, p.D - c0));  // 0: a lane without channels
  const bool vec = kVec && n == NV;
  const long long first = ((long long)(blockIdx.x / p.nblk) * blockDim.y + threadIdx.y) * p.L;
  pdl_wait();
  pdl_trigger();
  if (first >= p.q.T) return;
  int t = (int)first;
  int t1 = (int)min((long long)p.q.T, first + p.L);
  const T* xg = reinterpret_cast<const T*>(p.x) + c0;
  T* yg = reinterpret_cast<T*>(p.y) + c0;
  extern __shared__ float4 ring_smem[];
  ConvRing<T, NV> ring;
  ring.mine = reinterpret_cast<Pack<T, NV>*>(reinterpret_cast<char*>(ring_smem) +
                                             threadIdx.y * ConvRing<T, NV>::kBytes) + lane;
  ring.g = xg;
  ring.ld = p.ldx;
  ring.n = n;
  Chans<NV> w[MW], bias, win[MH];
  const SeqView sv(p.q, lane);
  Seg g = sv.at(t);

  int tend = t1;
  if (PACKED && H > 0) {
    // A request's first W-1 tokens stay with the run that has its first: that
    // run alone reads the slot (and writes it, below), so no other run's write
    // can come between.
    if (g.in && t > g.b && t - g.b < H) {
      const int skip = min(g.b + H, g.e);
      if (skip >= t1) return;
      t = skip;
      if (t == g.e) g = sv.next(g);
    }
    if (t1 < p.q.T && t1 != g.e) {
      const Seg last = g.in && g.e > t1 ? g : sv.at(t1);
      if (last.in && t1 > last.b && t1 - last.b < H) tend = min(last.b + H, last.e);
    }
  }
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) ring.fetch(i, t + i * kGroup, tend);
  conv_weights<T, NV>(p, c0, n, W, w, bias);
  conv_zero<NV>(win);
  // inside a sequence: the inputs ahead of the run (t - H + h >= 0 where kept)
  if (g.in && t > g.b) {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h >= MH - H && t - MH + h >= g.b)
        widen<T, NV>(load_part<T, NV>(xg + (long long)(t - MH + h) * p.ldx, n, vec), win[h]);
  }
  int slot = -1;
  Pack<T, NV> old[MH];  // the slot's inputs of a request that begins here
#pragma unroll
  for (int h = 0; h < MH; ++h) zero(old[h]);
  // the first token of sequence g
  auto begin = [&] {
    conv_zero<NV>(win);
    slot = -1;
    if (!PACKED || p.state == nullptr) return;
    const int raw = p.slots[g.s], initial = p.initial[g.s];
    if (raw >= p.num_slots && p.err != nullptr && c0 == 0) atomicOr(p.err, 1);
    slot = raw >= 0 && raw < p.num_slots ? raw : -1;
#pragma unroll
    for (int h = 0; h < MH; ++h) zero(old[h]);
    if (slot >= 0 && initial != 0) {
      conv_load_state<T, NV, MH>(p, slot, c0, n, H, old, WT > 1);
#pragma unroll
      for (int h = 0; h < MH; ++h)
        if (h >= MH - H) widen<T, NV>(old[h], win[h]);
    }
    if (slot >= 0 && g.e > tend) {
      // the request ends in a later run: its last W-1 inputs (it has more
      // than W-1) straight from x
      Pack<T, NV> fin[MH];
#pragma unroll
      for (int h = 0; h < MH; ++h) {
        zero(fin[h]);
        if (h >= MH - H) fin[h] = load_part<T, NV>(xg + (long long)(g.e - MH + h) * p.ldx, n, vec);
      }
      conv_store_state<T, NV, MH>(p, slot, c0, n, H, fin, WT > 1);
      slot = -1;
    }
  };
  // behind the last token of sequence g
  auto finish = [&] {
    if (!PACKED || slot < 0) return;
    // the last W-1 of (old inputs, the request's), copied bit for bit
    Pack<T, NV> fin[MH];
    const int len = g.e - g.b;
#pragma unroll
    for (int h = 0; h < MH; ++h) {
      zero(fin[h]);
      if (h < MH - H) continue;
      if (len - MH + h >= 0) {
        fin[h] = load_part<T, NV>(xg + (long long)(g.e - MH + h) * p.ldx, n, vec);
      } else {
#pragma unroll
        for (int k = 0; k < MH; ++k)
          if (k == h + len) fin[h] = old[k];
      }
    }
    conv_store_state<T, NV, MH>(p, slot, c0, n, H, fin, WT > 1);
    slot = -1;
  };
  auto token = [&](int at, const Pack<T, NV>& raw) {
    Chans<NV> x, o;
    widen<T, NV>(raw, x);
    conv_pre<NV>(w, bias, win, x, W, o);
    conv_push<NV>(win, x);
    if (p.silu) conv_silu<T, NV>(o);
    store_part<T, NV>(yg + (long long)at * p.D, narrow<T, NV>(o), n, vec);
  };

  for (int group = 0; t < tend; t += kGroup, ++group) {
    if (NV > 1) ring_wait();
    // (into the stage of the group before this one)
    ring.fetch(group + kStages - 1, t + (kStages - 1) * kGroup, tend);
    if (g.in && t > g.b && t + kGroup <= min(g.e - 1, tend)) {
      Pack<T, NV> x[kGroup];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) x[i] = ring.row(group, t, i);
#pragma unroll
      for (int i = 0; i < kGroup; ++i) token(t + i, x[i]);
    } else {
#pragma unroll 1
      for (int i = 0; i < kGroup && t + i < tend; ++i) {
        const int ti = t + i;
        if (ti >= g.e) g = sv.next(g);
        if (g.in) {
          if (ti == g.b) begin();
          token(ti, ring.row(group, t, i));
          if (ti + 1 == g.e) finish();
        } else if (p.zero_rest) {
          Pack<T, NV> z;
          zero(z);
          store_part<T, NV>(yg + (long long)ti * p.D, z, n, vec);
        }
      }
    }
  }
}

// Batches of (nearly) one token per request: a warp has the channels of one
// request and walks its tokens, with filters and window in the element type (a
// third of the registers, so that all of a step's warps run at once) and with
// the metadata, the first token's row and the filters asked for together.
template <typename T, int NV, int WT>
__global__ void __launch_bounds__(128) ssm_conv_decode_kernel(const ConvParams p) {
  constexpr int MW = WT > 0 ? WT : -WT;
  constexpr int MH = MW > 1 ? MW - 1 : 1;
  const int W = WT > 0 ? WT : p.W;
  const int H = W - 1;
  const int lane = threadIdx.x & 31;
  const int c0 = ((int)(blockIdx.x % p.nblk) * 32 + lane) * NV;
  const int n = max(0, min(NV, p.D - c0));
  const bool vec = NV > 1 && n == NV;
  const int r = (int)(blockIdx.x / p.nblk) * blockDim.y + threadIdx.y;
  const T* xg = reinterpret_cast<const T*>(p.x) + c0;
  T* yg = reinterpret_cast<T*>(p.y) + c0;
  const T* wg = reinterpret_cast<const T*>(p.w);
  pdl_wait();
  pdl_trigger();
  if (r >= p.q.nseq) return;
  const int b = seq_start(p.q, r), e = seq_start(p.q, r + 1), raw = p.slots[r], initial = p.initial[r];
  Pack<T, NV> x, w[MW], win[MH];
  zero(x);
  if (r < p.q.T) x = load_part<T, NV>(xg + (long long)r * p.ldx, n, vec);  // its row, in a batch of single tokens
  float bias[NV];
#pragma unroll
  for (int k = 0; k < MW; ++k) {
    zero(w[k]);
    const int tap = k - (MW - W);
    if (tap < 0) continue;
    if (p.vec_w) {
      w[k] = load_part<T, NV>(wg + (long long)tap * p.sw_k + c0, n, n == NV);
    } else {
#pragma unroll
      for (int c = 0; c < NV; ++c)
        if (c < n) w[k].v[c] = wg[(long long)tap * p.sw_k + (long long)(c0 + c) * p.sw_d];
    }
  }
#pragma unroll
  for (int c = 0; c < NV; ++c)
    bias[c] = p.bias != nullptr && c < n ? to_f(reinterpret_cast<const T*>(p.bias)[c0 + c]) : 0.f;
#pragma unroll
  for (int h = 0; h < MH; ++h) zero(win[h]);
  int slot = -1;
  if (p.state != nullptr && b < e) {
    if (raw >= p.num_slots && p.err != nullptr && c0 == 0) atomicOr(p.err, 1);
    slot = raw >= 0 && raw < p.num_slots ? raw : -1;
    if (slot >= 0 && initial != 0) conv_load_state<T, NV, MH>(p, slot, c0, n, H, win, WT > 1);
  }
  for (int t = b; t < e; ++t) {
    if (t != r || t != b) x = load_part<T, NV>(xg + (long long)t * p.ldx, n, vec);
    Pack<T, NV> o;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float s = bias[c];
#pragma unroll
      for (int k = 0; k < MW; ++k) {
        if (k == MW - 1)
          s = fma_io(w[k].v[c], x.v[c], s);
        else if (k >= MW - W)
          s = fma_io(w[k].v[c], win[k < MH ? k : 0].v[c], s);
      }
      o.v[c] = from_f<T>(p.silu ? s * sigmoid_t<T>(s) : s);
    }
    store_part<T, NV>(yg + (long long)t * p.D, o, n, vec);
#pragma unroll
    for (int h = 0; h < MH; ++h) win[h] = h + 1 < MH ? win[h + 1 < MH ? h + 1 : h] : x;
  }
  if (slot >= 0) conv_store_state<T, NV, MH>(p, slot, c0, n, H, win, WT > 1);
  if (p.zero_rest) {
    Pack<T, NV> z;
    zero(z);
    if (r == 0)
      for (int t = 0; t < b; ++t) store_part<T, NV>(yg + (long long)t * p.D, z, n, vec);
    if (r == p.q.nseq - 1)
      for (int t = e; t < p.q.T; ++t) store_part<T, NV>(yg + (long long)t * p.D, z, n, vec);
  }
}

// Backward (zero history):
//   dpre[t] = dout[t] (times SiLU'(pre[t]), pre recomputed from x)
//   dx[t]   = sum_k w[k] dpre[t + W-1-k]      over tokens of t's sequence
//   dw[k]   = sum_t dpre[t] x[t + k - W + 1],  dbias = sum_t dpre[t]
// A thread walks its run and the W-1 tokens behind it in order; token t adds
// w[k] dpre[t] to the open sums of tokens t-W+1 .. t that its sequence has, and
// the sum of token t-W+1 (of t-MW+1 with a runtime W) is then complete. dw and dbias of the run stay in
// registers, the block's four runs are added in shared memory, and one row of
// partial sums per block goes to `part`, which ssm_conv_reduce_kernel adds in
// a fixed order: the same call gives the same bits.
template <typename T, int NV, int WT>
__global__ void __launch_bounds__(128) ssm_conv_bwd_kernel(const ConvParams p) {
  constexpr int MW = WT > 0 ? WT : -WT;
  constexpr int MH = MW > 1 ? MW - 1 : 1;
  constexpr int NC = (NV + 1) / 2;
  extern __shared__ __align__(16) float red[];  // the rings; then [runs][W + 1][32 * NV]
  const int W = WT > 0 ? WT : p.W;
  const int H = W - 1;
  const int lane = threadIdx.x & 31;
  const int cb = (int)(blockIdx.x % p.nblk) * 32 * NV;
  const int c0 = cb + lane * NV;
  const int n = max(0, min(NV, p.D - c0));
  const bool vec = NV > 1 && n == NV;
  const long long first = ((long long)(blockIdx.x / p.nblk) * blockDim.y + threadIdx.y) * p.L;
  pdl_wait();
  pdl_trigger();
  Chans<NV> dw[MW], db;
  conv_zero<NV>(dw);
#pragma unroll
  for (int c = 0; c < NC; ++c) db[c] = 0ull;
  if (first < p.q.T) {
    const int t0 = (int)first;
    const int t1 = (int)min((long long)p.q.T, first + p.L);
    const T* xg = reinterpret_cast<const T*>(p.x) + c0;
    T* dxg = reinterpret_cast<T*>(p.dx) + c0;
    const int t2 = t1 + MW - 1;  // one behind the token that completes the run's last
    const int tin = min(t2, p.q.T);
    ConvRing<T, NV> rx, rd;
    char* mine = reinterpret_cast<char*>(red) + threadIdx.y * 2 * ConvRing<T, NV>::kBytes;
    rx.mine = reinterpret_cast<Pack<T, NV>*>(mine) + lane;
    rd.mine = reinterpret_cast<Pack<T, NV>*>(mine + ConvRing<T, NV>::kBytes) + lane;
    rx.g = xg;
    rd.g = reinterpret_cast<const T*>(p.dout) + c0;
    rx.ld = p.ldx;
    rd.ld = p.D;
    rx.n = rd.n = n;
    auto fetch = [&](int group, int t) {  // both operands' rows are one group of copies
      if (NV > 1) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          if (t + i < tin && n == NV) {
            const int at = (group % kStages * kGroup + i) * 32;
            copy_async<NV * (int)sizeof(T)>(rx.mine + at, rx.g + (long long)(t + i) * rx.ld, true);
            copy_async<NV * (int)sizeof(T)>(rd.mine + at, rd.g + (long long)(t + i) * rd.ld, true);
          }
        copy_commit();
      }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i, t0 + i * kGroup);
    Chans<NV> w[MW], bias, win[MH], acc[MW];
    conv_weights<T, NV>(p, c0, n, W, w, bias);
    conv_zero<NV>(win);
    conv_zero<NV>(acc);
    const SeqView sv(p.q, lane);
    Seg g = sv.at(t0);
    if (g.in && t0 > g.b) {
#pragma unroll
      for (int h = 0; h < MH; ++h)
        if (h >= MH - H && t0 - MH + h >= g.b)
          widen<T, NV>(load_part<T, NV>(xg + (long long)(t0 - MH + h) * p.ldx, n, vec), win[h]);
    }
    // Token ti of the sequence g: its dpre, what it adds, and the window. `all`:
    // a token of the run with all its W inputs in the sequence.
    auto token = [&](int ti, const Pack<T, NV>& xr, const Pack<T, NV>& dr, auto all) {
      constexpr bool kAll = decltype(all)::value;
      Chans<NV> x, d;
      widen<T, NV>(xr, x);
      widen<T, NV>(dr, d);
      if (p.silu) {
        Chans<NV> pre;
        conv_pre<NV>(w, bias, win, x, W, pre);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float v[2], o[2] = {0.f, 0.f};
          unpack2(pre[c], v[0], v[1]);
#pragma unroll
          for (int i = 0; i < (NV > 1 ? 2 : 1); ++i) {
            const float s = sigmoid_t<T>(v[i]);
            o[i] = s * fmaf(v[i], 1.f - s, 1.f);
          }
          d[c] = f2_mul(d[c], pack2(o[0], o[1]));
        }
      }
      const int pos = ti - g.b;
      const bool mine = kAll || ti < t1;
#pragma unroll
      for (int k = 0; k < MW; ++k) {
        // (a tap ahead of the sequence has no input and no token to add to)
        if (k >= MW - W && (kAll || MW - 1 - k <= pos)) {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            acc[k][c] = f2_fma(w[k][c], d[c], acc[k][c]);
            if (mine) dw[k][c] = f2_fma(d[c], k == MW - 1 ? x[c] : win[k < MH ? k : 0][c], dw[k][c]);
          }
        }
      }
      if (mine) {
#pragma unroll
        for (int c = 0; c < NC; ++c) db[c] = f2_add(db[c], d[c]);
      }
      conv_push<NV>(win, x);
    };
    // dx of token `to` is complete: store it and move the sums on
    auto complete = [&](int to, bool store) {
      if (store) store_part<T, NV>(dxg + (long long)to * p.D, narrow<T, NV>(acc[0]), n, vec);
#pragma unroll
      for (int k = 0; k < MW; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          acc[k][c] = k + 1 < MW ? acc[k + 1 < MW ? k + 1 : k][c] : 0ull;
        }
    };
    int group = 0;
    for (int t = t0; t < t2; t += kGroup, ++group) {
      if (NV > 1) ring_wait();
      fetch(group + kStages - 1, t + (kStages - 1) * kGroup);
      if (g.in && t + kGroup <= min(g.e, t1) && t - g.b >= H && t - (MW - 1) >= t0) {
        Pack<T, NV> x[kGroup], dy[kGroup];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          x[i] = rx.row(group, t, i);
          dy[i] = rd.row(group, t, i);
        }
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          token(t + i, x[i], dy[i], std::true_type());
          complete(t + i - (MW - 1), true);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kGroup && t + i < t2; ++i) {
          const int ti = t + i;
          if (ti < tin && ti >= g.e) g = sv.next(g);
          if (ti < tin && g.in) {
            if (ti == g.b) conv_zero<NV>(win);
            token(ti, rx.row(group, t, i), rd.row(group, t, i), std::false_type());
          }
          complete(ti - (MW - 1), ti - (MW - 1) >= t0 && ti - (MW - 1) < t1);
        }
      }
    }
  }
  __syncthreads();  // (every warp is done with its ring)
  constexpr int CW = 32 * NV;
  float* mine = red + (long long)threadIdx.y * (W + 1) * CW + lane * NV;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    float v[2];
#pragma unroll
    for (int k = 0; k < MW; ++k) {
      unpack2(dw[k][c / 2], v[0], v[1]);
      if (k >= MW - W) mine[(k - (MW - W)) * CW + c] = v[c % 2];
    }
    unpack2(db[c / 2], v[0], v[1]);
    mine[W * CW + c] = v[c % 2];
  }
  __syncthreads();
  const long long row = blockIdx.x / p.nblk;
  for (int i = threadIdx.y * 32 + lane; i < (W + 1) * CW; i += 32 * blockDim.y) {
    float s = 0.f;
    for (int r = 0; r < (int)blockDim.y; ++r) s += red[(long long)r * (W + 1) * CW + i];
    const int c = cb + i % CW;
    if (c < p.D) p.part[(row * (W + 1) + i / CW) * p.D + c] = s;
  }
}

// dw[k, d], dbias[d] = the sums of `part` over its rows. 32 columns per block,
// eight threads a column, added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) ssm_conv_reduce_kernel(const float* part, T* dw, T* dbias, long long rows,
                                                              int D, int W) {
  __shared__ float red[8][33];
  pdl_wait();
  pdl_trigger();
  const long long cols = (long long)(W + 1) * D;
  const long long col = (long long)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (col < cols)
#pragma unroll 4
    for (long long r = threadIdx.y; r < rows; r += 8) s += part[r * cols + col];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
    if (col < (long long)W * D)
      dw[col] = from_f<T>(s);
    else if (dbias != nullptr)
      dbias[col - (long long)W * D] = from_f<T>(s);
  }
}

}  // namespace greta
