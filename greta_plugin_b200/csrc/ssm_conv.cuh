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
// by renaming registers. 16288 x 4096, 4 taps, bf16: 53 us, 5.0 TB/s; 898 tokens
// of 8 requests 9.1 us.
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

// NV channels of a row for a lane that has them (n != 0), else zeros; and back.
// (The host takes NV > 1 only where every row is whole aligned vectors: a lane
// has all of its channels or none.)
template <typename T, int NV>
__device__ __forceinline__ Pack<T, NV> get_row(const T* g, int n) {
  Pack<T, NV> r;
  zero(r);
  if (n != 0) r = load_part<T, NV>(g, NV, true);
  return r;
}
template <typename T, int NV>
__device__ __forceinline__ void put_row(T* g, const Pack<T, NV>& r, int n) {
  if (n != 0) store_part<T, NV>(g, r, NV, true);
}

// A lane's part of the ring for one operand: [stage][token][lane] vectors.
// Single elements (rows that are not whole vectors) are loaded when the group
// is due. Stages are byte offsets, rows a pointer that moves on: with products
// of token and stride a row took as many instructions for addresses as for sums.
template <typename T, int NV>
struct ConvRing {
  static constexpr int kRow = 32 * NV * (int)sizeof(T), kStage = kGroup * kRow;
  static constexpr int kBytes = kStages * kStage;  // of a warp, a power of two
  static __device__ __forceinline__ int after(int stage) { return (stage + kStage) & (kBytes - 1); }
  const char* mine;
  unsigned to;    // the same in the shared window
  const T* next;  // the lane's first channel of the next row to be fetched
  const T* g;     // ... of row 0
  long long ld;
  int n;
  __device__ __forceinline__ ConvRing(char* s, int lane, const void* base, long long ld_, int c0, int n_, int t) {
    mine = s + lane * (NV * (int)sizeof(T));
    to = (unsigned)__cvta_generic_to_shared(mine);
    g = reinterpret_cast<const T*>(base) + c0;
    next = g + t * ld_;
    ld = ld_;
    n = n_;
  }
  // Rows t .. t + 3 that are below `end`, the next ones, into a stage.
  __device__ __forceinline__ void fetch(int stage, int t, int end) {
    if constexpr (NV > 1) {
      constexpr int B = NV * (int)sizeof(T);
      static_assert(kGroup == 4, "written out");
      const T *r0 = next, *r1 = r0 + ld, *r2 = r1 + ld, *r3 = r2 + ld;
      next = r3 + ld;
      if (n == 0) return;
      const unsigned s = to + stage;
      if (t + kGroup <= end) {
        copy_async_to<B, 0>(s, r0);
        copy_async_to<B, kRow>(s, r1);
        copy_async_to<B, 2 * kRow>(s, r2);
        copy_async_to<B, 3 * kRow>(s, r3);
      } else {
        if (t < end) copy_async_to<B, 0>(s, r0);
        if (t + 1 < end) copy_async_to<B, kRow>(s, r1);
        if (t + 2 < end) copy_async_to<B, 2 * kRow>(s, r2);
      }
    }
  }
  // Row t + i of the group that begins at t.
  __device__ __forceinline__ Pack<T, NV> row(int stage, int t, int i) const {
    if constexpr (NV > 1) return load_part<T, NV>(reinterpret_cast<const T*>(mine + stage + i * kRow), NV, true);
    return get_row<T, NV>(g + (t + i) * ld, n);
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
  for (int c = 0; c < NV; c += 2) {
    if constexpr (NV % 4 == 0) {
      if (c % 4 == 0) {
        Pack<T, 4> four;
#pragma unroll
        for (int e = 0; e < 4; ++e) four.v[e] = r.v[c + e];
        const float4 v = widen4(four);
        o[c / 2] = pack2(v.x, v.y);
        o[c / 2 + 1] = pack2(v.z, v.w);
      }
    } else {
      o[c / 2] = pack2(to_f(r.v[c]), c + 1 < NV ? to_f(r.v[c + 1 < NV ? c + 1 : c]) : 0.f);
    }
  }
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
__device__ __forceinline__ void conv_weights(const ConvParams& p, int c0, int n, int W, Pack<T, NV> (&w)[MW],
                                             float (&bias)[NV]) {
  const T* wg = reinterpret_cast<const T*>(p.w);
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

// The same from operands in the element type (fma_io: exact products, fp32 sums),
// with SiLU, rounded to the output.
template <typename T, int NV, int MW, int MH>
__device__ __forceinline__ Pack<T, NV> conv_out(const Pack<T, NV> (&w)[MW], const float (&bias)[NV],
                                                const Pack<T, NV> (&win)[MH], const Pack<T, NV>& x, int W, bool silu) {
  float s[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    s[c] = bias[c];
#pragma unroll
    for (int k = 0; k < MW; ++k) {
      if (k == MW - 1)
        s[c] = fma_io(w[k].v[c], x.v[c], s[c]);
      else if (k >= MW - W)
        s[c] = fma_io(w[k].v[c], win[k < MH ? k : 0].v[c], s[c]);
    }
  }
  Chans<NV> o;
#pragma unroll
  for (int c = 0; c < NV; c += 2) {
    o[c / 2] = pack2(s[c], c + 1 < NV ? s[c + 1 < NV ? c + 1 : c] : 0.f);
    if (silu) o[c / 2] = f2_mul(o[c / 2], sigmoid2<T>(o[c / 2]));
  }
  return narrow<T, NV>(o);
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

// PACKED: history from and to the requests' cache slots; else zero history.
template <typename T, int NV, int WT, bool PACKED>
__global__ void __launch_bounds__(128, WT > -16 ? 4 : 2) ssm_conv_fwd_kernel(const ConvParams p) {
  constexpr int MW = WT > 0 ? WT : -WT;
  constexpr int MH = MW > 1 ? MW - 1 : 1;
  const int W = WT > 0 ? WT : p.W;
  const int H = W - 1;
  const int lane = threadIdx.x & 31;
  const int c0 = ((int)(blockIdx.x % p.nblk) * 32 + lane) * NV;
  const int n = max(0, min(NV, p.D - c0));  // 0: a lane without channels
  const long long first = ((long long)(blockIdx.x / p.nblk) * blockDim.y + threadIdx.y) * p.L;
  pdl_wait();
  pdl_trigger();
  if (first >= p.q.T) return;
  int t = (int)first;
  int t1 = (int)min((long long)p.q.T, first + p.L);
  const T* xg = reinterpret_cast<const T*>(p.x) + c0;
  extern __shared__ float4 ring_smem[];
  using Ring = ConvRing<T, NV>;
  // filters and window in the element type: nothing to widen or to narrow
  Pack<T, NV> w[MW], win[MH];
  float bias[NV];
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
  Ring ring(reinterpret_cast<char*>(ring_smem) + threadIdx.y * Ring::kBytes, lane, p.x, p.ldx, c0, n, t);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    ring.fetch(i * Ring::kStage, t + i * kGroup, tend);
    copy_commit();
  }
  conv_weights<T, NV>(p, c0, n, W, w, bias);
  auto forget = [&] {
#pragma unroll
    for (int h = 0; h < MH; ++h) zero(win[h]);
  };
  forget();
  // inside a sequence: the inputs ahead of the run (t - H + h >= 0 where kept)
  if (g.in && t > g.b) {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h >= MH - H && t - MH + h >= g.b)
        win[h] = get_row<T, NV>(xg + (long long)(t - MH + h) * p.ldx, n);
  }
  int slot = -1;
  Pack<T, NV> old[MH];  // the slot's inputs of a request that begins here
#pragma unroll
  for (int h = 0; h < MH; ++h) zero(old[h]);
  // the first token of sequence g
  auto begin = [&] {
    forget();
    slot = -1;
    if (!PACKED || (p.state == nullptr && p.err == nullptr)) return;
    const int raw = p.slots[g.s], initial = p.initial[g.s];
    if (raw >= p.num_slots && p.err != nullptr && c0 == 0) atomicOr(p.err, 1);
    if (p.state == nullptr) return;  // (no slots, or no history: asked for the check alone)
    slot = raw >= 0 && raw < p.num_slots ? raw : -1;
#pragma unroll
    for (int h = 0; h < MH; ++h) zero(old[h]);
    if (slot >= 0 && initial != 0) {
      conv_load_state<T, NV, MH>(p, slot, c0, n, H, old, WT > 1);
#pragma unroll
      for (int h = 0; h < MH; ++h)
        if (h >= MH - H) win[h] = old[h];
    }
    if (slot >= 0 && g.e > tend) {
      // the request ends in a later run: its last W-1 inputs (it has more
      // than W-1) straight from x
      Pack<T, NV> fin[MH];
#pragma unroll
      for (int h = 0; h < MH; ++h) {
        zero(fin[h]);
        // (offsets that fall may give it fewer: no row ahead of x all the same)
        if (h >= MH - H) fin[h] = get_row<T, NV>(xg + (long long)max(g.e - MH + h, 0) * p.ldx, n);
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
        fin[h] = get_row<T, NV>(xg + (long long)(g.e - MH + h) * p.ldx, n);
      } else {
#pragma unroll
        for (int k = 0; k < MH; ++k)
          if (k == h + len) fin[h] = old[k];
      }
    }
    conv_store_state<T, NV, MH>(p, slot, c0, n, H, fin, WT > 1);
    slot = -1;
  };
  T* y = reinterpret_cast<T*>(p.y) + t * (long long)p.D + c0;  // the next token's
  auto token = [&](const Pack<T, NV>& raw) {
    put_row<T, NV>(y, conv_out<T, NV>(w, bias, win, raw, W, p.silu), n);
#pragma unroll
    for (int h = 0; h < MH; ++h) win[h] = h + 1 < MH ? win[h + 1 < MH ? h + 1 : h] : raw;
    y += p.D;
  };

  // groups from `lo` + 1 up to `hi` lie in g behind its first and ahead of its
  // last token
  int lo = g.in ? g.b : INT_MAX, hi = min(g.e - 1, tend);
  int get = 0, put = (kStages - 1) * Ring::kStage;
  for (; t < tend; t += kGroup, get = Ring::after(get), put = Ring::after(put)) {
    if (NV > 1) ring_wait();
    // (into the stage of the group before this one)
    ring.fetch(put, t + (kStages - 1) * kGroup, tend);
    if (NV > 1) copy_commit();
    if (t > lo && t + kGroup <= hi) {
      Pack<T, NV> x[kGroup];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) x[i] = ring.row(get, t, i);
#pragma unroll
      for (int i = 0; i < kGroup; ++i) token(x[i]);
    } else {
#pragma unroll 1
      for (int i = 0; i < kGroup && t + i < tend; ++i) {
        const int ti = t + i;
        if (ti >= g.e) g = sv.next(g);
        if (g.in) {
          if (ti == g.b) begin();
          token(ring.row(get, t, i));
          if (ti + 1 == g.e) finish();
        } else {
          Pack<T, NV> z;
          zero(z);
          if (p.zero_rest) put_row<T, NV>(y, z, n);
          y += p.D;
        }
      }
      lo = g.in ? g.b : INT_MAX;
      hi = min(g.e - 1, tend);
    }
  }
}

// Batches of (nearly) one token per request: a warp has the channels of one
// request and walks its tokens, with all of a step's warps running at once and
// the metadata, the first token's row and the filters asked for together: three
// latencies in a row. 256 requests of 4096 channels, 4 taps, bf16: 7.6 us.
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
  pdl_wait();
  pdl_trigger();
  if (r >= p.q.nseq) return;
  const int b = seq_start(p.q, r), e = seq_start(p.q, r + 1), raw = p.slots[r], initial = p.initial[r];
  Pack<T, NV> x, w[MW], win[MH];
  zero(x);
  if (r < p.q.T) x = load_part<T, NV>(xg + (long long)r * p.ldx, n, vec);  // its row, in a batch of single tokens
  float bias[NV];
  conv_weights<T, NV>(p, c0, n, W, w, bias);
#pragma unroll
  for (int h = 0; h < MH; ++h) zero(win[h]);
  int slot = -1;
  if (b < e && raw >= p.num_slots && p.err != nullptr && c0 == 0) atomicOr(p.err, 1);
  if (p.state != nullptr && b < e) {
    slot = raw >= 0 && raw < p.num_slots ? raw : -1;
    if (slot >= 0 && initial != 0) conv_load_state<T, NV, MH>(p, slot, c0, n, H, win, WT > 1);
  }
  for (int t = b; t < e; ++t) {
    if (t != r || t != b) x = load_part<T, NV>(xg + (long long)t * p.ldx, n, vec);
    const Pack<T, NV> o = conv_out<T, NV>(w, bias, win, x, W, p.silu);
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
// a fixed order: the same call gives the same bits. Four channels a thread (sums,
// filters and windows of eight in fp32 do not fit 128 registers): 102 instructions
// a token for 12 elements read and written, so issue and fp32 pipe (45 and 44 %
// busy at 16 warps an SM) are ahead of HBM: 16288 x 4096, 4 taps, bf16 100 us,
// 4.0 TB/s.
template <typename T, int NV, int WT>
__global__ void __launch_bounds__(128, WT > -16 ? 4 : 2) ssm_conv_bwd_kernel(const ConvParams p) {
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
    const int t2 = t1 + MW - 1;  // one behind the token that completes the run's last
    const int tin = min(t2, p.q.T);
    using Ring = ConvRing<T, NV>;
    char* mine = reinterpret_cast<char*>(red) + threadIdx.y * 2 * Ring::kBytes;
    Ring rx(mine, lane, p.x, p.ldx, c0, n, t0), rd(mine + Ring::kBytes, lane, p.dout, p.D, c0, n, t0);
    auto fetch = [&](int stage, int t) {  // both operands' rows are one group of copies
      rx.fetch(stage, t, tin);
      rd.fetch(stage, t, tin);
      if (NV > 1) copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i * Ring::kStage, t0 + i * kGroup);
    Chans<NV> w[MW], bias, win[MH], acc[MW];
    {
      Pack<T, NV> raw[MW];
      float b[NV];
      conv_weights<T, NV>(p, c0, n, W, raw, b);
#pragma unroll
      for (int k = 0; k < MW; ++k) widen<T, NV>(raw[k], w[k]);
#pragma unroll
      for (int c = 0; c < NC; ++c) bias[c] = pack2(b[2 * c], 2 * c + 1 < NV ? b[2 * c + 1 < NV ? 2 * c + 1 : 0] : 0.f);
    }
    conv_zero<NV>(win);
    conv_zero<NV>(acc);
    const SeqView sv(p.q, lane);
    Seg g = sv.at(t0);
    if (g.in && t0 > g.b) {
#pragma unroll
      for (int h = 0; h < MH; ++h)
        if (h >= MH - H && t0 - MH + h >= g.b)
          widen<T, NV>(get_row<T, NV>(xg + (long long)(t0 - MH + h) * p.ldx, n), win[h]);
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
          const f2 one = pack2(1.f, 1.f), s = sigmoid2<T>(pre[c]);
          d[c] = f2_mul(d[c], f2_mul(s, f2_fma(pre[c], f2_fma(s, pack2(-1.f, -1.f), one), one)));
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
    // dx of the next token is complete: store it and move the sums on
    T* dx = reinterpret_cast<T*>(p.dx) + (t0 - (MW - 1)) * (long long)p.D + c0;
    auto complete = [&](bool store) {
      if (store) put_row<T, NV>(dx, narrow<T, NV>(acc[0]), n);
      dx += p.D;
#pragma unroll
      for (int k = 0; k < MW; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          acc[k][c] = k + 1 < MW ? acc[k + 1 < MW ? k + 1 : k][c] : 0ull;
        }
    };
    // groups from `lo` up to `hi` lie in g and in the run, with all their inputs,
    // and complete tokens of the run
    auto from = [&] { return g.in ? max(g.b + H, t0 + MW - 1) : INT_MAX; };
    int lo = from(), hi = min(g.e, t1);
    int get = 0, put = (kStages - 1) * Ring::kStage;
    for (int t = t0; t < t2; t += kGroup, get = Ring::after(get), put = Ring::after(put)) {
      if (NV > 1) ring_wait();
      fetch(put, t + (kStages - 1) * kGroup);
      if (t >= lo && t + kGroup <= hi) {
        Pack<T, NV> x[kGroup], dy[kGroup];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          x[i] = rx.row(get, t, i);
          dy[i] = rd.row(get, t, i);
        }
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          token(t + i, x[i], dy[i], std::true_type());
          complete(true);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kGroup && t + i < t2; ++i) {
          const int ti = t + i;
          if (ti < tin && ti >= g.e) g = sv.next(g);
          if (ti < tin && g.in) {
            if (ti == g.b) conv_zero<NV>(win);
            token(ti, rx.row(get, t, i), rd.row(get, t, i), std::false_type());
          }
          complete(ti - (MW - 1) >= t0 && ti - (MW - 1) < t1);
        }
        lo = from();
        hi = min(g.e, t1);
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
