// Short causal depthwise convolution with static filters:
//
//   pre[t, d] = bias[d] + sum_k w[k, d] x[t + k - W + 1, d]   (tap W-1 = current token)
//   out[t, d] = pre or SiLU(pre)
//
// Bound by HBM: 2 W + 4 operations per element read and written. A thread owns
// NV channels (16 bytes of a row) of a run of L consecutive tokens of the
// packed stream and keeps the last W-1 inputs in registers, so a row is read
// once, plus W-1 rows ahead of each run from L2. Runs are cut by position, so
// ragged batches are balanced; a run's warp follows the sequence borders in
// it (ssm_common.cuh). W is a template parameter for 2, 3 and 4 (the kernel
// sizes in use); WT = -8 and -16 take any W up to that.
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
  int vec;    // rows of x and y are whole aligned vectors
  int vec_w;  // the filters' rows too (sw_d == 1)
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

// The filters of this thread's channels in their own type (the mixed-precision
// FMA widens them) and the bias.
template <typename T, int NV, int MW>
__device__ __forceinline__ void conv_weights(const ConvParams& p, int c0, int n, int W, Pack<T, NV> (&w)[MW],
                                             float (&bias)[NV]) {
  const T* wg = reinterpret_cast<const T*>(p.w);
#pragma unroll
  for (int k = 0; k < MW; ++k) {
    zero(w[k]);
    if (k < W) {
      if (p.vec_w) {
        w[k] = load_part<T, NV>(wg + (long long)k * p.sw_k + c0, n, n == NV);
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c)
          if (c < n) w[k].v[c] = wg[(long long)k * p.sw_k + (long long)(c0 + c) * p.sw_d];
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NV; ++c)
    bias[c] = p.bias != nullptr && c < n ? to_f(reinterpret_cast<const T*>(p.bias)[c0 + c]) : 0.f;
}

// The slot's W-1 inputs of this thread's channels, oldest first.
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
      if (h < H) win[h] = load_part<T, NV>(base + (long long)h * p.s_h + c0, NV, true);
  } else {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h < H) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
          win[h].v[c] = c < n ? base[(long long)(c0 + c) * p.s_d + (long long)h * p.s_h] : from_f<T>(0.f);
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
      if (h < H) store_part<T, NV>(base + (long long)h * p.s_h + c0, win[h], NV, true);
  } else {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h < H) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
          if (c < n) base[(long long)(c0 + c) * p.s_d + (long long)h * p.s_h] = win[h].v[c];
      }
  }
}

// Pre-activation of one token: taps oldest first, win[h] under tap h, the
// token itself under tap W-1.
template <typename T, int NV, int MW, int MH>
__device__ __forceinline__ void conv_pre(const Pack<T, NV> (&w)[MW], const float (&bias)[NV],
                                         const Pack<T, NV> (&win)[MH], const Pack<T, NV>& x, int W,
                                         float (&pre)[NV]) {
#pragma unroll
  for (int c = 0; c < NV; ++c) pre[c] = bias[c];
#pragma unroll
  for (int k = 0; k < MW; ++k) {
    if (k < W - 1) {
#pragma unroll
      for (int c = 0; c < NV; ++c) pre[c] = fma_io(w[k].v[c], win[k < MH ? k : 0].v[c], pre[c]);
    } else if (k == W - 1) {
#pragma unroll
      for (int c = 0; c < NV; ++c) pre[c] = fma_io(w[k].v[c], x.v[c], pre[c]);
    }
  }
}

template <typename T, int NV, int MH>
__device__ __forceinline__ void conv_push(Pack<T, NV> (&win)[MH], const Pack<T, NV>& x, int H) {
#pragma unroll
  for (int h = 0; h < MH; ++h) {
    if (h < H - 1 && h + 1 < MH) win[h] = win[h + 1 < MH ? h + 1 : h];
    if (h == H - 1) win[h] = x;
  }
}

// PACKED: history from and to the requests' cache slots; else zero history.
template <typename T, int NV, int WT, bool PACKED>
__global__ void __launch_bounds__(128) ssm_conv_fwd_kernel(const ConvParams p) {
  constexpr int MW = WT > 0 ? WT : -WT;
  constexpr int MH = MW > 1 ? MW - 1 : 1;
  const int W = WT > 0 ? WT : p.W;
  const int H = W - 1;
  const int lane = threadIdx.x & 31;
  const int c0 = ((int)(blockIdx.x % p.nblk) * 32 + lane) * NV;
  const int n = min(NV, p.D - c0);  // may be <= 0: a lane without channels
  const bool vec = p.vec && n == NV;
  const long long first = ((long long)(blockIdx.x / p.nblk) * blockDim.y + threadIdx.y) * p.L;
  pdl_wait();
  pdl_trigger();
  if (first >= p.q.T) return;
  int t = (int)first;
  int t1 = (int)min((long long)p.q.T, first + p.L);
  Seg g;
  // one token per run: in a batch of single tokens, token t is sequence t
  if (PACKED && p.L == 1 && t < p.q.nseq && seq_start(p.q, t) == t && seq_start(p.q, t + 1) == t + 1)
    g = Seg{t, t, t + 1, true};
  else
    g = seg_at(p.q, t, lane);

  Pack<T, NV> w[MW];
  float bias[NV];
  conv_weights(p, c0, n, W, w, bias);
  const T* xg = reinterpret_cast<const T*>(p.x) + c0;
  T* yg = reinterpret_cast<T*>(p.y) + c0;
  Pack<T, NV> win[MH];
#pragma unroll
  for (int h = 0; h < MH; ++h) zero(win[h]);

  int tend = t1;
  if (PACKED && H > 0) {
    // A request's first W-1 tokens stay with the run that has its first: that
    // run alone reads the slot (and writes it, below), so no other run's write
    // can come between.
    if (g.in && t > g.b && t - g.b < H) {
      const int skip = min(g.b + H, g.e);
      if (skip >= t1) return;
      t = skip;
      if (t == g.e) g = seg_next(p.q, g);
    }
    if (t1 < p.q.T) {
      const Seg last = seg_at(p.q, t1, lane);
      if (last.in && t1 > last.b && t1 - last.b < H) tend = min(last.b + H, last.e);
    }
  }
  // inside a sequence: the inputs ahead of the run (t - H + h >= 0 where kept)
  if (g.in && t > g.b) {
#pragma unroll
    for (int h = 0; h < MH; ++h)
      if (h < H && t - H + h >= g.b) win[h] = load_part<T, NV>(xg + (long long)(t - H + h) * p.ldx, n, vec);
  }
  int slot = -1;
  while (t < tend) {
    if (t == g.b && g.in) {
#pragma unroll
      for (int h = 0; h < MH; ++h) zero(win[h]);
      slot = -1;
      if (PACKED && p.state != nullptr) {
        const int raw = p.slots[g.s];
        if (raw >= p.num_slots && p.err != nullptr && c0 == 0) atomicOr(p.err, 1);
        slot = raw >= 0 && raw < p.num_slots ? raw : -1;
        if (slot >= 0 && p.initial[g.s] != 0) conv_load_state<T, NV, MH>(p, slot, c0, n, H, win, WT > 1);
        if (slot >= 0 && g.e > tend) {
          // the request ends in a later run: its last W-1 inputs (it has more
          // than W-1) straight from x
          Pack<T, NV> fin[MH];
#pragma unroll
          for (int h = 0; h < MH; ++h) {
            zero(fin[h]);
            if (h < H) fin[h] = load_part<T, NV>(xg + (long long)(g.e - H + h) * p.ldx, n, vec);
          }
          conv_store_state<T, NV, MH>(p, slot, c0, n, H, fin, WT > 1);
          slot = -1;
        }
      }
    }
    const int stop = min(g.e, tend);
    if (!g.in) {
      if (p.zero_rest) {
        Pack<T, NV> z;
        zero(z);
        for (; t < stop; ++t) store_part<T, NV>(yg + (long long)t * p.D, z, n, vec);
      }
      t = stop;
    } else {
      while (t < stop) {
        constexpr int U = 4;  // rows in flight
        Pack<T, NV> x[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (t + i < stop) x[i] = load_part<T, NV>(xg + (long long)(t + i) * p.ldx, n, vec);
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (t + i < stop) {
            float pre[NV];
            conv_pre(w, bias, win, x[i], W, pre);
            conv_push<T, NV, MH>(win, x[i], H);
            Pack<T, NV> o;
#pragma unroll
            for (int c = 0; c < NV; ++c) o.v[c] = from_f<T>(p.silu ? pre[c] * sigmoidf_(pre[c]) : pre[c]);
            store_part<T, NV>(yg + (long long)(t + i) * p.D, o, n, vec);
          }
        t = min(t + U, stop);
      }
      if (PACKED && t == g.e && slot >= 0) {
        conv_store_state<T, NV, MH>(p, slot, c0, n, H, win, WT > 1);
        slot = -1;
      }
    }
    if (t < tend) g = seg_next(p.q, g);
  }
}

// Backward (zero history):
//   dpre[t] = dout[t] (times SiLU'(pre[t]), pre recomputed from x)
//   dx[t]   = sum_k w[k] dpre[t + W-1-k]      over tokens of t's sequence
//   dw[k]   = sum_t dpre[t] x[t + k - W + 1],  dbias = sum_t dpre[t]
// A thread walks its run and the W-1 tokens behind it in order; token t adds
// w[k] dpre[t] to the open sums of tokens t-W+1 .. t that its sequence has, and
// the sum of token t-W+1 is then complete. dw and dbias of the run stay in
// registers, the block's four runs are added in shared memory, and one row of
// partial sums per block goes to `part`, which ssm_conv_reduce_kernel adds in
// a fixed order: the same call gives the same bits.
template <typename T, int NV, int WT>
__global__ void __launch_bounds__(128) ssm_conv_bwd_kernel(const ConvParams p) {
  constexpr int MW = WT > 0 ? WT : -WT;
  constexpr int MH = MW > 1 ? MW - 1 : 1;
  extern __shared__ float red[];  // [runs][W + 1][32 * NV]
  const int W = WT > 0 ? WT : p.W;
  const int H = W - 1;
  const int lane = threadIdx.x & 31;
  const int cb = (int)(blockIdx.x % p.nblk) * 32 * NV;
  const int c0 = cb + lane * NV;
  const int n = min(NV, p.D - c0);
  const bool vec = p.vec && n == NV;
  const long long first = ((long long)(blockIdx.x / p.nblk) * blockDim.y + threadIdx.y) * p.L;
  pdl_wait();
  pdl_trigger();
  float dw[MW][NV], db[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    db[c] = 0.f;
#pragma unroll
    for (int k = 0; k < MW; ++k) dw[k][c] = 0.f;
  }
  if (first < p.q.T) {
    const int t0 = (int)first;
    const int t1 = (int)min((long long)p.q.T, first + p.L);
    Pack<T, NV> w[MW];
    float bias[NV];
    conv_weights(p, c0, n, W, w, bias);
    const T* xg = reinterpret_cast<const T*>(p.x) + c0;
    const T* gg = reinterpret_cast<const T*>(p.dout) + c0;
    T* dxg = reinterpret_cast<T*>(p.dx) + c0;
    Seg g = seg_at(p.q, t0, lane);
    Pack<T, NV> win[MH];
    float acc[MW][NV];
#pragma unroll
    for (int h = 0; h < MH; ++h) zero(win[h]);
#pragma unroll
    for (int k = 0; k < MW; ++k)
#pragma unroll
      for (int c = 0; c < NV; ++c) acc[k][c] = 0.f;
    if (g.in && t0 > g.b) {
#pragma unroll
      for (int h = 0; h < MH; ++h)
        if (h < H && t0 - H + h >= g.b) win[h] = load_part<T, NV>(xg + (long long)(t0 - H + h) * p.ldx, n, vec);
    }
    const int t2 = t1 + H;  // one behind the last token that reaches a token of the run
    const int tin = min(t2, p.q.T);
    constexpr int U = 4;
    for (int t = t0; t < t2; t += U) {
      Pack<T, NV> x[U], dy[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        zero(x[i]);
        zero(dy[i]);
        if (t + i < tin) {
          x[i] = load_part<T, NV>(xg + (long long)(t + i) * p.ldx, n, vec);
          dy[i] = load_part<T, NV>(gg + (long long)(t + i) * p.D, n, vec);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int ti = t + i;
        if (ti < t2) {
          if (ti < tin && ti >= g.e) g = seg_next(p.q, g);
          if (ti < tin && g.in) {
            if (ti == g.b) {
#pragma unroll
              for (int h = 0; h < MH; ++h) zero(win[h]);
            }
            float d[NV];
            if (p.silu) {
              float pre[NV];
              conv_pre(w, bias, win, x[i], W, pre);
#pragma unroll
              for (int c = 0; c < NV; ++c) {
                const float sg = sigmoidf_(pre[c]);
                d[c] = to_f(dy[i].v[c]) * sg * (1.f + pre[c] * (1.f - sg));
              }
            } else {
#pragma unroll
              for (int c = 0; c < NV; ++c) d[c] = to_f(dy[i].v[c]);
            }
            const int pos = ti - g.b;
#pragma unroll
            for (int k = 0; k < MW; ++k)
              if (k < W && W - 1 - k <= pos) {
#pragma unroll
                for (int c = 0; c < NV; ++c) acc[k][c] = fmaf(to_f(w[k].v[c]), d[c], acc[k][c]);
              }
            if (ti < t1) {
#pragma unroll
              for (int c = 0; c < NV; ++c) db[c] += d[c];
#pragma unroll
              for (int k = 0; k < MW; ++k) {
                // a tap ahead of the sequence has no input (and its place in
                // the window may hold none)
                if (k < W && W - 1 - k <= pos) {
#pragma unroll
                  for (int c = 0; c < NV; ++c)
                    dw[k][c] = fmaf(d[c], to_f(k == W - 1 ? x[i].v[c] : win[k < MH ? k : 0].v[c]), dw[k][c]);
                }
              }
            }
            conv_push(win, x[i], H);
          }
          const int to = ti - H;
          if (to >= t0 && to < t1) {
            Pack<T, NV> o;
#pragma unroll
            for (int c = 0; c < NV; ++c) o.v[c] = from_f<T>(acc[0][c]);
            store_part<T, NV>(dxg + (long long)to * p.D, o, n, vec);
          }
#pragma unroll
          for (int k = 0; k < MW; ++k) {
#pragma unroll
            for (int c = 0; c < NV; ++c) {
              if (k < W - 1) acc[k][c] = acc[k + 1 < MW ? k + 1 : k][c];
              if (k == W - 1) acc[k][c] = 0.f;
            }
          }
        }
      }
    }
  }
  constexpr int CW = 32 * NV;
  float* mine = red + (long long)threadIdx.y * (W + 1) * CW + lane * NV;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
#pragma unroll
    for (int k = 0; k < MW; ++k)
      if (k < W) mine[k * CW + c] = dw[k][c];
    mine[W * CW + c] = db[c];
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
