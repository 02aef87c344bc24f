// Shared device code of the state-space operators (short causal convolution,
// selective scan): where a packed stream's sequences begin, vector loads of
// channel rows, and the packed fp32 pipe on 64-bit register pairs.
//
// Both operators cut the packed stream of T tokens into ranges by position,
// not by sequence: a range may begin inside a sequence and hold any number of
// them, so one long sequence and thousands of one-token ones give the same
// grid. A warp walks its range segment by segment (Seg); what it asks of the
// offsets is the same in all lanes.
#pragma once

#include <climits>

#include "dynconv_common.cuh"

namespace greta {

// The sequences of a packed stream: token offsets starts[0 .. nseq] (null: one
// sequence of all T tokens). Offsets are clamped to [0, T].
struct Seqs {
  const void* starts;
  int is64;
  int nseq;
  int T;
};

__device__ __forceinline__ int seq_start(const Seqs& q, int i) {
  if (q.starts == nullptr) return i <= 0 ? 0 : q.T;
  return (int)clampll(load_idx(q.starts, i, q.is64), 0, q.T);
}

// A run of tokens [b, e) that one sequence s holds (in), or that none does
// (ahead of the first sequence, s = -1, or behind the last, s = nseq).
struct Seg {
  int s, b, e;
  bool in;
};

// The offsets as a warp asks for them; every lane asks the same. Up to 31
// sequences are read once, an offset per lane (a question is then a ballot or a
// shuffle: a lookup's loads one after another are what short runs wait for).
struct SeqView {
  Seqs q;
  int lane, mine;
  bool held;

  __device__ __forceinline__ SeqView(const Seqs& seqs, int lane_) : q(seqs), lane(lane_) {
    held = q.nseq < 32;
    mine = held && lane <= q.nseq ? seq_start(q, lane) : INT_MAX;
  }

  __device__ __forceinline__ int start(int i) const {
    return held ? __shfl_sync(0xffffffffu, mine, i) : seq_start(q, i);
  }

  // The largest s in [-1, nseq] with start(s) <= t (-1: t is ahead of the first
  // sequence, nseq: behind the last). 32 probes a round, so two rounds for a
  // thousand sequences. Ends on any contents of the offsets.
  __device__ __forceinline__ int find(int t) const {
    if (held) return __popc(__ballot_sync(0xffffffffu, mine <= t)) - 1;
    int lo = -1, hi = q.nseq + 1;
    while (hi - lo > 1) {
      const int step = (hi - lo - 1 + 31) / 32;
      const int idx = lo + step * (lane + 1);
      const bool ok = idx < hi && seq_start(q, idx) <= t;
      const int cnt = __popc(__ballot_sync(0xffffffffu, ok));
      lo += step * cnt;
      hi = min(hi, lo + step);
    }
    return lo;
  }

  __device__ __forceinline__ Seg make(int s, int t) const {
    Seg g;
    g.s = s;
    g.in = s >= 0 && s < q.nseq;
    g.b = s >= 0 ? start(s) : 0;
    g.e = s < q.nseq ? start(s + 1) : q.T;
    if (g.e <= t) g.e = t + 1;  // offsets that fall: stay on the way forward
    return g;
  }
  __device__ __forceinline__ Seg at(int t) const { return make(find(t), t); }

  // The segment that begins where `g` ends (sequences of no tokens are passed).
  __device__ __forceinline__ Seg next(const Seg& g) const {
    const int t = g.e;
    int s = g.s + 1;
    while (s < q.nseq && start(s + 1) <= t) ++s;
    Seg n = make(s, t);
    n.b = t;
    return n;
  }
};

// The ranges that a packed stream is cut into. Split: by position, L tokens
// each; a sequence over several ranges needs carries between them. Whole: range
// i takes the sequences that begin in its L tokens, so none needs a carry, but
// the longest sequence is one warp's walk, as are the rows ahead of the first and
// behind the last; taken where each is at most `limit` tokens (up to 31
// sequences; the carries of many short ones cost little).
struct Ranges {
  int L;
  bool whole;

  __device__ __forceinline__ Ranges(const SeqView& v, int L_, int limit) : L(L_), whole(false) {
    if (!v.held) return;
    const int next = __shfl_down_sync(0xffffffffu, v.mine, 1);
    int run = v.lane < v.q.nseq ? next - v.mine : v.lane == v.q.nseq ? v.q.T - v.mine : 0;
    if (v.lane == 0) run = max(run, v.mine);
    whole = __reduce_max_sync(0xffffffffu, run) <= limit;
  }

  // The first token of range i.
  __device__ __forceinline__ int begin(const SeqView& v, int i) const {
    const int p = (int)min((long long)i * L, (long long)v.q.T);
    if (!whole || i == 0) return p;
    const unsigned m = __ballot_sync(0xffffffffu, v.lane <= v.q.nseq && v.mine >= p);
    return m == 0 ? v.q.T : min(v.q.T, __shfl_sync(0xffffffffu, v.mine, __ffs(m) - 1));
  }
};

// NV consecutive elements of a row as fp32. vec: the row starts on a whole
// vector and all NV are there; else one by one, `n` of them, the rest zero.
template <typename T, int NV>
__device__ __forceinline__ Pack<T, NV> load_part(const T* ptr, int n, bool vec) {
  Pack<T, NV> r;
  if (vec) {
    constexpr int kBytes = sizeof(T) * NV;
    if constexpr (kBytes % 16 == 0) {
      const uint4* s = reinterpret_cast<const uint4*>(ptr);
      uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) d[i] = s[i];
    } else {
      r = ld<T, NV>(ptr);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NV; ++c) r.v[c] = c < n ? ptr[c] : from_f<T>(0.f);
  }
  return r;
}

template <typename T, int NV>
__device__ __forceinline__ void store_part(T* ptr, const Pack<T, NV>& r, int n, bool vec) {
  if (vec) {
    constexpr int kBytes = sizeof(T) * NV;
    if constexpr (kBytes % 16 == 0) {
      uint4* d = reinterpret_cast<uint4*>(ptr);
      const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) d[i] = s[i];
    } else {
      st<T, NV>(ptr, r);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NV; ++c)
      if (c < n) ptr[c] = r.v[c];
  }
}

// Asynchronous copies of 4, 8 or 16 bytes into shared memory; zeros where !ok
// (the address is not read then, but has to be one).
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool ok) {
  const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
  const int n = ok ? BYTES : 0;
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
// ... to shared memory at the 32-bit address d + OFF.
template <int BYTES, int OFF>
__device__ __forceinline__ void copy_async_to(unsigned d, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1], 16;" ::"r"(d), "l"(src), "n"(OFF) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0+%2], [%1], %3;" ::"r"(d), "l"(src), "n"(OFF), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All of this thread's copies have landed.
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A whole aligned vector of NV elements into shared memory.
template <typename T, int NV>
__device__ __forceinline__ void copy_vec(T* dst, const T* src) {
  constexpr int kBytes = sizeof(T) * NV;
  if constexpr (kBytes <= 16) {
    copy_async<kBytes>(dst, src, true);
  } else {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      copy_async<16>(dst + i * (16 / sizeof(T)), src + i * (16 / sizeof(T)), true);
  }
}

// NV elements of a row into shared memory: asynchronously when the operand's rows
// are whole aligned vectors (vec), zeros from `base` where n <= 0; else n of them
// one by one and zeros. An asynchronous copy of nothing, too, needs an address
// aligned to its size, which only vec gives `base`.
template <typename T, int NV>
__device__ __forceinline__ void copy_part(T* dst, const T* src, const T* base, int n, bool vec) {
  constexpr int kBytes = sizeof(T) * NV;
  if (vec) {
    const bool ok = n > 0;
    const T* s = ok ? src : base;
    if constexpr (kBytes <= 16) {
      copy_async<kBytes>(dst, s, ok);
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        copy_async<16>(dst + i * (16 / sizeof(T)), ok ? s + i * (16 / sizeof(T)) : s, ok);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NV; ++c) dst[c] = c < n ? src[c] : from_f<T>(0.f);
  }
}

// Four elements in fp32. For bf16 two shifts and two masks, written out.
template <typename T>
__device__ __forceinline__ float4 widen4(const Pack<T, 4>& v) {
  return make_float4(to_f(v.v[0]), to_f(v.v[1]), to_f(v.v[2]), to_f(v.v[3]));
}
template <>
__device__ __forceinline__ float4 widen4(const Pack<__nv_bfloat16, 4>& v) {
  const uint2 w = *reinterpret_cast<const uint2*>(&v);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u));
}

// ---------------------------------------------------------------------------
// fp32 pairs in 64-bit registers (one instruction for two lanes; each lane is
// rounded like the scalar operation)
// ---------------------------------------------------------------------------
using f2 = unsigned long long;

__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float f2_sum(f2 a) {
  float x, y;
  unpack2(a, x, y);
  return x + y;
}

// 2^x by the special-function unit.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 f2_ex2(f2 x) {
  float a, b;
  unpack2(x, a, b);
  return pack2(ex2(a), ex2(b));
}

// 2^(d a) of two pairs: a decay. ex2's results are low by 0.6e-8 to 2.6e-8 of
// their value on average between -0.1 and 0 (measured; an ulp is 6e-8), and a
// state that remembers a thousand tokens adds that up a thousand times. kLift in
// the exponent, which the multiplication takes for nothing, brings the average
// to within 1.3e-8 there and leaves 2^0 at 1 (error of dA over 16384 tokens:
// 1.8e-6 without, 0.8e-6 with it).
constexpr float kLift = 2e-8f;
// (Scalar, with the lift as an immediate: as a packed operation it takes a third
// register pair, and the backward 2150 us instead of 1680.)
__device__ __forceinline__ f2 f2_decay(f2 d, f2 a) {
  float d0, d1, a0, a1;
  unpack2(d, d0, d1);
  unpack2(a, a0, a1);
  return pack2(ex2(fmaf(d0, a0, kLift)), ex2(fmaf(d1, a1, kLift)));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// e^x for x <= 0 to about an ulp: ex2 of the rounded product x log2(e), times
// 1 + what the rounding lost (the product's error and log2(e)'s low part).
__device__ __forceinline__ float exp_neg(float x) {
  if (x < -150.f) x = -150.f;  // 0; keeps -inf out of the product's error
  const float t = x * kLog2e;
  const float lost = fmaf(x, kLog2e, -t) + x * 1.925963033e-8f;
  const float e = ex2(t);
  return fmaf(e, lost * kLn2, e);
}

// max(x, 0) that keeps NaN.
__device__ __forceinline__ float max0(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
  return r;
}

// log(1 + e^x) of two values, with a small relative error also where it is
// small (steps of 1e-3 and less): max(x, 0) + log1p(e) for e = e^-|x| in
// (0, 1], and log1p(e) = e P(e) with the polynomial of degree 8 that fits
// log1p(e) / e on [0, 1] best (3e-8; 1.9e-7 with the fp32 roundings). e is
// ex2's of the rounded product: off by 2^-24 |x| beside ex2's own ulp, 4e-7 for
// a step of 1e-3. (0 from |x| = 120 on at the latest, so that -inf gives 0 and
// no NaN.) e: the two values of e.
__device__ __forceinline__ f2 softplus2(float x0, float x1, f2& e) {
  const f2 x = pack2(fminf(fabsf(x0), 120.f), fminf(fabsf(x1), 120.f));
  e = f2_ex2(f2_mul(x, pack2(-kLog2e, -kLog2e)));
  constexpr float c[9] = {0.9999999403953552f, -0.4999949336051941f, 0.3331909477710724f,
                          -0.24842970073223114f, 0.19105957448482513f, -0.13663139939308167f,
                          0.07822470366954803f, -0.029504472389817238f, 0.005232503172010183f};
  f2 q = pack2(c[8], c[8]);
#pragma unroll
  for (int i = 7; i >= 0; --i) q = f2_fma(q, e, pack2(c[i], c[i]));
  return f2_fma(q, e, pack2(max0(x0), max0(x1)));
}

// Its derivative, 1 / (1 + e^-x), from that e.
__device__ __forceinline__ float softplus_slope(float x, float e) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return x >= 0.f ? r : e * r;
}

// 1 / (1 + e^-x), to a few ulp at both ends; sigmoid_fast to about 1e-6, for
// results that are rounded to 16 bits (2^-12 and more).
__device__ __forceinline__ float sigmoid_exact(float x) {
  const float e = exp_neg(-fabsf(x));
  const float r = __fdividef(1.f, 1.f + e);
  return x >= 0.f ? r : e * r;
}
__device__ __forceinline__ float sigmoid_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(-kLog2e * x)));
  return r;
}
// The sigmoid for inputs and outputs of type T.
template <typename T>
__device__ __forceinline__ float sigmoid_t(float x) {
  if constexpr (sizeof(T) == 4)
    return sigmoid_exact(x);
  else
    return sigmoid_fast(x);
}
// Two of them.
template <typename T>
__device__ __forceinline__ f2 sigmoid2(f2 x) {
  float a, b;
  if constexpr (sizeof(T) == 4) {
    unpack2(x, a, b);
    return pack2(sigmoid_exact(a), sigmoid_exact(b));
  } else {
    unpack2(f2_mul(x, pack2(-kLog2e, -kLog2e)), a, b);
    unpack2(f2_add(pack2(ex2(a), ex2(b)), pack2(1.f, 1.f)), a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    return pack2(a, b);
  }
}

}  // namespace greta
