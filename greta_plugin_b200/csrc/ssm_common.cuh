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

// The largest s in [-1, nseq] with seq_start(s) <= t (-1: t is ahead of the
// first sequence, nseq: behind the last). 32 probes a round, so two rounds for
// a thousand sequences; every lane of the warp calls it with the same t. Ends
// on any contents of `starts`.
__device__ __forceinline__ int warp_find(const Seqs& q, int t, int lane) {
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

// A run of tokens [b, e) that one sequence s holds (in), or that none does
// (ahead of the first sequence, s = -1, or behind the last, s = nseq).
struct Seg {
  int s, b, e;
  bool in;
};

__device__ __forceinline__ Seg seg_make(const Seqs& q, int s, int t) {
  Seg g;
  g.s = s;
  g.in = s >= 0 && s < q.nseq;
  g.b = s >= 0 ? seq_start(q, s) : 0;
  g.e = s < q.nseq ? seq_start(q, s + 1) : q.T;
  if (g.e <= t) g.e = t + 1;  // offsets that fall: stay on the way forward
  return g;
}

__device__ __forceinline__ Seg seg_at(const Seqs& q, int t, int lane) {
  return seg_make(q, warp_find(q, t, lane), t);
}

// The segment that begins where `g` ends (sequences of no tokens are passed).
__device__ __forceinline__ Seg seg_next(const Seqs& q, const Seg& g) {
  const int t = g.e;
  int s = g.s + 1;
  while (s < q.nseq && seq_start(q, s + 1) <= t) ++s;
  Seg n = seg_make(q, s, t);
  n.b = t;
  return n;
}

// Where range i of R ranges of about L tokens begins: i * L, or the nearest
// sequence start within half a range of it. A range that begins with a
// sequence needs nothing from the range before; the moved borders stay in
// order, since each moves by less than half a range.
__device__ __forceinline__ int range_begin(const Seqs& q, int i, int R, int L, int lane) {
  if (i <= 0) return 0;
  if (i >= R) return q.T;
  const int p = (int)min((long long)i * L, (long long)q.T);
  const int s = warp_find(q, p, lane);
  const int before = s >= 0 ? seq_start(q, s) : 0;
  const int after = s < q.nseq ? seq_start(q, s + 1) : q.T;
  const bool nb = before <= p && p - before <= L / 2 && before > 0;
  const bool na = after > p && after - p < L / 2;
  if (nb && (!na || p - before <= after - p)) return before;
  if (na) return after;
  return p;
}

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

// log(1 + e^x), with a small relative error also where it is small (steps of
// 1e-3 and less): max(x, 0) + log1p(e) for e = e^-|x| in (0, 1], and
// log1p(e) = 2 atanh(v), v = e / (2 + e) <= 1/3, by atanh's series up to v^15
// (the next term is below 2^-28 of the sum). x itself above 20, where the
// rest is less than half an ulp, and for NaN the NaN.
__device__ __forceinline__ float softplusf_(float x) {
  const float e = exp_neg(-fabsf(x));
  const float v = __fdividef(e, 2.f + e);
  const float q = v * v;
  float s = 1.f / 15.f;
  s = fmaf(s, q, 1.f / 13.f);
  s = fmaf(s, q, 1.f / 11.f);
  s = fmaf(s, q, 1.f / 9.f);
  s = fmaf(s, q, 1.f / 7.f);
  s = fmaf(s, q, 1.f / 5.f);
  s = fmaf(s, q, 1.f / 3.f);
  const float l = 2.f * fmaf(s * q, v, v);
  return x > 20.f ? x : (x > 0.f ? x + l : l);
}

// 1 / (1 + e^-x), to a few ulp at both ends.
__device__ __forceinline__ float sigmoid_exact(float x) {
  const float e = exp_neg(-fabsf(x));
  const float r = __fdividef(1.f, 1.f + e);
  return x >= 0.f ? r : e * r;
}

}  // namespace greta
