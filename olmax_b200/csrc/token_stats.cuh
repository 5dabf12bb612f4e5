// Statistics of a row of logits on the way through it, shared by the kernels that read logits (token_probs.cu) and by the GEMM whose epilogue
// sees them in registers (gemm.cu).  All exponentials and logarithms are to the base 2, of differences t = (z - m) c of capped
// logits with c = log2(e) / T: the difference is formed before the product, so that the lowest values of a type do not overflow.
#pragma once
#include <float.h>
#include <math.h>

#include "sm100.cuh"

namespace ob {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// 2^x by the hardware: 0 at -inf, off by at most 1.4e-7 of the value over 2^20 points of [-20, 0), low by 5e-8 in the mean
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (fminf would drop a NaN)
__device__ __forceinline__ float min_nan(float x, float y) {
  float z;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// The capped logit cap(z) = softcap * tanh(z / softcap).  tanh(u) = 1 - 2 r and 1 - tanh^2(u) = 4 r (1 - r) with r = 1 / a, a = 1 + e^2u: the
// approximate tanh instruction's error of 5e-4 would show in every log probability, this form's is below 8e-7 (the roundings of r <= 1 and the
// exponential's; 3e-7 is the largest seen), so that a cap of 256 costs a logit no more than 2e-4.  It takes two special-function operations beside the exponential of the softmax, of which an SM does sixteen a clock: they
// bound the kernels.  So four classes share a reciprocal, that of the product of their a; a <= 2^30 changes no tanh and keeps the product
// finite.  What follows is linear in r: t = (cap(z) - m) c is one multiply-add.
struct Scaling {
  float cap, k;     // k = 2 log2(e) / cap
  float c;          // log2(e) / T
  float inv_temp;   // 1 / T

  __device__ __forceinline__ float2 denominators(float z0, float z1) const {
    const float2 x = mul2(make_float2(z0, z1), make_float2(k, k));
    return add2(make_float2(exp2_fast(min_nan(x.x, 30.f)), exp2_fast(min_nan(x.y, 30.f))), make_float2(1.f, 1.f));
  }
  // f <- r of the logits f (one, or a multiple of four)
  template <int E>
  __device__ __forceinline__ void reciprocals(float (&f)[E]) const {
    if constexpr (E == 1) {
      f[0] = rcp_fast(1.f + exp2_fast(min_nan(f[0] * k, 30.f)));
    }
#pragma unroll
    for (int j = 0; j < E / 4 * 4; j += 4) {
      const float2 a = denominators(f[j], f[j + 1]), b = denominators(f[j + 2], f[j + 3]);
      const float2 p = mul2(make_float2(a.x, b.x), make_float2(a.y, b.y));
      const float all = rcp_fast(p.x * p.y);
      const float2 q = mul2(make_float2(all, all), make_float2(p.y, p.x));   // 1 / (a.x a.y), 1 / (b.x b.y)
      const float2 ra = mul2(make_float2(q.x, q.x), make_float2(a.y, a.x)), rb = mul2(make_float2(q.y, q.y), make_float2(b.y, b.x));
      f[j] = ra.x;
      f[j + 1] = ra.y;
      f[j + 2] = rb.x;
      f[j + 3] = rb.y;
    }
  }
  __device__ __forceinline__ float of_r(float r) const { return fmaf(-2.f * cap, r, cap); }
  // one class, whether there is a cap or not: its capped logit, and dy / dz
  __device__ __forceinline__ float capped(float z, float* slope) const {
    *slope = inv_temp;
    if (!(cap > 0.f)) return z;
    float f[1] = {z};
    reciprocals(f);
    *slope *= 4.f * fmaf(-f[0], f[0], f[0]);
    return of_r(f[0]);
  }
  __device__ __forceinline__ float capped(float z) const {
    float slope;
    return capped(z, &slope);
  }
};

// Of some classes: their largest capped logit m, s = sum 2^t, w = sum 2^t t with t = (z - m) c.
// log p = ln 2 (t - log2 s), entropy = ln 2 (log2 s - w / s).
struct Stats {
  float m, s, w;
};
__device__ __forceinline__ Stats empty_stats() { return Stats{-INFINITY, 0.f, 0.f}; }
// the sums of `a` with respect to the maximum m >= a.m; m = -inf: no class has been seen
__device__ __forceinline__ Stats shifted(Stats a, float m, float c) {
  if (a.m == m || a.s == 0.f) return Stats{m, a.s, a.w};
  const float d = fmaxf((a.m - m) * c, -FLT_MAX), f = exp2_fast(d);
  return Stats{m, a.s * f, f > 0.f ? (a.w + a.s * d) * f : 0.f};
}
__device__ __forceinline__ Stats combine(Stats a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  a = shifted(a, m, c);
  b = shifted(b, m, c);
  return Stats{m, a.s + b.s, a.w + b.w};
}
__device__ __forceinline__ bool no_class(Stats a) { return a.m == -INFINITY && a.s == 0.f; }   // (a NaN makes the sum NaN)

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <int E>
__device__ __forceinline__ float largest(const float (&f)[E]) {
  float mx = f[0];
#pragma unroll
  for (int j = 1; j + 1 < E; j += 2) mx = max3(mx, f[j], f[j + 1]);
  return E % 2 ? mx : fmaxf(mx, f[E - 1]);
}
constexpr float ABSENT = 1e20f;   // the r of a class that is not there: its exponent is far below any, and finite
// Adds E classes of logits f with the largest (capped) logit mx, known first so that the exponentials do not wait for one another.  A masked class
// (-inf) adds nothing: its exponent is kept finite where 0 * infinity would come up.  With CAP f are the classes' r (ABSENT for one that is
// not there).  Two-wide arithmetic halves the instructions beside the exponentials, which the issue slots are short of at two bytes a class.
template <bool CAP, bool W, int E>
__device__ __forceinline__ void add_classes(Stats& a, const float (&f)[E], float mx, const Scaling& sc) {
  if (mx > a.m) a = shifted(a, mx, sc.c);
  const float ref = a.m == -INFINITY ? 0.f : a.m;
  const float t0 = (sc.cap - ref) * sc.c, t1 = -2.f * sc.cap * sc.c;
  float2 s = make_float2(0.f, 0.f), w = s;
#pragma unroll
  for (int j = 0; j + 1 < E; j += 2) {
    const float2 x = make_float2(f[j], f[j + 1]);
    const float2 t = CAP ? fma2(x, make_float2(t1, t1), make_float2(t0, t0))
                         : mul2(add2(x, make_float2(-ref, -ref)), make_float2(sc.c, sc.c));
    const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
    s = add2(s, e);
    if (W) w = fma2(e, CAP ? t : make_float2(fmaxf(t.x, -FLT_MAX), fmaxf(t.y, -FLT_MAX)), w);
  }
  if (E % 2) {
    const float t = CAP ? fmaf(f[E - 1], t1, t0) : (f[E - 1] - ref) * sc.c, e = exp2_fast(t);
    s.x += e;
    if (W) w.x = fmaf(e, fmaxf(t, -FLT_MAX), w.x);
  }
  a.s += s.x + s.y;
  if (W) a.w += w.x + w.y;
}
// one class of capped logit y
__device__ __forceinline__ void add_class(Stats& a, float y, const Scaling& sc) {
  const float f[1] = {y};
  add_classes<false, true, 1>(a, f, y, sc);
}

__device__ __forceinline__ Stats shuffle_combine(Stats a, int first, float c) {
  for (int off = first; off > 0; off >>= 1)
    a = combine(a, Stats{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off),
                         __shfl_xor_sync(0xffffffffu, a.w, off)}, c);
  return a;
}
static inline Scaling scaling(float softcap, double inv_temp) {
  const double k = softcap > 0.f ? 2.0 * 1.4426950408889634 / (double)softcap : 0.0;
  return Scaling{softcap, (float)k, (float)(1.4426950408889634 * inv_temp), (float)inv_temp};
}

}  // namespace ob
