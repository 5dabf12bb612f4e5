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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The capped logit y = cap tanh(u), u = z / cap.  Up to |u| = 3/4, where almost all logits lie, tanh(u) / u is a polynomial g in s = u^2, so that
// y = z g(s) is relatively as exact as fp32 arithmetic is (off by at most 2.3 times 2^-24, 0.65 in the root of the mean square) and takes no special-function
// operation, of which an SM does sixteen a clock; beyond, tanh|u| = 1 - 2 w with w = e / (1 + e) <= 0.19, e = e^-2|u|, whose error arrives at a third.
// 1 - tanh^2(u) is formed of tanh(u) or as 4 w (1 - w).  The coefficients are the minimax fit of tanh(sqrt s) / sqrt s on [0, 9/16] by a polynomial that is 1
// at 0 (relative error 3.3e-8, Remez exchange in 80-bit floats, then rounded).  w for every logit was off by 3e-7 cap, near zero
// too: 1e-5 of a probability at a cap of 30.
struct Scaling {
  float cap, minus_s;   // -1 / cap^2
  float k;              // 2 log2(e) / cap
  float c;              // log2(e) / T
  float inv_temp;       // 1 / T

  // w of four logits, which share a reciprocal: that of the product of their denominators
  __device__ __forceinline__ void far_tails(const float (&z)[4], float (&w)[4]) const {
    float a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = exp2_fast(-fabsf(z[j]) * k);
      a[j] = 1.f + w[j];
    }
    const float p = a[0] * a[1], q = a[2] * a[3], all = rcp_fast(p * q), x = all * q, y = all * p;
    w[0] *= x * a[1];
    w[1] *= x * a[0];
    w[2] *= y * a[3];
    w[3] *= y * a[2];
  }
  // f <- capped logits, and with SLOPE slope <- dy / dz, of E logits (one, or a multiple of four)
  template <bool SLOPE, int E>
  __device__ __forceinline__ void cap_logits(float (&f)[E], float (&slope)[E]) const {
    // (signs for a polynomial in -s)
    constexpr float G[6] = {1.f, 0.33333068381f, 0.13326521175f, 0.05339025875f, 0.019664913816f, 0.0047694904028f};
    constexpr float FAR = -0.5625f;
    constexpr int Q = E < 4 ? E : 4;
#pragma unroll
    for (int j = 0; j < E; j += Q) {
      float z[4], s[4], y[4], d[4];   // s: -u^2
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = f[i < Q ? j + i : j];
#pragma unroll
      for (int i = 0; i < Q; i += 2) {
        const float2 v = make_float2(z[i], z[i + 1]), t = mul2(mul2(v, v), make_float2(minus_s, minus_s));
        float2 g = make_float2(G[5], G[5]);
#pragma unroll
        for (int n = 4; n >= 0; --n) g = fma2(g, t, make_float2(G[n], G[n]));
        const float2 o = mul2(v, g);
        s[i] = t.x;
        s[i + 1] = t.y;
        y[i] = o.x;
        y[i + 1] = o.y;
        if (SLOPE) {
          const float2 e = fma2(mul2(o, o), make_float2(minus_s, minus_s), make_float2(1.f, 1.f));
          d[i] = e.x;
          d[i + 1] = e.y;
        }
      }
      if ((Q == 1 ? s[0] : fminf(min3(s[0], s[1], s[2]), s[3])) < FAR) {   // (a NaN goes through the polynomial)
        float w[4];
        far_tails(z, w);
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          if (!(s[i] < FAR)) continue;
          y[i] = copysignf(fmaf(-2.f * cap, w[i], cap), z[i]);
          if (SLOPE) d[i] = 4.f * fmaf(-w[i], w[i], w[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        f[j + i] = y[i];
        if (SLOPE) slope[j + i] = d[i];
      }
    }
  }
  template <int E>
  __device__ __forceinline__ void cap_logits(float (&f)[E]) const {
    float none[E];
    cap_logits<false>(f, none);
  }
  // one class, whether there is a cap or not: its capped logit, and dy / dz with the temperature
  __device__ __forceinline__ float capped(float z, float* slope) const {
    *slope = inv_temp;
    if (!(cap > 0.f)) return z;
    float f[1] = {z}, d[1];
    cap_logits<true>(f, d);
    *slope *= d[0];
    return f[0];
  }
  __device__ __forceinline__ float capped(float z) const {
    if (!(cap > 0.f)) return z;
    float f[1] = {z};
    cap_logits(f);
    return f[0];
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

template <int E>
__device__ __forceinline__ float largest(const float (&f)[E]) {
  float mx = f[0];
#pragma unroll
  for (int j = 1; j + 1 < E; j += 2) mx = max3(mx, f[j], f[j + 1]);
  return E % 2 ? mx : fmaxf(mx, f[E - 1]);
}
constexpr float ABSENT = -1e30f;   // the capped logit of a class that is not there: far below any, and finite
// Adds E classes of (capped) logits f with the largest one mx, known first so that the exponentials do not wait for one another.  A masked class (-inf)
// adds nothing: its exponent is kept finite where 0 * infinity would come up.  CAP: there are no infinities among f.  Two-wide arithmetic halves the
// instructions beside the exponentials, which the issue slots are short of at two bytes a class.
template <bool CAP, bool W, int E>
__device__ __forceinline__ void add_classes(Stats& a, const float (&f)[E], float mx, const Scaling& sc) {
  if (mx > a.m) a = shifted(a, mx, sc.c);
  const float ref = a.m == -INFINITY ? 0.f : a.m;
  float2 s = make_float2(0.f, 0.f), w = s;
#pragma unroll
  for (int j = 0; j + 1 < E; j += 2) {
    const float2 t = mul2(add2(make_float2(f[j], f[j + 1]), make_float2(-ref, -ref)), make_float2(sc.c, sc.c));
    const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
    s = add2(s, e);
    if (W) w = fma2(e, CAP ? t : make_float2(fmaxf(t.x, -FLT_MAX), fmaxf(t.y, -FLT_MAX)), w);
  }
  if (E % 2) {
    const float t = (f[E - 1] - ref) * sc.c, e = exp2_fast(t);
    s.x += e;
    if (W) w.x = fmaf(e, fmaxf(t, -FLT_MAX), w.x);
  }
  a.s += s.x + s.y;
  if (W) a.w += w.x + w.y;
}
// ... of capped logits, ABSENT ones among them
template <bool W, int E>
__device__ __forceinline__ void add_capped(Stats& a, const float (&f)[E], const Scaling& sc) {
  const float mx = largest(f);
  add_classes<true, W, E>(a, f, mx == ABSENT ? -INFINITY : mx, sc);
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
  return Scaling{softcap, softcap > 0.f ? (float)(-1.0 / ((double)softcap * softcap)) : 0.f, (float)k, (float)(1.4426950408889634 * inv_temp), (float)inv_temp};
}

}  // namespace ob
