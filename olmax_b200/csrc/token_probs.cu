// The distribution of an LM head: log probabilities of given tokens, entropy and top classes; distillation from a teacher's top
// classes; the gradients of both with respect to the logits.  See token_probs.h for the definitions.
//
// One block per row.  Statistics are kept as (maximum, sum of exponentials) so that a row is read once whatever its range is.
#include "token_probs.h"
#include "host_common.h"

#include <float.h>
#include <limits.h>
#include "sm100.cuh"

namespace ob {

constexpr int TP_THREADS = 512;

template <class T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16(x); }

// y(z) and dy/dz.  tanh(u) = 1 - 2 r and 1 - tanh^2(u) = 4 r (1 - r) with r = 1 / (1 + e^2u): two hardware approximations, absolute error of
// the tanh below 2e-7 (the approximate tanh instruction's 5e-4 would show in every log probability).
struct Scaling {
  float cap, inv_cap, inv_temp;
  __device__ __forceinline__ float y(float z) const {
    if (cap > 0.f) z = cap * (1.f - 2.f * __fdividef(1.f, 1.f + __expf(2.f * z * inv_cap)));
    return z * inv_temp;
  }
  __device__ __forceinline__ float y(float z, float* slope) const {
    *slope = inv_temp;
    if (cap > 0.f) {
      const float r = __fdividef(1.f, 1.f + __expf(2.f * z * inv_cap));
      z = cap * (1.f - 2.f * r);
      *slope *= 4.f * r * (1.f - r);
    }
    return z * inv_temp;
  }
};

// (maximum, sum e^(y - m), sum e^(y - m) (y - m)): log-sum-exp = m + log s, entropy = log s - w / s
struct Stats {
  float m, s, w;
};
__device__ __forceinline__ Stats empty_stats() { return Stats{-INFINITY, 0.f, 0.f}; }
// the sums of `a` with respect to the maximum m >= a.m; m = -inf: no class has been seen
__device__ __forceinline__ Stats shifted(Stats a, float m) {
  if (a.m == m || a.s == 0.f) return Stats{m, a.s, a.w};
  const float d = fmaxf(a.m - m, -FLT_MAX), f = __expf(d);
  return Stats{m, a.s * f, f > 0.f ? (a.w + a.s * d) * f : 0.f};
}
__device__ __forceinline__ Stats combine(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  a = shifted(a, m);
  b = shifted(b, m);
  return Stats{m, a.s + b.s, a.w + b.w};
}
// a class that is masked (-inf) adds nothing, not a product of 0 and infinity
__device__ __forceinline__ void add_class(Stats& a, float y) {
  if (y > a.m) a = shifted(a, y);
  const float d = fmaxf(y - (a.m == -INFINITY ? 0.f : a.m), -FLT_MAX), e = y == y ? __expf(d) : y;
  a.s += e;
  a.w += e * d;
}

__device__ __forceinline__ Stats block_combine(Stats a, Stats* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    a = combine(a, Stats{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off),
                         __shfl_xor_sync(0xffffffffu, a.w, off)});
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
  a = red[0];
  for (int i = 1; i < (int)blockDim.x / 32; ++i) a = combine(a, red[i]);
  return a;
}

// Order of the classes: larger logits first (NaN before all, -0 equal to 0), then lower classes.
__device__ __forceinline__ unsigned order_key(float z) {
  if (z != z) return 0xffffffffu;
  const unsigned u = __float_as_uint(z + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int block_sum(int c, int* red) {
  c = __reduce_add_sync(0xffffffffu, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = c;
  __syncthreads();
  int t = 0;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) t += red[i];
  return t;
}

template <class T>
__global__ void __launch_bounds__(TP_THREADS)
    token_log_probs_fwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ ids,
                               float* __restrict__ log_probs, float* __restrict__ entropy, float* __restrict__ lse_out,
                               int top_k, float* __restrict__ top_log_probs, long long* __restrict__ top_ids, int V,
                               int ignore_index, Scaling sc) {
  __shared__ Stats red[TP_THREADS / 32];
  __shared__ int redi[TP_THREADS / 32];
  __shared__ unsigned keys[OB_TOP_K_MAX];
  __shared__ int idx[OB_TOP_K_MAX];
  __shared__ int found;
  const long long row = blockIdx.x;
  const T* z = logits + row * ld;
  Stats a = empty_stats();
  for (int i = threadIdx.x; i < V; i += TP_THREADS) add_class(a, sc.y(to_f(z[i])));
  a = block_combine(a, red);
  const float log_s = logf(a.s);
  const bool none = a.m == -INFINITY && a.s == 0.f;   // (a NaN makes the sum NaN)
  auto log_p = [&](float y) { return y == -INFINITY ? (log_s == log_s ? y : log_s) : (y - a.m) - log_s; };
  if (threadIdx.x == 0) {
    if (log_probs != nullptr) {
      const long long id = ids[row];
      log_probs[row] = id != (long long)ignore_index && id >= 0 && id < V ? log_p(sc.y(to_f(z[id]))) : 0.f;
    }
    if (entropy != nullptr) entropy[row] = none ? 0.f : log_s - a.w / a.s;
    if (lse_out != nullptr) lse_out[row] = none ? -INFINITY : a.m + log_s;
    found = 0;
  }
  if (top_k <= 0) return;
  // the top_k-th largest key, by bits
  unsigned cut = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned c = cut | (1u << bit);
    int n = 0;
    for (int i = threadIdx.x; i < V; i += TP_THREADS) n += order_key(to_f(z[i])) >= c;
    if (block_sum(n, redi) >= top_k) cut = c;
  }
  int n = 0;
  for (int i = threadIdx.x; i < V; i += TP_THREADS) n += order_key(to_f(z[i])) > cut;
  const int equal = top_k - block_sum(n, redi);
  // the lowest class up to which `equal` classes have that key
  int last = 0;
  for (int bit = 30; bit >= 0; --bit) {
    const int c = last | (1 << bit);   // classes below c
    n = 0;
    for (int i = threadIdx.x; i < V && i < c; i += TP_THREADS) n += order_key(to_f(z[i])) == cut;
    if (block_sum(n, redi) < equal) last = c;
  }
  for (int i = threadIdx.x; i < V; i += TP_THREADS) {
    const unsigned key = order_key(to_f(z[i]));
    if (key > cut || (key == cut && i <= last)) {
      const int at = atomicAdd(&found, 1);
      keys[at] = key;
      idx[at] = i;
    }
  }
  __syncthreads();
  if (threadIdx.x < top_k) {
    const unsigned key = keys[threadIdx.x];
    const int i = idx[threadIdx.x];
    int rank = 0;
    for (int j = 0; j < top_k; ++j) rank += keys[j] > key || (keys[j] == key && idx[j] < i);
    top_log_probs[row * top_k + rank] = log_p(sc.y(to_f(z[i])));
    top_ids[row * top_k + rank] = i;
  }
}

template <class T, class D>
__global__ void __launch_bounds__(TP_THREADS)
    token_log_probs_bwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ ids,
                               const float* __restrict__ lse_in, const float* __restrict__ entropy,
                               const float* __restrict__ g_log_probs, long long stride_lp,
                               const float* __restrict__ g_entropy, long long stride_ent, D* __restrict__ dlogits,
                               long long ld_d, int V, int ignore_index, Scaling sc) {
  const long long row = blockIdx.x;
  const T* z = logits + row * ld;
  D* d = dlogits + row * ld_d;
  const float lse = lse_in[row];
  const float ge = g_entropy != nullptr ? g_entropy[row * stride_ent] : 0.f;
  float gl = 0.f;
  long long id = -1;
  if (g_log_probs != nullptr) {
    id = ids[row];
    if (id != (long long)ignore_index && id >= 0 && id < V) gl = g_log_probs[row * stride_lp];
    else id = -1;
  }
  const bool none = lse == -INFINITY;
  const float h = entropy != nullptr ? entropy[row] : 0.f;
  for (int i = threadIdx.x; i < V; i += TP_THREADS) {
    float slope;
    const float y = sc.y(to_f(z[i]), &slope);
    const float lp = y - lse, p = __expf(lp);
    float g = -p * (gl + ge * (p > 0.f ? lp + h : 0.f));
    if (i == id) g += gl;
    d[i] = from_f<D>(none ? 0.f : g * slope);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Distillation.  S: the classes that the teacher names, t_i its values, q_i its masses; L the log-sum-exp of the student's other classes.
//   loss = sum_S q (log q - log p) + rest_q (log rest_q - (L - lse)),   M = sum_S q + rest_q
//   d/dy_j = M p_j - q_j in S,   e^(y_j - L) (M e^(L - lse) - rest_q) outside
// L has its own maximum and sum over the classes outside S: 1 - sum_S p would lose what a confident student leaves to the rest.
// The teacher's masses are summed in 64 bits for the same reason.
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ long long teacher_id(const void* ids, int ids_64, long long at) {
  return ids_64 ? reinterpret_cast<const long long*>(ids)[at] : (long long)reinterpret_cast<const int*>(ids)[at];
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

template <class T>
__global__ void __launch_bounds__(TP_THREADS)
    distill_fwd_kernel(const T* __restrict__ logits, long long ld, const void* __restrict__ teacher_ids, int ids_64,
                       const float* __restrict__ teacher_log_probs, long long ld_t, int k, int renormalize,
                       float* __restrict__ row_loss, float* __restrict__ row_stats, float* __restrict__ q_out, int V,
                       Scaling sc) {
  extern __shared__ unsigned named[];   // one bit per class
  __shared__ Stats red[TP_THREADS / 32];
  __shared__ long long id_s[OB_TOP_K_MAX];
  const long long row = blockIdx.x;
  const T* z = logits + row * ld;
  for (int i = threadIdx.x; i < (V + 31) / 32; i += TP_THREADS) named[i] = 0;
  if (threadIdx.x < k) id_s[threadIdx.x] = teacher_id(teacher_ids, ids_64, row * ld_t + threadIdx.x);
  __syncthreads();
  bool counts = false;
  if (threadIdx.x < k) {
    const long long id = id_s[threadIdx.x];
    counts = id >= 0 && id < V;
    for (int j = 0; j < (int)threadIdx.x; ++j) counts &= id_s[j] != id;
    if (counts) atomicOr(&named[id >> 5], 1u << (id & 31));
  }
  __syncthreads();
  if (threadIdx.x < k && !counts) id_s[threadIdx.x] = -1;
  Stats a = empty_stats();
  for (int i = threadIdx.x; i < V; i += TP_THREADS)
    if (!((named[i >> 5] >> (i & 31)) & 1)) add_class(a, sc.y(to_f(z[i])));
  a = block_combine(a, red);
  if (threadIdx.x >= 32) return;
  // the first warp: up to four of the teacher's pairs per lane
  constexpr int N = OB_TOP_K_MAX / 32;
  float t[N], y[N];
  bool in[N];
  Stats st = empty_stats();
  float t_max = -INFINITY;
  bool any = false;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = n * 32 + threadIdx.x;
    in[n] = i < k && id_s[i] >= 0;
    t[n] = in[n] ? teacher_log_probs[row * ld_t + i] : -INFINITY;
    y[n] = in[n] ? sc.y(to_f(z[id_s[i]])) : -INFINITY;
    if (in[n]) add_class(st, y[n]);
    t_max = fmaxf(t_max, t[n]);
    any |= in[n] && !(renormalize && t[n] == -INFINITY);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    st = combine(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, off), __shfl_xor_sync(0xffffffffu, st.s, off),
                           __shfl_xor_sync(0xffffffffu, st.w, off)});
    t_max = fmaxf(t_max, __shfl_xor_sync(0xffffffffu, t_max, off));
  }
  any = __any_sync(0xffffffffu, any);
  const Stats all = combine(st, a);
  const bool none = all.m == -INFINITY && all.s == 0.f;
  const float lse = none ? -INFINITY : all.m + logf(all.s);
  const bool others = !(a.m == -INFINITY && a.s == 0.f);
  const float rest_lse = others ? a.m + logf(a.s) : -INFINITY;
  const double shift = renormalize && t_max > -INFINITY ? (double)t_max : 0.0;
  double q[N], sum = 0.0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    q[n] = in[n] ? exp((double)t[n] - shift) : 0.0;
    sum += q[n];
  }
  sum = warp_sum(sum);
  double log_norm = shift, mass = sum, rest = 0.0;
  if (renormalize) {
    log_norm += log(sum);
    mass = 1.0;
  } else if (others) {
    rest = fmax(0.0, 1.0 - sum);
  }
  double loss = 0.0;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (renormalize) q[n] /= sum;
    const double lp = y[n] == -INFINITY ? -INFINITY : (double)y[n] - lse;
    if (in[n] && q[n] != 0.0) loss += q[n] * ((double)t[n] - log_norm - lp);
    const int i = n * 32 + threadIdx.x;
    if (i < k) q_out[row * k + i] = in[n] && any ? (float)q[n] : -1.f;
  }
  loss = warp_sum(loss);
  if (threadIdx.x == 0) {
    const double rest_lp = (double)rest_lse - lse;
    if (rest > 0.0) loss += rest * (log(rest) - rest_lp);
    row_loss[row] = any ? (float)loss : 0.f;
    const double total = mass + rest;
    float4 o = make_float4(rest_lse, others && any ? (float)(total * exp(rest_lp) - rest) : 0.f, lse, any ? (float)total : -1.f);
    *reinterpret_cast<float4*>(row_stats + row * 4) = o;
  }
}

template <class T, class D>
__global__ void __launch_bounds__(TP_THREADS)
    distill_bwd_kernel(const T* __restrict__ logits, long long ld, const void* __restrict__ teacher_ids, int ids_64,
                       long long ld_t, int k, const float* __restrict__ row_stats, const float* __restrict__ q,
                       const float* __restrict__ g, long long stride_g, const float* __restrict__ inv_count, float scale,
                       D* __restrict__ dlogits, long long ld_d, int V, Scaling sc) {
  const long long row = blockIdx.x;
  const T* z = logits + row * ld;
  D* d = dlogits + row * ld_d;
  const float4 st = *reinterpret_cast<const float4*>(row_stats + row * 4);
  const float gs = (g != nullptr ? g[row * stride_g] : 1.f) * scale * (inv_count != nullptr ? *inv_count : 1.f);
  const bool nothing = st.w < 0.f || st.z == -INFINITY;
  const float rest_lse = st.x == -INFINITY ? 0.f : st.x;
  const float coef = st.y * gs;
  for (int i = threadIdx.x; i < V; i += TP_THREADS) {
    float slope;
    const float y = sc.y(to_f(z[i]), &slope);
    d[i] = from_f<D>(nothing ? 0.f : __expf(y - rest_lse) * coef * slope);
  }
  __syncthreads();
  if (threadIdx.x < k && !nothing) {
    const float qi = q[row * k + threadIdx.x];
    if (!(qi < 0.f)) {
      const long long i = teacher_id(teacher_ids, ids_64, row * ld_t + threadIdx.x);
      float slope;
      const float y = sc.y(to_f(z[i]), &slope);
      d[i] = from_f<D>((st.w * __expf(y - st.z) - qi) * gs * slope);
    }
  }
}

// One block: the order of the sum does not depend on the launch.
__global__ void __launch_bounds__(1024)
    distill_reduce_kernel(const float* __restrict__ row_loss, const float* __restrict__ row_stats, long long rows, int mean,
                          float* __restrict__ loss, float* __restrict__ inv_count) {
  __shared__ double red[32];
  __shared__ int redi[32];
  double sum = 0.0;
  int n = 0;
  for (long long r = threadIdx.x; r < rows; r += 1024) {
    const bool counted = !(row_stats[r * 4 + 3] < 0.f);
    if (counted) sum += (double)row_loss[r];
    n += counted;
  }
  sum = warp_sum(sum);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = sum;
    redi[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = warp_sum(red[threadIdx.x]);
    n = __reduce_add_sync(0xffffffffu, redi[threadIdx.x]);
    if (threadIdx.x == 0) {
      const double inv = 1.0 / (double)(n > 0 ? n : 1);
      *loss = (float)(mean ? sum * inv : sum);
      if (inv_count != nullptr) *inv_count = (float)inv;
    }
  }
}

__global__ void __launch_bounds__(1024)
    distill_count_kernel(const void* __restrict__ teacher_ids, int ids_64, const float* __restrict__ teacher_log_probs,
                         long long ld_t, int k, int renormalize, long long rows, int V, float* __restrict__ inv_count) {
  __shared__ int redi[32];
  int n = 0;
  for (long long r = threadIdx.x; r < rows; r += 1024) {
    bool any = false;
    for (int i = 0; i < k && !any; ++i) {
      const long long id = teacher_id(teacher_ids, ids_64, r * ld_t + i);
      any = id >= 0 && id < V && !(renormalize && teacher_log_probs[r * ld_t + i] == -INFINITY);
    }
    n += any;
  }
  n = block_sum(n, redi);
  if (threadIdx.x == 0) *inv_count = 1.f / (float)(n > 0 ? n : 1);
}

static inline int check_logits(const char* what, const void* logits, int dtype, long long ld, long long rows, int V) {
  if (logits == nullptr) OB_FAIL(-1, "%s: no logits", what);
  if (dtype != OB_F32 && dtype != OB_BF16) OB_FAIL(-2, "%s: unknown type of logits %d", what, dtype);
  if (V < 1 || rows > INT_MAX || ld < 0) OB_FAIL(-3, "%s: %lld rows of %d classes, %lld apart", what, rows, V, ld);
  return 0;
}

static inline Scaling scaling(float softcap, float inv_temp) {
  return Scaling{softcap, softcap > 0.f ? 1.f / softcap : 0.f, inv_temp};
}

}  // namespace ob

using namespace ob;

extern "C" int ob_token_log_probs_fwd(const void* logits, int dtype, long long ld, const long long* ids, float* log_probs,
                                      float* entropy, float* lse, int top_k, float* top_log_probs, long long* top_ids,
                                      long long rows, int V, int ignore_index, float softcap, float inv_temp,
                                      cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("token_log_probs", logits, dtype, ld, rows, V)) return rc;
  if (top_k < 0 || top_k > OB_TOP_K_MAX || top_k > V) OB_FAIL(-4, "token_log_probs: top_k %d outside [0, min(%d, %d)]", top_k, OB_TOP_K_MAX, V);
  if ((log_probs != nullptr && ids == nullptr) || (top_k > 0 && (top_log_probs == nullptr || top_ids == nullptr)))
    OB_FAIL(-5, "token_log_probs: missing tensor");
  const Scaling sc = scaling(softcap, inv_temp);
  if (dtype == OB_F32)
    token_log_probs_fwd_kernel<float><<<(unsigned)rows, TP_THREADS, 0, stream>>>(
        (const float*)logits, ld, ids, log_probs, entropy, lse, top_k, top_log_probs, top_ids, V, ignore_index, sc);
  else
    token_log_probs_fwd_kernel<bf16><<<(unsigned)rows, TP_THREADS, 0, stream>>>(
        (const bf16*)logits, ld, ids, log_probs, entropy, lse, top_k, top_log_probs, top_ids, V, ignore_index, sc);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int ob_token_log_probs_bwd(const void* logits, int dtype, long long ld, const long long* ids, const float* lse,
                                      const float* entropy, const float* g_log_probs, long long stride_lp,
                                      const float* g_entropy, long long stride_ent, void* dlogits, int dtype_d, long long ld_d,
                                      long long rows, int V, int ignore_index, float softcap, float inv_temp,
                                      cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("token_log_probs backward", logits, dtype, ld, rows, V)) return rc;
  if (lse == nullptr || dlogits == nullptr || (g_log_probs != nullptr && ids == nullptr) || (g_entropy != nullptr && entropy == nullptr))
    OB_FAIL(-5, "token_log_probs backward: missing tensor");
  const Scaling sc = scaling(softcap, inv_temp);
#define OB_LAUNCH(T, D)                                                                                                     \
  token_log_probs_bwd_kernel<T, D><<<(unsigned)rows, TP_THREADS, 0, stream>>>((const T*)logits, ld, ids, lse, entropy,      \
                                                                              g_log_probs, stride_lp, g_entropy, stride_ent, \
                                                                              (D*)dlogits, ld_d, V, ignore_index, sc)
  if (dtype == OB_F32 && dtype_d == OB_F32) OB_LAUNCH(float, float);
  else if (dtype == OB_F32 && dtype_d == OB_BF16) OB_LAUNCH(float, bf16);
  else if (dtype == OB_BF16 && dtype_d == OB_BF16) OB_LAUNCH(bf16, bf16);
  else OB_FAIL(-2, "token_log_probs backward: no gradient of type %d for logits of type %d", dtype_d, dtype);
#undef OB_LAUNCH
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int ob_distill_fwd(const void* logits, int dtype, long long ld, const void* teacher_ids, int ids_64,
                              const float* teacher_log_probs, long long ld_t, int k, int renormalize, float* row_loss,
                              float* row_stats, float* q, long long rows, int V, float softcap, float inv_temp,
                              cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("distillation", logits, dtype, ld, rows, V)) return rc;
  if (k < 1 || k > OB_TOP_K_MAX) OB_FAIL(-4, "distillation: %d teacher classes outside [1, %d]", k, OB_TOP_K_MAX);
  if (teacher_ids == nullptr || teacher_log_probs == nullptr || row_loss == nullptr || row_stats == nullptr || q == nullptr)
    OB_FAIL(-5, "distillation: missing tensor");
  const int bytes = (V + 31) / 32 * 4;
  if (bytes > 160 * 1024) OB_FAIL(-6, "distillation: more than %d classes", 160 * 1024 * 8);
  const Scaling sc = scaling(softcap, inv_temp);
  auto launch = [&](auto kernel, auto* z) -> int {
    OB_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    kernel<<<(unsigned)rows, TP_THREADS, bytes, stream>>>(z, ld, teacher_ids, ids_64, teacher_log_probs, ld_t, k, renormalize,
                                                          row_loss, row_stats, q, V, sc);
    OB_CUDA_OK(cudaGetLastError());
    return 0;
  };
  return dtype == OB_F32 ? launch(distill_fwd_kernel<float>, (const float*)logits)
                         : launch(distill_fwd_kernel<bf16>, (const bf16*)logits);
}

extern "C" int ob_distill_bwd(const void* logits, int dtype, long long ld, const void* teacher_ids, int ids_64, long long ld_t,
                              int k, const float* row_stats, const float* q, const float* g, long long stride_g,
                              const float* inv_count, float scale, void* dlogits, int dtype_d, long long ld_d, long long rows,
                              int V, float softcap, float inv_temp, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int rc = check_logits("distillation backward", logits, dtype, ld, rows, V)) return rc;
  if (k < 1 || k > OB_TOP_K_MAX) OB_FAIL(-4, "distillation backward: %d teacher classes outside [1, %d]", k, OB_TOP_K_MAX);
  if (teacher_ids == nullptr || row_stats == nullptr || q == nullptr || dlogits == nullptr)
    OB_FAIL(-5, "distillation backward: missing tensor");
  const Scaling sc = scaling(softcap, inv_temp);
#define OB_LAUNCH(T, D)                                                                                                   \
  distill_bwd_kernel<T, D><<<(unsigned)rows, TP_THREADS, 0, stream>>>((const T*)logits, ld, teacher_ids, ids_64, ld_t, k, \
                                                                      row_stats, q, g, stride_g, inv_count, scale,        \
                                                                      (D*)dlogits, ld_d, V, sc)
  if (dtype == OB_F32 && dtype_d == OB_F32) OB_LAUNCH(float, float);
  else if (dtype == OB_F32 && dtype_d == OB_BF16) OB_LAUNCH(float, bf16);
  else if (dtype == OB_BF16 && dtype_d == OB_BF16) OB_LAUNCH(bf16, bf16);
  else OB_FAIL(-2, "distillation backward: no gradient of type %d for logits of type %d", dtype_d, dtype);
#undef OB_LAUNCH
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int ob_distill_reduce(const float* row_loss, const float* row_stats, long long rows, int mean, float* loss,
                                 float* inv_count, cudaStream_t stream) {
  if (loss == nullptr || (rows > 0 && (row_loss == nullptr || row_stats == nullptr))) OB_FAIL(-5, "distillation sum: missing tensor");
  distill_reduce_kernel<<<1, 1024, 0, stream>>>(row_loss, row_stats, rows, mean, loss, inv_count);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int ob_distill_count(const void* teacher_ids, int ids_64, const float* teacher_log_probs, long long ld_t, int k,
                                int renormalize, long long rows, int V, float* inv_count, cudaStream_t stream) {
  if (inv_count == nullptr || (rows > 0 && (teacher_ids == nullptr || teacher_log_probs == nullptr)))
    OB_FAIL(-5, "distillation count: missing tensor");
  distill_count_kernel<<<1, 1024, 0, stream>>>(teacher_ids, ids_64, teacher_log_probs, ld_t, k, renormalize, rows, V, inv_count);
  OB_CUDA_OK(cudaGetLastError());
  return 0;
}
