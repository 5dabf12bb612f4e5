// C interface of the kernels over the distribution of an LM head (token_probs.cu): log probabilities of given tokens with
// entropy and top classes, and distillation from a teacher's top classes, each with its gradient.
//
// logits: [rows, V] of `dtype` (OB_F32 / OB_BF16), row stride ld elements, classes contiguous; rows may start at any multiple of
// the element size.  The distribution of a row is p = softmax(y), y = cap(z) * inv_temp with cap(z) = softcap * tanh(z / softcap)
// for softcap > 0, else z.  A row whose y are all -inf has log p = -inf, entropy 0 and no gradient.
#pragma once
#include <cuda_runtime.h>

#ifdef __cplusplus
extern "C" {
#endif

#define OB_F32 0
#define OB_BF16 1
#define OB_TOP_K_MAX 128

// log_probs[r] = log p of class ids[r] (0 where ids[r] == ignore_index or lies outside [0, V); both may be null), entropy[r],
// norm[r] = two floats (8-byte aligned) that the backward pass reads: the largest capped logit and log2 sum exp(y - its y) (may be null).  top_k > 0: top_log_probs / top_ids [rows, top_k] = the classes with the largest logits
// in order, equal logits by their class (top_k <= min(V, OB_TOP_K_MAX)).
int ob_token_log_probs_fwd(const void* logits, int dtype, long long ld, const long long* ids, float* log_probs, float* entropy,
                           float* norm, int top_k, float* top_log_probs, long long* top_ids, long long rows, int V,
                           int ignore_index, float softcap, double inv_temp, cudaStream_t stream);
// The same of logits that exist as statistics of `n` groups of classes only: parts[i * stride + r] = four floats (largest capped logit m, sum 2^t, sum
// 2^t t, unused) with t = (cap(z) - m) log2(e) inv_temp over group i, target[r] = the logit of class ids[r] (undefined where it is not scored).
int ob_join_scores(const float* parts, const float* target, long long stride, int n, const long long* ids, float* log_probs,
                   float* entropy, float* norm, long long rows, int V, int ignore_index, float softcap, double inv_temp,
                   cudaStream_t stream);
// dlogits (of dtype_d, row stride ld_d) = g_log_probs[r * stride_lp] * d log_probs[r] + g_entropy[r * stride_ent] * d entropy[r]
// over d logits; either upstream gradient may be null.
int ob_token_log_probs_bwd(const void* logits, int dtype, long long ld, const long long* ids, const float* norm,
                           const float* entropy, const float* g_log_probs, long long stride_lp, const float* g_entropy,
                           long long stride_ent, void* dlogits, int dtype_d, long long ld_d, long long rows, int V,
                           int ignore_index, float softcap, double inv_temp, cudaStream_t stream);

// Teacher of a row: k <= OB_TOP_K_MAX pairs (teacher_ids, int32 or int64 by ids_64; teacher_log_probs fp32), rows ld_t apart.  A pair whose id
// lies outside [0, V) is padding; of several pairs with one id the first counts.
//   renormalize != 0: q = softmax of the row's values;  loss = sum q (log q - log p)
//   else:             q = exp(value); the classes the teacher does not name are one further class with what is left of one:
//                     loss = sum q (log q - log p) + rest_q (log rest_q - log rest_p)
// row_loss[r]; row_stats[r] = eight floats (16-byte aligned): the teacher's total mass (-1 for a row without a teacher: loss 0, gradient 0), the
// coefficient of the other classes' gradient, two unused, the largest capped logit and log2 sum exp(y - its y) of all classes, the same
// of the other classes; q [rows, k] = the teacher's masses, -1 for pairs that do not count.
int ob_distill_fwd(const void* logits, int dtype, long long ld, const void* teacher_ids, int ids_64,
                   const float* teacher_log_probs, long long ld_t, int k, int renormalize, float* row_loss, float* row_stats,
                   float* q, long long rows, int V, float softcap, double inv_temp, cudaStream_t stream);
// dlogits = scale * (*inv_count, if given) * g[r * stride_g] * d row_loss[r] / d logits
int ob_distill_bwd(const void* logits, int dtype, long long ld, const void* teacher_ids, int ids_64, long long ld_t, int k,
                   const float* row_stats, const float* q, const float* g, long long stride_g, const float* inv_count, float scale,
                   void* dlogits, int dtype_d, long long ld_d, long long rows, int V, float softcap, double inv_temp,
                   cudaStream_t stream);
// *loss = sum of row_loss, divided by the number of rows with a teacher if mean; *inv_count (may be null) = 1 / max(1, that number)
int ob_distill_reduce(const float* row_loss, const float* row_stats, long long rows, int mean, float* loss, float* inv_count,
                      cudaStream_t stream);
// *inv_count alone, from the teacher
int ob_distill_count(const void* teacher_ids, int ids_64, const float* teacher_log_probs, long long ld_t, int k, int renormalize,
                     long long rows, int V, float* inv_count, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
