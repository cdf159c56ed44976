/*
 * sqb_train.h - helpers of the GPT training caller (not part of the attention
 * operator's drop-in boundary, which is sqrtblock.h).
 *
 * Token cross-entropy over a (N, V) block of logits, fused: the forward reads
 * each row once (fp32 max / sum-of-exp), the backward writes each row's
 * gradient once in the logits' dtype.  It computes what the reference's
 * calculate_loss (training_utils.py:8-17: F.cross_entropy over the flattened
 * logits under bf16 autocast, fp32 softmax math) computes, per token; the mean
 * over the non-ignored tokens is taken by the caller.  A LayerNorm with one
 * warp per row and a fixed-order weight gradient.  For training on answers:
 * token log-probabilities, a preference loss, a clipped policy loss, gradient
 * clipping, and a residual step between two norms.
 *
 * Conventions as in sqrtblock.h: caller-owned device pointers, asynchronous on
 * `stream` (a cudaStream_t; NULL = legacy default stream), return SQB_OK or an
 * SQB_ERR_* code.  From the token log-probabilities on, every pointer off its type's
 * boundary is refused with SQB_ERR_ALIGN.  logits / dlogits are (N, ld) row-major with ld >= V,
 * dtype SQB_BF16 or SQB_F32; columns [V, ld) of logits are not read.  A column
 * holding -inf takes no probability and gets a zero gradient.
 */
#ifndef SQB_TRAIN_H_
#define SQB_TRAIN_H_

#include <stddef.h>
#include <stdint.h>

#include "sqrtblock.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Forward, per row r: lse[r] = log sum_{c < V} exp(logits[r, c]) and
 * loss[r] = lse[r] - logits[r, targets[r]]; a row with targets[r] < 0 is
 * ignored (loss[r] = 0).  targets are int64 in [0, V) or negative.  loss and
 * lse are fp32 arrays of N. */
int sqb_xent_fwd(const void* logits, const int64_t* targets, float* loss, float* lse, int64_t N,
                 int64_t V, int64_t ld, int dtype, void* stream);

/* Backward: dlogits[r, c] = (exp(logits[r, c] - lse[r]) - [c == targets[r]]) * scale[0]
 * for c < V and 0 for V <= c < ld; an ignored row is all zero.  `scale` points
 * to one fp32 on the device (d loss / d loss[r]: the upstream gradient over
 * the number of counted tokens), read there so the host never waits. */
int sqb_xent_bwd(const void* logits, const int64_t* targets, const float* lse, const float* scale,
                 void* dlogits, int64_t N, int64_t V, int64_t ld, int dtype, void* stream);

/* LayerNorm over the last dimension of N contiguous fp32 rows of C (C a
 * multiple of 128, at most 1024; else SQB_ERR_UNSUPPORTED):
 *   y = (x - mean) / sqrt(var + eps) * weight + bias   (var biased; bias may be NULL),
 * as torch.nn.LayerNorm computes it (the reference's LayerNorm module,
 * model/layer_norm.py:4-13).  y has y_dtype: fp32, or bf16 - what a bf16
 * autocast consumer of an fp32 LayerNorm would cast it to.  mean and rstd
 * (1 / sqrt(var + eps)) are fp32 arrays of N for the backward.  x, weight,
 * bias and y 16-byte aligned (else SQB_ERR_ALIGN). */
int sqb_layernorm_fwd(const float* x, const float* weight, const float* bias, void* y, int y_dtype,
                      float* mean, float* rstd, int64_t N, int64_t C, float eps, void* stream);

/* Scratch bytes sqb_layernorm_bwd needs for N rows of C. */
size_t sqb_layernorm_workspace_bytes(int64_t N, int64_t C);

/* Backward: dx (fp32, N x C) from dy (dy_dtype) and the forward's x, mean and
 * rstd; dweight and, unless dbias is NULL, dbias (fp32, C) are overwritten with
 * their column sums, added in a fixed order (bit-reproducible). */
int sqb_layernorm_bwd(const void* dy, int dy_dtype, const float* x, const float* weight,
                      const float* mean, const float* rstd, float* dx, float* dweight,
                      float* dbias, void* workspace, size_t ws_bytes, int64_t N, int64_t C,
                      void* stream);

/* Residual add fused into the LayerNorm that reads its sum (the GPT caller's
 * x = x + block(...) followed by the next LayerNorm):
 *   x_out = x + h   (h: fp32 or bf16 rows by h_dtype, e.g. a bf16 autocast
 *                    Linear's output; the sum in fp32 as torch adds them),
 *   y     = LayerNorm(x_out) as sqb_layernorm_fwd, mean and rstd of x_out.
 * x_out and h 16-byte aligned like the other rows. */
int sqb_add_layernorm_fwd(const float* x, const void* h, int h_dtype, float* x_out,
                          const float* weight, const float* bias, void* y, int y_dtype,
                          float* mean, float* rstd, int64_t N, int64_t C, float eps,
                          void* stream);

/* Its backward: dx = (LayerNorm's input gradient from dy) + dres, where dres
 * (fp32, N x C, may be NULL) is the gradient reaching x_out from its other
 * uses; dx is the gradient of both x and h, written as fp32 and, unless dh_bf16
 * is NULL, also as bf16 (for a bf16 h).  dweight / dbias and the workspace as
 * sqb_layernorm_bwd (x_out is the LayerNorm's input). */
int sqb_add_layernorm_bwd(const void* dy, int dy_dtype, const float* x_out, const float* weight,
                          const float* mean, const float* rstd, const float* dres, float* dx,
                          void* dh_bf16, float* dweight, float* dbias, void* workspace,
                          size_t ws_bytes, int64_t N, int64_t C, void* stream);

/* ---- Token log-probabilities and the losses on them -------------------------
 * logits are an (S, T, V) view, unit stride on V, element strides ss (sequence)
 * and st (token), any alignment of the element's size; row r is sequence r / T,
 * token r % T (a packed batch: S = 1, T = all rows).  targets (S * T) are int64; a
 * negative one leaves its row out: the row is not read, its log-probability is 0
 * and its gradient row zero.  One of V or more gives NaN.  S * T < 2^31. */

/* Per row: logp = log softmax(logits)[target], and stats = (m, sum of exp(x - m)) with m
 * a number near the row's maximum, fp32 (S * T, 2), 8-byte aligned (a row left out:
 * (0, 0), which no other row has; a target of V or more: the sum is NaN). */
int sqb_logp_fwd(const void* logits, const int64_t* targets, float* logp, float* stats, int64_t S,
                 int64_t T, int64_t V, int64_t ss, int64_t st, int dtype, void* stream);

/* dlogits[r, c] = g_row[r] * scale[0] * ([c == target] - softmax(logits)[r, c]) in the
 * logits' dtype, strides dss and dst; scale (one fp32 on the device) may be NULL.  Zero for
 * rows whose target is negative or whose statistics say that they are left out, whatever
 * their target, factor and logits.  Rows whose 16-byte phase is the logits' are written with
 * vector stores. */
int sqb_logp_bwd(const void* logits, const int64_t* targets, const float* stats,
                 const float* g_row, const float* scale, void* dlogits, int64_t S, int64_t T,
                 int64_t V, int64_t ss, int64_t st, int64_t dss, int64_t dst, int dtype,
                 void* stream);

/* Sequences: with cu_seqlens (S = 1) sequence i has rows [cu_seqlens[i],
 * cu_seqlens[i + 1]), non-decreasing and held inside [0, N], N = S * T; rows of no
 * sequence are left out.  NULL: sequence i has rows [i * T, (i + 1) * T). */

/* Preference loss over P pairs: sequence p < P is chosen, P + p its rejected one.  With
 * r = sum of the sequence's logp - ref_logps[i] (fp32, NULL: 0) and
 * z = beta * (r_chosen - r_rejected):
 *   loss = mean of -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z),
 *   rewards (2P, fp32) = beta * r,   g_row (N, fp32) = d loss / d logp,
 * stats as sqb_logp_fwd: the gradient is sqb_logp_bwd's from stats and g_row.  T may be 0
 * (logits, targets, stats and g_row then unused).  The sums and the loss are computed in
 * 64 bits, in a fixed order; the workspace (8-byte aligned) needs no initialisation. */
size_t sqb_preference_workspace_bytes(int64_t N, int64_t P);
int sqb_preference_fwd(const void* logits, const int64_t* targets, const int64_t* cu_seqlens,
                       const float* ref_logps, int64_t P, double beta, double label_smoothing,
                       float* loss, float* rewards, float* stats, float* g_row, int64_t S,
                       int64_t T, int64_t V, int64_t ss, int64_t st, int dtype, void* workspace,
                       size_t ws_bytes, void* stream);

/* Clipped policy loss over `seqs` sequences.  Per counted row, with
 * r = exp(logp - old_logp) (1 for NULL), A = adv[row] (adv_by_seq: adv[sequence]) and
 * ref_logp (NULL: no KL):
 *   policy = -min(r A, held A), held = r kept in [1 - clip_low, 1 + clip_high],
 *   KL = exp(ref - logp) - (ref - logp) - 1,   clipped = [held A < r A];
 *   loss = sum of w (policy + kl_coef KL),   statistics (3) = sums of w (policy, KL, clipped)
 * with w = 1 / counted rows, or per_sequence 1 / (counted rows of its sequence * sequences
 * that have any); 0 where no row is counted.  logp as sqb_logp_fwd; stats and g_row (each
 * may be NULL) as sqb_preference_fwd.  With dlogits also the gradient of
 * grad_scale * loss, as sqb_logp_bwd writes it, in the same pass over the logits. */
size_t sqb_policy_workspace_bytes(int64_t N, int64_t seqs);
int sqb_policy_fwd(const void* logits, const int64_t* targets, const int64_t* cu_seqlens,
                   int64_t seqs, const float* old_logp, const float* ref_logp, const float* adv,
                   int adv_by_seq, double clip_low, double clip_high, double kl_coef,
                   int per_sequence, float* loss, float* statistics, float* logp, float* stats,
                   float* g_row, void* dlogits, float grad_scale, int64_t S, int64_t T, int64_t V,
                   int64_t ss, int64_t st, int64_t dss, int64_t dst, int dtype, void* workspace,
                   size_t ws_bytes, void* stream);

/* ---- Global gradient norm and clipping ---------------------------------------
 * n tensors as host arrays of device pointers (element-aligned), element counts (0
 * allowed) and dtypes; the arrays are read before the call returns.
 * norm: one fp32 on the device, sqrt of the sum of squares, summed in 64 bits in a
 * fixed order.  The workspace is 8-byte aligned. */
size_t sqb_grad_norm_workspace_bytes(int64_t n_tensors);
int sqb_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes,
                  int64_t n, void* workspace, size_t ws_bytes, float* norm, void* stream);

/* outs[i] = grads[i] * min(1, max_norm / (norm + 1e-6)) in out_dtypes[i], the factor and
 * the product in fp32.  outs[i] is grads[i] (same dtype) or memory apart from every
 * gradient; where all are in place and the factor is 1 nothing is written. */
int sqb_grad_clip(const void* const* grads, void* const* outs, const int64_t* numel,
                  const int32_t* dtypes, const int32_t* out_dtypes, int64_t n, float max_norm,
                  void* workspace, size_t ws_bytes, float* norm, void* stream);

/* ---- Residual step between two norms -----------------------------------------
 * On N contiguous rows of C <= 4096 (else SQB_ERR_UNSUPPORTED), x and h each fp32 or bf16:
 *   n = Norm(h; post_weight, post_bias)   (h itself for a NULL post_weight)
 *   x_out = x + scale * gate * n          (x's dtype; a NULL gate is ones)
 *   y = Norm(x_out; weight, bias)         (y_dtype; of x_out before its rounding)
 * Norm: LayerNorm, or with `rms` an RMS norm; biases may be NULL.  gate: (gates, C), each
 * row shared by N / gates rows in turn.  Parameters are fp32.  stats: fp32 (N, 4), the
 * mean and 1/std of h and of x_out, 16-byte aligned. */
int sqb_residual_norm_fwd(const void* x, int x_dtype, const void* h, int h_dtype,
                          const float* weight, const float* bias, const float* post_weight,
                          const float* post_bias, const float* gate, int64_t gates, float scale,
                          float eps, int rms, void* x_out, void* y, int y_dtype, float* stats,
                          int64_t N, int64_t C, void* stream);

size_t sqb_residual_norm_workspace_bytes(int64_t N, int64_t C, int64_t gates);

/* Backward from x, h and the forward's stats: dy (y_dtype), dx_out (x's dtype; NULL: 0)
 * -> dx, dh in x's and h's dtypes and the gradient of every parameter given (fp32,
 * overwritten; dgate (gates, C)), summed in a fixed order.  At most 65530 gates.  The
 * workspace is 16-byte aligned. */
int sqb_residual_norm_bwd(const void* dy, int y_dtype, const void* dx_out, const void* x,
                          int x_dtype, const void* h, int h_dtype, const float* weight,
                          const float* bias, const float* post_weight, const float* post_bias,
                          const float* gate, int64_t gates, float scale, float eps, int rms,
                          const float* stats, void* dx, void* dh, float* dweight, float* dbias,
                          float* dpost_weight, float* dpost_bias, float* dgate, void* workspace,
                          size_t ws_bytes, int64_t N, int64_t C, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SQB_TRAIN_H_ */
