/* C-ABI of the operators of an LM's training and scoring step around the
 * mixer in libgmdn_scan.so (MI355X, gfx950): layer norm, 8-bit activation
 * checkpoints, and log probabilities of given tokens.
 *
 * Matrices are (rows, d) with unit-stride rows; inputs take a row stride in
 * elements (any value >= 0: a slice of a wider tensor, a broadcast row),
 * outputs are contiguous.  No alignment beyond the element's is needed.
 * Types are GMDN_DTYPE_BF16 or GMDN_DTYPE_F32; all sums and statistics are
 * float32.  Error codes are those of gmdn_scan.h; calls are asynchronous on
 * `stream`, allocate nothing, and give the same bits on every run.
 *
 * The 8-bit checkpoint of a (rows, d) matrix is q (rows, d) int8 and scale
 * (rows, ceil(d / 128)) float32, one for each group of 128 consecutive values
 * of a row: with amax the group's largest magnitude, scale = amax times the
 * float32 below 1 / 127, q = rint(x * (127 / amax)) and x reads back as
 * q * scale, within amax / 254.  A group below 2^-100 reads back as zeros, one
 * that holds an infinity or a NaN as NaN.
 */
#ifndef GMDN_LM_H
#define GMDN_LM_H

#include <stddef.h>
#include <stdint.h>

#include "gmdn_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------- layer norm
 * y = (x - mean) rstd weight + bias over rows of d <= 16384 values, with
 * rstd = 1 / sqrt(var + eps).  weight (and with it bias, of the same type) may
 * be NULL: 1 and 0.  (x_type, y_type) is (bf16, bf16), (f32, f32) or
 * (f32, bf16).  mean and rstd (rows) are kept for the backward; where q and
 * scale are given they receive x's checkpoint. */
int gmdn_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                        int8_t* q, float* scale, int64_t rows, int64_t d, int64_t x_stride, float eps,
                        int32_t x_type, int32_t y_type, int32_t w_type, void* stream);

/* Floats of the backward's workspace (sums of the weight's gradient); 0 for few
 * rows. */
size_t gmdn_layer_norm_bwd_workspace_floats(int64_t rows, int64_t d);

/* dx (x_type), dweight and dbias (w_type; where weight is given) from dy
 * (y_type) and x, or with x NULL its checkpoint q, scale. */
int gmdn_layer_norm_bwd(const void* dy, const void* x, const int8_t* q, const float* scale, const void* weight,
                        const float* mean, const float* rstd, void* dx, void* dweight, void* dbias, float* workspace,
                        size_t workspace_floats, int64_t rows, int64_t d, int64_t dy_stride, int64_t x_stride,
                        int32_t x_type, int32_t y_type, int32_t w_type, void* stream);

/* y again, from x's checkpoint and the forward's statistics: the operand of
 * the following product's weight gradient. */
int gmdn_layer_norm8_rebuild(const int8_t* q, const float* scale, const void* weight, const void* bias,
                             const float* mean, const float* rstd, void* y, int64_t rows, int64_t d, int32_t y_type,
                             int32_t w_type, void* stream);

/* ------------------------------------------------------- 8-bit checkpoints */
/* Groups of a row: ceil(d / 128). */
int64_t gmdn_act8_groups(int64_t d);

int gmdn_act8_pack(const void* x, int8_t* q, float* scale, int64_t rows, int64_t d, int64_t x_stride, int32_t dtype,
                   void* stream);
int gmdn_act8_unpack(const int8_t* q, const float* scale, void* x, int64_t rows, int64_t d, int32_t dtype,
                     void* stream);

/* a = GELU(h) = h Phi(h) (Phi the normal distribution function), and h's
 * checkpoint (none where q and scale are NULL). */
int gmdn_gelu8_fwd(const void* h, void* a, int8_t* q, float* scale, int64_t rows, int64_t d, int64_t h_stride,
                   int32_t dtype, void* stream);

/* dh = da GELU'(h) and, where a is not NULL, a = GELU(h) again, with h as its
 * checkpoint reads back. */
int gmdn_gelu8_bwd(const void* da, const int8_t* q, const float* scale, void* dh, void* a, int64_t rows, int64_t d,
                   int64_t da_stride, int32_t dtype, void* stream);

/* -------------------------------------------------------- log probabilities
 * Over rows of `vocab` logits: logprob (rows), the log probability of the
 * row's token (0 where it is ignore_index, NaN where it is outside the
 * vocabulary); entropy (rows) in nats; the top <= 32 likeliest tokens (larger
 * logit first, equal ones by index) and their log probabilities, (rows, top);
 * stats (rows, 2), the largest logit and the log of the sum of e^(logit -
 * largest), kept for the backward.
 * Masked logits are -inf.  A row of nothing else has log probabilities -inf
 * and entropy 0, and no gradient.  A NaN or +inf in a row makes it NaN (its
 * alternatives are then ordered with NaN first). */
int gmdn_logprobs_fwd(const void* logits, const int64_t* tokens, float* logprob, float* entropy, float* top_logprobs,
                      int64_t* top_tokens, float* stats, void* workspace, size_t workspace_bytes, int64_t rows,
                      int64_t vocab, int64_t stride, int32_t top, int64_t ignore_index, int32_t dtype, void* stream);

/* Bytes of the forward's workspace (8-byte aligned): 0 but for few rows of
 * large vocabularies, whose columns several workgroups share. */
size_t gmdn_logprobs_fwd_workspace_bytes(int64_t rows, int64_t vocab, int32_t top);

/* dlogits (rows, vocab) from the cotangents of logprob, entropy and
 * top_logprobs, each of which may be NULL. */
int gmdn_logprobs_bwd(const void* logits, const int64_t* tokens, const float* stats, const float* entropy,
                      const int64_t* top_tokens, const float* dlogprob, const float* dentropy, const float* dtop,
                      void* dlogits, int64_t rows, int64_t vocab, int64_t stride, int32_t top, int64_t ignore_index,
                      int32_t dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GMDN_LM_H */
