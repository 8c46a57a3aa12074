/* C ABI of token log probabilities (libmoe_b200.so, sm_100a): what a language model answers with, and the
 * gradient that a loss on it sends back.  It stands beside the fused head + cross-entropy of transformer_b200.h,
 * which keeps the loss only (reference causal_lm_loss.rs:66-150).
 *
 *   lse[r]     = log sum_v exp(x[r, v])
 *   logprob[r] = x[r, target[r]] - lse[r]
 *   entropy[r] = - sum_v p[r, v] log p[r, v],   p = exp(x - lse)
 *   top        = the top_n largest logits of the row, larger first, the lower index first among equal ones
 *
 *   grad_x[r, v] = grad_logprob[r] * (1[v == target[r]] - p[r, v]) - grad_entropy[r] * p[r, v] * (log p[r, v] + entropy[r])
 *
 * Sums are f32 whatever the logits' type.  Log probabilities are never above 0; the one of a near-certain token is off by about 2^-23, not by a
 * part of itself.  Edge values:
 *   - a masked logit is -inf: probability 0, nothing added to the entropy, gradient 0; it may appear among the
 *     alternatives (with log probability -inf) once the others are used up.  Lowest finite values are ordinary values.
 *   - a row of -inf only has no distribution: lse = logprob = -inf, entropy 0, gradient 0.
 *   - a negative target means "no token": logprob 0, and grad_logprob of that row is not used.
 *   - a target >= vocab gives logprob NaN and a gradient row of NaN.
 *   - a row with a NaN or a +inf has NaN results; its alternatives are ids of the row, or -1.
 *
 * Stateless: all pointers are device pointers of the current device, owned by the caller; nothing is allocated, no scratch is
 * kept, every call can be captured into a CUDA graph, and calls on different streams do not meet.  x is f32 (MOE_PRECISION_F32)
 * or bf16 (MOE_PRECISION_BF16), rows `row_stride` elements apart (>= vocab; any alignment of the element type).  Status codes are the
 * moe_status values of moe_b200.h; on failure `message` (optional) receives the reason.  rows == 0 is a call that does nothing.
 */
#ifndef LOGPROBS_B200_H
#define LOGPROBS_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LOGPROBS_MAX_TOP 32

/* targets [rows] (null: every row has no token); logprob, entropy, lse [rows] f32; top_logprob f32 and top_ids i32 [rows, top_n],
 * 0 <= top_n <= min(vocab, LOGPROBS_MAX_TOP) (both null when top_n is 0).  Any of logprob, entropy and lse may be null. */
int32_t logprobs_forward(const void* x, int64_t row_stride, const int32_t* targets, int32_t rows, int32_t vocab, int32_t top_n,
                         int32_t precision, float* logprob, float* entropy, float* lse, float* top_logprob, int32_t* top_ids,
                         void* stream, char* message, int32_t message_len);

/* grad_x has x's type, its rows grad_stride elements apart; it may be x itself (same stride); otherwise the two share
 * nothing, though their rows may lie between one another, and an overlap is InvalidInput.
 * lse and entropy are the forward call's.  grad_logprob or grad_entropy may be null: no such term (entropy may then be null too). */
int32_t logprobs_backward(const void* x, int64_t row_stride, const int32_t* targets, const float* lse, const float* entropy,
                          const float* grad_logprob, const float* grad_entropy, int32_t rows, int32_t vocab, int32_t precision,
                          void* grad_x, int64_t grad_stride, void* stream, char* message, int32_t message_len);

#ifdef __cplusplus
}
#endif
#endif
