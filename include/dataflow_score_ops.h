/*
 * Scoring ops: what is computed from a model's logits besides the softmax and
 * the cross-entropy of dataflow_ops.h. No reference counterpart.
 *
 *   token_logprobs       log-probabilities of given tokens, the entropy, the
 *                        log-sum-exp and the likeliest columns of each row
 *   token_logprobs_bwd   the logits' gradient from those of the
 *                        log-probabilities and of the entropy
 *   distillation_loss    loss against a teacher's top logits, with the
 *                        logits' gradient
 *
 * They are registered by register_native_score_ops
 * (set_native_score_op_skeletons.h). dt is DATAFLOW_FP32, DATAFLOW_FP16 or
 * DATAFLOW_BF16. Row r of the logits is the n_cols elements from
 * logits + r * row_stride on (row_stride >= n_cols, in elements; the elements
 * between n_cols and row_stride are neither read nor written); rows need no
 * more alignment than their elements. `scale` is 1 / temperature, within
 * [1e-6, 1e6]: the probabilities of a row are p = softmax(scale * x).
 * Statistics, losses and the gradients of the loss are fp32.
 *
 * Each call returns 0, or -1 with a message on stderr and nothing launched.
 * Zero rows or columns launch nothing. Ops keep no state between calls, and
 * calls on different streams need no ordering: what a call needs besides its
 * operands is in `workspace`, whose size the _workspace functions give (0:
 * workspace may be NULL). A workspace is 256-byte aligned device memory of
 * any content; calls that may run at the same time need one each, and so
 * does each captured graph that may run beside another.
 */
#ifndef DATAFLOW_SCORE_OPS_H
#define DATAFLOW_SCORE_OPS_H

#include "dataflow.h"
#include "ops.h"
#include "dataflow_handle.h"
#include "set_native_score_op_skeletons.h"

#ifdef __cplusplus
extern "C" {
#endif

/* at most so many given tokens, alternatives and teacher logits per row */
#define SCORE_MAX_TOKENS_PER_ROW 1024
#define SCORE_MAX_TOP_K 256
#define SCORE_MAX_TEACHER_K 1024

/* Workspace bytes of submit_token_logprobs for these sizes. */
uint64_t dataflow_token_logprobs_workspace(DataflowDatatype dt, int n_rows, int n_cols, int top_k);

/* With z = scale * x_r:
 *   lse[r]          = log sum_j exp(z_j)
 *   logprobs[r, m]  = z[tokens[r, m]] - lse[r]          m < tokens_per_row
 *   entropy[r]      = -sum_j p_j log p_j                (natural logarithms)
 *   top_ids[r, i]   = the columns of the top_k largest logits, largest first,
 *                     of equal ones the lowest column first
 *   top_logprobs[r, i] = z[top_ids[r, i]] - lse[r]      i < top_k
 * entropy and lse may be NULL; tokens and logprobs too with tokens_per_row 0,
 * top_ids and top_logprobs with top_k 0. top_k may not exceed n_cols. A token
 * that is no column (>= n_cols) gets log-probability 0. Columns of -inf have
 * probability 0. A row of -inf alone has lse -inf, entropy 0 and
 * log-probabilities -inf. A row that holds NaN or +inf has NaN for its
 * statistics; its top_ids are ordered with every NaN below -inf. */
int submit_token_logprobs(Dataflow_Handle * handle, int stream_id,
							DataflowDatatype dt,
							int n_rows, int n_cols, uint64_t row_stride, float scale,
							int tokens_per_row, int top_k,
							void * logits, uint32_t * tokens,
							float * logprobs, float * entropy, float * lse,
							uint32_t * top_ids, float * top_logprobs,
							uint64_t workspaceBytes, void * workspace);

/* The gradient of a loss L with respect to the logits, from
 * d_logprobs[r, m] = dL/dlogprobs[r, m], d_entropy[r] = dL/dentropy[r] and
 * what submit_token_logprobs wrote (same scale and tokens):
 *   dlogits[r, j] = scale * (sum_m d_logprobs[r, m] * [tokens[r, m] == j]
 *                   - p_j * (sum_m d_logprobs[r, m] + d_entropy[r] * (log p_j + entropy[r])))
 * with log p_j = scale * x_j - lse[r]; tokens that are no column contribute
 * nothing, a token given twice contributes twice. d_entropy may be NULL (no
 * such term; entropy may be NULL then), tokens and d_logprobs with
 * tokens_per_row 0. dlogits has rows grad_stride elements apart and either is
 * the logits themselves (with grad_stride == row_stride: in place) or does
 * not overlap them. A row whose upstream gradients are all 0, or whose lse is
 * -inf, gets gradient 0, whatever its logits hold. */
int submit_token_logprobs_bwd(Dataflow_Handle * handle, int stream_id,
							DataflowDatatype dt,
							int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float scale,
							int tokens_per_row,
							void * logits, uint32_t * tokens, float * lse, float * entropy,
							float * d_logprobs, float * d_entropy, void * dlogits);

/* Workspace bytes of submit_distillation_loss for these sizes. */
uint64_t dataflow_distillation_loss_workspace(DataflowDatatype dt, int n_rows, int n_cols, int top_k);

/* Distillation from a teacher's top_k logits (or log-probabilities: a constant
 * added to a row's values changes nothing), e.g. the top_ids and top_logprobs
 * of submit_token_logprobs at scale 1. With T = 1 / scale, the student's
 * p = softmax(scale * x_r) over all columns and the teacher's
 * q = softmax(scale * teacher_logits[r, :]) over its top_k entries:
 *   loss[r]       = T^2 * sum_k q_k * (log q_k - log p[teacher_ids[r, k]])
 *   mean_loss     = sum_r row_weights[r] * loss[r] / n_rows
 *   dlogits[r, j] = row_weights[r] * T * (p_j - sum_k q_k * [teacher_ids[r, k] == j])
 * dlogits is the gradient of sum_r row_weights[r] * loss[r]. Entries whose id
 * is no column are left out of q (0xffffffff pads short lists), and so are
 * values of -inf; a column given twice counts as two entries.
 * row_weights may be NULL (all 1), mean_loss NULL (not wanted), dlogits NULL
 * (the loss alone). dlogits has rows grad_stride elements apart and either is
 * the logits themselves (with grad_stride == row_stride: in place) or does
 * not overlap them. A row of weight 0 has loss 0 and gradient 0 whatever its
 * logits hold, and so has a row without a teacher entry. A row of -inf alone
 * has loss +inf and gradient 0; NaN or +inf make their row's loss and
 * gradient NaN. */
int submit_distillation_loss(Dataflow_Handle * handle, int stream_id,
							DataflowDatatype dt,
							int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float scale,
							int top_k,
							void * logits, uint32_t * teacher_ids, float * teacher_logits, float * row_weights,
							float * loss, float * mean_loss, void * dlogits,
							uint64_t workspaceBytes, void * workspace);

#ifdef __cplusplus
}
#endif

#endif
