/*
 * Skeletons and registration of the scoring ops (dataflow_score_ops.h). No
 * reference counterpart. set_native_op_skeleton knows them by name too.
 */
#ifndef SET_NATIVE_SCORE_OPS_H
#define SET_NATIVE_SCORE_OPS_H

#include "dataflow.h"
#include "ops.h"
#include "dataflow_handle.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Registers the scoring ops in fp32, fp16 and bf16 from their code object and
 * the launch-configuration library of the native ops. Returns the number of
 * functions added (9) or -1. Call once per handle. */
int register_native_score_ops(Dataflow_Handle * dataflow_handle, char * score_function_code_filename, char * native_function_config_filename);

/* "token_logprobs_<DT>", 15 args: (INT_SCALAR n_rows, INT_SCALAR n_cols,
 * UINT64_SCALAR row_stride, FP32_SCALAR scale, INT_SCALAR tokens_per_row,
 * INT_SCALAR top_k, dt logits, UINT32 tokens, FP32 logprobs, FP32 entropy,
 * FP32 lse, UINT32 top_ids, FP32 top_logprobs, UINT64_SCALAR workspaceBytes,
 * VOID workspace) */
void set_native_token_logprobs_skeleton(Op_Skeleton * skeleton, DataflowDatatype datatype);

/* "token_logprobs_bwd_<DT>", 13 args: (INT_SCALAR n_rows, INT_SCALAR n_cols,
 * UINT64_SCALAR row_stride, UINT64_SCALAR grad_stride, FP32_SCALAR scale,
 * INT_SCALAR tokens_per_row, dt logits, UINT32 tokens, FP32 lse, FP32 entropy,
 * FP32 d_logprobs, FP32 d_entropy, dt dlogits) */
void set_native_token_logprobs_bwd_skeleton(Op_Skeleton * skeleton, DataflowDatatype datatype);

/* "distillation_loss_<DT>", 15 args: (INT_SCALAR n_rows, INT_SCALAR n_cols,
 * UINT64_SCALAR row_stride, UINT64_SCALAR grad_stride, FP32_SCALAR scale,
 * INT_SCALAR top_k, dt logits, UINT32 teacher_ids, FP32 teacher_logits,
 * FP32 row_weights, FP32 loss, FP32 mean_loss, dt dlogits,
 * UINT64_SCALAR workspaceBytes, VOID workspace) */
void set_native_distillation_loss_skeleton(Op_Skeleton * skeleton, DataflowDatatype datatype);

#ifdef __cplusplus
}
#endif

#endif
