/*
 * Op API of the scoring ops (dataflow_score_ops.h): build an Op on the stack
 * and submit it. The arguments are checked where the launch is configured, so
 * an Op that is submitted by hand is checked too.
 */
#include "dataflow_score_ops.h"
#include "score_geometry.h"

static int submit_score_op(Dataflow_Handle * handle, Op * op, int stream_id, const char * what) {
	if (!handle || !handle->submit_op) {
		fprintf(stderr, "Error: cannot submit %s op: handle is not initialised...\n", what);
		return -1;
	}
	if (handle->submit_op(handle, op, stream_id)) {
		fprintf(stderr, "Error: failed to submit %s op...\n", what);
		return -1;
	}
	return 0;
}

uint64_t dataflow_token_logprobs_workspace(DataflowDatatype dt, int n_rows, int n_cols, int top_k) {
	return score_logprobs_workspace(n_rows, n_cols, (int) dataflow_sizeof_element(dt), top_k);
}

uint64_t dataflow_distillation_loss_workspace(DataflowDatatype dt, int n_rows, int n_cols, int top_k) {
	return score_distill_workspace(n_rows, n_cols, (int) dataflow_sizeof_element(dt), top_k);
}

int submit_token_logprobs(Dataflow_Handle * handle, int stream_id,
							DataflowDatatype dt,
							int n_rows, int n_cols, uint64_t row_stride, float scale,
							int tokens_per_row, int top_k,
							void * logits, uint32_t * tokens,
							float * logprobs, float * entropy, float * lse,
							uint32_t * top_ids, float * top_logprobs,
							uint64_t workspaceBytes, void * workspace) {
	Op op;
	set_native_token_logprobs_skeleton(&op.op_skeleton, dt);
	void ** a = op.op_args;
	a[0] = &n_rows; a[1] = &n_cols; a[2] = &row_stride; a[3] = &scale;
	a[4] = &tokens_per_row; a[5] = &top_k;
	a[6] = &logits; a[7] = &tokens; a[8] = &logprobs; a[9] = &entropy; a[10] = &lse;
	a[11] = &top_ids; a[12] = &top_logprobs;
	a[13] = &workspaceBytes; a[14] = &workspace;
	return submit_score_op(handle, &op, stream_id, "token logprobs");
}

int submit_token_logprobs_bwd(Dataflow_Handle * handle, int stream_id,
							DataflowDatatype dt,
							int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float scale,
							int tokens_per_row,
							void * logits, uint32_t * tokens, float * lse, float * entropy,
							float * d_logprobs, float * d_entropy, void * dlogits) {
	Op op;
	set_native_token_logprobs_bwd_skeleton(&op.op_skeleton, dt);
	void ** a = op.op_args;
	a[0] = &n_rows; a[1] = &n_cols; a[2] = &row_stride; a[3] = &grad_stride; a[4] = &scale;
	a[5] = &tokens_per_row;
	a[6] = &logits; a[7] = &tokens; a[8] = &lse; a[9] = &entropy;
	a[10] = &d_logprobs; a[11] = &d_entropy; a[12] = &dlogits;
	return submit_score_op(handle, &op, stream_id, "token logprobs bwd");
}

int submit_distillation_loss(Dataflow_Handle * handle, int stream_id,
							DataflowDatatype dt,
							int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float scale,
							int top_k,
							void * logits, uint32_t * teacher_ids, float * teacher_logits, float * row_weights,
							float * loss, float * mean_loss, void * dlogits,
							uint64_t workspaceBytes, void * workspace) {
	Op op;
	set_native_distillation_loss_skeleton(&op.op_skeleton, dt);
	void ** a = op.op_args;
	a[0] = &n_rows; a[1] = &n_cols; a[2] = &row_stride; a[3] = &grad_stride; a[4] = &scale;
	a[5] = &top_k;
	a[6] = &logits; a[7] = &teacher_ids; a[8] = &teacher_logits; a[9] = &row_weights;
	a[10] = &loss; a[11] = &mean_loss; a[12] = &dlogits;
	a[13] = &workspaceBytes; a[14] = &workspace;
	return submit_score_op(handle, &op, stream_id, "distillation loss");
}
