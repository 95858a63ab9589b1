/*
 * token_logprobs: log-probabilities of given tokens, entropy, log-sum-exp and
 * the k likeliest columns of each row of logits (formulas and odd cases in
 * dataflow_score_ops.h). One workgroup per row.
 */
#include "score_rows.h"

template <typename T>
__device__ __forceinline__ void token_logprobs_run(int n_rows, int n_cols, uint64_t row_stride, float s, int tokens_per_row, int top_k,
												   const T * logits, const uint32_t * tokens, float * logprobs, float * entropy, float * lse,
												   uint32_t * top_ids, float * top_logprobs) {
	__shared__ float cells[SCORE_MAX_WAVES];
	__shared__ ScoreTop top;
	for (long r = blockIdx.x; r < n_rows; r += gridDim.x) {
		const T * row = logits + (uint64_t) r * row_stride;
		const RowStats st = score_row_stats(row, n_cols, s, cells);
		if (threadIdx.x == 0) {
			if (entropy) entropy[r] = st.entropy();
			if (lse) lse[r] = st.lse(s);
		}
		for (int m = (int) threadIdx.x; m < tokens_per_row; m += (int) blockDim.x) {
			const uint32_t t = tokens[r * tokens_per_row + m];
			logprobs[r * tokens_per_row + m] = t < (uint32_t) n_cols ? st.log_p(to_f(row[t]), s) : 0.0f;
		}
		if (top_k > 0) {
			score_select(row, n_cols, top_k, top);
			for (int i = (int) threadIdx.x; i < top_k; i += (int) blockDim.x) {
				const long at = r * top_k + score_rank(top, top_k, i);
				top_ids[at] = top.id[i];
				top_logprobs[at] = st.log_p(to_f(row[top.id[i]]), s);
			}
		}
	}
}

#define TOKEN_LOGPROBS_KERNEL(SUF, T)                                                                                            \
	extern "C" __global__ void __launch_bounds__(SCORE_THREADS) token_logprobs_##SUF##_kernel(int n_rows, int n_cols,            \
			uint64_t row_stride, float scale, int tokens_per_row, int top_k, T * logits, uint32_t * tokens, float * logprobs,    \
			float * entropy, float * lse, uint32_t * top_ids, float * top_logprobs, uint64_t workspace_bytes, void * workspace) { \
		token_logprobs_run<T>(n_rows, n_cols, row_stride, scale, tokens_per_row, top_k, logits, tokens, logprobs, entropy, lse,  \
							  top_ids, top_logprobs);                                                                            \
	}

TOKEN_LOGPROBS_KERNEL(fp32, float)
TOKEN_LOGPROBS_KERNEL(fp16, f16_t)
TOKEN_LOGPROBS_KERNEL(bf16, bf16_t)
