/*
 * token_logprobs_bwd: the logits' gradient from those of the log-probabilities
 * and of the entropy (formula in dataflow_score_ops.h). With G = sum_m g_m over
 * the tokens that are columns, h the entropy's gradient and H the entropy,
 *   dx_j = -s p_j (G + h (log p_j + H)) + s sum_m g_m [t_m = j].
 * Every column gets the first term; the tokens' columns, whose logits are set
 * aside before the first store (the gradient may lie in the logits' place),
 * are then stored once more, whole, so that they are rounded once. p_j is
 * exp(s x_j - lse) with the forward pass' lse, which is all that the row needs:
 * nothing is reduced over columns.
 *
 * Bound by reading the logits and writing as much: 2048 x 128256 bf16 189 us
 * (5.6 TB/s), 8192 x 32000 180 us (5.8 TB/s), 509 x 50257 fp16 22.0 us (4.7
 * TB/s); 16 x 32000 fp32 5.5 us, a launch. Stores are aligned, loads lie as they
 * do (8192 x 32001 186 us, with chunks from the rows' first elements on 223).
 */
#include "score_rows.h"

struct GradTokens {
	uint32_t id[SCORE_TOKENS_MAX];
	float g[SCORE_TOKENS_MAX], x[SCORE_TOKENS_MAX];
};
#define SCORE_NO_TOKEN 0xffffffffu

/* -s p (G + h (log p + H)) of a column */
template <bool ENTROPY>
struct GradTerm {
	float s, lse, down, h, H;
	__device__ __forceinline__ float operator()(float x) const {
		const float lp = fmaf(s, x, -lse);
		const float p = __builtin_amdgcn_exp2f(lp * SCORE_LOG2E);
		/* the bound, below which p is 0, keeps -inf * 0 out */
		return p * (ENTROPY ? -s * fmaf(h, fmaxf(lp, SCORE_FAR_BELOW) + H, down) : -s * down);
	}
};

template <typename T>
struct GradRow {
	const T * row;
	T * out;
	int tokens_per_row;
	RowSlice sl;
	GradTokens & tok;

	template <typename F>
	__device__ __forceinline__ void run(const F & term, float s) const {
		score_map(row, out, sl, term);
		if (tokens_per_row == 0) return;
		score_stores_done();
		for (int m = (int) threadIdx.x; m < tokens_per_row; m += (int) blockDim.x) {
			const uint32_t t = tok.id[m];
			if (t == SCORE_NO_TOKEN || !sl.holds(t, VecOf<T>::N)) continue;
			float g = 0.0f;
			bool first = true;
			for (int o = 0; o < tokens_per_row; o++)
				if (tok.id[o] == t) {
					first = first && o >= m;
					g += tok.g[o];
				}
			if (first) out[t] = from_f<T>(fmaf(s, g, term(tok.x[m])));
		}
	}
};

template <typename T>
__device__ __forceinline__ void token_logprobs_bwd_run(int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float s,
													   int tokens_per_row, const T * logits, const uint32_t * tokens, const float * lse,
													   const float * entropy, const float * d_logprobs, const float * d_entropy, T * dlogits) {
	constexpr int V = VecOf<T>::N;
	__shared__ float cells[SCORE_MAX_WAVES];
	__shared__ GradTokens tok;
	const Score_Plan plan = score_map_plan(n_rows, n_cols, (int) sizeof(T));
	for (long w = blockIdx.x; w < (long) n_rows * plan.slices; w += gridDim.x) {
		const long r = plan.slices == 1 ? w : w / plan.slices;
		const int slice = plan.slices == 1 ? 0 : (int) (w - r * plan.slices);
		const T * row = logits + (uint64_t) r * row_stride;
		T * out = dlogits + (uint64_t) r * grad_stride;
		const RowSlice sl(n_cols, V, score_head(out, n_cols), slice, plan.slices, plan.slice_chunks);   /* stores aligned */
		__syncthreads();
		float down = 0.0f, any = 0.0f;
		for (int m = (int) threadIdx.x; m < tokens_per_row; m += (int) blockDim.x) {
			const uint32_t t = tokens[r * tokens_per_row + m];
			const bool is = t < (uint32_t) n_cols;
			const float g = is ? d_logprobs[r * tokens_per_row + m] : 0.0f;
			tok.id[m] = is ? t : SCORE_NO_TOKEN;
			tok.g[m] = g;
			tok.x[m] = is && sl.holds(t, V) ? to_f(row[t]) : 0.0f;
			down += g;
			any = g != 0.0f ? 1.0f : any;
		}
		if (tokens_per_row == 1) {
			__syncthreads();
			down = tok.g[0];
			any = down != 0.0f ? 1.0f : 0.0f;
		}
		else {
			down = score_group_sum(down, cells);
			any = score_group_max(any, cells);
		}
		const float row_lse = lse[r], h = d_entropy ? d_entropy[r] : 0.0f, H = d_entropy ? entropy[r] : 0.0f;
		const GradRow<T> g = {row, out, tokens_per_row, sl, tok};
		if ((any == 0.0f && h == 0.0f) || row_lse == -__builtin_inff()) score_clear(out, sl);
		else if (h != 0.0f) g.run(GradTerm<true>{s, row_lse, down, h, H}, s);
		else g.run(GradTerm<false>{s, row_lse, down, h, H}, s);
	}
}

#define TOKEN_LOGPROBS_BWD_KERNEL(SUF, T)                                                                                      \
	extern "C" __global__ void __launch_bounds__(64 * SCORE_MAX_WAVES, 8) token_logprobs_bwd_##SUF##_kernel(int n_rows, int n_cols,      \
			uint64_t row_stride, uint64_t grad_stride, float scale, int tokens_per_row, T * logits, uint32_t * tokens,         \
			float * lse, float * entropy, float * d_logprobs, float * d_entropy, T * dlogits) {                                \
		token_logprobs_bwd_run<T>(n_rows, n_cols, row_stride, grad_stride, scale, tokens_per_row, logits, tokens, lse,         \
								  entropy, d_logprobs, d_entropy, dlogits);                                                    \
	}

TOKEN_LOGPROBS_BWD_KERNEL(fp32, float)
TOKEN_LOGPROBS_BWD_KERNEL(fp16, f16_t)
TOKEN_LOGPROBS_BWD_KERNEL(bf16, bf16_t)
