/*
 * distillation_loss: loss of a student's logits against a teacher's top
 * logits, and the logits' gradient (formulas in dataflow_score_ops.h). With
 * q = softmax(s v) over the teacher's entries and T = 1 / s,
 *   loss = T^2 sum_k q_k (log q_k - log p_k),  dx_j = w T (p_j - sum_k q_k [i_k = j]).
 * The teacher's columns, whose logits are set aside before the first store
 * (the gradient may lie in the logits' place), are stored once more, whole,
 * after the others, so that they are rounded once.
 */
#include "score_rows.h"

struct Teacher {
	uint32_t id[SCORE_TEACHER_MAX];
	float q[SCORE_TEACHER_MAX], x[SCORE_TEACHER_MAX];
};

template <typename T>
__device__ __forceinline__ void distillation_loss_run(int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float s, int top_k,
													  const T * logits, const uint32_t * teacher_ids, const float * teacher_logits,
													  const float * row_weights, float * loss, T * dlogits) {
	__shared__ float cells[3 * SCORE_MAX_WAVES];
	__shared__ Teacher te;
	const float temperature = 1.0f / s;
	for (long r = blockIdx.x; r < n_rows; r += gridDim.x) {
		const T * row = logits + (uint64_t) r * row_stride;
		T * out = dlogits ? dlogits + (uint64_t) r * grad_stride : nullptr;
		const float w = row_weights ? row_weights[r] : 1.0f;
		__syncthreads();
		/* the teacher's entries: columns, and not -inf */
		float vmax = -__builtin_inff(), entries = 0.0f;
		for (int k = (int) threadIdx.x; k < top_k; k += (int) blockDim.x) {
			const uint32_t id = teacher_ids[r * top_k + k];
			const float v = teacher_logits[r * top_k + k];
			const bool is = id < (uint32_t) n_cols && v != -__builtin_inff();
			te.id[k] = is ? id : 0xffffffffu;
			te.q[k] = v;
			te.x[k] = is ? to_f(row[id]) : 0.0f;
			if (is) { vmax = fmaxf(vmax, v); entries = 1.0f; }
		}
		vmax = score_group_max(vmax, cells);
		entries = score_group_max(entries, cells);
		if (w == 0.0f || entries == 0.0f) {
			if (threadIdx.x == 0) loss[r] = 0.0f;
			if (out)
				for (long j = threadIdx.x; j < n_cols; j += blockDim.x) out[j] = from_f<T>(0.0f);
			continue;
		}
		float zq = 0.0f;
		for (int k = (int) threadIdx.x; k < top_k; k += (int) blockDim.x)
			if (te.id[k] != 0xffffffffu) zq += __builtin_amdgcn_exp2f((te.q[k] - vmax) * (s * SCORE_LOG2E));
		zq = score_group_sum(zq, cells);
		const RowStats st = score_row_stats(row, n_cols, s, cells);
		const float log_zq = logf(zq);
		float l = 0.0f;
		for (int k = (int) threadIdx.x; k < top_k; k += (int) blockDim.x)
			if (te.id[k] != 0xffffffffu) {
				const float d = s * (te.q[k] - vmax);
				const float q = __builtin_amdgcn_exp2f(d * SCORE_LOG2E) / zq;
				if (!(q == 0.0f)) l = fmaf(q, (d - log_zq) - (st.none() ? -__builtin_inff() : st.log_p(te.x[k], s)), l);
				te.q[k] = q;
			}
		l = score_group_sum(l, cells);
		if (threadIdx.x == 0) loss[r] = l * temperature * temperature;
		if (!out) continue;
		const float wt = w * temperature;
		if (st.none()) {
			for (long j = threadIdx.x; j < n_cols; j += blockDim.x) out[j] = from_f<T>(0.0f);
			continue;
		}
		const float s_log2e = s * SCORE_LOG2E, a = wt * st.inv_z;
		for (long j = threadIdx.x; j < n_cols; j += blockDim.x) out[j] = from_f<T>(a * __builtin_amdgcn_exp2f((to_f(row[j]) - st.max) * s_log2e));
		__threadfence_block();
		__builtin_amdgcn_s_waitcnt(0);
		__syncthreads();
		for (int k = (int) threadIdx.x; k < top_k; k += (int) blockDim.x) {
			const uint32_t id = te.id[k];
			if (id == 0xffffffffu) continue;
			float q = 0.0f;
			bool first = true;
			for (int o = 0; o < top_k; o++)
				if (te.id[o] == id) {
					first = first && o >= k;
					q += te.q[o];
				}
			const float p = __builtin_amdgcn_exp2f((te.x[k] - st.max) * s_log2e) * st.inv_z;
			if (first) out[id] = from_f<T>(wt * (p - q));
		}
	}
}

/* mean_loss = sum_r w_r loss_r / n_rows in 64 bits, in a fixed order */
__device__ __forceinline__ void distillation_loss_mean(int n_rows, const float * row_weights, const float * loss, float * mean_loss) {
	__shared__ double part[SCORE_THREADS];
	double sum = 0.0;
	for (long r = threadIdx.x; r < n_rows; r += blockDim.x) {
		const float w = row_weights ? row_weights[r] : 1.0f;
		if (w != 0.0f) sum += (double) w * (double) loss[r];
	}
	part[threadIdx.x] = sum;
	for (int step = SCORE_THREADS / 2; step > 0; step /= 2) {
		__syncthreads();
		if ((int) threadIdx.x < step) part[threadIdx.x] += part[threadIdx.x + step];
	}
	if (threadIdx.x == 0) *mean_loss = (float) (part[0] / (double) n_rows);
}

#define DISTILLATION_ARGS(T)                                                                                                     \
	int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float scale, int top_k, T * logits,                       \
		uint32_t * teacher_ids, float * teacher_logits, float * row_weights, float * loss, float * mean_loss, T * dlogits,       \
		uint64_t workspace_bytes, void * workspace
#define DISTILLATION_LOSS_KERNEL(SUF, T)                                                                                         \
	extern "C" __global__ void __launch_bounds__(SCORE_THREADS) distillation_loss_##SUF##_kernel(DISTILLATION_ARGS(T)) {         \
		distillation_loss_run<T>(n_rows, n_cols, row_stride, grad_stride, scale, top_k, logits, teacher_ids, teacher_logits,     \
								 row_weights, loss, dlogits);                                                                    \
	}                                                                                                                            \
	extern "C" __global__ void __launch_bounds__(SCORE_THREADS) distillation_loss_##SUF##_kernel_finish(DISTILLATION_ARGS(T)) {  \
		distillation_loss_mean(n_rows, row_weights, loss, mean_loss);                                                            \
	}

DISTILLATION_LOSS_KERNEL(fp32, float)
DISTILLATION_LOSS_KERNEL(fp16, f16_t)
DISTILLATION_LOSS_KERNEL(bf16, bf16_t)
