/*
 * distillation_loss: loss of a student's logits against a teacher's top
 * logits, and the logits' gradient (formulas in dataflow_score_ops.h). With
 * q = softmax(s v) over the teacher's entries and T = 1 / s,
 *   loss = T^2 sum_k q_k (log q_k - log p_k),  dx_j = w T (p_j - sum_k q_k [i_k = j]).
 * Every column gets the first term of the gradient; the teacher's columns,
 * whose logits are set aside before the first store (the gradient may lie in
 * the logits' place), are stored once more, whole, when the others are there,
 * so that they are rounded once.
 *
 * Two ways. Where a workgroup can hold a row in its registers and rows are
 * many (distill_held), a row is read once and written once; otherwise
 * (distill_parts, distill_out) one launch finds the statistics of the rows'
 * slices and a second one reads them again for the gradient.
 *
 * Bound by reading the logits and writing as much, held: 4096 x 128256 bf16 with
 * 64 entries 365 us (5.8 TB/s), 1024 x 50257 fp16 with 128 45 us (4.5 TB/s),
 * 8192 x 32000 205 us (5.1 TB/s); 2048 x 151936 230 us, read twice 335. Longer
 * rows are read twice: 2600 x 200000 519 us. The loss alone reads once: 256 x
 * 151936 bf16 18.5 us with the mean, which is a launch of its own. Few rows are
 * bound by the launches: 1 x 128256 14.1 us, 7 x 1000 fp32 8.4 us.
 */
#include "score_rows.h"

#define SCORE_NO_COLUMN 0xffffffffu

struct DistillArgs {
	int n_rows, n_cols;
	uint64_t row_stride, grad_stride;
	float s;
	int top_k;
	const void * logits;
	const uint32_t * ids;
	const float * values;
	const float * weights;
	float * loss;
	void * dlogits;
	Score_Part * parts;   /* of a row's slices, row after row */
	float * picked;       /* the logits of a row's teacher columns, row after row */
};

/* sums that a teacher's entries leave: shift and sum of exp(s (v - max)) */
__device__ __forceinline__ RowPart teacher_entry(float v, bool is) {
	RowPart p;
	if (is) {
		/* NaN makes the sum NaN, and so does +inf, which has no difference to itself */
		p.m = fmaxf(v, -__builtin_inff());
		p.z = __builtin_amdgcn_exp2f(v - p.m);
	}
	return p;
}

/* ---------------- rows held in registers ---------------- */

/* what a workgroup's waves tell each other of a row; rows alternate between
 * two of them, so one barrier a row is enough */
struct DistillCells {
	float m[SCORE_MAX_WAVES], z[SCORE_MAX_WAVES], vm[SCORE_MAX_WAVES], vz[SCORE_MAX_WAVES], loss[SCORE_MAX_WAVES];
};

template <typename T> __device__ __forceinline__ float buf_load_elem(__amdgpu_buffer_rsrc_t r, uint32_t off);
template <> __device__ __forceinline__ float buf_load_elem<float>(__amdgpu_buffer_rsrc_t r, uint32_t off) {
	return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}
template <> __device__ __forceinline__ float buf_load_elem<f16_t>(__amdgpu_buffer_rsrc_t r, uint32_t off) {
	return to_f(f16_t{(uint16_t) __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0)});
}
template <> __device__ __forceinline__ float buf_load_elem<bf16_t>(__amdgpu_buffer_rsrc_t r, uint32_t off) {
	return to_f(bf16_t{(uint16_t) __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0)});
}
template <typename T> __device__ __forceinline__ void buf_store_elem(__amdgpu_buffer_rsrc_t r, uint32_t off, float v);
template <> __device__ __forceinline__ void buf_store_elem<float>(__amdgpu_buffer_rsrc_t r, uint32_t off, float v) {
	__builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, off, 0, 0);
}
template <> __device__ __forceinline__ void buf_store_elem<f16_t>(__amdgpu_buffer_rsrc_t r, uint32_t off, float v) {
	__builtin_amdgcn_raw_buffer_store_b16(from_f<f16_t>(v).bits, r, off, 0, 0);
}
template <> __device__ __forceinline__ void buf_store_elem<bf16_t>(__amdgpu_buffer_rsrc_t r, uint32_t off, float v) {
	__builtin_amdgcn_raw_buffer_store_b16(from_f<bf16_t>(v).bits, r, off, 0, 0);
}
/* past every range: loads give 0, stores are dropped */
#define SCORE_NOWHERE 0xfffffff0u

/* A workgroup walks rows a grid apart and holds one of them: thread t has its
 * chunks t + j blockDim.x, j < CH. Behind a thread's last store of a row's outputs
 * its registers take the next row's logits, so the next row arrives while this
 * one leaves and its statistics are formed as it arrives. Stores and loads each
 * go out together: memory does worse by them in turn (4096 x 128256 bf16 365 us;
 * by fours 385, by ones 402). All memory
 * accesses are unconditional (buffer ranges drop what is not there), so the
 * waits count them exactly. Vector-memory operations complete in order, so
 * when a thread has a row's last chunk its stores of the row before are done;
 * behind the next barrier everybody's are, and there the teacher's columns of
 * that row are stored, and its loss. */
template <typename T, int CH, int NT>
__device__ __forceinline__ void distill_held(const DistillArgs & a) {
	constexpr int V = VecOf<T>::N;
	constexpr uint32_t E = (uint32_t) sizeof(T);
	constexpr int B = CH < 4 ? CH : 4;   /* chunks that share a shift */
	__shared__ DistillCells both[2];
	extern __shared__ uint4 entries[];   /* ids and values of two rows */
	const int tid = (int) threadIdx.x, nt = NT ? NT : (int) blockDim.x, wave = tid >> 6, waves = nt >> 6, K = a.top_k;
	const float s_log2e = a.s * SCORE_LOG2E, temperature = 1.0f / a.s;
	const uint32_t voff = (uint32_t) tid * 16u;
	const uint32_t row_bytes = (uint32_t) a.n_cols * E;
	const uint32_t entry_off = tid < K ? (uint32_t) tid * 4u : SCORE_NOWHERE;

	const auto row_ptr = [&](long r) { return static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride; };
	const auto out_ptr = [&](long r) { return static_cast<T *>(a.dlogits) + (uint64_t) r * a.grad_stride; };
	/* chunks lie as the gradient's do */
	const auto head_of = [&](long r) { return score_head(out_ptr(r), a.n_cols); };
	/* this thread's element of a row's head or tail */
	const auto single_off = [&](int head) {
		const int tail = head + (a.n_cols - head) / V * V, e = tid < head ? tid : tail + tid - head;
		return e < a.n_cols ? (uint32_t) e * E : SCORE_NOWHERE;
	};
	const auto weight = [&](long r) { return r >= a.n_rows ? 0.0f : a.weights ? load_scalar(a.weights + r) : 1.0f; };
	const auto ids_rsrc = [&](long r) { return make_rsrc(a.ids + (uint64_t) r * K, r < a.n_rows ? (uint32_t) K * 4u : 0u); };
	const auto values_rsrc = [&](long r) { return make_rsrc(a.values + (uint64_t) r * K, r < a.n_rows ? (uint32_t) K * 4u : 0u); };
	const auto pick_off = [&](uint32_t id) { return tid < K && id < (uint32_t) a.n_cols ? id * E : SCORE_NOWHERE; };

	long r = blockIdx.x;
	float w = weight(r);
	int head = head_of(r), chunks = (a.n_cols - head) / V;
	uint32_t single = single_off(head);
	R16 x[CH];
	uint32_t id;
	float v, xk, xt;
	{
		id = __builtin_amdgcn_raw_buffer_load_b32(ids_rsrc(r), entry_off, 0, 0);
		v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(values_rsrc(r), entry_off, 0, 0));
		const bool there = w != 0.0f;
		const __amdgpu_buffer_rsrc_t rs = make_rsrc(row_ptr(r) + head, there ? (uint32_t) chunks * 16u : 0u);
#pragma unroll
		for (int j = 0; j < CH; j++) x[j] = buf_load16_nt(rs, voff, (uint32_t) (j * nt) * 16u);
		const __amdgpu_buffer_rsrc_t re = make_rsrc(row_ptr(r), there ? row_bytes : 0u);
		xt = buf_load_elem<T>(re, single);
		xk = buf_load_elem<T>(re, pick_off(id));
	}
	long before = -1;                        /* the row whose teacher columns and loss are still to be stored */
	uint32_t fix_off = SCORE_NOWHERE;
	float fix = 0.0f;
	int turn = 0;
	for (; r < a.n_rows; turn ^= 1) {
		DistillCells & cells = both[turn];
		uint32_t * ids = reinterpret_cast<uint32_t *>(entries) + turn * 2 * score_entries(K);
		float * values = reinterpret_cast<float *>(ids + score_entries(K));
		const long next = r + gridDim.x;
		const float next_w = weight(next);
		const uint32_t next_id = __builtin_amdgcn_raw_buffer_load_b32(ids_rsrc(next), entry_off, 0, 0);
		const float next_v = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(values_rsrc(next), entry_off, 0, 0));

		/* statistics */
		RowPart p;
		const float xs = single != SCORE_NOWHERE ? xt : -__builtin_inff();
		p.m = fmaxf(xs, -__builtin_inff());
		p.z = __builtin_amdgcn_exp2f((xs - (p.m == -__builtin_inff() ? 0.0f : p.m)) * s_log2e);
#pragma unroll
		for (int j0 = 0; j0 < CH; j0 += B) {
			float m = -__builtin_inff();
#pragma unroll
			for (int j = j0; j < j0 + B; j++) {
				if (j * nt + tid >= chunks) continue;
				float f[V];
				unpack16<T>(x[j], f);
#pragma unroll
				for (int i = 0; i < V; i++) m = fmaxf(m, f[i]);
			}
			p.shift(fmaxf(p.m, m), s_log2e);
			const float ref = p.m == -__builtin_inff() ? 0.0f : p.m;
			float z[2] = {0.0f, 0.0f};
#pragma unroll
			for (int j = j0; j < j0 + B; j++) {
				if (j * nt + tid >= chunks) continue;
				__builtin_amdgcn_sched_barrier(0);
				reg_barrier(x[j]);
				float f[V];
				unpack16<T>(x[j], f);
#pragma unroll
				for (int i = 0; i < V; i++) z[i & 1] += __builtin_amdgcn_exp2f((f[i] - ref) * s_log2e);
			}
			p.z += z[0] + z[1];
		}
		p.shift(wave_max(p.m), s_log2e);
		p.z = wave_sum(p.z);
		const bool is = tid < K && id < (uint32_t) a.n_cols && v != -__builtin_inff();
		RowPart te = teacher_entry(v, is);
		if (wave * 64 < K) {
			te.shift(wave_max(te.m), s_log2e);
			te.z = wave_sum(te.z);
		}
		if (tid < score_entries(K)) {
			ids[tid] = is ? id : SCORE_NO_COLUMN;
			values[tid] = v;
		}
		if ((tid & 63) == 0) {
			cells.m[wave] = p.m;
			cells.z[wave] = p.z;
			cells.vm[wave] = te.m;
			cells.vz[wave] = te.z;
		}
		__builtin_amdgcn_s_waitcnt(0x0F70);   /* vmcnt(0): all of it is behind the last chunk, which is here */
		lds_barrier();
		if (before >= 0) {
			buf_store_elem<T>(make_rsrc(out_ptr(before), row_bytes), fix_off, fix);
			if (tid == 0) {
				float l = 0.0f;
				for (int i = 0; i * 64 < K; i++) l += both[turn ^ 1].loss[i];
				a.loss[before] = l * temperature * temperature;
			}
		}
		p = score_join_cells(cells.m, cells.z, nullptr, waves, s_log2e);
		const int teacher_waves = K == 0 ? 0 : (K + 63) >> 6;
		te = score_join_cells(cells.vm, cells.vz, nullptr, teacher_waves, s_log2e);
		const RowStats st(p.m, p.z, 0.0f);
		const bool counts = w != 0.0f && !(te.z == 0.0f);
		const float wt = w * temperature;

		/* this thread's entry: its term of the loss, and its column's gradient
		 * if no entry before it has the same column */
		fix_off = SCORE_NOWHERE;
		float l = 0.0f;
		if (wave * 64 < K) {
			if (is && counts) {
				const float d = a.s * (v - te.m);
				const float q = __builtin_amdgcn_exp2f(d * SCORE_LOG2E) / te.z;
				if (!(q == 0.0f)) l = q * ((d - logf(te.z)) - (st.none() ? -__builtin_inff() : st.log_p(xk, a.s)));
				/* columns given twice: counted first, since there hardly are any */
				int same = 0;
#pragma unroll 4
				for (int o = 0; o < score_entries(K) / 4; o++) {
					const uint4 i4 = reinterpret_cast<const uint4 *>(ids)[o];
					same += (i4.x == id) + (i4.y == id) + (i4.z == id) + (i4.w == id);
				}
				bool first = true;
				float sum = q;
				if (same > 1) {
					sum = 0.0f;
#pragma unroll 1
					for (int o = 0; o < K; o++) {
						if (ids[o] != id) continue;
						if (o < tid) first = false;
						sum += __builtin_amdgcn_exp2f(a.s * (values[o] - te.m) * SCORE_LOG2E) / te.z;
					}
				}
				if (first) fix_off = id * E;
				fix = st.none() ? 0.0f : wt * (__builtin_amdgcn_exp2f((xk - st.max) * s_log2e) * st.inv_z - sum);
			}
			l = wave_sum(l);
			if ((tid & 63) == 0) cells.loss[wave] = l;
		}

		/* the gradient, and the next row */
		const bool zero = !counts || st.none();
		const float scale = zero ? 0.0f : wt * st.inv_z, ref = st.max;
		const int next_head = next < a.n_rows ? head_of(next) : 0, next_chunks = (a.n_cols - next_head) / V;
		const __amdgpu_buffer_rsrc_t rs = make_rsrc(row_ptr(next) + next_head, next_w != 0.0f ? (uint32_t) next_chunks * 16u : 0u);
		const __amdgpu_buffer_rsrc_t re = make_rsrc(row_ptr(next), next_w != 0.0f ? row_bytes : 0u);
		T * out = out_ptr(r);
		const __amdgpu_buffer_rsrc_t ro = make_rsrc(out + head, (uint32_t) chunks * 16u);
		const auto grad = [&](float f) { return zero ? 0.0f : scale * __builtin_amdgcn_exp2f((f - ref) * s_log2e); };
#pragma unroll
		for (int j = 0; j < CH; j++) {
			__builtin_amdgcn_sched_barrier(0);
			reg_barrier(x[j]);
			float f[V];
			unpack16<T>(x[j], f);
#pragma unroll
			for (int i = 0; i < V; i++) f[i] = grad(f[i]);
			buf_store16_nt(ro, voff, (uint32_t) (j * nt) * 16u, pack16<T>(f));
		}
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int j = 0; j < CH; j++) x[j] = buf_load16_nt(rs, voff, (uint32_t) (j * nt) * 16u);
		buf_store_elem<T>(make_rsrc(out, row_bytes), single, grad(xs));
		head = next_head;
		chunks = next_chunks;
		single = single_off(head);
		xt = buf_load_elem<T>(re, single);
		xk = buf_load_elem<T>(re, pick_off(next_id));
		before = r;
		r = next;
		w = next_w;
		id = next_id;
		v = next_v;
	}
	__builtin_amdgcn_s_waitcnt(0x0F70);
	lds_barrier();
	if (before >= 0) {
		buf_store_elem<T>(make_rsrc(out_ptr(before), row_bytes), fix_off, fix);
		if (tid == 0) {
			float l = 0.0f;
			for (int i = 0; i * 64 < K; i++) l += both[turn ^ 1].loss[i];
			a.loss[before] = l * temperature * temperature;
		}
	}
}

/* ---------------- slices of rows, read twice ---------------- */

struct Teacher {
	uint32_t id[SCORE_TEACHER_MAX];
	float q[SCORE_TEACHER_MAX], x[SCORE_TEACHER_MAX];
};

/* A row's loss, and in te what its gradient needs, from the row's statistics;
 * picked(k, id): the logit of an entry's column. False where the row has no
 * entry (its loss is 0). */
template <typename Picked>
__device__ __forceinline__ bool distill_teacher(const DistillArgs & a, long r, const RowStats & st, bool write_loss, Teacher & te, float * cells, const Picked & picked) {
	const int K = a.top_k, nt = (int) blockDim.x;
	RowPart sum;
	__syncthreads();
	for (int k = (int) threadIdx.x; k < K; k += nt) {
		const uint32_t id = a.ids[r * K + k];
		const float v = a.values[r * K + k];
		const bool is = id < (uint32_t) a.n_cols && v != -__builtin_inff();
		te.id[k] = is ? id : SCORE_NO_COLUMN;
		te.q[k] = v;
		te.x[k] = is ? picked(k, id) : 0.0f;
		const RowPart one = teacher_entry(v, is);
		const float m = fmaxf(sum.m, one.m);
		sum.shift(m, a.s * SCORE_LOG2E);
		sum.z += is ? one.z * __builtin_amdgcn_exp2f(fmaxf((one.m - m) * a.s * SCORE_LOG2E, SCORE_FAR_BELOW)) : 0.0f;
	}
	sum = score_group_join<false>(sum, a.s * SCORE_LOG2E, cells);
	if (sum.z == 0.0f) {
		if (threadIdx.x == 0 && write_loss) a.loss[r] = 0.0f;
		return false;
	}
	const float log_z = logf(sum.z);
	float l = 0.0f;
	for (int k = (int) threadIdx.x; k < K; k += nt) {
		if (te.id[k] == SCORE_NO_COLUMN) continue;
		const float d = a.s * (te.q[k] - sum.m);
		const float q = __builtin_amdgcn_exp2f(d * SCORE_LOG2E) / sum.z;
		if (!(q == 0.0f)) l = fmaf(q, (d - log_z) - (st.none() ? -__builtin_inff() : st.log_p(te.x[k], a.s)), l);
		te.q[k] = q;
	}
	if (write_loss) {
		l = score_group_sum(l, cells);
		if (threadIdx.x == 0) a.loss[r] = l / (a.s * a.s);
	}
	else __syncthreads();
	return true;
}

/* statistics of the slices; where that is all there is to a row (one slice,
 * no gradient) its loss too */
template <typename T>
__device__ __forceinline__ void distill_parts(const DistillArgs & a) {
	__shared__ float cells[3 * SCORE_MAX_WAVES];
	__shared__ Teacher te;
	const Score_Plan plan = score_stream_plan(a.n_rows, a.n_cols, (int) sizeof(T), 0);
	const float s_log2e = a.s * SCORE_LOG2E;
	for (long u = blockIdx.x; u < (long) a.n_rows * plan.slices; u += gridDim.x) {
		const long r = plan.slices == 1 ? u : u / plan.slices;
		const int slice = plan.slices == 1 ? 0 : (int) (u - r * plan.slices);
		const T * row = static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride;
		const bool alone = plan.slices == 1 && !a.dlogits;
		if ((a.weights ? a.weights[r] : 1.0f) == 0.0f) {
			if (alone && threadIdx.x == 0) a.loss[r] = 0.0f;
			continue;
		}
		const RowSlice sl(a.n_cols, VecOf<T>::N, score_head(row, a.n_cols), slice, plan.slices, plan.slice_chunks);
		const RowPart p = score_group_join<false>(a.dlogits ? score_stream<T, false, true>(row, sl, s_log2e, nullptr)
																  : score_stream<T, false, false>(row, sl, s_log2e, nullptr), s_log2e, cells);
		if (alone) {
			distill_teacher(a, r, RowStats(p.m, p.z, 0.0f), true, te, cells, [&](int, uint32_t id) { return to_f(row[id]); });
			continue;
		}
		if (threadIdx.x == 0) a.parts[u] = Score_Part{p.m, p.z, 0.0f, 0.0f};
		/* the gradient may be written over them */
		if (slice == 0)
			for (int k = (int) threadIdx.x; k < a.top_k; k += (int) blockDim.x) {
				const uint32_t id = a.ids[r * a.top_k + k];
				a.picked[r * a.top_k + k] = id < (uint32_t) a.n_cols ? to_f(row[id]) : 0.0f;
			}
		__syncthreads();
	}
}

/* losses and gradients from the slices' statistics */
template <typename T>
__device__ __forceinline__ void distill_out(const DistillArgs & a) {
	__shared__ float cells[3 * SCORE_MAX_WAVES];
	__shared__ Teacher te;
	const Score_Plan plan = score_stream_plan(a.n_rows, a.n_cols, (int) sizeof(T), 0);
	const float s_log2e = a.s * SCORE_LOG2E, temperature = 1.0f / a.s;
	for (long u = blockIdx.x; u < (long) a.n_rows * plan.slices; u += gridDim.x) {
		const long r = plan.slices == 1 ? u : u / plan.slices;
		const int slice = plan.slices == 1 ? 0 : (int) (u - r * plan.slices);
		const T * row = static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride;
		T * out = a.dlogits ? static_cast<T *>(a.dlogits) + (uint64_t) r * a.grad_stride : nullptr;
		if (!out && slice > 0) continue;
		const RowSlice sl(a.n_cols, VecOf<T>::N, out ? score_head(out, a.n_cols) : 0, slice, plan.slices, plan.slice_chunks);
		const float w = a.weights ? a.weights[r] : 1.0f;
		if (w == 0.0f) {
			if (slice == 0 && threadIdx.x == 0) a.loss[r] = 0.0f;
			if (out) score_clear(out, sl);
			continue;
		}
		RowPart p;
		const Score_Part * parts = a.parts + r * plan.slices;
		for (int i = 0; i < plan.slices; i++) p.m = fmaxf(p.m, parts[i].max);
		for (int i = 0; i < plan.slices; i++) {
			RowPart q;
			q.m = parts[i].max;
			q.z = parts[i].z;
			q.shift(p.m, s_log2e);
			p.z += q.z;
		}
		const RowStats st(p.m, p.z, 0.0f);
		const bool counts = distill_teacher(a, r, st, slice == 0, te, cells, [&](int k, uint32_t) { return a.picked[r * a.top_k + k]; });
		if (!out) continue;
		if (!counts || st.none()) {
			score_clear(out, sl);
			continue;
		}
		const float wt = w * temperature, scale = wt * st.inv_z, ref = st.max;
		score_map(row, out, sl, [&](float f) { return scale * __builtin_amdgcn_exp2f((f - ref) * s_log2e); });
		score_stores_done();
		for (int k = (int) threadIdx.x; k < a.top_k; k += (int) blockDim.x) {
			const uint32_t id = te.id[k];
			if (id == SCORE_NO_COLUMN || !sl.holds(id, VecOf<T>::N)) continue;
			float q = 0.0f;
			bool first = true;
			for (int o = 0; o < a.top_k; o++)
				if (te.id[o] == id) {
					first = first && o >= k;
					q += te.q[o];
				}
			if (first) out[id] = from_f<T>(wt * (__builtin_amdgcn_exp2f((te.x[k] - ref) * s_log2e) * st.inv_z - q));
		}
	}
}

/* mean_loss = sum_r w_r loss_r / n_rows in 64 bits, in a fixed order */
__device__ __forceinline__ void distillation_loss_mean(int n_rows, const float * row_weights, const float * loss, float * mean_loss) {
	__shared__ double part[SCORE_MAX_WAVES];
	double sum = 0.0;
#pragma unroll 4
	for (long r = threadIdx.x; r < n_rows; r += SCORE_MEAN_THREADS) {
		const float w = row_weights ? row_weights[r] : 1.0f, l = loss[r];
		sum += w != 0.0f ? (double) w * (double) l : 0.0;
	}
	for (int step = 32; step > 0; step >>= 1) sum += __shfl_xor(sum, step);
	if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
	__syncthreads();
	if (threadIdx.x == 0) {
		sum = 0.0;
		for (int i = 0; i < SCORE_MEAN_THREADS / 64; i++) sum += part[i];
		*mean_loss = (float) (sum / (double) n_rows);
	}
}

#define DISTILLATION_ARGS(T)                                                                                                     \
	int n_rows, int n_cols, uint64_t row_stride, uint64_t grad_stride, float scale, int top_k, T * logits,                       \
		uint32_t * teacher_ids, float * teacher_logits, float * row_weights, float * loss, float * mean_loss, T * dlogits,       \
		uint64_t workspace_bytes, void * workspace
#define DISTILLATION_PACK                                                                                                        \
	DistillArgs a = {n_rows, n_cols, row_stride, grad_stride, scale, top_k, logits, teacher_ids, teacher_logits, row_weights,    \
					 loss, dlogits, static_cast<Score_Part *>(workspace), nullptr};                                              \
	a.picked = reinterpret_cast<float *>(a.parts + (uint64_t) n_rows * score_stream_plan(n_rows, n_cols, (int) sizeof(*logits), 0).slices);
#define DISTILLATION_LOSS_KERNEL(SUF, T)                                                                                         \
	extern "C" __global__ void __launch_bounds__(1024) distillation_loss_##SUF##_kernel_any_rows(DISTILLATION_ARGS(T)) { \
		DISTILLATION_PACK \
		distill_held<T, SCORE_HELD_MOST, 1024>(a); \
	} \
	extern "C" __global__ void __launch_bounds__(1024) distillation_loss_##SUF##_kernel_long_rows(DISTILLATION_ARGS(T)) { \
		DISTILLATION_PACK \
		distill_held<T, SCORE_HELD_MORE, 1024>(a); \
	} \
	extern "C" __global__ void __launch_bounds__(512, 4) distillation_loss_##SUF##_kernel_wide_rows(DISTILLATION_ARGS(T)) { \
		DISTILLATION_PACK \
		distill_held<T, SCORE_HELD_MORE, 0>(a); \
	} \
	extern "C" __global__ void __launch_bounds__(1024, 8) distillation_loss_##SUF##_kernel_rows(DISTILLATION_ARGS(T)) { \
		DISTILLATION_PACK \
		distill_held<T, SCORE_HELD, 0>(a); \
	} \
	extern "C" __global__ void __launch_bounds__(64 * SCORE_MAX_WAVES, 8) distillation_loss_##SUF##_kernel(DISTILLATION_ARGS(T)) { \
		DISTILLATION_PACK                                                                                                        \
		distill_parts<T>(a);                                                                                                     \
	}                                                                                                                            \
	extern "C" __global__ void __launch_bounds__(64 * SCORE_MAX_WAVES, 8) distillation_loss_##SUF##_kernel_split_out(DISTILLATION_ARGS(T)) { \
		DISTILLATION_PACK                                                                                                        \
		distill_out<T>(a);                                                                                                       \
	}                                                                                                                            \
	extern "C" __global__ void __launch_bounds__(SCORE_MEAN_THREADS) distillation_loss_##SUF##_kernel_finish(DISTILLATION_ARGS(T)) {  \
		distillation_loss_mean(n_rows, row_weights, loss, mean_loss);                                                            \
	}

DISTILLATION_LOSS_KERNEL(fp32, float)
DISTILLATION_LOSS_KERNEL(fp16, f16_t)
DISTILLATION_LOSS_KERNEL(bf16, bf16_t)
