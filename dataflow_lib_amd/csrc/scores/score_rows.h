/*
 * What the scoring kernels share: a row's statistics in one pass over its
 * logits, and its k largest logits.
 *
 * A row is shifted by its largest logit M before anything is exponentiated:
 *   Z = sum exp(s (x - M)),  E = sum s (x - M) exp(s (x - M))
 *   lse = s M + log Z,  log p_j = s (x_j - M) - log Z,  entropy = log Z - E / Z
 * The difference x - M is formed first: it is exact next to the maximum, and
 * it cannot overflow where s x can (rows of the type's lowest value). In one
 * pass every thread shifts by the largest logit that it has met so far and
 * moves its sums when that grows, from a to b:
 *   Z <- f Z,  E <- f (E + s (a - b) Z),  f = exp(s (a - b))
 * where all terms of E have one sign, so nothing cancels; threads, waves and
 * slices are joined in the same way, in a fixed order: results do not change
 * from call to call. Exponents are in units of log 2 (t = s log2(e) (x - M)),
 * and so is E until the end. All of it is fp32; logits are widened exactly, and
 * only gradients are rounded to their type, once.
 */
#pragma once

#include "dtypes.h"
#include "reduce.h"
#include "score_geometry.h"

#define SCORE_LOG2E 1.4426950408889634f
#define SCORE_LN2 0.6931471805599453f
#define SCORE_MAX_WAVES 16
/* exp2 of it is 0; finite, so that it times 0 is 0 */
#define SCORE_FAR_BELOW -1e4f

/* what a row's log-probabilities are formed from */
struct RowStats {
	float max;      /* M */
	float log_z;    /* log Z; +inf for a row of -inf alone, NaN with NaN or +inf */
	float inv_z;    /* 1 / Z; 0 for a row of -inf alone */
	float e_z;      /* E / Z */
	__device__ __forceinline__ RowStats() {}
	/* e in units of log 2 */
	__device__ __forceinline__ RowStats(float m, float z, float e) {
		const bool none = z == 0.0f;
		max = none ? 0.0f : m;
		log_z = none ? __builtin_inff() : logf(z);
		inv_z = none ? 0.0f : 1.0f / z;
		e_z = none ? 0.0f : e / z * SCORE_LN2;
	}
	__device__ __forceinline__ bool none() const { return inv_z == 0.0f; }
	__device__ __forceinline__ float lse(float s) const { return none() ? -__builtin_inff() : fmaf(s, max, log_z); }
	__device__ __forceinline__ float entropy() const { return none() ? 0.0f : log_z - e_z; }
	__device__ __forceinline__ float log_p(float x, float s) const { return s * (x - max) - log_z; }
};

/* maximum and sums of a part of a row */
struct RowPart {
	float m, z, e;
	__device__ __forceinline__ RowPart() { m = -__builtin_inff(); z = 0.0f; e = 0.0f; }
	/* shifted by a larger maximum. Maxima that differ by infinity or are both
	 * -inf (NaN) give the far-below shift, whose sums are 0. */
	__device__ __forceinline__ void shift(float to, float s_log2e) {
		const float t = fmaxf((m - to) * s_log2e, SCORE_FAR_BELOW);
		const float f = __builtin_amdgcn_exp2f(t);
		e = f * fmaf(t, z, e);
		z = f * z;
		m = to;
	}
};

/* What a workgroup's waves have left in one cell each, joined by the lanes of
 * every wave alike: lane i takes cell i (of SCORE_MAX_WAVES, as many as a row
 * of lanes for the DPP steps), one LDS access for all of them. */
template <typename Op>
__device__ __forceinline__ float score_row16(float v, const Op & op) {
	v = op(v, dpp_f32<DPP_QUAD_1032>(v));
	v = op(v, dpp_f32<DPP_QUAD_2301>(v));
	v = op(v, dpp_f32<DPP_ROW_HALF_MIRROR>(v));
	return op(v, dpp_f32<DPP_ROW_MIRROR>(v));
}
struct ScoreMax { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct ScoreSum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
template <typename Op>
__device__ __forceinline__ float score_cells(const float * cells, float none, const Op & op) {
	const int i = (int) threadIdx.x & (SCORE_MAX_WAVES - 1);
	return readlane_f32(score_row16(i < (int) (blockDim.x >> 6) ? cells[i] : none, op), 0);
}
/* maximum or sum over a workgroup; `cells`: SCORE_MAX_WAVES floats of LDS */
__device__ __forceinline__ float score_group_max(float v, float * cells) {
	v = wave_max(v);
	if (blockDim.x == 64) return v;
	__syncthreads();
	if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = v;
	__syncthreads();
	return score_cells(cells, -__builtin_inff(), ScoreMax());
}
__device__ __forceinline__ float score_group_sum(float v, float * cells) {
	v = wave_sum(v);
	if (blockDim.x == 64) return v;
	__syncthreads();
	if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = v;
	__syncthreads();
	return score_cells(cells, 0.0f, ScoreSum());
}
/* parts of a row, one per wave: maxima, and sums shifted by them */
__device__ __forceinline__ RowPart score_join_cells(const float * m, const float * z, const float * e, int waves, float s_log2e) {
	const int i = (int) threadIdx.x & (SCORE_MAX_WAVES - 1);
	RowPart p;
	if (i < waves) {
		p.m = m[i];
		p.z = z[i];
		if (e) p.e = e[i];
	}
	p.shift(score_row16(p.m, ScoreMax()), s_log2e);
	p.z = readlane_f32(score_row16(p.z, ScoreSum()), 0);
	if (e) p.e = readlane_f32(score_row16(p.e, ScoreSum()), 0);
	p.m = readlane_f32(p.m, 0);
	return p;
}
/* the parts of a workgroup's threads, joined (every thread gets the result);
 * `cells`: 5 SCORE_MAX_WAVES floats of LDS. With TOP also the threads that have
 * met a column above -inf: how many, and the least of their maxima. */
template <bool TOP>
__device__ __forceinline__ RowPart score_group_join(RowPart p, float s_log2e, float * cells, float * met = nullptr, float * least = nullptr) {
	const int wave = (int) (threadIdx.x >> 6), waves = (int) (blockDim.x >> 6);
	float n = 0.0f, l = 0.0f;
	if (TOP) {
		const bool has = p.m > -__builtin_inff();
		n = (float) __popcll(__ballot(has));
		l = wave_max(has ? -p.m : -__builtin_inff());
	}
	p.shift(wave_max(p.m), s_log2e);
	p.z = wave_sum(p.z);
	p.e = wave_sum(p.e);
	if (waves > 1) {
		__syncthreads();
		if ((threadIdx.x & 63) == 0) {
			cells[wave] = p.m;
			cells[SCORE_MAX_WAVES + wave] = p.z;
			cells[2 * SCORE_MAX_WAVES + wave] = p.e;
			if (TOP) {
				cells[3 * SCORE_MAX_WAVES + wave] = n;
				cells[4 * SCORE_MAX_WAVES + wave] = l;
			}
		}
		__syncthreads();
		p = score_join_cells(cells, cells + SCORE_MAX_WAVES, cells + 2 * SCORE_MAX_WAVES, waves, s_log2e);
		if (TOP) {
			n = score_cells(cells + 3 * SCORE_MAX_WAVES, 0.0f, ScoreSum());
			l = score_cells(cells + 4 * SCORE_MAX_WAVES, -__builtin_inff(), ScoreMax());
		}
	}
	if (TOP) {
		*met = n;
		*least = -l;
	}
	return p;
}

/* 16 bytes of a row, which need no more alignment than its elements (of two
 * bytes at least) */
typedef uint32_t score_vec __attribute__((ext_vector_type(4), aligned(2)));
template <typename T, bool AGAIN = false>
__device__ __forceinline__ R16 score_load(const T * row, uint64_t uniform_chunk, uint32_t lane_chunk) {
	const score_vec * p = reinterpret_cast<const score_vec *>(reinterpret_cast<const char *>(row) + uniform_chunk * 16u + lane_chunk * 16u);
	/* read once: with the streaming hint */
	const score_vec v = AGAIN ? *p : __builtin_nontemporal_load(p);
	R16 r;
	r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
	return r;
}

/* A row's chunks begin where memory has a multiple of SCORE_ALIGN bytes, so
 * that a wave's accesses share no more lines with others than they have to
 * (rows of odd lengths begin anywhere: distillation_loss 4096 x 50257 bf16 174
 * us, with chunks from the rows' first elements on 198; token_logprobs 4096 x
 * 128257 167 and 216). The elements before them, the head, and those behind the
 * last whole chunk, the tail, are a thread's each (SCORE_ALIGN / 2 + 6 at
 * most, less than a wave). */
#define SCORE_ALIGN 64
template <typename T>
__device__ __forceinline__ int score_head(const T * row, int n_cols) {
	const int head = (int) ((-(uintptr_t) row & (SCORE_ALIGN - 1)) / sizeof(T));
	return head < n_cols ? head : n_cols;
}

/* the elements of a row that a workgroup works on: of the chunks behind the
 * head, [first, last), and with the first slice the head, with the last one
 * the tail */
struct RowSlice {
	int head, first, last, tail, end;   /* tail: where it begins; the row's end in other slices */
	bool with_head;
	__device__ __forceinline__ RowSlice(int n_cols, int vec, int row_head, int slice, int slices, int slice_chunks) {
		const int chunks = (n_cols - row_head) / vec;
		head = row_head;
		with_head = slice == 0;
		/* the plan counts a row's chunks without its head */
		first = slice * slice_chunks < chunks ? slice * slice_chunks : chunks;
		last = slice + 1 == slices || first + slice_chunks > chunks ? chunks : first + slice_chunks;
		tail = slice + 1 == slices ? head + chunks * vec : n_cols;
		end = n_cols;
	}
	/* the columns of the slice are [begin, behind) */
	__device__ __forceinline__ int begin(int vec) const { return with_head ? 0 : head + first * vec; }
	__device__ __forceinline__ int behind(int vec) const { return tail < end ? end : head + last * vec; }
	__device__ __forceinline__ bool holds(uint32_t column, int vec) const { return column >= (uint32_t) begin(vec) && column < (uint32_t) behind(vec); }
	/* this thread's element of the head or the tail, or -1 */
	__device__ __forceinline__ int single() const {
		int t = (int) threadIdx.x;
		if (with_head) {
			if (t < head) return t;
			t -= head;
		}
		return t < end - tail ? tail + t : -1;
	}
};

/* N chunks (c + tid, a workgroup's threads apart) into a thread's part: their
 * maximum, the part's shift to it, then their terms. -inf makes E's term NaN
 * (-inf * 0): a wave that finds NaN in its sum forms the terms again, with
 * exponents that are far below 0 but finite. Returns the chunks' maximum. */
template <typename T, int N, bool ENTROPY, bool AGAIN>
__device__ __forceinline__ float score_chunks(const T * row, int c, float s_log2e, RowPart & p) {
	constexpr int V = VecOf<T>::N;
	R16 x[N];
#pragma unroll
	for (int u = 0; u < N; u++) x[u] = score_load<T, AGAIN>(row, (uint64_t) (c + u * (int) blockDim.x), threadIdx.x);
	float m = -__builtin_inff();
#pragma unroll
	for (int u = 0; u < N; u++) {
		float f[V];
		unpack16<T>(x[u], f);
#pragma unroll
		for (int i = 0; i < V; i++) m = fmaxf(m, f[i]);
	}
	p.shift(fmaxf(p.m, m), s_log2e);
	/* a thread that has met -inf alone keeps its differences from being NaN */
	const float ref = p.m == -__builtin_inff() ? 0.0f : p.m;
	float z[2] = {0.0f, 0.0f}, e[2] = {0.0f, 0.0f};
#pragma unroll
	for (int u = 0; u < N; u++) {
		/* a chunk at a time: left to itself the compiler keeps all chunks' terms
		 * at once, at twice the registers */
		__builtin_amdgcn_sched_barrier(0);
		reg_barrier(x[u]);
		float f[V];
		unpack16<T>(x[u], f);
#pragma unroll
		for (int i = 0; i < V; i++) {
			const float t = (f[i] - ref) * s_log2e;
			const float q = __builtin_amdgcn_exp2f(t);
			z[i & 1] += q;
			if (ENTROPY) e[i & 1] = fmaf(t, q, e[i & 1]);
		}
	}
	float eb = e[0] + e[1], zb = z[0] + z[1];
	/* or the sum of z is moved behind the branch, and all its terms are kept */
	__asm__ volatile("" : "+v"(zb));
	if (ENTROPY && __builtin_expect(__any(eb != eb), 0)) {
		eb = 0.0f;
#pragma unroll
		for (int u = 0; u < N; u++) {
			__builtin_amdgcn_sched_barrier(0);
			reg_barrier(x[u]);
			float f[V];
			unpack16<T>(x[u], f);
#pragma unroll
			for (int i = 0; i < V; i++) {
				const float t = fmaxf((f[i] - ref) * s_log2e, SCORE_FAR_BELOW);
				eb = fmaf(t, __builtin_amdgcn_exp2f(t), eb);
			}
		}
	}
	p.z += zb;
	p.e += eb;
	return m;
}

/* A thread's part of a slice: batches of SCORE_BATCH chunks, and what is left
 * in batches of 2 and 1, so that only the last chunk has to ask whether it is
 * there. The maximum of the thread's b-th batch (what is left being one) goes
 * to groups[(b % SCORE_GROUP_SLOTS) * blockDim.x + tid] (LDS; null: not
 * wanted); the thread's element of the head or the tail counts to batch 0.
 * AGAIN: the logits, or some of them, are read again soon, and come without the
 * streaming hint (token_logprobs 1021 x 50257 bf16 with 64 alternatives 33.2 us,
 * with the hint 41.3; distillation_loss of 300 x 128256 fp32, in two launches,
 * 89 and 110). */
template <typename T, bool ENTROPY, bool AGAIN>
__device__ __forceinline__ RowPart score_stream(const T * row, const RowSlice & sl, float s_log2e, float * groups) {
	const int nt = (int) blockDim.x, tid = (int) threadIdx.x;
	RowPart p;
	float before = -__builtin_inff();
	const int single = sl.single();
	if (single >= 0) {
		const float x = to_f(row[single]);
		p.m = before = fmaxf(x, -__builtin_inff());   /* NaN: -inf */
		p.z = __builtin_amdgcn_exp2f((x - (p.m == -__builtin_inff() ? 0.0f : p.m)) * s_log2e);
	}
	row += sl.head;
	int slot = 0;
	bool again = false;
	for (int c = sl.first;;) {
		float m;
		const bool whole = c + SCORE_BATCH * nt <= sl.last;
		if (whole) {
			m = score_chunks<T, SCORE_BATCH, ENTROPY, AGAIN>(row, c, s_log2e, p);
			c += SCORE_BATCH * nt;
		}
		else {
			m = -__builtin_inff();
			if (c + 2 * nt <= sl.last) { m = fmaxf(m, score_chunks<T, 2, ENTROPY, AGAIN>(row, c, s_log2e, p)); c += 2 * nt; }
			if (c + nt <= sl.last) { m = fmaxf(m, score_chunks<T, 1, ENTROPY, AGAIN>(row, c, s_log2e, p)); c += nt; }
			if (c + tid < sl.last) m = fmaxf(m, score_chunks<T, 1, ENTROPY, AGAIN>(row, c, s_log2e, p));
		}
		if (groups) {
			float * g = groups + slot * nt + tid;
			*g = fmaxf(m, again ? *g : before);
			before = -__builtin_inff();
		}
		if (!whole || c >= sl.last) break;
		if (++slot == SCORE_GROUP_SLOTS) { slot = 0; again = true; }
	}
	return p;
}

__device__ __forceinline__ void score_store(void * row, uint64_t uniform_chunk, uint32_t lane_chunk, const R16 & r) {
	const score_vec v = {r.w[0], r.w[1], r.w[2], r.w[3]};
	char * p = static_cast<char *>(row) + uniform_chunk * 16u;
	__builtin_nontemporal_store(v, reinterpret_cast<score_vec *>(p + lane_chunk * 16u));
}

/* N chunks of out = f(row) */
template <typename T, int N, typename F>
__device__ __forceinline__ void score_map_chunks(const T * row, T * out, int c, const F & f) {
	constexpr int V = VecOf<T>::N;
	R16 x[N];
#pragma unroll
	for (int u = 0; u < N; u++) x[u] = score_load(row, (uint64_t) (c + u * (int) blockDim.x), threadIdx.x);
#pragma unroll
	for (int u = 0; u < N; u++) {
		__builtin_amdgcn_sched_barrier(0);
		float v[V];
		unpack16<T>(x[u], v);
#pragma unroll
		for (int i = 0; i < V; i++) v[i] = f(v[i]);
		score_store(out, (uint64_t) (c + u * (int) blockDim.x), threadIdx.x, pack16<T>(v));
	}
}
/* out = f(row) over a slice; out may be row */
template <typename T, typename F>
__device__ __forceinline__ void score_map(const T * row, T * out, const RowSlice & sl, const F & f) {
	const int nt = (int) blockDim.x, tid = (int) threadIdx.x;
	const int single = sl.single();
	if (single >= 0) out[single] = from_f<T>(f(to_f(row[single])));
	row += sl.head;
	out += sl.head;
	int c = sl.first;
	for (; c + SCORE_BATCH * nt <= sl.last; c += SCORE_BATCH * nt) score_map_chunks<T, SCORE_BATCH>(row, out, c, f);
	if (c + 2 * nt <= sl.last) { score_map_chunks<T, 2>(row, out, c, f); c += 2 * nt; }
	if (c + nt <= sl.last) { score_map_chunks<T, 1>(row, out, c, f); c += nt; }
	if (c + tid < sl.last) score_map_chunks<T, 1>(row, out, c, f);
}
/* out = 0 over a slice */
template <typename T>
__device__ __forceinline__ void score_clear(T * out, const RowSlice & sl) {
	R16 zero;
	zero.w[0] = zero.w[1] = zero.w[2] = zero.w[3] = 0u;
	for (int c = sl.first + (int) threadIdx.x; c < sl.last; c += (int) blockDim.x) score_store(out + sl.head, (uint64_t) c, 0u, zero);
	const int single = sl.single();
	if (single >= 0) out[single] = from_f<T>(0.0f);
}
/* every store that this workgroup has made so far is done before any that it
 * makes after this */
__device__ __forceinline__ void score_stores_done() {
	__builtin_amdgcn_s_waitcnt(0x0F70);   /* vmcnt(0) */
	__syncthreads();
}

/* Whole numbers that lie as floats do: -0 with +0, NaN below -inf. */
__device__ __forceinline__ uint32_t score_key(float x) {
	const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
	if (x != x) return 0u;
	return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float score_key_value(uint32_t key) {
	if (key == 0u) return __builtin_nanf("");
	return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}
/* An alternative as one number: larger logits are larger numbers, and of equal
 * ones the lower column's; 0 is none. */
__device__ __forceinline__ uint64_t score_alternative(uint32_t key, uint32_t id) { return ((uint64_t) key << 32) | (0xffffffffu - id); }
__device__ __forceinline__ uint32_t score_alternative_id(uint64_t a) { return 0xffffffffu - (uint32_t) a; }
__device__ __forceinline__ float score_alternative_value(uint64_t a) { return score_key_value((uint32_t) (a >> 32)); }
