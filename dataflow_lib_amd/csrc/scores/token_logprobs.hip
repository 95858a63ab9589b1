/*
 * token_logprobs: log-probabilities of given tokens, entropy, log-sum-exp and
 * the k likeliest columns of each row of logits (formulas and odd cases in
 * dataflow_score_ops.h).
 *
 * A workgroup streams a row, or a slice of it where rows are few, once
 * (score_stream). What it remembers for the alternatives is the maximum of
 * each batch of each thread ("groups" of 64 16-bit or 32 fp32 logits). Any
 * bound that k groups' maxima reach is at most the k-th largest logit, so the
 * logits that reach it hold the k largest: a bisection over the maxima finds
 * such a bound that not many more than k reach, and only the groups that
 * reach it are read again. Their logits that do, the candidates, are ranked by
 * counting. Where candidates are too many (ties, above all), the k largest are
 * found digit by digit (score_select).
 */
#include "score_rows.h"

struct TopState {
	float cells[3 * SCORE_MAX_WAVES];
	uint32_t counts[2 * SCORE_MAX_WAVES];
	uint32_t hist[256];
	uint32_t prefix, need, count;
};

/* a count over a workgroup of a wave's count; calls alternate between two
 * sets of cells, so one barrier each is enough */
__device__ __forceinline__ uint32_t score_group_count(uint32_t n, TopState & t, int & turn) {
	const int waves = (int) (blockDim.x >> 6);
	if (waves == 1) return n;
	uint32_t * cells = t.counts + (turn ^= SCORE_MAX_WAVES);
	if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = n;
	__syncthreads();
	n = 0;
	for (int w = 0; w < waves; w++) n += cells[w];
	return n;
}

/* Of the columns [first, end) those whose key is `key`, by rising column, the
 * first `most` of them, into list[0..); returns how many there were. */
template <typename T>
__device__ __forceinline__ uint32_t score_equal(const T * row, int first, int end, uint32_t key, uint32_t most, uint64_t * list, TopState & t) {
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x, lane = tid & 63, wave = tid >> 6, waves = nt >> 6;
	uint32_t have = 0;
	for (long base = first; base < end && have < most; base += nt) {
		const long j = base + tid;
		const bool is = j < end && score_key(to_f(row[j < end ? j : first])) == key;
		const unsigned long long ballot = __ballot(is);
		__syncthreads();
		if (lane == 0) t.counts[wave] = (uint32_t) __popcll(ballot);
		__syncthreads();
		uint32_t before = have + (uint32_t) __popcll(ballot & ((1ull << lane) - 1ull));
		for (int w = 0; w < waves; w++) {
			if (w < wave) before += t.counts[w];
			have += t.counts[w];
		}
		if (is && before < most) list[before] = score_alternative(key, (uint32_t) j);
	}
	return have < most ? have : most;
}

/* The k largest of the columns [first, end) (at least k) into list[0..k), in
 * any order: the k-th largest key digit by digit (8 bits of it a pass over the
 * columns, counted in LDS), then the larger ones, and of the equal ones as
 * many, by rising column, as are left. */
template <typename T>
__device__ __forceinline__ void score_select(const T * row, int first, int end, int k, uint64_t * list, TopState & t) {
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x;
	__syncthreads();
	if (tid == 0) { t.prefix = 0u; t.need = (uint32_t) k; t.count = 0u; }
	for (int shift = 24; shift >= 0; shift -= 8) {
		for (int b = tid; b < 256; b += nt) t.hist[b] = 0u;
		__syncthreads();
		const uint32_t prefix = t.prefix;
		const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
		for (long j = first + tid; j < end; j += nt) {
			const uint32_t key = score_key(to_f(row[j]));
			if ((key & above) == prefix) atomicAdd(&t.hist[(key >> shift) & 255u], 1u);
		}
		__syncthreads();
		if (tid == 0) {
			uint32_t need = t.need;
			int b = 255;
			while (b > 0 && t.hist[b] < need) need -= t.hist[b--];
			t.prefix = prefix | ((uint32_t) b << shift);
			t.need = need;
		}
		__syncthreads();
	}
	const uint32_t last = t.prefix, equal = t.need;
	for (long j = first + tid; j < end; j += nt) {
		const uint32_t key = score_key(to_f(row[j]));
		if (key > last) list[atomicAdd(&t.count, 1u)] = score_alternative(key, (uint32_t) j);
	}
	score_equal(row, first, end, last, equal, list + (k - (int) equal), t);
	__syncthreads();
}

/* Candidates of a slice into list[0..n): the k largest of its columns among
 * them (all of them where there are fewer than k). `groups`: the maxima that
 * the thread's batches left, SCORE_GROUP_SLOTS rows of blockDim.x. Returns n. */
template <typename T>
__device__ __forceinline__ int score_candidates(const T * row, const RowSlice & sl, int k, float row_max, const float * groups, uint64_t * list, TopState & t) {
	constexpr int V = VecOf<T>::N;
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x;
	const int batches = (sl.last - sl.first + SCORE_BATCH * nt - 1) / (SCORE_BATCH * nt);
	const int col0 = sl.first * V, col1 = sl.last * V + (sl.end - sl.tail);
	const bool tail = sl.tail + tid < sl.end;
	if (sl.columns(V) <= SCORE_CANDIDATES) {
		__syncthreads();
		for (int c = sl.first + tid; c < sl.last; c += nt) {
			R16 x = score_load(row, (uint64_t) c, 0u);
			float f[V];
			unpack16<T>(x, f);
#pragma unroll
			for (int i = 0; i < V; i++) list[(c - sl.first) * V + i] = score_alternative(score_key(f[i]), (uint32_t) (c * V + i));
		}
		if (tail) list[(sl.last - sl.first) * V + tid] = score_alternative(score_key(to_f(row[sl.tail + tid])), (uint32_t) (sl.tail + tid));
		__syncthreads();
		return (int) sl.columns(V);
	}
	float g[SCORE_GROUP_SLOTS];
	float mine = -__builtin_inff();
#pragma unroll
	for (int i = 0; i < SCORE_GROUP_SLOTS; i++) {
		g[i] = i < batches || i == 0 ? groups[i * nt + tid] : -__builtin_inff();
		mine = fmaxf(mine, g[i]);
	}
	int turn = 0;
	__syncthreads();
	if (tid == 0) t.count = 0u;
	/* as many threads as have a column above -inf reach the least of their maxima */
	const bool has = mine > -__builtin_inff();
	float lo = -score_group_max(has ? -mine : -__builtin_inff(), t.cells);
	float hi = row_max;
	if (score_group_count((uint32_t) __popcll(__ballot(has)), t, turn) >= (uint32_t) k) {
		/* lo is reached by k groups or more, hi not known to be */
		for (int step = 0; step < 24; step++) {
			const float mid = 0.5f * lo + 0.5f * hi;
			if (!(mid > lo)) break;
			uint32_t n = 0;
#pragma unroll
			for (int i = 0; i < SCORE_GROUP_SLOTS; i++) n += (uint32_t) __popcll(__ballot(g[i] >= mid));
			n = score_group_count(n, t, turn);
			if (n < (uint32_t) k) hi = mid;
			else {
				lo = mid;
				if (n <= (uint32_t) (k + (k >> 1) + 8)) break;
			}
		}
	}
	else lo = -3.402823466e38f;   /* few columns are above -inf: all of them */
#pragma unroll 1
	for (int i = 0; i < SCORE_GROUP_SLOTS; i++) {
		if (!((i < batches || i == 0 ? groups[i * nt + tid] : -__builtin_inff()) >= lo)) continue;
#pragma unroll 1
		for (int b = i; b < batches; b += SCORE_GROUP_SLOTS)
#pragma unroll 1
			for (int u = 0; u < SCORE_BATCH; u++) {
				const int c = sl.first + (b * SCORE_BATCH + u) * nt + tid;
				if (c >= sl.last) break;
				const R16 x = score_load(row, (uint64_t) c, 0u);
				float f[V];
				unpack16<T>(x, f);
#pragma unroll
				for (int v = 0; v < V; v++)
					if (f[v] >= lo) {
						const uint32_t at = atomicAdd(&t.count, 1u);
						if (at < SCORE_CANDIDATES) list[at] = score_alternative(score_key(f[v]), (uint32_t) (c * V + v));
					}
			}
		if (i == 0 && tail && to_f(row[sl.tail + tid]) >= lo) {
			const uint32_t at = atomicAdd(&t.count, 1u);
			if (at < SCORE_CANDIDATES) list[at] = score_alternative(score_key(to_f(row[sl.tail + tid])), (uint32_t) (sl.tail + tid));
		}
	}
	__syncthreads();
	const int n = (int) t.count;
	__syncthreads();
	if (n > SCORE_CANDIDATES) {
		score_select(row, col0, col1, k, list, t);
		return k;
	}
	if (n < k) {
		/* then columns of -inf, and then those of NaN */
		uint32_t have = (uint32_t) n;
		have += score_equal(row, col0, col1, score_key(-__builtin_inff()), (uint32_t) k - have, list + have, t);
		if (have < (uint32_t) k) score_equal(row, col0, col1, 0u, (uint32_t) k - have, list + have, t);
		__syncthreads();
		return k;
	}
	return n;
}

/* how many of a list's n numbers exceed one of them */
__device__ __forceinline__ int score_rank(const uint64_t * list, int n, uint64_t a) {
	int r = 0;
	for (int o = 0; o < n; o++) r += list[o] > a ? 1 : 0;
	return r;
}

struct LogprobsArgs {
	int n_rows, n_cols;
	uint64_t row_stride;
	float s;
	int tokens_per_row, top_k;
	const void * logits;
	const uint32_t * tokens;
	float * logprobs, * entropy, * lse;
	uint32_t * top_ids;
	float * top_logprobs;
	Score_Part * parts;     /* of a row's slices, row after row */
	uint64_t * lists;       /* their alternatives, largest first */
};

/* the outputs of a row whose statistics are known, but for the alternatives */
template <typename T>
__device__ __forceinline__ void token_logprobs_row(const LogprobsArgs & a, long r, const T * row, const RowStats & st) {
	if (threadIdx.x == 0) {
		if (a.entropy) a.entropy[r] = st.entropy();
		if (a.lse) a.lse[r] = st.lse(a.s);
	}
	for (int m = (int) threadIdx.x; m < a.tokens_per_row; m += (int) blockDim.x) {
		const uint32_t t = a.tokens[r * a.tokens_per_row + m];
		a.logprobs[r * a.tokens_per_row + m] = t < (uint32_t) a.n_cols ? st.log_p(to_f(row[t]), a.s) : 0.0f;
	}
}

template <typename T>
__device__ __forceinline__ void token_logprobs_run(const LogprobsArgs & a) {
	constexpr int V = VecOf<T>::N;
	__shared__ TopState t;
	extern __shared__ uint64_t list[];
	float * groups = reinterpret_cast<float *>(list + SCORE_CANDIDATES);
	const Score_Plan plan = score_stream_plan(a.n_rows, a.n_cols, (int) sizeof(T));
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x;
	const float s_log2e = a.s * SCORE_LOG2E;
	for (long w = blockIdx.x; w < (long) a.n_rows * plan.slices; w += gridDim.x) {
		const long r = plan.slices == 1 ? w : w / plan.slices;
		const int slice = plan.slices == 1 ? 0 : (int) (w - r * plan.slices);
		const T * row = static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride;
		const RowSlice sl(a.n_cols, V, slice, plan.slices, plan.slice_chunks);
		RowPart p = score_stream<T, true>(row, sl, s_log2e, a.top_k > 0 ? groups : nullptr);
		p = score_group_join(p, s_log2e, t.cells);
		const RowStats st(p.m, p.z, p.e);
		if (plan.slices == 1) token_logprobs_row<T>(a, r, row, st);
		else if (tid == 0) a.parts[w] = Score_Part{p.m, p.z, p.e, 0.0f};
		if (a.top_k > 0) {
			const int k = a.top_k;
			const int n = score_candidates(row, sl, k, p.m, groups, list, t);
			for (int i = tid; i < n; i += nt) {
				const uint64_t alt = list[i];
				const int rank = score_rank(list, n, alt);
				if (rank >= k) continue;
				if (plan.slices == 1) {
					a.top_ids[r * k + rank] = score_alternative_id(alt);
					a.top_logprobs[r * k + rank] = st.log_p(score_alternative_value(alt), a.s);
				}
				else a.lists[w * k + rank] = alt;
			}
			if (plan.slices > 1)
				for (int i = n + tid; i < k; i += nt) a.lists[w * k + i] = 0u;
		}
		__syncthreads();
	}
}

/* A row's slices, joined: one workgroup per row. An alternative's rank is the
 * sum over the slices' sorted lists of how many of each exceed it. */
template <typename T>
__device__ __forceinline__ void token_logprobs_join(const LogprobsArgs & a) {
	extern __shared__ uint64_t list[];
	const Score_Plan plan = score_stream_plan(a.n_rows, a.n_cols, (int) sizeof(T));
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x, k = a.top_k, slices = plan.slices;
	const float s_log2e = a.s * SCORE_LOG2E;
	for (long r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
		const T * row = static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride;
		const Score_Part * parts = a.parts + r * slices;
		float m = -__builtin_inff();
		for (int i = 0; i < slices; i++) m = fmaxf(m, parts[i].max);
		RowPart p;
		p.m = m;
		for (int i = 0; i < slices; i++) {
			RowPart q;
			q.m = parts[i].max;
			q.z = parts[i].z;
			q.e = parts[i].e;
			q.shift(m, s_log2e);
			p.z += q.z;
			p.e += q.e;
		}
		const RowStats st(p.m, p.z, p.e);
		token_logprobs_row<T>(a, r, row, st);
		__syncthreads();
		for (int i = tid; i < slices * k; i += nt) list[i] = a.lists[r * slices * k + i];
		__syncthreads();
		for (int i = tid; i < slices * k; i += nt) {
			const uint64_t alt = list[i];
			const int own = i / k;
			int rank = i - own * k;
			if (alt == 0u) continue;
			for (int o = 0; o < slices && rank < k; o++) {
				if (o == own) continue;
				const uint64_t * other = list + o * k;
				int from = 0, to = k;
				while (from < to) {
					const int mid = (from + to) >> 1;
					if (other[mid] > alt) from = mid + 1;
					else to = mid;
				}
				rank += from;
			}
			if (rank < k) {
				a.top_ids[r * k + rank] = score_alternative_id(alt);
				a.top_logprobs[r * k + rank] = st.log_p(score_alternative_value(alt), a.s);
			}
		}
	}
}

#define TOKEN_LOGPROBS_ARGS(T)                                                                                                   \
	int n_rows, int n_cols, uint64_t row_stride, float scale, int tokens_per_row, int top_k, T * logits, uint32_t * tokens,      \
		float * logprobs, float * entropy, float * lse, uint32_t * top_ids, float * top_logprobs, uint64_t workspace_bytes,      \
		void * workspace
#define TOKEN_LOGPROBS_PACK                                                                                                      \
	LogprobsArgs a = {n_rows, n_cols, row_stride, scale, tokens_per_row, top_k, logits, tokens, logprobs, entropy, lse, top_ids, \
					  top_logprobs, nullptr, nullptr};                                                                           \
	const Score_Plan plan = score_stream_plan(n_rows, n_cols, (int) sizeof(*logits));                                            \
	a.lists = static_cast<uint64_t *>(workspace);                                                                                \
	a.parts = reinterpret_cast<Score_Part *>(a.lists + (uint64_t) n_rows * plan.slices * top_k);
#define TOKEN_LOGPROBS_KERNEL(SUF, T)                                                                                            \
	extern "C" __global__ void __launch_bounds__(64 * SCORE_STREAM_WAVES, 2) token_logprobs_##SUF##_kernel(TOKEN_LOGPROBS_ARGS(T)) { \
		TOKEN_LOGPROBS_PACK                                                                                                      \
		token_logprobs_run<T>(a);                                                                                                \
	}                                                                                                                            \
	extern "C" __global__ void __launch_bounds__(SCORE_THREADS) token_logprobs_##SUF##_kernel_finish(TOKEN_LOGPROBS_ARGS(T)) {   \
		TOKEN_LOGPROBS_PACK                                                                                                      \
		token_logprobs_join<T>(a);                                                                                               \
	}

TOKEN_LOGPROBS_KERNEL(fp32, float)
TOKEN_LOGPROBS_KERNEL(fp16, f16_t)
TOKEN_LOGPROBS_KERNEL(bf16, bf16_t)
