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
 *
 * Without alternatives: bound by reading the logits once, 16 bytes a thread and
 * four of them under way (4096 x 128256 bf16 159 us, 6.6 TB/s; 8 under way 167
 * us: half the waves fit). One exp2 and three operations per logit stay below
 * that. With them: 1021 x 50257 bf16, 64 alternatives, 32 us, without 22.7:
 * the bound, the second reading (out of L2) and the ranking are latency; 6
 * waves to a SIMD, whose registers hold everything (in 8 the compiler spills:
 * 42.4 us; 5: 39.4). Few rows are bound by latency:
 * 1 x 128256 with 20 alternatives 14.4 us, in two launches of about 5 us of host
 * time each, 64 x 128256 fp16 with 5 17.6 us.
 */
#include "score_rows.h"

struct TopState {
	float cells[5 * SCORE_MAX_WAVES];
	float counts[2 * SCORE_MAX_WAVES];
	uint32_t hist[256];
	uint32_t prefix, need, count, n_groups;
};

/* a count over a workgroup of a wave's count; calls alternate between two
 * sets of cells, so one barrier each is enough */
__device__ __forceinline__ uint32_t score_group_count(uint32_t n, TopState & t, int & turn) {
	if (blockDim.x == 64) return n;
	float * cells = t.counts + (turn ^= SCORE_MAX_WAVES);
	if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = (float) n;
	lds_barrier();
	return (uint32_t) score_cells(cells, 0.0f, ScoreSum());
}

/* Of the columns [first, end) those whose key is `key`, by rising column, the
 * first `most` of them, into list[0..); returns how many there were. */
template <typename T>
__device__ __forceinline__ uint32_t score_equal(const T * row, int first, int end, uint32_t key, uint32_t most, uint64_t * list, TopState & t) {
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x, lane = tid & 63, wave = tid >> 6, waves = nt >> 6;
	uint32_t have = 0;
#pragma unroll 1
	for (long base = first; base < end && have < most; base += nt) {
		const long j = base + tid;
		const bool is = j < end && score_key(to_f(row[j < end ? j : first])) == key;
		const unsigned long long ballot = __ballot(is);
		__syncthreads();
		if (lane == 0) t.counts[wave] = (float) __popcll(ballot);
		__syncthreads();
		uint32_t before = have + (uint32_t) __popcll(ballot & ((1ull << lane) - 1ull));
#pragma unroll 1
		for (int w = 0; w < waves; w++) {
			if (w < wave) before += (uint32_t) t.counts[w];
			have += (uint32_t) t.counts[w];
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
#pragma unroll 1
	for (int shift = 24; shift >= 0; shift -= 8) {
#pragma unroll 1
		for (int b = tid; b < 256; b += nt) t.hist[b] = 0u;
		__syncthreads();
		const uint32_t prefix = t.prefix;
		const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
#pragma unroll 1
		for (long j = first + tid; j < end; j += nt) {
			const uint32_t key = score_key(to_f(row[j]));
			if ((key & above) == prefix) atomicAdd(&t.hist[(key >> shift) & 255u], 1u);
		}
		__syncthreads();
		if (tid == 0) {
			uint32_t need = t.need;
			int b = 255;
#pragma unroll 1
			while (b > 0 && t.hist[b] < need) need -= t.hist[b--];
			t.prefix = prefix | ((uint32_t) b << shift);
			t.need = need;
		}
		__syncthreads();
	}
	const uint32_t last = t.prefix, equal = t.need;
#pragma unroll 1
	for (long j = first + tid; j < end; j += nt) {
		const uint32_t key = score_key(to_f(row[j]));
		if (key > last) list[atomicAdd(&t.count, 1u)] = score_alternative(key, (uint32_t) j);
	}
	score_equal(row, first, end, last, equal, list + (k - (int) equal), t);
	__syncthreads();
}

/* A bound that `reach` numbers reach at `lo` (k or more of them) and none
 * beyond `hi`, moved up until not many more than k reach it. Far from a row's
 * bulk the logarithm of how many reach a bound falls about evenly, so every
 * other step interpolates there; the others halve the interval. count(bound):
 * how many reach it, over the workgroup. */
template <typename Count>
__device__ __forceinline__ float score_bound(float lo, float hi, uint32_t & reach, int k, const Count & count) {
	const float aim = __builtin_amdgcn_logf(1.25f * (float) k + 2.0f);
	float at_hi = 0.0f;
#pragma unroll 1
	for (int step = 0; step < 24 && reach > (uint32_t) (k + (k >> 1) + 8); step++) {
		const float at_lo = __builtin_amdgcn_logf((float) reach);
		float part = 0.5f;
		if (!(step & 1)) part = fminf(fmaxf((at_lo - aim) / (at_lo - at_hi), 0.02f), 0.98f);
		const float mid = lo + part * (hi - lo);
		if (!(mid > lo && mid <= hi)) break;
		const uint32_t n = count(mid);
		if (n < (uint32_t) k) {
			hi = mid;
			at_hi = n == 0u ? 0.0f : __builtin_amdgcn_logf((float) n);
		}
		else {
			lo = mid;
			reach = n;
		}
	}
	return lo;
}

/* Where many more than k of a list's n numbers are left (all of which reach lo,
 * if any k do), those that reach a bound that not many more than k reach, moved
 * to the list's front. Returns how many. */
__device__ __forceinline__ int score_thin(int n, int k, float lo, float hi, uint64_t * list, TopState & t, int & turn) {
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x;
	if (n <= 2 * k + 64) return n;
	const uint32_t * keys = reinterpret_cast<const uint32_t *>(list) + 1;   /* the numbers' upper halves */
	uint32_t reach = (uint32_t) n;
	if (tid == 0) t.count = 0u;
	lo = score_bound(lo, hi, reach, k, [&](float mid) {
		const uint32_t key = score_key(mid);
		uint32_t c = 0u;
#pragma unroll 1
		for (int i = tid; i < n + tid; i += nt) c += (uint32_t) __popcll(__ballot(i < n && keys[i < n ? 2 * i : 0] >= key));
		return score_group_count(c, t, turn);
	});
	if (reach == (uint32_t) n) return n;
	/* what is kept of a step's numbers lies no further than the step's end */
	const uint32_t key = score_key(lo);
#pragma unroll 1
	for (int i = tid; i < n + tid; i += nt) {
		const uint64_t alt = i < n ? list[i] : 0u;
		lds_barrier();
		if ((uint32_t) (alt >> 32) >= key) list[atomicAdd(&t.count, 1u)] = alt;
		lds_barrier();
	}
	return (int) t.count;
}

/* Candidates of a slice into list[0..n): the k largest of its columns among
 * them (all of them where there are fewer than k). `groups`: the maxima that
 * the thread's batches left, SCORE_GROUP_SLOTS rows of blockDim.x. Returns n. */
template <typename T>
__device__ __forceinline__ int score_candidates(const T * row, const RowSlice & sl, int k, float row_max, float met, float least, const float * groups, uint16_t * reached, uint64_t * list, TopState & t) {
	constexpr int V = VecOf<T>::N;
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x, lane = tid & 63;
	const int batches = (sl.last - sl.first + SCORE_BATCH * nt - 1) / (SCORE_BATCH * nt);
	const int col0 = sl.begin(V), col1 = sl.behind(V), single = sl.single();
	const T * chunks = row + sl.head;
	int turn = 0;
	if (col1 - col0 <= SCORE_CANDIDATES) {
		__syncthreads();
#pragma unroll 1
		for (int c = sl.first + tid; c < sl.last; c += nt) {
			R16 x = score_load(chunks, (uint64_t) c, 0u);
			float f[V];
			unpack16<T>(x, f);
#pragma unroll
			for (int i = 0; i < V; i++) list[sl.head + c * V + i - col0] = score_alternative(score_key(f[i]), (uint32_t) (sl.head + c * V + i));
		}
		if (single >= 0) list[single - col0] = score_alternative(score_key(to_f(row[single])), (uint32_t) single);
		__syncthreads();
		return met < (float) k ? col1 - col0 : score_thin(col1 - col0, k, least, row_max, list, t, turn);
	}
	float g[SCORE_GROUP_SLOTS];
#pragma unroll
	for (int i = 0; i < SCORE_GROUP_SLOTS; i++) g[i] = i < batches || i == 0 ? groups[i * nt + tid] : -__builtin_inff();
	/* as many threads as have a column above -inf reach the least of their maxima,
	 * and most of their groups do */
	float lo = least;
	uint32_t reach = (uint32_t) met * (uint32_t) (batches < SCORE_GROUP_SLOTS ? batches > 1 ? batches : 1 : SCORE_GROUP_SLOTS);   /* groups, at most */
	if (tid == 0) t.count = t.n_groups = 0u;
	lds_barrier();
	if (met >= (float) k) {
		lo = score_bound(lo, row_max, reach, k, [&](float mid) {
			uint32_t n = 0;
#pragma unroll
			for (int i = 0; i < SCORE_GROUP_SLOTS; i++) n += (uint32_t) __popcll(__ballot(g[i] >= mid));
			return score_group_count(n, t, turn);
		});
	}
	else lo = -3.402823466e38f;   /* few columns are above -inf: all of them */
	/* the groups that reach it, and then a thread for each of their chunks */
#pragma unroll
	for (int i = 0; i < SCORE_GROUP_SLOTS; i++) {
		const unsigned long long hit = __ballot(g[i] >= lo);
		if (hit == 0ull) continue;
		uint32_t at = 0u;
		if (lane == 0) at = atomicAdd(&t.n_groups, (uint32_t) __popcll(hit));
		at = __builtin_amdgcn_readfirstlane(at);
		if (g[i] >= lo) reached[at + (uint32_t) __popcll(hit & ((1ull << lane) - 1ull))] = (uint16_t) (i * nt + tid);
	}
	lds_barrier();
	const int items = (int) t.n_groups * SCORE_BATCH;
#pragma unroll 1
	for (int item = tid; item < items; item += nt) {
		const int group = reached[item / SCORE_BATCH], slot = group / nt, owner = group - slot * nt;
#pragma unroll 1
		for (int b = slot; b < batches || b == 0; b += SCORE_GROUP_SLOTS) {
			const int c = sl.first + (b * SCORE_BATCH + item % SCORE_BATCH) * nt + owner;
			if (c >= sl.last) continue;
			const R16 x = score_load<T, true>(chunks, (uint64_t) c, 0u);
			float f[V];
			unpack16<T>(x, f);
			uint32_t hits = 0u;
#pragma unroll
			for (int v = 0; v < V; v++) hits |= f[v] >= lo ? 1u << v : 0u;
			if (hits == 0u) continue;
			uint32_t at = atomicAdd(&t.count, (uint32_t) __popc(hits));
#pragma unroll
			for (int v = 0; v < V; v++)
				if (hits >> v & 1u) {
					if (at < SCORE_CANDIDATES) list[at] = score_alternative(score_key(f[v]), (uint32_t) (sl.head + c * V + v));
					at++;
				}
		}
	}
	if (single >= 0) {
		const float x = to_f(row[single]);
		if (x >= lo) {
			const uint32_t at = atomicAdd(&t.count, 1u);
			if (at < SCORE_CANDIDATES) list[at] = score_alternative(score_key(x), (uint32_t) single);
		}
	}
	lds_barrier();
	const int n = (int) t.count;
	lds_barrier();
	if (n > SCORE_CANDIDATES) {
		score_select(row, col0, col1, k, list, t);
		return k;
	}
	if (n < k) {
		/* then columns of -inf, and then those of NaN; a slice may have fewer than k */
		uint32_t have = (uint32_t) n;
		have += score_equal(row, col0, col1, score_key(-__builtin_inff()), (uint32_t) k - have, list + have, t);
		if (have < (uint32_t) k) have += score_equal(row, col0, col1, 0u, (uint32_t) k - have, list + have, t);
		__syncthreads();
		return (int) have;
	}
	return score_thin(n, k, lo, row_max, list, t, turn);
}

/* The place of each of a list's n numbers among them, by counting the larger
 * ones: four threads a number, each over a quarter of the list. put(place,
 * number) is called by one of them. */
template <typename Put>
__device__ __forceinline__ void score_rank(const uint64_t * list, int n, const Put & put) {
#pragma unroll 1
	for (int i = (int) threadIdx.x >> 2; i < n; i += (int) (blockDim.x >> 2)) {
		const uint64_t alt = list[i];
		int r = 0;
#pragma unroll 4
		for (int o = (int) threadIdx.x & 3; o < n; o += 4) r += list[o] > alt ? 1 : 0;
		r += __builtin_amdgcn_update_dpp(0, r, DPP_QUAD_1032, 0xf, 0xf, false);
		r += __builtin_amdgcn_update_dpp(0, r, DPP_QUAD_2301, 0xf, 0xf, false);
		if ((threadIdx.x & 3) == 0) put(r, alt);
	}
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
#pragma unroll 1
	for (int m = (int) threadIdx.x; m < a.tokens_per_row; m += (int) blockDim.x) {
		const uint32_t t = a.tokens[r * a.tokens_per_row + m];
		a.logprobs[r * a.tokens_per_row + m] = t < (uint32_t) a.n_cols ? st.log_p(to_f(row[t]), a.s) : 0.0f;
	}
}

template <typename T, bool TOP>
__device__ __forceinline__ void token_logprobs_run(const LogprobsArgs & a) {
	constexpr int V = VecOf<T>::N;
	__shared__ TopState t;
	const Score_Plan plan = score_stream_plan(a.n_rows, a.n_cols, (int) sizeof(T), a.top_k);
	extern __shared__ uint64_t list[];
	float * groups = reinterpret_cast<float *>(list + SCORE_CANDIDATES);
	uint16_t * reached = reinterpret_cast<uint16_t *>(groups + SCORE_GROUP_SLOTS * blockDim.x);
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x;
	const float s_log2e = a.s * SCORE_LOG2E;
#pragma unroll 1
	for (long w = blockIdx.x; w < (long) a.n_rows * plan.slices; w += gridDim.x) {
		const long r = plan.slices == 1 ? w : w / plan.slices;
		const int slice = plan.slices == 1 ? 0 : (int) (w - r * plan.slices);
		const T * row = static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride;
		const RowSlice sl(a.n_cols, V, score_head(row, a.n_cols), slice, plan.slices, plan.slice_chunks);
		float met, least;
		const RowPart p = score_group_join<TOP>(score_stream<T, true, TOP>(row, sl, s_log2e, TOP ? groups : nullptr), s_log2e, t.cells, &met, &least);
		const RowStats st(p.m, p.z, p.e);
		if (plan.slices == 1) token_logprobs_row<T>(a, r, row, st);
		else if (tid == 0) a.parts[w] = Score_Part{p.m, p.z, p.e, 0.0f};
		if (TOP) {
			const int k = a.top_k;
			const int n = score_candidates(row, sl, k, p.m, met, least, groups, reached, list, t);
			score_rank(list, n, [&](int rank, uint64_t alt) {
				if (rank >= k) return;
				if (plan.slices == 1) {
					a.top_ids[r * k + rank] = score_alternative_id(alt);
					a.top_logprobs[r * k + rank] = st.log_p(score_alternative_value(alt), a.s);
				}
				else a.lists[w * k + rank] = alt;
			});
			if (plan.slices > 1)
				for (int i = n + tid; i < k; i += nt) a.lists[w * k + i] = 0u;
		}
		__syncthreads();
	}
}

/* A row's slices, joined: one workgroup per row. k of the slices' alternatives
 * or more reach any slice's k-th, and the least of their p-th ones with
 * p = k / slices, rounded up: those that reach both are ranked by counting. */
template <typename T>
__device__ __forceinline__ void token_logprobs_join(const LogprobsArgs & a) {
	extern __shared__ uint64_t list[];
	__shared__ uint32_t count;
	__shared__ unsigned long long all_reach, one_reaches;
	const Score_Plan plan = score_stream_plan(a.n_rows, a.n_cols, (int) sizeof(T), a.top_k);
	const int tid = (int) threadIdx.x, nt = (int) blockDim.x, lane = tid & 63, k = a.top_k, slices = plan.slices;
	const float s_log2e = a.s * SCORE_LOG2E;
	for (long r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
		const T * row = static_cast<const T *>(a.logits) + (uint64_t) r * a.row_stride;
		const uint64_t * lists = a.lists + r * slices * k;
		RowPart p;   /* a lane of each wave for a slice (SCORE_MAX_SLICES are fewer than lanes) */
		if (lane < slices) {
			const Score_Part q = a.parts[r * slices + lane];
			p.m = q.max;
			p.z = q.z;
			p.e = q.e;
		}
		if (k > 0) {
			if (tid == 0) { count = 0u; all_reach = ~0ull; one_reaches = 0ull; }
			__syncthreads();
			if (tid < slices) {
				atomicMax(&one_reaches, (unsigned long long) lists[tid * k + k - 1]);
				atomicMin(&all_reach, (unsigned long long) lists[tid * k + (k + slices - 1) / slices - 1]);
			}
		}
		p.shift(wave_max(p.m), s_log2e);
		p.z = wave_sum(p.z);
		p.e = wave_sum(p.e);
		const RowStats st(p.m, p.z, p.e);
		token_logprobs_row<T>(a, r, row, st);
		if (k == 0) continue;
		__syncthreads();
		const uint64_t bound = all_reach > one_reaches ? all_reach : one_reaches;
		for (int i = tid; i < slices * k; i += nt) {
			const uint64_t alt = lists[i];
			if (alt != 0u && alt >= bound) list[atomicAdd(&count, 1u)] = alt;
		}
		__syncthreads();
		score_rank(list, (int) count, [&](int rank, uint64_t alt) {
			if (rank >= k) return;
			a.top_ids[r * k + rank] = score_alternative_id(alt);
			a.top_logprobs[r * k + rank] = st.log_p(score_alternative_value(alt), a.s);
		});
		__syncthreads();
	}
}

#define TOKEN_LOGPROBS_ARGS(T)                                                                                                   \
	int n_rows, int n_cols, uint64_t row_stride, float scale, int tokens_per_row, int top_k, T * logits, uint32_t * tokens,      \
		float * logprobs, float * entropy, float * lse, uint32_t * top_ids, float * top_logprobs, uint64_t workspace_bytes,      \
		void * workspace
#define TOKEN_LOGPROBS_PACK                                                                                                      \
	LogprobsArgs a = {n_rows, n_cols, row_stride, scale, tokens_per_row, top_k, logits, tokens, logprobs, entropy, lse, top_ids, \
					  top_logprobs, nullptr, nullptr};                                                                           \
	const Score_Plan plan = score_stream_plan(n_rows, n_cols, (int) sizeof(*logits), top_k);                                            \
	a.lists = static_cast<uint64_t *>(workspace);                                                                                \
	a.parts = reinterpret_cast<Score_Part *>(a.lists + (uint64_t) n_rows * plan.slices * top_k);
#define TOKEN_LOGPROBS_KERNEL(SUF, T)                                                                                            \
	extern "C" __global__ void __launch_bounds__(64 * SCORE_MAX_WAVES, 8) token_logprobs_##SUF##_kernel(TOKEN_LOGPROBS_ARGS(T)) { \
		TOKEN_LOGPROBS_PACK                                                                                                      \
		token_logprobs_run<T, false>(a);                                                                                                \
	}                                                                                                                            \
	extern "C" __global__ void __launch_bounds__(64 * SCORE_STREAM_WAVES, 6) token_logprobs_##SUF##_kernel_top(TOKEN_LOGPROBS_ARGS(T)) { \
		TOKEN_LOGPROBS_PACK                                                                                                      \
		token_logprobs_run<T, true>(a);                                                                                          \
	}                                                                                                                            \
	extern "C" __global__ void __launch_bounds__(SCORE_JOIN_THREADS) token_logprobs_##SUF##_kernel_finish(TOKEN_LOGPROBS_ARGS(T)) {   \
		TOKEN_LOGPROBS_PACK                                                                                                      \
		token_logprobs_join<T>(a);                                                                                               \
	}

TOKEN_LOGPROBS_KERNEL(fp32, float)
TOKEN_LOGPROBS_KERNEL(fp16, f16_t)
TOKEN_LOGPROBS_KERNEL(bf16, bf16_t)
