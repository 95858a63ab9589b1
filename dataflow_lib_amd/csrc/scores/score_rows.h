/*
 * What the scoring kernels share: a row's statistics and its k largest
 * logits, each found by one workgroup.
 *
 * A row is shifted by its largest logit M before anything is exponentiated:
 *   Z = sum exp(s (x - M)),  E = sum s (x - M) exp(s (x - M))
 *   lse = s M + log Z,  log p_j = s (x_j - M) - log Z,  entropy = log Z - E / Z
 * The difference x - M is formed first: it is exact next to the maximum, and
 * it cannot overflow where s x can (rows of the type's lowest value).
 */
#pragma once

#include "dtypes.h"
#include "reduce.h"
#include "score_geometry.h"

#define SCORE_LOG2E 1.4426950408889634f
#define SCORE_MAX_WAVES 16

/* what a row's log-probabilities are formed from */
struct RowStats {
	float max;      /* M; 0 for a row of -inf alone */
	float log_z;    /* log Z; +inf for a row of -inf alone, NaN with NaN or +inf */
	float inv_z;    /* 1 / Z; 0 for a row of -inf alone */
	float e_z;      /* E / Z */
	__device__ __forceinline__ RowStats() {}
	__device__ __forceinline__ RowStats(float m, float z, float e) {
		max = m;
		const bool none = z == 0.0f;
		log_z = none ? __builtin_inff() : logf(z);
		inv_z = none ? 0.0f : 1.0f / z;
		e_z = none ? 0.0f : e / z;
	}
	__device__ __forceinline__ bool none() const { return inv_z == 0.0f; }
	__device__ __forceinline__ float lse(float s) const { return none() ? -__builtin_inff() : fmaf(s, max, log_z); }
	__device__ __forceinline__ float entropy() const { return none() ? 0.0f : log_z - e_z; }
	__device__ __forceinline__ float log_p(float x, float s) const { return s * (x - max) - log_z; }
};

/* a term of Z (into z) and of E (into e): t = s (x - M) in units of log2, and a
 * column of -inf counts nothing (-inf * 0 is kept out of E) */
__device__ __forceinline__ void score_add(float d, float s_log2e, float s, float & z, float & e) {
	const float p = __builtin_amdgcn_exp2f(d * s_log2e);
	z += p;
	e = fmaf(fmaxf(d, -1e30f) * s, p, e);
}

/* sums and maxima over a workgroup; `cells`: SCORE_MAX_WAVES floats of LDS */
__device__ __forceinline__ float score_group_max(float v, float * cells) {
	v = wave_max(v);
	const int waves = (int) (blockDim.x >> 6);
	__syncthreads();
	if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = v;
	__syncthreads();
	v = cells[0];
	for (int w = 1; w < waves; w++) v = fmaxf(v, cells[w]);
	return v;
}
__device__ __forceinline__ float score_group_sum(float v, float * cells) {
	v = wave_sum(v);
	const int waves = (int) (blockDim.x >> 6);
	__syncthreads();
	if ((threadIdx.x & 63) == 0) cells[threadIdx.x >> 6] = v;
	__syncthreads();
	v = cells[0];
	for (int w = 1; w < waves; w++) v += cells[w];
	return v;
}

template <typename T>
__device__ __forceinline__ RowStats score_row_stats(const T * row, int n_cols, float s, float * cells) {
	float m = -__builtin_inff();
	for (long j = threadIdx.x; j < n_cols; j += blockDim.x) m = fmaxf(m, to_f(row[j]));
	m = score_group_max(m, cells);
	if (m == -__builtin_inff()) m = 0.0f;
	float z = 0.0f, e = 0.0f;
	for (long j = threadIdx.x; j < n_cols; j += blockDim.x) score_add(to_f(row[j]) - m, s * SCORE_LOG2E, s, z, e);
	z = score_group_sum(z, cells);
	e = score_group_sum(e, cells);
	return RowStats(m, z, e);
}

/* Whole numbers that lie as floats do: -0 with +0, NaN below -inf. */
__device__ __forceinline__ uint32_t score_key(float x) {
	const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
	if (x != x) return 0u;
	return (u >> 31) ? ~u : (u | 0x80000000u);
}

/* A row's k largest logits, found exactly: the k-th largest key digit by digit
 * (8 bits of it a pass over the row, counted in LDS), then the larger ones and
 * as many of the equal ones, by rising column, as are left. */
struct ScoreTop {
	uint32_t hist[256];
	uint32_t prefix, need, count;
	uint32_t waves[SCORE_MAX_WAVES];
	uint32_t key[SCORE_TOP_MAX], id[SCORE_TOP_MAX];
};

template <typename T>
__device__ __forceinline__ void score_select(const T * row, int n_cols, int k, ScoreTop & t) {
	const int tid = (int) threadIdx.x, lane = tid & 63, wave = tid >> 6, n_waves = (int) (blockDim.x >> 6);
	__syncthreads();
	if (tid == 0) { t.prefix = 0u; t.need = (uint32_t) k; t.count = 0u; }
	for (int shift = 24; shift >= 0; shift -= 8) {
		for (int b = tid; b < 256; b += (int) blockDim.x) t.hist[b] = 0u;
		__syncthreads();
		const uint32_t prefix = t.prefix;
		const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
		for (long j = tid; j < n_cols; j += blockDim.x) {
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
	for (long j = tid; j < n_cols; j += blockDim.x) {
		const uint32_t key = score_key(to_f(row[j]));
		if (key > last) {
			const uint32_t at = atomicAdd(&t.count, 1u);
			t.key[at] = key;
			t.id[at] = (uint32_t) j;
		}
	}
	/* the equal ones in the order of their columns */
	uint32_t have = 0;
	for (long base = 0; base < n_cols && have < equal; base += blockDim.x) {
		const long j = base + tid;
		const bool is = j < n_cols && score_key(to_f(row[j < n_cols ? j : 0])) == last;
		const unsigned long long ballot = __ballot(is);
		__syncthreads();
		if (lane == 0) t.waves[wave] = (uint32_t) __popcll(ballot);
		__syncthreads();
		uint32_t before = have + (uint32_t) __popcll(ballot & ((1ull << lane) - 1ull));
		for (int w = 0; w < n_waves; w++) {
			if (w < wave) before += t.waves[w];
			have += t.waves[w];
		}
		if (is && before < equal) {
			t.key[(uint32_t) k - equal + before] = last;
			t.id[(uint32_t) k - equal + before] = (uint32_t) j;
		}
	}
	__syncthreads();
}

/* the place of each chosen logit among the k: by falling key, equal keys by
 * rising column */
__device__ __forceinline__ int score_rank(const ScoreTop & t, int k, int i) {
	const uint32_t key = t.key[i], id = t.id[i];
	int r = 0;
	for (int o = 0; o < k; o++) r += (t.key[o] > key || (t.key[o] == key && t.id[o] < id)) ? 1 : 0;
	return r;
}
