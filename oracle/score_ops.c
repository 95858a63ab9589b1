/*
 * Oracle of the scoring ops (include/dataflow_score_ops.h) — TEST
 * INFRASTRUCTURE ONLY: their definitions in fp64, nothing rounded on the way,
 * and the adapters through which the CPU test backend runs them. They have no
 * reference counterpart.
 */
#include "oracle.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

static size_t elem_bytes(int dt) { return dt == ORACLE_FP32 ? 4 : 2; }

static const void * at(const void * p, int dt, uint64_t elems) { return (const char *) p + elems * elem_bytes(dt); }

static int supported(int dt) { return dt == ORACLE_FP32 || dt == ORACLE_FP16 || dt == ORACLE_BF16; }

/* log p of every column into lp; returns the log-sum-exp. A row of -inf alone
 * gives -inf everywhere, one with NaN or +inf NaN. */
static double log_probs(const double * x, int n, double s, double * lp) {
	double m = -INFINITY, z = 0.0;
	int bad = 0;
	for (int j = 0; j < n; j++) {
		if (isnan(x[j]) || x[j] == INFINITY) bad = 1;
		if (x[j] > m) m = x[j];
	}
	if (bad || m == -INFINITY) {
		for (int j = 0; j < n; j++) lp[j] = bad ? NAN : -INFINITY;
		return bad ? NAN : -INFINITY;
	}
	for (int j = 0; j < n; j++) z += exp(s * (x[j] - m));
	const double lz = log(z);
	for (int j = 0; j < n; j++) lp[j] = s * (x[j] - m) - lz;
	return s * m + lz;
}

typedef struct { double v; uint32_t id; } Alternative;
static int by_value(const void * pa, const void * pb) {
	const Alternative * a = pa, * b = pb;
	const int an = isnan(a->v), bn = isnan(b->v);
	if (an != bn) return an - bn;
	if (!an && a->v != b->v) return a->v > b->v ? -1 : 1;
	return a->id < b->id ? -1 : 1;
}

int oracle_token_logprobs(int dt, int n_rows, int n_cols, uint64_t row_stride, float scale, int tokens_per_row, int top_k, const void * logits,
						  const uint32_t * tokens, double * logprobs, double * entropy, double * lse, uint32_t * top_ids, double * top_logprobs) {
	if (!supported(dt) || n_rows < 0 || n_cols <= 0 || top_k > n_cols) return -1;
#pragma omp parallel for schedule(dynamic)
	for (int r = 0; r < n_rows; r++) {
		double * x = malloc(sizeof(double) * (size_t) n_cols), * lp = malloc(sizeof(double) * (size_t) n_cols);
		oracle_load(dt, at(logits, dt, (uint64_t) r * row_stride), n_cols, x);
		const double l = log_probs(x, n_cols, scale, lp);
		if (lse) lse[r] = l;
		if (entropy) {
			double h = isnan(l) ? NAN : 0.0;
			for (int j = 0; j < n_cols; j++)
				if (lp[j] != -INFINITY) h -= exp(lp[j]) * lp[j];
			entropy[r] = h;
		}
		for (int m = 0; m < tokens_per_row; m++) {
			const uint32_t t = tokens[(size_t) r * tokens_per_row + m];
			logprobs[(size_t) r * tokens_per_row + m] = t < (uint32_t) n_cols ? lp[t] : 0.0;
		}
		if (top_k > 0) {
			Alternative * a = malloc(sizeof(Alternative) * (size_t) n_cols);
			for (int j = 0; j < n_cols; j++) a[j] = (Alternative) {x[j], (uint32_t) j};
			qsort(a, (size_t) n_cols, sizeof(Alternative), by_value);
			for (int k = 0; k < top_k; k++) {
				top_ids[(size_t) r * top_k + k] = a[k].id;
				top_logprobs[(size_t) r * top_k + k] = lp[a[k].id];
			}
			free(a);
		}
		free(x);
		free(lp);
	}
	return 0;
}

int oracle_token_logprobs_bwd(int dt, int n_rows, int n_cols, uint64_t row_stride, float scale, int tokens_per_row, const void * logits,
							  const uint32_t * tokens, const float * lse, const float * entropy, const float * d_logprobs, const float * d_entropy,
							  double * dx) {
	if (!supported(dt) || n_rows < 0 || n_cols <= 0) return -1;
#pragma omp parallel for schedule(dynamic)
	for (int r = 0; r < n_rows; r++) {
		double * x = malloc(sizeof(double) * (size_t) n_cols), * out = dx + (size_t) r * n_cols;
		const double s = scale, h = d_entropy ? d_entropy[r] : 0.0, H = d_entropy ? entropy[r] : 0.0;
		double down = 0.0;
		int any = h != 0.0;
		oracle_load(dt, at(logits, dt, (uint64_t) r * row_stride), n_cols, x);
		for (int m = 0; m < tokens_per_row; m++) {
			const size_t i = (size_t) r * tokens_per_row + m;
			if (tokens[i] >= (uint32_t) n_cols) continue;
			down += d_logprobs[i];
			any |= d_logprobs[i] != 0.0f;
		}
		for (int j = 0; j < n_cols; j++) {
			const double lp = s * x[j] - lse[r], p = exp(lp);
			out[j] = !any || lse[r] == -INFINITY ? 0.0 : p == 0.0 ? 0.0 : -s * p * (down + (h != 0.0 ? h * (lp + H) : 0.0));
		}
		if (any && lse[r] != -INFINITY)
			for (int m = 0; m < tokens_per_row; m++) {
				const size_t i = (size_t) r * tokens_per_row + m;
				if (tokens[i] < (uint32_t) n_cols) out[tokens[i]] += s * d_logprobs[i];
			}
		free(x);
	}
	return 0;
}

int oracle_distillation_loss(int dt, int n_rows, int n_cols, uint64_t row_stride, float scale, int top_k, const void * logits,
							 const uint32_t * teacher_ids, const float * teacher_logits, const float * row_weights, double * loss, double * mean_loss,
							 double * dx) {
	if (!supported(dt) || n_rows < 0 || n_cols <= 0) return -1;
	const double s = scale, T = 1.0 / s;
#pragma omp parallel for schedule(dynamic)
	for (int r = 0; r < n_rows; r++) {
		double * out = dx ? dx + (size_t) r * n_cols : NULL;
		const uint32_t * ids = teacher_ids + (size_t) r * top_k;
		const float * v = teacher_logits + (size_t) r * top_k;
		const double w = row_weights ? row_weights[r] : 1.0;
		double vmax = -INFINITY, zq = 0.0;
		int entries = 0;
		for (int k = 0; k < top_k; k++) {
			if (ids[k] >= (uint32_t) n_cols || v[k] == -INFINITY) continue;
			entries++;
			if (isnan(v[k]) || v[k] > vmax) vmax = v[k];
			if (isnan(vmax)) break;
		}
		if (out) memset(out, 0, sizeof(double) * (size_t) n_cols);
		loss[r] = 0.0;
		if (w == 0.0 || entries == 0) continue;
		double * x = malloc(sizeof(double) * (size_t) n_cols), * lp = malloc(sizeof(double) * (size_t) n_cols);
		oracle_load(dt, at(logits, dt, (uint64_t) r * row_stride), n_cols, x);
		const double lse = log_probs(x, n_cols, s, lp);
		for (int k = 0; k < top_k; k++)
			if (ids[k] < (uint32_t) n_cols && v[k] != -INFINITY) zq += exp(s * (v[k] - vmax));
		if (out && lse != -INFINITY)
			for (int j = 0; j < n_cols; j++) out[j] = w * T * exp(lp[j]);
		for (int k = 0; k < top_k; k++) {
			if (ids[k] >= (uint32_t) n_cols || v[k] == -INFINITY) continue;
			const double lq = s * (v[k] - vmax) - log(zq), q = exp(lq);
			if (q != 0.0) loss[r] += T * T * q * (lq - lp[ids[k]]);
			if (out && lse != -INFINITY) out[ids[k]] -= w * T * q;
		}
		free(x);
		free(lp);
	}
	if (mean_loss) {
		double sum = 0.0;
		for (int r = 0; r < n_rows; r++) {
			const double w = row_weights ? row_weights[r] : 1.0;
			if (w != 0.0) sum += w * loss[r];
		}
		*mean_loss = sum / n_rows;
	}
	return 0;
}

/* ---- adapters of the CPU test backend ---- */

#define A(i, type) (*((type *) op_args[(i)]))

static double * dbuf(size_t n) { return (double *) malloc(sizeof(double) * (n > 0 ? n : 1)); }

static void to_f32(const double * v, size_t n, float * out) {
	for (size_t i = 0; out && i < n; i++) out[i] = (float) v[i];
}

static int token_logprobs_adapter(int dt, void ** op_args) {
	const int n_rows = A(0, int), n_cols = A(1, int), M = A(4, int), K = A(5, int);
	const size_t nm = (size_t) n_rows * M, nk = (size_t) n_rows * K;
	double * lp = dbuf(nm), * h = dbuf(n_rows), * l = dbuf(n_rows), * tl = dbuf(nk);
	const int ret = oracle_token_logprobs(dt, n_rows, n_cols, A(2, uint64_t), A(3, float), M, K, A(6, void *), A(7, uint32_t *), lp, h, l,
										  A(11, uint32_t *), tl);
	if (!ret) {
		to_f32(lp, nm, A(8, float *));
		to_f32(h, n_rows, A(9, float *));
		to_f32(l, n_rows, A(10, float *));
		to_f32(tl, nk, A(12, float *));
	}
	free(lp); free(h); free(l); free(tl);
	return ret;
}

static void store_rows(int dt, int n_rows, int n_cols, uint64_t stride, const double * v, void * out) {
	for (int r = 0; out && r < n_rows; r++)
		oracle_store(dt, v + (size_t) r * n_cols, n_cols, (void *) at(out, dt, (uint64_t) r * stride));
}

static int token_logprobs_bwd_adapter(int dt, void ** op_args) {
	const int n_rows = A(0, int), n_cols = A(1, int);
	double * dx = dbuf((size_t) n_rows * n_cols);
	const int ret = oracle_token_logprobs_bwd(dt, n_rows, n_cols, A(2, uint64_t), A(4, float), A(5, int), A(6, void *), A(7, uint32_t *), A(8, float *),
											  A(9, float *), A(10, float *), A(11, float *), dx);
	if (!ret) store_rows(dt, n_rows, n_cols, A(3, uint64_t), dx, A(12, void *));
	free(dx);
	return ret;
}

static int distillation_loss_adapter(int dt, void ** op_args) {
	const int n_rows = A(0, int), n_cols = A(1, int);
	double * dx = dbuf((size_t) n_rows * n_cols), * l = dbuf(n_rows), mean = 0.0;
	const int ret = oracle_distillation_loss(dt, n_rows, n_cols, A(2, uint64_t), A(4, float), A(5, int), A(6, void *), A(7, uint32_t *), A(8, float *),
											 A(9, float *), l, &mean, dx);
	if (!ret) {
		to_f32(l, n_rows, A(10, float *));
		to_f32(&mean, 1, A(11, float *));
		store_rows(dt, n_rows, n_cols, A(3, uint64_t), dx, A(12, void *));
	}
	free(dx); free(l);
	return ret;
}

#define ADAPT_SCORES(sfx, code)                                                                        \
	int token_logprobs_##sfx##_kernel(void ** a) { return token_logprobs_adapter(code, a); }           \
	int token_logprobs_bwd_##sfx##_kernel(void ** a) { return token_logprobs_bwd_adapter(code, a); }   \
	int distillation_loss_##sfx##_kernel(void ** a) { return distillation_loss_adapter(code, a); }

ADAPT_SCORES(fp32, ORACLE_FP32)
ADAPT_SCORES(fp16, ORACLE_FP16)
ADAPT_SCORES(bf16, ORACLE_BF16)
