/*
 * Launch rules of the scoring ops, shared by the kernels, the
 * launch-configuration library and the workspace functions (plain C on the
 * host side).
 */
#ifndef SCORE_GEOMETRY_H
#define SCORE_GEOMETRY_H

#ifndef GEOM_FN
#define GEOM_FN static inline
#endif

/* limits of the public interface (dataflow_score_ops.h) */
#define SCORE_TOKENS_MAX 1024
#define SCORE_TOP_MAX 256
#define SCORE_TEACHER_MAX 1024
#define SCORE_SCALE_MIN 1e-6f
#define SCORE_SCALE_MAX 1e6f

/* one workgroup per row, walking rows a grid apart: so many workgroups at
 * most, which keeps every launch below 2^32 threads */
#define SCORE_THREADS 256
#define SCORE_MAX_GROUPS (1 << 20)

GEOM_FN unsigned long score_logprobs_workspace(int n_rows, int n_cols, int elem_bytes, int top_k) {
	(void) n_rows; (void) n_cols; (void) elem_bytes; (void) top_k;
	return 0;
}

GEOM_FN unsigned long score_distill_workspace(int n_rows, int n_cols, int elem_bytes, int top_k) {
	(void) n_rows; (void) n_cols; (void) elem_bytes; (void) top_k;
	return 0;
}

#endif
