/*
 * Launch geometry of the scoring ops (dataflow_score_ops.h), and the checks of
 * their arguments: whatever the kernels rely on is refused here with a
 * message, before anything is launched.
 */
#include "hip_ops_config.h"
#include "score_geometry.h"

#include <math.h>

#define ARG(op, i, type) (*((type *) (op)->op_args[(i)]))

static void set_1d(Hip_Launch_Config * c, unsigned grid, unsigned block, unsigned lds) {
	c->gridDimX = grid;
	c->gridDimY = 1;
	c->gridDimZ = 1;
	c->blockDimX = block;
	c->blockDimY = 1;
	c->blockDimZ = 1;
	c->sharedMemBytes = lds;
}

/* an operand that the kernels access: there, and aligned to its elements */
static int score_pointer(const char * what, const char * name, const void * p, size_t elem) {
	if (!p || ((uintptr_t) p % elem) != 0) {
		fprintf(stderr, "Error: %s: %s is %s...\n", what, name, p ? "not aligned to its elements" : "missing");
		return -1;
	}
	return 0;
}

/* -1 refused, 0 nothing to do, 1 checked */
static int score_check(const char * what, int n_rows, int n_cols, uint64_t stride, float scale, const void * logits, size_t elem) {
	if (n_rows < 0 || n_cols < 0 || elem == 0) {
		fprintf(stderr, "Error: %s: invalid shape (%d x %d) or dtype...\n", what, n_rows, n_cols);
		return -1;
	}
	if (!(scale >= SCORE_SCALE_MIN && scale <= SCORE_SCALE_MAX)) {
		fprintf(stderr, "Error: %s: scale %g is outside [%g, %g]...\n", what, (double) scale, (double) SCORE_SCALE_MIN, (double) SCORE_SCALE_MAX);
		return -1;
	}
	if (n_rows == 0 || n_cols == 0) return 0;
	/* the whole tensor within 2^60 bytes: byte offsets do not wrap */
	if (stride < (uint64_t) n_cols || stride > (1ull << 60) / elem / (uint64_t) n_rows) {
		fprintf(stderr, "Error: %s: rows of %d columns cannot be %lu elements apart...\n", what, n_cols, (unsigned long) stride);
		return -1;
	}
	return score_pointer(what, "the logits pointer", logits, elem) ? -1 : 1;
}

/* the gradient's rows: the logits' own place, or apart from them */
static int score_check_grad(const char * what, int n_rows, int n_cols, uint64_t stride, uint64_t grad_stride, const void * logits, const void * grad, size_t elem) {
	if (grad_stride < (uint64_t) n_cols || grad_stride > (1ull << 60) / elem / (uint64_t) n_rows) {
		fprintf(stderr, "Error: %s: gradient rows of %d columns cannot be %lu elements apart...\n", what, n_cols, (unsigned long) grad_stride);
		return -1;
	}
	if (score_pointer(what, "the gradient pointer", grad, elem)) return -1;
	const uintptr_t x = (uintptr_t) logits, g = (uintptr_t) grad;
	const uint64_t x_bytes = ((uint64_t) (n_rows - 1) * stride + (uint64_t) n_cols) * elem;
	const uint64_t g_bytes = ((uint64_t) (n_rows - 1) * grad_stride + (uint64_t) n_cols) * elem;
	if (x == g ? (stride != grad_stride && n_rows > 1) : (x < g ? g - x < x_bytes : x - g < g_bytes)) {
		fprintf(stderr, "Error: %s: the gradient overlaps the logits without being in their place...\n", what);
		return -1;
	}
	return 0;
}

static int score_check_workspace(const char * what, uint64_t needed, uint64_t bytes, const void * workspace) {
	if (needed > 0 && (bytes < needed || !workspace || ((uintptr_t) workspace & 255u) != 0)) {
		fprintf(stderr, "Error: %s: needs a 256-byte aligned workspace of %lu bytes, got %lu bytes at %p...\n", what,
				(unsigned long) needed, (unsigned long) bytes, workspace);
		return -1;
	}
	return 0;
}

static size_t logits_elem(Hip_Function * f) { return dataflow_sizeof_element(f->op_skeleton.header.arg_dtypes[6]); }

/* a workgroup per slice */
static void plan_config(Hip_Launch_Config * c, Score_Plan plan, int n_rows, unsigned lds) {
	set_1d(c, (unsigned) MY_MIN((long) n_rows * plan.slices, (long) SCORE_MAX_GROUPS), (unsigned) (64 * plan.waves), lds);
}

/* workgroups of one of this function's kernels that are resident on the whole
 * device at once; the occupancy query is remembered per kernel for the last
 * (block, LDS) pair asked */
static long resident_groups(Dataflow_Handle * h, Hip_Function * f, unsigned variant, int block, unsigned lds) {
	uint64_t * slot = &f->function_config.occupancy_memo[variant];
	const uint64_t key = ((uint64_t) (unsigned) block << 40) | ((uint64_t) lds << 16);
	const uint64_t memo = __atomic_load_n(slot, __ATOMIC_RELAXED);
	int per_cu = 0;
	if (memo != 0 && (memo & ~0xffffull) == key) per_cu = (int) (memo & 0xffffull);
	else {
		const hipFunction_t fn = f->variant_handles[variant - 1];
		if (!fn || hipModuleOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, fn, block, lds) != hipSuccess || per_cu < 1) per_cu = 1;
		if (per_cu <= 0xffff) __atomic_store_n(slot, key | (uint64_t) per_cu, __ATOMIC_RELAXED);
	}
	return (long) per_cu * (long) ((const Hip_Device_Info *) h->device_info)->cu_count;
}

int token_logprobs_set_launch_config(Hip_Launch_Config * hip_launch_config, Dataflow_Handle * dataflow_handle, Hip_Function * hip_function, Op * op) {
	(void) dataflow_handle;
	const char * what = "token logprobs";
	const int n_rows = ARG(op, 0, int), n_cols = ARG(op, 1, int), tokens_per_row = ARG(op, 4, int), top_k = ARG(op, 5, int);
	const size_t elem = logits_elem(hip_function);
	if (tokens_per_row < 0 || tokens_per_row > SCORE_TOKENS_MAX || top_k < 0 || top_k > SCORE_TOP_MAX) {
		fprintf(stderr, "Error: %s: %d tokens per row (0 to %d) or top_k %d (0 to %d) out of range...\n", what, tokens_per_row, SCORE_TOKENS_MAX,
				top_k, SCORE_TOP_MAX);
		return -1;
	}
	const int checked = score_check(what, n_rows, n_cols, ARG(op, 2, uint64_t), ARG(op, 3, float), ARG(op, 6, void *), elem);
	if (checked < 0) return -1;
	if (checked == 0) {
		set_1d(hip_launch_config, 0, 1, 0);
		return 0;
	}
	if (top_k > n_cols) {
		fprintf(stderr, "Error: %s: top_k %d exceeds the %d columns...\n", what, top_k, n_cols);
		return -1;
	}
	if (tokens_per_row > 0 && (score_pointer(what, "the token pointer", ARG(op, 7, void *), 4) ||
							   score_pointer(what, "the log-probability pointer", ARG(op, 8, void *), 4))) return -1;
	if (ARG(op, 9, void *) && score_pointer(what, "the entropy pointer", ARG(op, 9, void *), 4)) return -1;
	if (ARG(op, 10, void *) && score_pointer(what, "the log-sum-exp pointer", ARG(op, 10, void *), 4)) return -1;
	if (top_k > 0 && (score_pointer(what, "the top id pointer", ARG(op, 11, void *), 4) ||
					  score_pointer(what, "the top log-probability pointer", ARG(op, 12, void *), 4))) return -1;
	if (score_check_workspace(what, score_logprobs_workspace(n_rows, n_cols, (int) elem, top_k), ARG(op, 13, uint64_t), ARG(op, 14, void *))) return -1;
	const Score_Plan plan = score_stream_plan(n_rows, n_cols, (int) elem, top_k);
	plan_config(hip_launch_config, plan, n_rows, top_k > 0 ? score_top_lds(plan.waves) : 0);
	if (top_k > 0) hip_launch_config->variant = HIP_VARIANT_TOP;
	return 0;
}

/* rows of several slices: their join */
int token_logprobs_set_finish_launch_config(Hip_Launch_Config * hip_launch_config, Dataflow_Handle * dataflow_handle, Hip_Function * hip_function, Op * op) {
	(void) dataflow_handle;
	const int n_rows = ARG(op, 0, int), top_k = ARG(op, 5, int);
	const Score_Plan plan = score_stream_plan(n_rows, ARG(op, 1, int), (int) logits_elem(hip_function), top_k);
	set_1d(hip_launch_config, plan.slices > 1 ? (unsigned) n_rows : 0u, SCORE_JOIN_THREADS, (unsigned) (8 * plan.slices * top_k));
	return 0;
}

int token_logprobs_bwd_set_launch_config(Hip_Launch_Config * hip_launch_config, Dataflow_Handle * dataflow_handle, Hip_Function * hip_function, Op * op) {
	(void) dataflow_handle;
	const char * what = "token logprobs bwd";
	const int n_rows = ARG(op, 0, int), n_cols = ARG(op, 1, int), tokens_per_row = ARG(op, 5, int);
	const size_t elem = logits_elem(hip_function);
	if (tokens_per_row < 0 || tokens_per_row > SCORE_TOKENS_MAX) {
		fprintf(stderr, "Error: %s: %d tokens per row (0 to %d) out of range...\n", what, tokens_per_row, SCORE_TOKENS_MAX);
		return -1;
	}
	const int checked = score_check(what, n_rows, n_cols, ARG(op, 2, uint64_t), ARG(op, 4, float), ARG(op, 6, void *), elem);
	if (checked < 0) return -1;
	if (checked == 0) {
		set_1d(hip_launch_config, 0, 1, 0);
		return 0;
	}
	if (tokens_per_row > 0 && (score_pointer(what, "the token pointer", ARG(op, 7, void *), 4) ||
							   score_pointer(what, "the log-probability gradient pointer", ARG(op, 10, void *), 4))) return -1;
	if (score_pointer(what, "the log-sum-exp pointer", ARG(op, 8, void *), 4)) return -1;
	if (ARG(op, 11, void *) && (score_pointer(what, "the entropy gradient pointer", ARG(op, 11, void *), 4) ||
								score_pointer(what, "the entropy pointer", ARG(op, 9, void *), 4))) return -1;
	if (score_check_grad(what, n_rows, n_cols, ARG(op, 2, uint64_t), ARG(op, 3, uint64_t), ARG(op, 6, void *), ARG(op, 12, void *), elem)) return -1;
	plan_config(hip_launch_config, score_map_plan(n_rows, n_cols, (int) elem), n_rows, 0);
	return 0;
}

int distillation_loss_set_launch_config(Hip_Launch_Config * hip_launch_config, Dataflow_Handle * dataflow_handle, Hip_Function * hip_function, Op * op) {
	const char * what = "distillation loss";
	const int n_rows = ARG(op, 0, int), n_cols = ARG(op, 1, int), top_k = ARG(op, 5, int);
	const size_t elem = logits_elem(hip_function);
	if (top_k < 0 || top_k > SCORE_TEACHER_MAX) {
		fprintf(stderr, "Error: %s: top_k %d (0 to %d) out of range...\n", what, top_k, SCORE_TEACHER_MAX);
		return -1;
	}
	const int checked = score_check(what, n_rows, n_cols, ARG(op, 2, uint64_t), ARG(op, 4, float), ARG(op, 6, void *), elem);
	if (checked < 0) return -1;
	if (checked == 0) {
		set_1d(hip_launch_config, 0, 1, 0);
		return 0;
	}
	if (top_k > 0 && (score_pointer(what, "the teacher id pointer", ARG(op, 7, void *), 4) ||
					  score_pointer(what, "the teacher logit pointer", ARG(op, 8, void *), 4))) return -1;
	if (ARG(op, 9, void *) && score_pointer(what, "the row weight pointer", ARG(op, 9, void *), 4)) return -1;
	if (score_pointer(what, "the loss pointer", ARG(op, 10, void *), 4)) return -1;
	if (ARG(op, 11, void *) && score_pointer(what, "the mean loss pointer", ARG(op, 11, void *), 4)) return -1;
	if (ARG(op, 12, void *) && score_check_grad(what, n_rows, n_cols, ARG(op, 2, uint64_t), ARG(op, 3, uint64_t), ARG(op, 6, void *), ARG(op, 12, void *), elem)) return -1;
	if (score_check_workspace(what, score_distill_workspace(n_rows, n_cols, (int) elem, top_k), ARG(op, 13, uint64_t), ARG(op, 14, void *))) return -1;
	const int held = ARG(op, 12, void *) ? score_held(n_rows, n_cols, (int) elem, top_k) : 0;
	if (held) {
		const int waves = score_held_waves(held, n_cols, (int) elem, top_k);
		const unsigned lds = (unsigned) (2 * 8 * score_entries(top_k));
		const unsigned variant = held == SCORE_HELD_ROWS ? HIP_VARIANT_ROWS : held == SCORE_HELD_WIDE_ROWS ? HIP_VARIANT_WIDE_ROWS :
								 held == SCORE_HELD_LONG_ROWS ? HIP_VARIANT_LONG_ROWS : HIP_VARIANT_ANY_ROWS;
		set_1d(hip_launch_config, (unsigned) MY_MIN((long) n_rows, resident_groups(dataflow_handle, hip_function, variant, 64 * waves, lds)), (unsigned) (64 * waves), lds);
		hip_launch_config->variant = variant;
		return 0;
	}
	Score_Plan plan = score_stream_plan(n_rows, n_cols, (int) elem, 0);
	/* rows that are read and written, and too long to be held: as in
	 * score_map_plan (2600 x 200000 bf16 549 -> 519 us) */
	if (plan.slices == 1 && ARG(op, 12, void *)) plan.waves = 2 * SCORE_STREAM_WAVES;
	plan_config(hip_launch_config, plan, n_rows, 0);
	if (plan.slices > 1 || ARG(op, 12, void *)) hip_launch_config->then_variant = HIP_VARIANT_SPLIT_OUT;
	return 0;
}

/* the mean loss: one workgroup, after the rows' losses */
int distillation_loss_set_finish_launch_config(Hip_Launch_Config * hip_launch_config, Dataflow_Handle * dataflow_handle, Hip_Function * hip_function, Op * op) {
	(void) dataflow_handle;
	(void) hip_function;
	set_1d(hip_launch_config, ARG(op, 11, void *) ? 1u : 0u, SCORE_MEAN_THREADS, 0);
	return 0;
}
