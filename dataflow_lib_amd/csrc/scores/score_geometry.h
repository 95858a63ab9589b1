/*
 * Launch rules of the scoring ops, shared by the kernels, the
 * launch-configuration library and the workspace functions (plain C on the
 * host side).
 */
#ifndef SCORE_GEOMETRY_H
#define SCORE_GEOMETRY_H

#ifndef GEOM_FN
#ifdef __HIPCC__
#define GEOM_FN __host__ __device__ static inline
#else
#define GEOM_FN static inline
#endif
#endif

/* limits of the public interface (dataflow_score_ops.h) */
#define SCORE_TOKENS_MAX 1024
#define SCORE_TOP_MAX 256
#define SCORE_TEACHER_MAX 1024
#define SCORE_SCALE_MIN 1e-6f
#define SCORE_SCALE_MAX 1e6f

/* so many workgroups at most, which walk what is left: every launch stays
 * below 2^32 threads */
#define SCORE_MAX_GROUPS (1 << 20)
#define SCORE_MEAN_THREADS 1024

/* Streaming kernels: a row is cut into slices of whole 16-byte chunks (the
 * first one takes the elements before the first chunk too, the last one those
 * behind the last), a workgroup per slice, whose threads take SCORE_BATCH chunks
 * at a time (4096 x 128256 bf16 logprobs 162 us, 8 at a time 167). */
#define SCORE_BATCH 4
#define SCORE_STREAM_WAVES 8
#define SCORE_MAP_BATCH 2
/* few rows: slices until the chip has this many waves (twice as many: 64 x
 * 128256 bf16 18.9 -> 19.5 us), each of at least SCORE_SLICE_BATCH chunks per
 * thread (1 x 128256 14.6 us, of 2 15.3, of 1 17.2). Fewer than SCORE_MIN_SLICES
 * are not worth the second launch that joins them (two for 256 x 151936: 20.4
 * -> 23.9 us). */
#define SCORE_FILL_WAVES 2048
#define SCORE_SLICE_BATCH 4
#define SCORE_MIN_SLICES 3
#define SCORE_MAX_SLICES 32   /* fewer than a wave's lanes, one of which joins each */
#define SCORE_JOIN_THREADS 512

/* how a call's rows are cut */
typedef struct {
	int waves;          /* per workgroup */
	int slices;         /* per row */
	int slice_chunks;   /* per slice; the last may have fewer */
} Score_Plan;

/* waves that a row fills with `batch` chunks per thread, at most max_waves of
 * them to a workgroup; few rows are cut into slices of SCORE_SLICE_BATCH chunks
 * per thread or more until the chip has SCORE_FILL_WAVES waves */
GEOM_FN Score_Plan score_plan(int n_rows, int n_cols, int elem_bytes, int batch, int max_waves) {
	Score_Plan p;
	const long chunks = (long) n_cols * elem_bytes / 16;
	long waves = (chunks + 64 * batch - 1) / (64 * batch);
	if (waves < 1) waves = 1;
	p.waves = (int) (waves < max_waves ? waves : max_waves);
	p.slices = 1;
	const long most = chunks / (64 * SCORE_SLICE_BATCH * max_waves);
	long want = SCORE_FILL_WAVES / ((long) n_rows * p.waves);
	if (want > most) want = most;
	if (want > SCORE_MAX_SLICES) want = SCORE_MAX_SLICES;
	if (want >= SCORE_MIN_SLICES) p.slices = (int) want;
	p.slice_chunks = (int) ((chunks + p.slices - 1) / p.slices);
	if (p.slices > 1) p.slices = (int) ((chunks + p.slice_chunks - 1) / p.slice_chunks);
	return p;
}

/* A wave of a workgroup that finds alternatives keeps so many maxima ("groups")
 * per thread, and takes so many chunks per thread where rows are many. */
#define SCORE_GROUP_SLOTS 4
#define SCORE_TOP_CHUNKS 32
#define SCORE_TOP_WAVES 2
GEOM_FN long score_groups(int waves, long chunks) {
	const long batches = (chunks + 64 * SCORE_BATCH * waves - 1) / (64 * SCORE_BATCH * waves);
	return 64l * waves * (batches < SCORE_GROUP_SLOTS ? batches : SCORE_GROUP_SLOTS);
}

/* token_logprobs and the statistics of distillation_loss.
 * With alternatives, whose second phase is latency, more rows at a time hide
 * more of it: rows in one slice take SCORE_TOP_WAVES waves, or as many more as
 * give a thread no more than SCORE_TOP_CHUNKS chunks and the chip
 * SCORE_FILL_WAVES waves (bf16, 20 alternatives, next to up to 8 waves of
 * SCORE_BATCH chunks: 8192 x 12000 127 -> 58 us, 8192 x 32000 150 -> 119, 8192 x
 * 65000 216 -> 203); and, where there are as many chunks as alternatives, twice
 * as many groups as alternatives (600 x 4096 with 100 95 -> 22 us).
 * Where no alternatives are to be found, rows in one slice that would leave half of the chip's waves
 * free take workgroups of twice as many (256 x 151936 bf16 20.4 -> 18.5 us; with
 * alternatives, 300 x 32000 fp32, 17.6 -> 20.0). */
GEOM_FN Score_Plan score_stream_plan(int n_rows, int n_cols, int elem_bytes, int top_k) {
	Score_Plan p = score_plan(n_rows, n_cols, elem_bytes, SCORE_BATCH, SCORE_STREAM_WAVES);
	if (top_k == 0 && p.slices == 1 && (long) n_rows * SCORE_STREAM_WAVES <= 2 * SCORE_FILL_WAVES && p.slice_chunks >= 64 * 4 * SCORE_STREAM_WAVES)
		p.waves = 2 * SCORE_STREAM_WAVES;
	if (top_k > 0 && p.slices == 1) {
		const long chunks = p.slice_chunks;
		int waves = SCORE_TOP_WAVES;
		while (waves < p.waves && (64l * SCORE_TOP_CHUNKS * waves < chunks || (long) n_rows * waves < SCORE_FILL_WAVES)) waves *= 2;
		if (waves > p.waves) waves = p.waves;
		while (waves < SCORE_STREAM_WAVES && 64 * waves < chunks && chunks >= top_k && (64 * waves < top_k || score_groups(waves, chunks) < 2 * top_k)) waves *= 2;
		p.waves = waves < SCORE_STREAM_WAVES ? waves : SCORE_STREAM_WAVES;
	}
	return p;
}

/* token_logprobs_bwd, which reads and writes a row once. Rows that fill 16 waves
 * with SCORE_BATCH chunks per thread take as many: fewer rows under way at once
 * lie closer together, which reading with writing gains by (2048 x 128256 bf16
 * 204 -> 190 us, 8192 x 16384 fp32 198 -> 187; shorter ones lose, 8192 x 16384
 * bf16 93 -> 115 us, and so does reading alone: token_logprobs 4096 x 128256
 * bf16 162 -> 171 us). */
#define SCORE_MAP_WAVES 8
GEOM_FN Score_Plan score_map_plan(int n_rows, int n_cols, int elem_bytes) {
	Score_Plan p = score_plan(n_rows, n_cols, elem_bytes, SCORE_MAP_BATCH, SCORE_MAP_WAVES);
	if (p.slices == 1 && p.slice_chunks >= 64 * SCORE_BATCH * 2 * SCORE_MAP_WAVES) p.waves = 2 * SCORE_MAP_WAVES;
	return p;
}

/* what a slice of a row leaves in the workspace: its statistics, and its
 * top_k alternatives, largest first */
typedef struct {
	float max, z, e, unused;
} Score_Part;

GEOM_FN unsigned long score_logprobs_workspace(int n_rows, int n_cols, int elem_bytes, int top_k) {
	if (n_rows <= 0 || n_cols <= 0 || elem_bytes <= 0 || top_k < 0) return 0;
	const Score_Plan p = score_stream_plan(n_rows, n_cols, elem_bytes, top_k);
	if (p.slices == 1) return 0;
	return (unsigned long) n_rows * (unsigned long) p.slices * (sizeof(Score_Part) + 8ul * (unsigned long) top_k);
}

/* distillation_loss with a gradient: rows that a workgroup holds in its
 * registers, with a thread per teacher entry.
 * - SCORE_HELD_ROWS: SCORE_HELD chunks per thread in a wave or two, 32 and 16
 *   workgroups to a CU; up to 16 waves where rows are few (256 x 32000 bf16 13.3
 *   us, with fewer waves of more chunks 21.0);
 * - SCORE_HELD_WIDE_ROWS: SCORE_HELD_MORE chunks per thread in up to 8 waves, so
 *   that two rows or more share a CU (8192 x 32000 bf16 205 us; 16 waves of
 *   SCORE_HELD chunks, of which a CU has one workgroup, 365);
 * - SCORE_HELD_LONG_ROWS, SCORE_HELD_MOST_ROWS: 16 waves of SCORE_HELD_MORE chunks,
 *   and of SCORE_HELD_MOST, all that a CU's registers hold (2048 x 151936 bf16
 *   230 us; read twice, 335);
 * - longer rows, and a few of more than 8 waves, are cut into slices and read
 *   twice (40 x 128256 bf16 19.7 us, held 22.9; 100 rows 32.3 and 23.3). */
#define SCORE_HELD 4
#define SCORE_HELD_MORE 16
#define SCORE_HELD_MOST 20
#define SCORE_HELD_FEW 512
#define SCORE_HELD_NONE 0
#define SCORE_HELD_ROWS 1
#define SCORE_HELD_WIDE_ROWS 2
#define SCORE_HELD_LONG_ROWS 3
#define SCORE_HELD_MOST_ROWS 4
GEOM_FN int score_held(int n_rows, int n_cols, int elem_bytes, int top_k) {
	const long chunks = (long) n_cols * elem_bytes / 16;
	if (chunks <= (n_rows <= SCORE_HELD_FEW ? 16 : 2) * 64 * SCORE_HELD) return SCORE_HELD_ROWS;
	if (chunks <= 8 * 64 * SCORE_HELD_MORE && top_k <= 8 * 64) return SCORE_HELD_WIDE_ROWS;
	if (n_rows <= SCORE_HELD_FEW / 8) return SCORE_HELD_NONE;
	if (chunks <= 16 * 64 * SCORE_HELD_MORE) return SCORE_HELD_LONG_ROWS;
	return chunks <= 16 * 64 * SCORE_HELD_MOST ? SCORE_HELD_MOST_ROWS : SCORE_HELD_NONE;
}
GEOM_FN int score_held_waves(int held, int n_cols, int elem_bytes, int top_k) {
	if (held >= SCORE_HELD_LONG_ROWS) return 16;
	const int chunks = (int) ((long) n_cols * elem_bytes / 16), per_wave = 64 * (held == SCORE_HELD_ROWS ? SCORE_HELD : SCORE_HELD_MORE);
	const int waves = (chunks + per_wave - 1) / per_wave, entries = (top_k + 63) / 64;
	return waves > entries ? waves : entries > 0 ? entries : 1;
}
/* LDS: ids (padded to whole 16 bytes) and values of two rows' entries */
GEOM_FN int score_entries(int top_k) { return (top_k + 3) & ~3; }

/* a call may want the loss alone, whatever its sizes */
GEOM_FN unsigned long score_distill_workspace(int n_rows, int n_cols, int elem_bytes, int top_k) {
	if (n_rows <= 0 || n_cols <= 0 || elem_bytes <= 0 || top_k < 0) return 0;
	const Score_Plan p = score_stream_plan(n_rows, n_cols, elem_bytes, 0);
	if (p.slices == 1 && score_held(n_rows, n_cols, elem_bytes, top_k)) return 0;
	return (unsigned long) n_rows * ((unsigned long) p.slices * sizeof(Score_Part) + 4ul * (unsigned long) top_k);
}

/* token_logprobs: LDS of a workgroup with alternatives to find. Candidates,
 * group maxima (SCORE_GROUP_SLOTS per thread) and which of them reach a bound. */
#define SCORE_CANDIDATES 1024   /* all columns of a slice of so many */
GEOM_FN unsigned score_top_lds(int waves) {
	return (unsigned) (waves * 64 * SCORE_GROUP_SLOTS * 6 + SCORE_CANDIDATES * 8);
}

#endif
