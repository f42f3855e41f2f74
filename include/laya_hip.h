/*
 * liblaya_hip: C ABI of the MI355X (gfx950) encoder forward path.
 *
 * This is the drop-in boundary under laya-cuda's Python runtime.  The reference's Runtime
 * (laya_cuda/runtime.py:136-197) owns a CuPy memory pool, one stream, the resident weights and an
 * LRU of shape slots, each with a CUDA graph; Ops (laya_cuda/ops.py:19-71) owns NVRTC kernels and
 * cuBLAS.  Here one opaque engine handle owns all of that natively: an HBM arena per slot, one
 * non-blocking HIP stream, resident weights, and one hipGraph per shape slot.
 *
 * Conventions: every entry point returns 0 (LAYA_OK) or a LAYA_E* status; the message of the
 * last failure is laya_last_error(handle) (handle may be NULL for failures that have none).
 * Pointers named host_* are host memory; every other buffer pointer of the laya_op_* entry
 * points is device memory.  `stream` is a hipStream_t (NULL = the null stream).  A handle is
 * single-threaded: callers serialise access (as the reference's Engine and BatchEngine do).
 */
#ifndef LAYA_HIP_H
#define LAYA_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LAYA_ABI_VERSION 2

enum {
  LAYA_OK = 0,
  LAYA_EINVAL = 1,   /* bad argument, name, shape or configuration */
  LAYA_EDEVICE = 2,  /* HIP runtime failure */
  LAYA_ENOMEM = 3,   /* device or pinned allocation failed */
  LAYA_ESTATE = 4    /* call out of order (e.g. predict before finalize) */
};

/* Element types of host weights and of the 16-bit MFMA operand type. */
enum { LAYA_F32 = 0, LAYA_F16 = 1, LAYA_BF16 = 2 };
/* Output type of the 8-bit operators below (codes with scales; no host weights of this type). */
enum { LAYA_E4M3 = 3 };

/* Encoder variants (the reference's executor is pre-LN/RoPE/GeGLU, laya_cuda/laya.py:59-79). */
enum { LAYA_NORM_POST = 0, LAYA_NORM_PRE = 1 };
enum { LAYA_POS_LEARNED = 0, LAYA_POS_ROPE = 1 };
enum { LAYA_FFN_GELU = 0, LAYA_FFN_GEGLU = 1 };

/* Model configuration: the fields the reference's adapter exposes to Runtime
 * (width, heads, layers, intermediate, eps, max_len, n_act, ...; laya_cuda/laya.py:61-81). */
typedef struct LayaConfig {
  int32_t width;          /* d_model; heads * 64 */
  int32_t heads;
  int32_t layers;
  int32_t intermediate;   /* FFN width f */
  int32_t vocab;
  int32_t max_positions;  /* learned position rows */
  int32_t type_vocab;     /* token-type rows (row 0 is added) */
  int32_t norm_order;     /* LAYA_NORM_* */
  int32_t pos_kind;       /* LAYA_POS_* */
  int32_t ffn_kind;       /* LAYA_FFN_* */
  int32_t bias;           /* encoder linear layers carry biases */
  float eps;              /* encoder LayerNorm epsilon */
  int32_t window;         /* local attention half-window, -1 = global */
  int32_t global_every;
  int32_t head_layers;    /* decision-head transformer layers */
  int32_t n_act;          /* act-head outputs */
  int32_t act_hidden;     /* act-head hidden width (256 in Laya) */
  int32_t max_len;        /* longest sequence, tokens */
  int32_t mfma_dtype;     /* LAYA_BF16 or LAYA_F16: resident matrices and MFMA operands */
  float theta_global;     /* RoPE theta of global layers (LAYA_POS_ROPE; laya.py:72-78) */
  float theta_local;      /* RoPE theta of local (windowed) layers */
} LayaConfig;

/* Shape class of one predict: the reference's slot key (laya_cuda/runtime.py:20-25). */
typedef struct LayaShape {
  int32_t rows;     /* packed token rows m (multiple of 16) */
  int32_t batch;    /* question capacity b (also the sequence capacity) */
  int32_t options;  /* option capacity k per question */
} LayaShape;

typedef struct LayaMetrics {
  float gpu_ms;            /* stream time of the forward (graph replay or eager), events */
  int32_t cache_miss;      /* the slot was created by this call */
  int32_t graph_capture;   /* the slot's graph was captured by this call */
  int32_t graph_replay;    /* the forward ran as a graph replay */
  int64_t owned_gpu_bytes; /* weights + slot arenas */
} LayaMetrics;

/*
 * Packed int32 input block of a predict, laid out for shape (m, b, k):
 *   meta[4]          n_seq, n_questions, 0, 0
 *   ids[m] positions[m] rows[m] kinds[m]            per packed token (runtime.py:35-36)
 *   starts[b] lengths[b]                            per sequence
 *   counts[b] qkind[b]                              per question
 *   indices[b*(k+1)]                                per question: CLS row, then option rows,
 *                                                   absolute packed rows (runtime.py:63-66)
 * laya_packed_ints(shape) gives its length.  Sequences start at multiples of 16 rows; rows of
 * no sequence carry rows[i] = -1.
 */
int64_t laya_packed_ints(const LayaShape* shape);

/* One HIP device as the doctor reports it (laya_cuda/cli.py:118-176 reports CUDA devices through
 * CuPy; here the library itself answers, from hipGetDeviceProperties and hipMemGetInfo). */
typedef struct LayaDevice {
  char name[256];
  char arch[64];            /* gcnArchName, e.g. "gfx950:sramecc+:xnack-" */
  int64_t hbm_bytes;        /* total device memory */
  int64_t free_bytes;       /* free device memory now */
  int32_t compute_units;
  int32_t lds_bytes_per_cu;
  int32_t clock_khz;
  int32_t supported;        /* 1: gfx950, the architecture this library is built for */
} LayaDevice;

/* Number of HIP devices (0 without a driver or device: not an error); the doctor's
 * getDeviceCount (cli.py:140-141). */
int laya_device_count(int* count);
/* Properties of HIP device `device`; the doctor's getDeviceProperties (cli.py:142-147). */
int laya_device_info(int device, LayaDevice* out);

/* Runtime(adapter, device, max_cached_shapes) construction (runtime.py:137-146). */
int laya_create(const LayaConfig* cfg, int device, int max_slots, void** handle);

/* Upload one named checkpoint tensor (runtime.py:147-158): the name set and shapes are those of
 * the adapter's weight_shapes(); matrices feeding MFMA become resident in cfg->mfma_dtype, all
 * other tensors in fp32.  host_dtype is LAYA_F32/F16/BF16, shape has ndim entries. */
int laya_load_weight(void* handle, const char* name, const void* host_data, int host_dtype,
                     const int64_t* shape, int ndim);

/* Checks that every tensor is present (the name-set check of runtime.py:149-151) and resolves the
 * layer tables.  Required before predict. */
int laya_finalize(void* handle);

/* Runtime.predict / Slot.run (runtime.py:115-133, 171-186): find or create the shape slot (LRU
 * eviction at max_slots), upload the packed block, capture the slot's graph on first use when
 * capture != 0, replay (or run eagerly), and copy back host_logits [b][k] (option slots 1..k,
 * laya.py:208) and host_acts [b][n_act]. */
int laya_predict(void* handle, const int32_t* host_packed, const LayaShape* shape, int capture,
                 float* host_logits, float* host_acts, LayaMetrics* metrics);

/* No counterpart in the reference.  For callers that cannot allocate device or pinned memory
 * (tight serving loops, harnesses that forbid hipMalloc): the forward of laya_predict without a
 * shape slot.  Its arena (packed block, activations, split-K partials, head buffers) lives in a
 * fixed 64 MiB device array that every device running the library holds for the life of the
 * process; the packed block is staged through a fixed host array of 2^18 int32.  A shape class
 * whose arena or block does not fit is refused with LAYA_EINVAL (12L/768 requests of up to 1,024
 * packed rows fit).  The forward runs eagerly on the engine's stream (no graph), outputs and
 * metrics as laya_predict (cache_miss, graph_capture and graph_replay are 0).  The call makes no
 * allocation.  Calls share each device's array and the host staging: the library serialises them
 * with a process-wide lock, held until the outputs are on the host; calls that overlapped would
 * race on the array, and each call overwrites what the previous one left there. */
int laya_predict_static(void* handle, const int32_t* host_packed, const LayaShape* shape, float* host_logits,
                        float* host_acts, LayaMetrics* metrics);

/* Per-launch timing, the native counterpart of the reference's profiling hook that records events
 * around every Ops.call/linear (tools/profile_long.py:21-67).  The forward is a fixed list of
 * stages (embed_norm; per layer qkv, attention, attn_out, attn_norm, ffn_up, ffn_down, ffn_norm;
 * head_gather, head_scorer, head_tail).  laya_time_stage uploads the request like
 * laya_predict, runs one eager forward so every buffer holds this request's values, then launches
 * stage `stage` of layer `layer` `reps` times back to back between two events on the engine's
 * stream and stores the average per launch in *avg_ms.  Stages that normalise in place
 * (attn_norm, ffn_norm) change the residual on every repetition: time them, do not read results
 * afterwards.  layer = -1 times the stage where it runs: `reps` (at most 1000) eager forwards,
 * queued back to back, in which every kernel of the stage (all its layers) records the start and
 * end of its own execution (hipExtLaunchKernel events, the interval a kernel trace reports);
 * *avg_ms is their average. */
int laya_stage_count(void);
const char* laya_stage_name(int stage);
/* How many times this engine's forward launches `stage` (0: not part of this model) and the first
 * layer index it runs for, the `layer` argument of laya_time_stage.  Per-launch times times these
 * counts give the per-forward breakdown of tools/profile_long.py:21-67. */
int laya_stage_launches(void* handle, int stage, int* launches, int* first_layer);
int laya_time_stage(void* handle, const int32_t* host_packed, const LayaShape* shape, int stage, int layer,
                    int reps, float* avg_ms);

/* Read a resident tensor back as fp32 (runtime.weights[name], tests/test_custom_models.py:46). */
int laya_read_weight(void* handle, const char* name, float* host_out, int64_t count);
int64_t laya_used_bytes(void* handle);   /* weights + slots: CuPy pool used_bytes() */
int laya_slot_count(void* handle);       /* len(runtime.slots) */
int laya_destroy(void* handle);          /* Runtime.close (runtime.py:188-197) */
const char* laya_last_error(void* handle);  /* the exception text of ops.py:45-48, runtime.py:149-153 */
/* No counterpart in the reference: the version of the struct layouts above, which a binding
 * compares with the one it mirrors before it binds anything else. */
int laya_abi_version(void);

/* ------------------------------------------------------------------------------------------
 * Kernel-level entry points: the Ops surface the reference's kernel tests drive
 * (laya_cuda/ops.py:50-66; tests/test_gpu.py, tests/test_attention.py).
 * ------------------------------------------------------------------------------------------ */

/* Attention work list for packed sequences (Slot.attend's ragged rows, runtime.py:82-88): tiles of
 * up to `block` query rows of one sequence plus zero-tiles for rows of no sequence, as int32 quads
 * (row0, row1, kstart, klen) with klen = -1 for zero-tiles; all max_tiles quads are written (unused
 * ones as empty ranges).  Returns the used count, or -1 for a bad layout or too small a list.
 * Host-only. */
int laya_attention_tiles(const int32_t* starts, const int32_t* lengths, int n_seq, int m, int block,
                         int32_t* tiles, int max_tiles);
/* Query rows per tile of an attention kernel: mode 0 (K/V blocks staged once in LDS and shared by
 * `waves` = 1, 2, 4 or 8 waves of 32 queries each; large batches) -> 32*waves; mode 1 (one tile of
 * 32 queries whose keys are split across `waves` = 2, 4 or 8 waves; batch-1 latency) -> 32; mode 2
 * (64 queries as two 32-query groups sharing each of waves/2 key groups' blocks, waves = 4 or 8;
 * long batch-1 sequences) -> 64.  -1 for an invalid pair. */
int laya_attention_block(int mode, int waves);

/* embed (kernels.cu:16-19) fused with the embeddings norm (runtime.py:93-95):
 * v = table[ids] (+ pos_table[positions]) (+ type_row); LayerNorm if gamma; writes out32 and/or
 * out16 (dtype16 = LAYA_BF16/F16). */
int laya_op_embed(const int32_t* ids, const int32_t* positions, const float* table,
                  const float* pos_table, const float* type_row, const float* gamma,
                  const float* beta, float eps, float* out32, void* out16, int dtype16, int rows,
                  int width, int vocab, int n_positions, void* stream);

/* layer_norm (kernels.cu:20-49): v = residual + (sum of `splits` branch partials + bias);
 * sum_out = v; LayerNorm if gamma; out32/out16 = result.  out32 may alias residual. */
int laya_op_norm(float* residual, const float* branch, int splits, int64_t part_stride,
                 const float* bias, const float* gamma, const float* beta, float eps,
                 float* sum_out, float* out32, void* out16, int dtype16, int rows, int width,
                 void* stream);

/* Ops.linear (ops.py:58-66) with the activate modes (kernels.cu:59-67) as epilogues:
 * out[M][N] = x[M][K] w[N][K]^T (+ bias).  kind 0: fp32 out (split-K partials at out + z*M*N when
 * splits > 1, bias then must be NULL), 1: 16-bit out, 2: 16-bit exact-GELU out, 3: 16-bit ReLU out,
 * 4: GeGLU, out[M][N/2] = gelu(gate) * value with w's rows in the resident GeGLU interleave
 * (32-row groups: 16 gate rows, then their 16 value rows).  tile -1 lets the planner choose tile
 * and splits (splits ignored): for 16-bit outputs by its cost model, for fp32 by the measured plan
 * table when it holds the problem, else the heuristic; tile -2 takes the heuristic alone.  A planned
 * fp32 product without bias writes as many partials as the plan splits K: out must hold that many
 * times M*N floats.  laya_op_plan tells the number beforehand (at most 8). */
int laya_op_linear(const void* x, const void* w, const float* bias, void* out, int kind,
                   int dtype16, int M, int N, int K, int splits, int tile, void* stream);

/* The launch that tile -1 (or -2) stands for: *planned_tile and *planned_splits for laya_op_linear of
 * this kind (biased: with a bias), or for laya_op_qkv with N = 3 width, K = width (kind 5; 6 with RoPE); with
 * tile -3 the launch that a laya_predict slot of M rows takes.  Host arithmetic only: needs no device. */
int laya_op_plan(int kind, int dtype16, int M, int N, int K, int biased, int tile, int* planned_tile,
                 int* planned_splits);

/* QKV projection with the head-major epilogue that replaces `layout` (kernels.cu:68-82):
 * q, k [heads][M][64], vt [heads][64][M].  With rope_cos non-NULL, Q and K are rotated (rotate-half
 * RoPE, kernels.cu:73-77) in fp32 before rounding, by the [positions][32] cos/sin tables at each
 * row's positions[row].  M must be a multiple of 8.  tile -1 / -2 as for laya_op_linear. */
int laya_op_qkv(const void* x, const void* w, const float* bias, void* q, void* k, void* vt,
                const float* rope_cos, const float* rope_sin, const int32_t* positions, int dtype16,
                int M, int width, int tile, void* stream);

/* attention (kernels.cu:90-154) over a device copy (16-byte aligned) of a tile list from
 * laya_attention_tiles built with laya_attention_block(mode, waves) rows per tile; q, k [heads][m][64],
 * vt [heads][64][m], out [m][heads*64]; window >= 0 keeps only keys with |query - key| <= window (the
 * local layers, kernels.cu:106-107), window < 0 is global attention. */
int laya_op_attention(const void* q, const void* k, const void* vt, void* out, const int32_t* tiles,
                      int m, int heads, int max_tiles, int mode, int waves, int window, int dtype16,
                      void* stream);

/* gather / gather_half (kernels.cu:159-166), the option-position row gather of the decision head
 * (laya.py:226-227, 237): for r < *n_live, dst32[r] = src32[indices[r]] and dst16[r] =
 * src16[indices[r]] (16-bit rows of dtype16), bit-exact copies in the order of `indices`
 * (duplicates allowed); rows n_live..rows-1 are written as zeros.  n_live is a device int32 (the
 * forward reads the live row count on the device); either src/dst pair may be NULL to skip it. */
int laya_op_gather_rows(const float* src32, float* dst32, const void* src16, void* dst16, int dtype16,
                        const int32_t* indices, const int32_t* n_live, int rows, int width, void* stream);

/* The scorer input rows (type_add + gather, kernels.cu:155-162; laya.py:236-238): for r < *n_live,
 * selected[r] = src[src_rows[r]] + type_rows[question_kind[row_question[r]]] (the type row only
 * when type_rows is non-NULL; one fp32 add, bit-exact), and normed[r] = LayerNorm(selected[r];
 * gamma, beta, eps) (scorer.0).  All pointers are device memory; n_live a device int32. */
int laya_op_head_gather(const float* src, const int32_t* src_rows, const int32_t* row_question,
                        const int32_t* question_kind, const int32_t* n_live, const float* type_rows,
                        const float* gamma, const float* beta, float eps, float* selected, float* normed,
                        int rows, int width, void* stream);

/* ------------------------------------------------------------------------------------------
 * 8-bit rows and the operators on them (no counterpart in the reference, whose operands are 16-bit).
 *
 * A matrix of `rows` x `width` values in 8-bit rows is two device arrays, rows back to back:
 *   codes  [rows][laya_width8(width)]       e4m3 (OCP, no infinities), 16-byte aligned
 *   scales [rows][laya_width8(width) / 32]  uint8, 4-byte aligned
 * laya_width8 rounds the width up to a multiple of 128; the codes past the width are zeros (NaN codes where
 * a block, or for laya_op_linear8 a row, holds a NaN).  Code i of a row stands for
 * e4m3(code) * 2^(scale[i / 32] - 127).  A writer takes the smallest scale with which the block's largest
 * magnitude is at most 448 (2^-127 at the least; 0 for a block of zeros) and rounds each value once, to nearest
 * with ties to even; finite values stay finite (what would round to 2^128 goes to 240 * 2^120).  A block that holds
 * a NaN or an infinity gets the scale 255 and reads back as NaNs.  Codes that no writer makes, of 2^128 or more (scales
 * 247 to 254), read back as infinities, and exact products take them as such.
 *
 * Every operator runs on the current device, which owns the pointers and the stream; it makes no allocation, no
 * host synchronisation and keeps nothing between calls, so calls may be captured, replayed and run side by side.
 * An output overlaps no input and no other output unless its operator says so.  Zero rows are a call that does
 * nothing.  Bad sizes, types, missing or misaligned pointers: LAYA_EINVAL.
 * ------------------------------------------------------------------------------------------ */

enum { LAYA_LAYER_NORM = 0, LAYA_RMS_NORM = 1 };
enum { LAYA_ACT_NONE = 0, LAYA_ACT_GELU = 1, LAYA_ACT_RELU = 2, LAYA_ACT_GEGLU = 3, LAYA_ACT_SWIGLU = 4 };
enum { LAYA_TILE_EXACT = -1, LAYA_TILE_FAST = -2 };  /* planned tiles of laya_op_linear8 */

/* Codes per 8-bit row of `width` values; -1 for a width below 1 or above 2^30.  Host-only. */
int laya_width8(int width);

/* 8-bit rows of x (LAYA_F32/F16/BF16), whose rows of `width` values start `stride` elements apart (stride >=
 * width): weights once at load, or activations.  x needs its own element's alignment only; rows that start
 * and end on whole 16 bytes are read fastest.  At most 2^36 - 4096 codes, from values that span at
 * most 2^50 elements. */
int laya_op_quantize8(const void* x, int dtype, int64_t stride, void* codes, void* scales, int64_t rows, int width,
                      void* stream);

/* The values 8-bit rows stand for, as dtype with rows `stride` elements apart; what lies between the rows is left as it
 * was.  Exact in LAYA_F32, and in LAYA_BF16 but for blocks of scales below 2^-117; LAYA_F16 rounds once
 * (infinity past its range).  Extents as laya_op_quantize8's. */
int laya_op_dequantize8(const void* codes, const void* scales, void* out, int dtype, int64_t stride, int64_t rows,
                        int width, void* stream);

/* laya_op_norm with 8-bit output: v = residual + (sum of `splits` branch partials + bias); sum_out = v; then
 *   kind LAYA_LAYER_NORM  y = (v - mean(v)) / sqrt(var(v) + eps) * gamma + beta
 *   kind LAYA_RMS_NORM    y = v / sqrt(mean(v^2) + eps) * gamma + beta
 * in fp32, out32 = y, and codes, scales = the 8-bit rows of y.  branch (partials part_stride elements apart) is of
 * branch_dtype LAYA_F32/F16/BF16, or NULL (v = residual; bias must be NULL).  beta, bias, sum_out and
 * out32 may be NULL; either one of sum_out and out32 may be residual itself.  1 <= width <= 8192; fewer than 2^26 rows,
 * 2^24 of widths above 2048. */
int laya_op_norm8(const float* residual, const void* branch, int branch_dtype, int splits, int64_t part_stride,
                  const float* bias, const float* gamma, const float* beta, float eps, int kind, float* sum_out,
                  float* out32, void* codes, void* scales, int rows, int width, void* stream);

/* out = act(x w^T + bias) + residual: x [M][K] and w [N][K] in 8-bit rows, bias fp32 [N] or NULL, residual
 * [M][cols] of residual_dtype LAYA_F32/F16/BF16 or NULL, out [M][cols] of out_dtype LAYA_F32/F16/BF16, or 8-bit rows
 * (LAYA_E4M3: out takes the codes, out_scales the scales; out_scales is NULL otherwise).  cols is N, or N / 2
 * for the gated activations, whose w (and bias) come in groups of 32 rows: 16 gate rows, then their 16 value rows
 * (act(gate) * value; N a multiple of 32).  GELU is the exact-erf one, SWIGLU's gate x / (1 + exp(-x)).  The residual
 * is added in fp32 before the one rounding; it may be out itself when both have the same type (with another
 * it is refused), and nothing else may overlap out.
 * tile says how the sums are made:
 *   LAYA_TILE_EXACT  exact products (of values of at least 2^-126, smaller ones count as zero) and fp32 sums, whatever the
 *                    output's type; the planner chooses the tile, and with it the order of a sum.
 *   LAYA_TILE_FAST   16- and 8-bit outputs may take the 8-bit matrix unit, at up to twice the rate.  It cuts the products
 *                    of each group of 8 neighbours off, towards zero, 2^13 below the largest sum of two codes' exponents: a
 *                    sum loses up to 2^-10 of its products' magnitudes (2^-7 where the largest have a subnormal code),
 *                    one-sidedly where they have one sign.
 *   0 .. 14          that tile, refused where it cannot make the output; 5, 7 to 10 and 13 are of the 8-bit unit.
 * Activations are accurate to 1e-6 of the larger of 1 and their magnitude, a gated one's times its value. */
int laya_op_linear8(const void* x, const void* x_scales, const void* w, const void* w_scales, const float* bias,
                    const void* residual, int residual_dtype, void* out, void* out_scales, int out_dtype,
                    int activation, int M, int N, int K, int tile, void* stream);

/* ------------------------------------------------------------------------------------------
 * Rotary positions, and attention over packed sequences with masks, capped scores and distance biases (no counterpart in
 * the reference, whose rotation is part of its layout kernel and whose attention is bidirectional or windowed, of heads of 64).
 *
 * As above: the current device owns the pointers and the stream, no allocation, no host synchronisation, nothing kept
 * between calls, LAYA_EINVAL for bad arguments.  Rows of heads lie `row` elements apart and a row's heads `head` elements
 * apart, so that a projection's packed rows, caches and head-major planes are read and written where they are.
 * ------------------------------------------------------------------------------------------ */

enum { LAYA_ROTARY_HALF = 0, LAYA_ROTARY_INTERLEAVED = 1 };  /* pairs (i, i + rotated / 2), or (2 i, 2 i + 1) */
enum {
  LAYA_FREQ_PLAIN = 0,   /* theta^(-2 i / rotated) radians a position */
  LAYA_FREQ_LINEAR = 1,  /* that over factor: positions are squeezed */
  LAYA_FREQ_BASE = 2,    /* theta times factor^(rotated / (rotated - 2)) (times factor for rotated 2): the slowest pair
                            slows down by factor, the fastest stays */
  LAYA_FREQ_PARTS = 3    /* by the turns n that a pair makes over `original` positions: kept where n >= high, over factor
                            where n <= low, and between them mixed in proportion */
};

/* Frequencies of the rotated / 2 pairs in turns (2 pi) a position, 64 bits, for laya_op_rotary (copied to the device by the
 * caller).  original, low and high belong to LAYA_FREQ_PARTS.  theta > 0, factor >= 1, rotated even and from 2 to 8192,
 * original > 0, 0 <= low < high.  Host-only. */
int laya_rotary_frequencies(int kind, double theta, int rotated, double factor, double original, double low,
                            double high, double* host_turns);

/* out = x with each head's first `rotated` values turned by their row's position: with the angle 2 pi positions[row] turns[i]
 * of pair i, (a, b) -> amplitude (a cos - b sin, a sin + b cos); direction -1 turns back (the gradient of direction 1, and
 * its inverse where amplitude is 1).  Values rotated .. dim - 1 are copied.  dtype LAYA_F32/F16/BF16; positions
 * int32, of either sign; turns as laya_rotary_frequencies makes them.  Angles are exact to 2^-27 of a turn at any position (turns up to
 * 2^20 in size), arithmetic is fp32, and the output rounds once.  out may be x itself with the same strides, else it overlaps nothing;
 * what lies between rows and heads is left as it was.  rotated even, 2 <= rotated <= dim <= 8192, heads * dim <= 2^20, rows <= 2^23,
 * strides not negative and below 2^40, over at most 2^50 elements.  Whole 16 bytes of halves, strides and addresses are fastest. */
int laya_op_rotary(const void* x, int64_t x_row, int64_t x_head, void* out, int64_t out_row, int64_t out_head,
                   int dtype, const int32_t* positions, const double* turns, float amplitude, int layout,
                   int direction, int64_t rows, int heads, int dim, int rotated, void* stream);

/* Kernels of laya_op_attend: the planner's choice; a workgroup for 128 queries of a head (256 of heads above 128 and, of those above
 * 64, in long prompts), for many rows; a workgroup or, over long keys, several for 32 rows, for few. */
enum { LAYA_ATTEND_PLANNED = 0, LAYA_ATTEND_MANY = 1, LAYA_ATTEND_FEW = 2 };

/* Ranges of a document mask: bounds[row] = (first, end) of the run of equal neighbouring ids that holds the row, counted from
 * its sequence's start.  documents [rows], bounds [rows][2], starts and lengths [n_seq] are device memory; a
 * sequence's rows are starts[s] .. starts[s] + lengths[s] - 1, cut to the array and to max_length; rows of no sequence are left
 * as they were.  Sequences must not share rows.  Work is linear in the rows; max_length above 4,096 takes three launches for one.  One
 * call serves every layer and head of a batch. */
int laya_op_document_bounds(const int32_t* documents, const int32_t* starts, const int32_t* lengths, int n_seq,
                            int64_t rows, int max_length, int32_t* bounds, void* stream);

/* A call of laya_op_attend.  Sequence s has the queries of rows q_starts[s] .. + q_lengths[s] - 1 of q and the keys and values of
 * rows k_starts[s] .. + k_lengths[s] - 1 of k and v (device arrays, cut to the row counts and to max_q and max_k); its query i
 * stands at position p = i + k_lengths[s] - q_lengths[s].  Query head h reads key head h / (heads / kv_heads).  The query sees key j if
 *   j < prefix[s], or  bounds[row][0] <= j < bounds[row][1]  and  p - before <= j <= p + after
 * (prefix and bounds may be NULL: no prefix, no bounds; row counts q's rows; -1: no limit).  before = -1, after = 0 is causal, a prefix beside
 * it a prefix mask, bounds of laya_op_document_bounds a document mask.  Then
 *   t = scale q . k;  t = cap tanh(t / cap) if cap > 0;  t -= slopes[h] |j - p|  or  t += table[h][clamp(j - p, -span, span) + span];
 *   out = sum of softmax(t) v over the keys seen.
 * A query that sees no key, or whose scores are all below -1e30 (biases of a type's lowest value hide keys), gets zeros; what lies in
 * hidden keys, NaNs and infinities too, does not matter.  Other entries of a table are at most 1e27
 * in size.  out's rows of no query are left as they were.  Sequences may share keys, not queries. */
typedef struct LayaAttend {
  uint32_t struct_bytes;  /* sizeof(LayaAttend) */
  int32_t dtype;          /* LAYA_F16 or LAYA_BF16: q, k, v, out */
  const void* q;          /* [q_rows][heads][dim] */
  const void* k;          /* [k_rows][kv_heads][dim] */
  const void* v;          /* [k_rows][kv_heads][dim] */
  void* out;              /* [q_rows][heads][dim]; overlaps nothing */
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  /* strides in elements */
  int32_t heads, kv_heads, dim;
  int32_t q_rows, k_rows;
  int32_t n_seq, max_q, max_k;  /* sequences, and the most queries and keys that one has */
  const int32_t* q_starts;
  const int32_t* q_lengths;
  const int32_t* k_starts;
  const int32_t* k_lengths;
  float scale, cap;       /* cap 0: none */
  const float* slopes;    /* [heads], or NULL */
  const float* table;     /* [heads][2 span + 1], or NULL; not both */
  int32_t span;
  int32_t before, after;
  int32_t kernel;         /* a LAYA_ATTEND_* value */
  const int32_t* prefix;  /* [n_seq], or NULL */
  const int32_t* bounds;  /* [q_rows][2], or NULL */
} LayaAttend;

/* Bytes of workspace that laya_op_attend needs for this call: 0 unless long keys of few queries are shared by several
 * workgroups.  Depends on the sizes, before, after, kernel and whether there is a prefix, on no other pointer; -1 for sizes that are refused.  Host-only. */
int64_t laya_attend_workspace(const LayaAttend* call);

/* The attention described above, sums and softmax in fp32, weights rounded to dtype for the matrix unit, one rounding of the
 * output.  Lengths of zero are fine.  dim a multiple of 8 up to 256, heads a multiple of kv_heads; q, k, v and out and
 * their strides on whole 16 bytes, row strides of k and v at least dim and below 2^23; scale from 1e-10 to 1e10; cap 0 or
 * 1e-10 to 1024 (a capped score is exact to 2^-20 of the cap: from 512 on half a step of an fp16 weight and more); span 0 to
 * 1024 with a table; rows, max_q, max_k, before and after below 2^30, heads at most 2^16, and n_seq * heads * max_q, max_q counted as whole 128 (256 for heads above 64), at most about
 * 2^31 (one launch; the kernel for few rows, where it is named, takes about 2^28).  workspace: device memory, 16-byte aligned,
 * of the bytes that laya_attend_workspace tells (NULL for 0), written before it is read; calls that may run at the same time,
 * captured ones too, take different ones.  Equal calls give equal bits. */
int laya_op_attend(const LayaAttend* call, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LAYA_HIP_H */
