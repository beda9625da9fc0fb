/*
 * C-ABI of libwgp_int8.so, the gfx950 (MI355X) INT8 weight linear library.
 *
 * Drop-in for the reference library of the same name: every entry point below has the argument list, argument
 * meaning and return codes of the reference's wgpkernels/int8/int8_gemm.cu (cited as K8:<line>) as bound by its
 * ctypes layer wgpkernels/int8/__init__.py (cited as I:<line>), so that layer loads this library unchanged once
 * "gfx950" is in its HIP_ARCHS (I:47).
 *
 * Conventions (as the reference):
 *  - returns 0 on success, a HIP error code from the launch, or -1 (bad dtype / group / act), -2 (bad shape or
 *    operand combination), -3 (unknown variant), -4 (bad segments), -5 (workspace beyond the allocation-free
 *    entry point's array), -6 (allocation-free entry point first called on a device under graph capture);
 *    calls are asynchronous on `stream`;
 *  - dtype: 0 FP16, 1 BF16, 2 FP32 (activations only); group: 0, 16, 64 or 256 (ConvRot); act: 0 none,
 *    1 RMSNorm, 2 SwiGLU (rows hold [gate | value]), 3 GELU (tanh approximation);
 *  - every buffer belongs to the caller; y may alias residual.
 */
#ifndef WQ8_H
#define WQ8_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* wq8_stream_t; /* hipStream_t */

/* ABI version, 11. Replaces K8:1349; checked at I:69. */
int wq8_abi(void);

/* Feature bits; bit 0: per-(channel, 128-element K block) weight scales. Replaces K8:1352; read at I:71-72. */
int wq8_features(void);

/* Row INT8 of op(x) with optional hi/lo split: hi, lo (m, k) int8, scale (m) f32. Replaces K8:1404; bound at I:74. */
int wq8_quantize(const void* x, int8_t* hi, int8_t* lo, float* scale, int m, int k, int64_t ldx, int dtype, int group, int act,
                 const void* act_weight, float eps, wq8_stream_t stream);

/* Per-128-block INT8 of op(x): q (m, k) int8, scale (m, ceil(k/128)) f32; inv_rms: m floats, required for RMSNorm
 * with k > 16384. Replaces K8:1936; bound at I:75. */
int wq8_quantize_blocks(const void* x, int8_t* q, float* scale, int m, int k, int64_t ldx, int dtype, int group, int act,
                        const void* act_weight, float eps, float* inv_rms, wq8_stream_t stream);

/* wq8_quantize / wq8_quantize_blocks reading input rows first + counter[0] * step (counter: int64 on the GPU).
 * Replace K8:1396 and K8:1926 (not bound by I; called directly by graph-loop callers). */
int wq8_quantize_at(const void* x, int8_t* hi, int8_t* lo, float* scale, int m, int k, int64_t ldx, int dtype, int group, int act,
                    const void* act_weight, float eps, const long long* counter, long long first, long long step, wq8_stream_t stream);
int wq8_quantize_blocks_at(const void* x, int8_t* q, float* scale, int m, int k, int64_t ldx, int dtype, int group, int act,
                           const void* act_weight, float eps, float* inv_rms, const long long* counter, long long first, long long step,
                           wq8_stream_t stream);

/* rotate(op(x)) rounded once to x's dtype: out (m, k), which may be x itself where its rows are k values apart (or, with
 * one row, at the start of x), and overlaps x in no other way. Replaces K8:1971; bound at I:76. */
int wq8_transform_rows(const void* x, void* out, int m, int k, int64_t ldx, int dtype, int group, int act, const void* act_weight,
                       float eps, wq8_stream_t stream);

/* ConvRot rotation only (group 16, 64, 256), rounded once. Replaces K8:1871; bound at I:87. */
int wq8_rotate_groups(const void* x, void* out, int m, int k, int64_t ldx, int dtype, int group, wq8_stream_t stream);

/* Y (m, n) = epilogue(A (m, k) int8 [, A_lo], B (n, k) int8); variant ids keep the reference's modes: 0, 2, 6 row;
 * 1, 7 exact (a_lo required); 10, 11 block (sa (m, ceil(k/128))); 12, 13 block with weight scales sb (n, ceil(k/128));
 * 14 exact with such weight scales. Ids with no counterpart in the reference: 15 the short block tile with 10's biased
 * fold; 16 row, 17 exact, 18 block (biased fold), 19 block and 20 exact with weight scales sb, on tiles for launches of
 * about one tile per compute unit. k % 16 == 0. Replaces K8:1648; bound at I:79. */
int wq8_gemm(const int8_t* a, const int8_t* a_lo, const float* sa, const int8_t* b, const float* sb, const void* bias, const void* residual,
             const void* rscale, void* y, int m, int n, int k, int dtype, int variant, int sms, int split, int* workspace, int* counters,
             wq8_stream_t stream);

/* Workspace bytes {slots, counters} of a wq8_gemm call. Variants 0-15: slots = the block scales transposed (sa of the block
 * modes, sb where it is per k-block), then with split != 0 the split-K partial sums (per split tile, or whole m x n planes
 * per piece for launches of few tiles); counters = one int per tail-split tile (zero on entry, left zero). Variants 16-20
 * read the scales as they are: slots = whole m x n planes per K piece with split != 0 (0 bytes for one piece; two planes
 * a piece for 17), no counters. wq8_gemm returns -2 for a workspace that is not 16-byte aligned. Replaces K8:1506; bound at I:80-81. */
void wq8_gemm_workspace(int m, int n, int k, int variant, int sms, int split, int64_t* sizes);

/* Untuned variant choice for the row (hilo 0) or exact (hilo 1) mode. Replaces K8:1564; bound at I:82. */
int wq8_gemm_select(int m, int n, int k, int hilo, int sms);

/* wq8_gemm writing output / residual rows first + counter[0] * step, residual scales per span of rows, input rows from
 * in_first + counter[0] * in_step. Replaces K8:1637 (not bound by I). */
int wq8_gemm_at(const int8_t* a, const int8_t* a_lo, const float* sa, const int8_t* b, const float* sb, const void* bias, const void* residual,
                const void* rscale, void* y, int m, int n, int k, int dtype, int variant, int sms, int split, int* workspace, int* counters,
                const long long* counter, long long first, long long step, long long span, long long scale_step, long long in_first,
                long long in_step, wq8_stream_t stream);

/* 1 to 4 linears of one prepared input in one launch: ys[s] (m, rows) = A @ (bs[s] * sbs[s]).T + biases[s]; rows % 8 == 0,
 * per-channel scales, whole K whatever split says (size the workspace with split 0).
 * Replaces K8:1663; bound at I:88-89 (hasattr-gated). */
int wq8_gemm_segments(const int8_t* a, const int8_t* a_lo, const float* sa, const int8_t* const* bs, const float* const* sbs,
                      const void* const* biases, void* const* ys, int count, int rows, int m, int k, int dtype, int variant, int sms,
                      int split, int* workspace, int* counters, wq8_stream_t stream);

/* wq8_gemm for callers that cannot allocate (code under graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). No counterpart in the reference. The workspace and split counters wq8_gemm takes from its caller live in
 * a library-owned device array of WQ8_GEMM_NOALLOC_MAX_BYTES per GPU, held until the process ends; a call needing more
 * returns -5. It allocates nothing. Every call on a GPU shares that GPU's array: calls that overlap on one GPU (several
 * streams) race. Results equal wq8_gemm's bit for bit. The array's address is resolved by the first wq8_gemm_workspace
 * query on a device (outside capture); a first call on a device made under graph capture returns -6. */
#define WQ8_GEMM_NOALLOC_MAX_BYTES (32ll << 20)
int wq8_gemm_noalloc(const int8_t* a, const int8_t* a_lo, const float* sa, const int8_t* b, const float* sb, const void* bias,
                     const void* residual, const void* rscale, void* y, int m, int n, int k, int dtype, int variant, int sms, int split,
                     wq8_stream_t stream);

/* Few tokens (m <= 32, k % 64 == 0): unquantized activations, exact INT8 weights on BF16/FP16 matrix cores, split-K
 * with `slots` (f32 partials) sized by wq8_small_workspace; `counters` is accepted and unused (its size is 0). Replace K8:1752 / K8:1693;
 * bound at I:83-85. */
int wq8_small(const void* x, int64_t ldx, const int8_t* w, const float* sw, const void* bias, const void* residual, const void* rscale,
              void* y, int m, int n, int k, int dtype, int sms, float* slots, int* counters, wq8_stream_t stream);
void wq8_small_workspace(int m, int n, int k, int sms, int64_t* sizes);

/* One to four tokens (k % 4 == 0): FP32 GEMV streaming the weights. Replaces K8:1851; bound at I:86. */
int wq8_gemv_lines(const void* x, int64_t ldx, const int8_t* w, const float* sw, const void* bias, const void* residual, const void* rscale,
                   void* y, int m, int n, int k, int dtype, wq8_stream_t stream);

/* One token with its input operation (act 1-3) applied in the same launch: x one row of k values (2 k for SwiGLU), 16-byte
 * aligned, k a multiple of 16 up to 16384, dtype FP16 / BF16; the bits of wq8_transform_rows + wq8_gemv_lines. -2 where y
 * overlaps x (residual may be x). No reference counterpart. */
int wq8_gemv_line_act(const void* x, int act, const void* act_weight, float eps, const int8_t* w, const float* sw, const void* bias,
                      const void* residual, const void* rscale, void* y, int n, int k, int dtype, wq8_stream_t stream);

/* Rotary positions, no counterpart in the reference. count (1 to 4) tensors of rows (tokens, heads, head_dim) of one dtype (0-2), unit
 * channel stride, 16-byte aligned rows: shapes holds per tensor {heads, token stride and head stride of x, of y} in elements (xs, ys
 * and shapes are host arrays); ys[i] may be xs[i]. positions: int32, or int64 with wide, element (token, axis) at token *
 * pos_token + axis * pos_axis. Pair i (of pairs; 2 pairs <= head_dim, a multiple of 8) turns by position * turns[i] / 2^64 turns, position
 * on axis[i] (int32); style 0: channels 2 i, 2 i + 1; 1: i, i + pairs; the others are copied. inverse turns back. */
int wq8_rotary(const void* const* xs, void* const* ys, const long long* shapes, int count, const void* positions, int64_t pos_token, int64_t pos_axis,
               int wide, int64_t tokens, const long long* turns, const void* axis, int pairs, int head_dim, int style, int inverse, int dtype,
               wq8_stream_t stream);

/* The paged 8-bit key/value cache, no counterpart in the reference: codes (pages, heads, block, head_dim) int8, scales (pages, heads) f32.
 * kv_plan: past, fresh (requests) and pages (pages_count), used (1) int32; tables rows of `width` int32, table_stride apart, completed in
 * place; slots and positions (tokens), starts (requests + 1), lens (requests), used_out and missing (1) are written. */
int wq8_kv_plan(const void* past, const void* fresh, int32_t* tables, int64_t table_stride, const void* pages, int pages_count, const void* used,
                int requests, int width, int block, int64_t tokens, int64_t* slots, int32_t* positions, int32_t* starts, int32_t* lens, int32_t* used_out,
                int32_t* missing, wq8_stream_t stream);

/* Rows (tokens, heads, head_dim) of dtype 0-2 into the cache at slots; strides (host): {token, head} of k, of v, in elements; rows 16-byte
 * aligned; block a power of two up to 128, head_dim a multiple of 8 up to 1024; owner: pages * block int32 of scratch, never cleared. */
int wq8_kv_write(const void* k, const void* v, const long long* strides, const long long* slots, int64_t tokens, int8_t* k_codes, float* k_scales,
                 int8_t* v_codes, float* v_scales, int64_t pages, int heads, int block, int head_dim, int dtype, int32_t* owner, wq8_stream_t stream);

/* The values at slots: k, v (tokens, heads, head_dim) contiguous, of dtype 0-2; zeros for slots outside the cache. */
int wq8_kv_read(const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, const long long* slots, int64_t tokens, void* k,
                void* v, int64_t pages, int heads, int block, int head_dim, int dtype, wq8_stream_t stream);

/* Attention of q (tokens, heads * group, head_dim), dtype 0-1, over the cache: request r has rows starts[r] to starts[r + 1] and the
 * first lens[r] tokens of its row of tables (int32; width entries, table_stride apart); strides (host): {token, head} of q, of out;
 * head_dim 64, 128 or 256; block 16, 32, 64 or 128; workspace: of the bytes that the query
 * gives (sizes[0]; sizes[1] is 0), 16-byte aligned. */
int wq8_kv_attention(const void* q, void* out, const long long* strides, const int8_t* k_codes, const float* k_scales, const int8_t* v_codes,
                     const float* v_scales, const void* tables, int64_t table_stride, int width, const void* lens, const void* starts, int tokens,
                     int requests, int heads, int group, int head_dim, int block, int64_t pages, float scale, int causal, int window, int dtype, int sms,
                     void* workspace, wq8_stream_t stream);
void wq8_kv_attention_workspace(int tokens, int requests, int heads, int group, int head_dim, int sms, int64_t* sizes);

/* Cold-cache timing: reads `bytes` of a library-owned buffer on `stream` (nonzero if it cannot be allocated);
 * release frees it. Replace K8:1997-2016; bound at I:77-78. */
int wq8_l2_flush(int device, int64_t bytes, wq8_stream_t stream);
void wq8_l2_flush_release(void);

#ifdef __cplusplus
}
#endif
#endif
