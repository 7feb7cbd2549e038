/* libsslm_b200 -- the C ABI of the B200 (sm_100a) implementation of SuperSLM's
 * integer-only transformer forward pass.
 *
 * The first block re-declares, name for name and argument for argument, the verbs of the
 * reference's public ABI that lie on the forward-pass path, so that a program written
 * against the reference header links against this library unchanged. Each declaration
 * cites the reference declaration it replaces (paths inside the reference project).
 * Handles are opaque; statuses keep the reference's frozen ordinals
 * (include/superslm/sslm_abi.h:96-163).
 *
 * Differences a caller can observe, all inside the reference's contract:
 *  - model weights and KV live in GPU memory. The `buf` passed to sslm_kv_pool_create /
 *    sslm_workspace_create is still validated (non-null, size, 64-byte alignment) but is
 *    used only as the caller's reservation: device memory of the same capacity is
 *    allocated by the call (SSLM_ALLOCATION_FAILED if the device cannot provide it).
 *  - sslm_kv_block_size still returns layers*context_cap*kv_heads*head_dim*2 bytes; a
 *    pool of N blocks holds N full-length sequences, stored as 16-token pages.
 *  - the int16 KV precision is rejected at map time with SSLM_ARTIFACT_REJECTED; the
 *    Option-G header flag is ignored, as the reference's CPU ABI path ignores it
 *    (src/sslm_abi.cpp:1539, :2256 always run the legacy K landing).
 * There is no CPU fallback: every compute verb fails with SSLM_ALLOCATION_FAILED if no
 * CUDA device is usable.
 */
#ifndef SSLM_B200_H
#define SSLM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- types: include/superslm/sslm_abi.h:20-46, :96-224, :250 ---------------------- */
typedef struct sslm_model_s* sslm_model;
typedef struct sslm_seq_s* sslm_seq;
typedef struct sslm_adapter_s* sslm_adapter;
typedef struct sslm_prefix_s* sslm_prefix;
typedef struct sslm_schema_s* sslm_schema;     /* owned by the model; NULL = no schema */
typedef struct sslm_kv_pool_s* sslm_kv_pool;
typedef struct sslm_workspace_s* sslm_workspace;

typedef struct sslm_config {
	int32_t max_batch;        /* max sequences in one sslm_decode_step call, >= 1 */
	int32_t max_chunk_budget; /* max tokens in one sslm_prefill call, >= 1 */
	int32_t max_layer_budget; /* in [1, num_hidden_layers] */
	uint32_t reserved;        /* must be 0 */
} sslm_config;

typedef enum sslm_status {
	SSLM_OK = 0,
	SSLM_INVALID_ARGUMENT = 1,
	SSLM_BUFFER_TOO_SMALL = 2,
	SSLM_MISALIGNED_BUFFER = 3,
	SSLM_ARTIFACT_REJECTED = 4,
	SSLM_ADAPTER_MODEL_MISMATCH = 5,
	SSLM_RESTORE_MODEL_MISMATCH = 6,
	SSLM_RESTORE_KV_MISMATCH = 7,
	SSLM_MODEL_HAS_LIVE_SEQUENCES = 8,
	SSLM_POOL_HAS_LIVE_HANDLES = 9,
	SSLM_ADAPTER_HAS_LIVE_SEQUENCES = 10,
	SSLM_ADAPTER_SWAP_MIDTOKEN_REJECTED = 11,
	SSLM_SEQ_RESET_MIDTOKEN_REJECTED = 12,
	SSLM_PREFIX_FROZEN_REJECTED = 13,
	SSLM_KV_POOL_EXHAUSTED = 14,
	SSLM_TOKEN_ID_OUT_OF_RANGE = 15,
	SSLM_CONTEXT_CAP_EXCEEDED = 16,
	SSLM_TOKEN_ID_UNMAPPED = 17,
	SSLM_SCHEMA_NOT_FOUND = 18,
	SSLM_SCHEMA_BIND_REJECTED = 19,
	SSLM_SCHEMA_SPAN_UNBOUND = 20,
	SSLM_PREFIX_SCHEMA_MISMATCH = 21,
	SSLM_RESTORE_SCHEMA_MISMATCH = 22,
	SSLM_SCHEMA_SPAN_UNREACHABLE = 23,
	SSLM_SCHEMA_UNSATISFIABLE = 24,
	SSLM_ALLOCATION_FAILED = 25,
	SSLM_NUMERIC_STEP_REFUSED = 26,
	SSLM_STATUS_NEXT_FREE
} sslm_status;

typedef enum sslm_span_kind { SSLM_SPAN_PROMPT = 0, SSLM_SPAN_SCHEMA_CONTENT = 1 } sslm_span_kind;

/* sslm_decode_step reads layer_budget only (the v1.1 four-byte prefix); the remaining
 * fields exist so that the struct has the reference's size and layout. */
typedef struct sslm_decode_params {
	int32_t layer_budget;
	uint32_t struct_size;
	int32_t mode;
	int32_t alpha_q15;
	int32_t anti_lm_max_order;
	int32_t top_k;
	int64_t q_ln2;
	int64_t q_b;
	int64_t q_c;
} sslm_decode_params;

#define SSLM_ABI_ALIGNMENT_BYTES 64u

/* every entry point below has default visibility; the rest of the library is hidden */
#if defined(__GNUC__)
#define SSLM_API __attribute__((visibility("default")))
#else
#define SSLM_API
#endif

/* ---- model: include/superslm/sslm_abi_functions_g5_comparable.inc (sslm_model_map,
 *      sslm_model_unmap); src/sslm_abi.cpp:1058-1140. The artifact bytes are copied to the
 *      device during the call; the caller may free `data` afterwards. */
SSLM_API sslm_status sslm_model_map(const void* data, size_t size, sslm_model* out);
SSLM_API sslm_status sslm_model_unmap(sslm_model model);

/* ---- sizing + pool + workspace: sslm_abi_functions.inc (sslm_kv_block_size,
 *      sslm_kv_pool_overhead_size, sslm_kv_pool_create/destroy, sslm_workspace_size,
 *      sslm_workspace_create/destroy); src/sslm_abi.cpp:852-1051 */
SSLM_API size_t sslm_kv_block_size(sslm_model model);
SSLM_API size_t sslm_kv_pool_overhead_size(sslm_model model, uint32_t block_count);
SSLM_API sslm_status sslm_kv_pool_create(sslm_model model, void* buf, size_t buf_size, uint32_t block_count,
                                sslm_kv_pool* out);
SSLM_API sslm_status sslm_kv_pool_destroy(sslm_kv_pool pool);
SSLM_API size_t sslm_workspace_size(sslm_model model, const sslm_config* config);
SSLM_API sslm_status sslm_workspace_create(sslm_model model, const sslm_config* config, void* buf,
                                  size_t buf_size, sslm_workspace* out);
SSLM_API sslm_status sslm_workspace_destroy(sslm_workspace ws);

/* ---- sequences: sslm_abi_functions_g5_comparable.inc (sslm_seq_create, sslm_seq_release,
 *      sslm_prefill, sslm_decode_step); src/sslm_abi.cpp:1695-1760, :1950-1975, :1989-2449.
 *      sslm_prefill consumes min(count, chunk_budget) tokens as ONE chunk-batched pass;
 *      sslm_decode_step advances every sequence by params->layer_budget layers and writes
 *      the greedy token, or -1 while the token is in flight, -3 for a released handle. `ws`
 *      may be NULL (an internal workspace is used). */
SSLM_API sslm_status sslm_seq_create(sslm_model model, sslm_kv_pool* pool, sslm_seq* out);
SSLM_API sslm_status sslm_seq_release(sslm_seq seq);
SSLM_API sslm_status sslm_prefill(sslm_model model, sslm_seq seq, const int32_t* tokens, int32_t count,
                         int32_t chunk_budget, sslm_span_kind kind, sslm_workspace ws,
                         int32_t* consumed);
SSLM_API sslm_status sslm_decode_step(sslm_model model, sslm_seq* seqs, int32_t n,
                             const sslm_decode_params* params, sslm_workspace ws, int32_t* out_tokens);

/* ---- adapters: sslm_abi_functions.inc (sslm_adapter_map, sslm_adapter_release,
 *      sslm_adapter_residency, sslm_seq_set_adapter); src/sslm_abi.cpp:2990-3118 */
SSLM_API sslm_status sslm_adapter_map(const void* data, size_t size, sslm_model base, sslm_adapter* out);
SSLM_API sslm_status sslm_adapter_release(sslm_adapter adapter);
SSLM_API size_t sslm_adapter_residency(sslm_adapter adapter);
SSLM_API sslm_status sslm_seq_set_adapter(sslm_seq seq, sslm_adapter adapter /* NULL = detach */);

/* ---- state export: sslm_abi_functions.inc (sslm_seq_save); src/sslm_abi.cpp:2620-2716.
 *      Writes the reference's SSB3 blob, KV block in canonical
 *      [layer][K|V][kv_head][position][head_dim] order. */
SSLM_API sslm_status sslm_seq_save(sslm_seq seq, void* buf, size_t* n);

/* ---- state import and restart: sslm_abi_functions_g5_comparable.inc (sslm_seq_restore,
 *      sslm_seq_reset); src/sslm_abi.cpp:2722-2990, :1820-1860.
 *      Restore accepts the blobs sslm_seq_save writes here AND the ones the reference's CPU
 *      library writes (SSB3, and its SSB2 predecessor), so a sequence saved on either side
 *      continues bit-exactly on the other. Validation order and statuses follow the
 *      reference: bad magic / lengths -> SSLM_INVALID_ARGUMENT, other model ->
 *      SSLM_RESTORE_MODEL_MISMATCH, other KV precision -> SSLM_RESTORE_KV_MISMATCH, any
 *      schema binding that does not resolve in this model -> SSLM_RESTORE_SCHEMA_MISMATCH, pool of
 *      another model -> SSLM_INVALID_ARGUMENT, no free block -> SSLM_KV_POOL_EXHAUSTED.
 *      A blob that carries damped-greedy history (sslm_decode_step_v2 state) is refused with
 *      SSLM_INVALID_ARGUMENT: that decode mode is not part of this library.
 *      Reset returns a sequence to the state of a freshly created one (an attached adapter
 *      stays attached); mid-token -> SSLM_SEQ_RESET_MIDTOKEN_REJECTED. */
SSLM_API sslm_status sslm_seq_restore(sslm_model model, sslm_kv_pool* pool, const void* buf, size_t n,
                                      sslm_seq* out);
SSLM_API sslm_status sslm_seq_reset(sslm_seq seq);

/* ---- shared prompt prefixes: sslm_abi_functions_g5_comparable.inc (sslm_prefix_begin,
 *      sslm_prefix_prefill, sslm_prefix_freeze, sslm_prefix_release, sslm_seq_adopt_prefix);
 *      src/sslm_abi.cpp:1584-1694, :1870-1925.
 *      A prefix holds one block credit of the pool, is prefilled like a sequence, frozen, and
 *      then adopted by any number of sequences, each of which continues as if it had prefilled
 *      the same tokens itself (same tokens, same save blobs). The reference copies the whole KV
 *      block at adoption; this library shares the prefix's full 16-token pages between the
 *      prefix and its adopters and copies only the last, partly filled page. Prefill of a frozen
 *      prefix -> SSLM_PREFIX_FROZEN_REJECTED; adopting a prefix that is not frozen, or one of
 *      another model -> SSLM_INVALID_ARGUMENT. A prefix may be released while sequences that
 *      adopted it live on. */
SSLM_API sslm_status sslm_prefix_begin(sslm_model model, sslm_kv_pool* pool, sslm_prefix* out);
SSLM_API sslm_status sslm_prefix_prefill(sslm_model model, sslm_prefix prefix, const int32_t* tokens, int32_t count,
                                         int32_t chunk_budget, sslm_span_kind kind, sslm_workspace ws,
                                         int32_t* consumed);
SSLM_API sslm_status sslm_prefix_freeze(sslm_prefix prefix);
SSLM_API sslm_status sslm_prefix_release(sslm_prefix prefix);
SSLM_API sslm_status sslm_seq_adopt_prefix(sslm_seq seq, sslm_prefix prefix);

/* ---- constrained decoding: sslm_abi_functions_g5_comparable.inc (sslm_schema_lookup,
 *      sslm_schema_count, sslm_schema_name, sslm_seq_set_schema, sslm_prefix_set_schema);
 *      src/sslm_abi.cpp:1236-1264, :1791-1818, :1646-1654, :1486-1512, :2392-2424;
 *      include/superslm/schema_masks.h (the SCM1 section).
 *      An artifact may carry decode schemas: DFAs over token ids with one vocab-bit mask page
 *      per state. A sequence bound to a schema picks each token as the arg-max over the tokens
 *      its current state allows (the mask is applied inside the vocab-head kernel) and then
 *      follows the transition; a state that allows nothing yields -2 in out_tokens and the
 *      sequence stays where it is (later steps report SSLM_ARTIFACT_REJECTED, as the
 *      reference's do). sslm_prefill with SSLM_SPAN_SCHEMA_CONTENT walks the DFA with the given
 *      tokens and stops with SSLM_SCHEMA_SPAN_UNREACHABLE at the first one the schema does not
 *      allow; SSLM_SPAN_PROMPT never moves the walk. The binding, the walk state and the count
 *      of forced tokens travel in save blobs. Binding is possible only on a fresh (or reset)
 *      sequence: otherwise SSLM_SCHEMA_BIND_REJECTED. Damped-greedy decoding
 *      (sslm_decode_step_v2) is not part of this library. */
SSLM_API sslm_status sslm_schema_lookup(sslm_model model, const char* name, sslm_schema* out);
SSLM_API size_t sslm_schema_count(sslm_model model);
SSLM_API sslm_status sslm_schema_name(sslm_model model, int32_t index, char* buf, size_t* n);
SSLM_API sslm_status sslm_seq_set_schema(sslm_seq seq, sslm_schema schema);
SSLM_API sslm_status sslm_prefix_set_schema(sslm_prefix prefix, sslm_schema schema);

/* ======================================================================================
 * Entry points below have no counterpart in the reference; they exist for device
 * selection, for the standalone linear-layer workload and for measurement.
 * ====================================================================================== */

/* CUDA device ordinal used by subsequent sslm_model_map calls of this process (default 0,
 * or the SSLM_B200_DEVICE environment variable). */
SSLM_API sslm_status sslm_b200_set_device(int ordinal);

/* One int8 linear layer with the reference's full epilogue, on host buffers:
 *   acc = x[M,K] . w[N,K]^T ; folded = ApplyWeightScaleFold(acc, fold[N,3]) ;
 *   per row: RequantChainChecked(folded, incoming = {in_scale[m]}, site constant).
 * (GemmInt8Accumulate + FunnelProjectedRow, src/matmul.cpp:466-509,
 * src/forward/forward_sites.cpp:1114-1146, :1182-1203.) Outputs that are NULL are skipped.
 * in_scales: M pairs (m, e); out_scales: M pairs; row_status: M reference
 * SslmForwardStatus ordinals (0 = Ok). use_tensor_cores: 0 forces the streaming GEMV
 * kernel, 1 lets M > 8 take the activation-major tcgen05 kernel, 2 lets up to 256 rows take the
 * weights-first one where it is the better of the two, 3 up to eight rows the one whose weights wait in shared memory,
 * where they fit. */
SSLM_API sslm_status sslm_b200_linear(const int8_t* x, const int8_t* w, const int32_t* fold, int32_t M,
                             int32_t N, int32_t K, const int64_t* in_scales, int64_t site_m,
                             int64_t site_e, int32_t use_tensor_cores, int32_t* out_folded,
                             int8_t* out_codes, int64_t* out_scales, int32_t* row_status);

/* The same layer with operands resident in HBM, launched `iters` times back to back on one
 * stream; returns the average device time of one launch of the GEMM/GEMV kernel plus its
 * funnel kernel in microseconds through *avg_us (CUDA events). For the benchmark. */
SSLM_API sslm_status sslm_b200_linear_bench(int32_t M, int32_t N, int32_t K, int32_t use_tensor_cores,
                                   int32_t iters, uint64_t seed, double* avg_us_gemm,
                                   double* avg_us_total);

/* Device time (ms, CUDA events on the workspace stream) of the most recent sslm_prefill or
 * sslm_decode_step that ran on `ws`, and the number of kernels launched on it so far. */
SSLM_API sslm_status sslm_b200_last_call_ms(sslm_workspace ws, float* ms, uint64_t* kernel_launches);

/* Process-wide counters of the tensor-core linear kernels: launches of all of them, times one declined a shape
 * (another kernel ran instead) and the reason code of the last refusal. */
SSLM_API sslm_status sslm_b200_tc_stats(uint64_t* launches, uint64_t* refusals, int32_t* last_reason);
/* Launches of the tensor-core linear kernels, first n of: the activation-major one per tile shape (rows x weight
 * columns) 128 x 64, 128 x 128, 256 x 64, 256 x 128; the weights-first one; the one of up to eight rows. Lets a test assert which of them
 * served a shape. */
SSLM_API sslm_status sslm_b200_tc_variant_counts(uint64_t* counts, int32_t n);

/* Attention cuts a row along its context width into slices that run as the blocks of one
 * thread-block cluster. splits = 1, 2, 4, 8 or 16 fixes the slices per kv head of later calls
 * (rounded down to a power of two, limited by the row's width); 0 restores the automatic choice.
 * Results do not depend on it. For tuning and for tests that walk every cut. */
SSLM_API sslm_status sslm_b200_set_attention_splits(int32_t splits);

/* Decode rows whose sequences adopted the same frozen prefix are attended together, the prefix's K and V read and
 * multiplied once for all of them. mode 1 (the default): where that is faster; 0: never; 2: wherever two rows of a call share
 * a whole page. Results do not depend on it. For tuning and for tests; the second verb counts the launches so far. */
SSLM_API sslm_status sslm_b200_set_prefix_attention(int32_t mode);
SSLM_API uint64_t sslm_b200_prefix_attention_launches(void);

/* Bisection aid (the counterpart of the reference's per-site trace hook,
 * src/forward/checked_chain_funnel.cpp:338-361). With a buffer set, every later sslm_prefill /
 * sslm_decode_step on this workspace appends one record per traced site, layer and row:
 *   { int64 position; int32 layer; int32 site; int64 scale_m; int64 scale_e; int32 n; int32 row }
 * followed by the site's n int8 codes, padded to a multiple of 8 bytes. Sites: 0 attn_norm,
 * 2 rotated q (no scale), 3 attn_ctx, 5 attn_residual, 6 mlp_norm, 9 mlp_act, 11 mlp_residual.
 * Records that do not fit are dropped. buf = NULL ends the trace; *used (optional) receives the
 * bytes the trace held when this call was made. Slow (a copy per record); results are unchanged. */
SSLM_API sslm_status sslm_b200_trace(sslm_workspace ws, void* buf, size_t capacity, size_t* used);

/* Tests only: every wait of the kernels on an mbarrier is bounded, and this makes one run out on
 * purpose. The next `launches` (0..16) launches of the tensor-core linear kernel arm the barrier of
 * their first weight tile in block 0 without requesting the tile; the wait on it gives up after its
 * limit (a second or less), the rows of that tile end with an internal status, and the verb
 * that launched the kernel returns SSLM_ALLOCATION_FAILED like any other refusal (a prefill chunk
 * consumes nothing). Nothing faults and nothing spins without a limit; the next call works normally. */
SSLM_API sslm_status sslm_b200_debug_withhold_tc_load(int32_t launches);
/* The same for the words that the blocks of a cluster send each other: block 0 of the next launch of
 * `kernel` waits for more than will come in one of its exchanges. kernel 0: the weights-first linear kernel
 * where K is cut over a cluster (exchange 0); 1: attention of few rows (0 maxima, 1 sums, 2 contexts, 3 the
 * funnel's maximum); 2: attention of prefill chunks in tiles cut over a cluster (0 to 2); 3: the activation
 * site (0); 5: attention of few biased rows with the q/k/v site inside (0 the biased elements' maximum); 6: attention of
 * rows that share a prefix (0 to 2, 3 its copies of V); 7: the pick (0, 1 its first copy of logits); 8: the draw (0 maxima, 1 sums,
 * 2 lists, and of a window 3 its ends, 4 its sums, 5 its lists, 6 the last key, 7 what is kept; 3 and 6 in the second block). kernel -1 takes the request back. */
SSLM_API sslm_status sslm_b200_debug_withhold_exchange(int32_t kernel, int32_t exchange);
/* Tests only: the first kernel of each of the next `launches` (0..16) row groups counts as refused by the CUDA
 * runtime, as for want of resources. The verb returns SSLM_ALLOCATION_FAILED and launches nothing behind it. */
SSLM_API sslm_status sslm_b200_debug_refuse_launch(int32_t launches);

/* Tests only: the device integer library's primitives evaluated ON THE DEVICE over n operand
 * tuples (host arrays a, b, c, e; three host result arrays), so that their device-only halves
 * (reciprocal / root estimates, 32-bit short forms) are held to the CPU oracle as well. `which`:
 *   0 DynamicScaleReciprocal(a)            1 ISqrt(a)            2 floor((a << 32) / b), |a| <= 127
 *   3 RequantTokenCodeWide(x = a, R = b, s = c): out0 the code, out1 / out2 the per-row coders' code
 *   4 LandingRescale(code a, m b, R c, e_a = e >> 32, e_t = low half of e): out0 value, out1 flags
 *   5 a / b (unsigned, small quotient)     6 the funnel's scalars for a one-element row of magnitude a,
 *     incoming scale (b, c), site constant (e >> 32, low half of e): out0/out1 the output scale, out2 status
 *   7 one i-exp softmax element: shifted score a, constants (q_ln2 b, q_b c, q_c e >> 32), peak = low
 *     half of e << 16: out0 value, out1 refused, out2 the value rebuilt from its (shift, base) word
 *   8 Q15 probability floor((a << 15) / b)
 * and the short forms of the row and attention kernels (out1 = 0 where a form does not cover the operands):
 *   9 code of a in a row of maximum b: out0 32-bit, out1 64-bit elements, out2 0 if the signs agree
 *  10 the same for small integers in floats: out0 of a, out1 of -a
 *  11 residual landing of code a: branch scale (b, e >> 32), stream scale (c, low half of e): out0, out1 covered
 *  12 RMSNorm of code a, sum of squares b over c elements: out0 quotient, out1 covered, out2 root
 *  13 i-exp element: shifted score a, constants q_ln2 b, q_b c, q_c e: out0 value, out1 (shift, base)
 *  14 Q15 probability of a (shift, base) word a, row total b, q_c = c: out0, out1 settled exactly
 *  15 K/V landing as in 4: out0 value, out1 covered. */
SSLM_API sslm_status sslm_b200_int_sweep(int32_t which, const int64_t* a, const int64_t* b, const int64_t* c,
                                const int64_t* e, int64_t n, int64_t* out0, int64_t* out1, int64_t* out2);

/* The vocabulary head on host buffers: logits[m, n] = sum_k x[m,k] w[n,k] (int32, no fold), and per
 * row the greedy token = the lowest index of the row's maximum (LogitsSite + NarrowRowChecked +
 * ArgmaxLowestIndexTieBreak, src/forward/forward_sites.cpp:2412-2437). out_logits ([M,N], may be
 * NULL: the kernels then keep only the running maximum, as in a decode step) and out_tokens [M].
 * use_tensor_cores as for sslm_b200_linear. For the parity sweep of the logits form. */
SSLM_API sslm_status sslm_b200_logits(const int8_t* x, const int8_t* w, int32_t M, int32_t N, int32_t K,
                             int32_t use_tensor_cores, int32_t* out_logits, int32_t* out_tokens);

/* Per-kernel-class device timing of later calls on `ws` (CUDA events around every launch;
 * slows the call slightly). Classes, in order: begin, linear q/k/v, q/k/v post, attention,
 * context funnel, linear o, residual 1, linear gate/up, activation, linear down, residual 2,
 * head, LoRA u, other. profile_read returns accumulated milliseconds and launch counts of the
 * first n classes since profiling was enabled. */
SSLM_API sslm_status sslm_b200_profile(sslm_workspace ws, int32_t enable);
SSLM_API sslm_status sslm_b200_profile_read(sslm_workspace ws, double* ms, uint64_t* launches, int32_t n);

/* Tests only: capture the full int32 logit row of every token produced by later
 * sslm_decode_step calls on `ws` into host memory ([tokens in call order][vocab]);
 * pass NULL to stop. */
SSLM_API sslm_status sslm_b200_capture_logits(sslm_workspace ws, int32_t* host_rows);

/* Penalties for repeated tokens and biases of a sequence's picks. From this call on sslm_decode_step chooses the sequence's
 * tokens from its logit row as sslm_b200_pick_resident (below) changes it: the history is the tokens the sequence has
 * produced, and with count_given those it was given as well (prompts and an adopted prefix), since it was created, reset or
 * restored. A bound schema's mask applies as before, and where it allows nothing the step answers as before. Other sequences of a
 * call are chosen for as ever, and a save blob has nothing of this: a restored sequence has no controls and an empty history.
 * NULL takes the controls away; a second call replaces them; sslm_seq_reset leaves them attached and empties the history.
 * repetition below 1, more than 1,024 biases, or a missing list: SSLM_INVALID_ARGUMENT; a bias token outside the vocabulary:
 * SSLM_TOKEN_ID_OUT_OF_RANGE; nothing changes then. The first decode call of a workspace that has such a sequence allocates room
 * for the logit rows of max_batch sequences, and the first one of more sequences for the rows of as many as the workspace takes at once;
 * no other call allocates. */
typedef struct sslm_b200_controls {
	uint32_t struct_size;
	int32_t repetition;              /* Q15: 32,768 is 1.0 */
	int32_t presence, frequency;     /* logit units */
	int32_t count_given;
	int32_t n_bias;
	const int32_t* bias_tokens;
	const int32_t* bias_values;
} sslm_b200_controls;
SSLM_API sslm_status sslm_b200_seq_set_controls(sslm_seq seq, const sslm_b200_controls* controls);

/* Sampling: from this call on sslm_decode_step draws the sequence's tokens from its logit row as sslm_b200_sample_resident (below) does, after
 * its controls and its schema's mask if it has them (where that allows nothing the step answers as before). A logit unit is worth the scale of the row that the
 * head multiplies times that of the head's weights, (head_m, head_e), 2^30 <= head_m < 2^31 and |head_e| <= 4,096, or with head_m = 0 the
 * embedding's (a model whose head has weights of its own: SSLM_INVALID_ARGUMENT); a row's temperature divides it. The first n_draws tokens take draws[i]
 * (0 .. 2^31 - 1), later ones numbers made from the seed and how many tokens were drawn since this call, or since the last sslm_seq_reset. Other
 * sequences of a call are chosen for as ever, and a save blob has nothing of this. NULL goes back to the greedy token; a second call
 * replaces the first. Outside these ranges, with a list missing or a vocabulary above 2^20: SSLM_INVALID_ARGUMENT; nothing changes then. Room for logit rows as with controls. */
typedef struct sslm_b200_sampling {
	uint32_t struct_size;
	int32_t temperature;             /* Q16: 65,536 is 1.0 */
	int32_t top_k;                   /* 0: no limit */
	int32_t top_p, min_p;            /* shares of 2^30; 2^30 and 0: no limit */
	int32_t n_draws;
	int64_t head_m, head_e;
	uint64_t seed;
	const int32_t* draws;
	uint64_t reserved;
} sslm_b200_sampling;
SSLM_API sslm_status sslm_b200_seq_set_sampling(sslm_seq seq, const sslm_b200_sampling* sampling);

/* `seq` becomes a copy of `parent` as it is now, between two tokens (else SSLM_SEQ_RESET_MIDTOKEN_REJECTED, for either of them): several answers to
 * one question, the branches of a search. What it was is gone. It has the parent's adapter, schema and walk, and its history; its controls and its
 * sampling stay its own (its draws begin again). Both go on by themselves as if each had been given all that was before: same tokens, same save blobs. The
 * full 16-token pages are shared, the partly filled one is copied; the call does not wait for that. Sequences of one pool of one model
 * (else SSLM_INVALID_ARGUMENT). */
SSLM_API sslm_status sslm_b200_seq_fork(sslm_seq seq, sslm_seq parent);

/* Bytes of HBM held by the model's weights, tables and constants. */
SSLM_API size_t sslm_b200_model_device_bytes(sslm_model model);

/* The layer of sslm_b200_linear for operands that are already in device memory, for callers
 * that may not allocate (all HBM already assigned to their own pools, or no device-wide stall
 * allowed where they call from). This entry point has no counterpart in the reference. It
 * allocates nothing on the host or the device: the only scratch the layer needs, the per-row
 * peak of the folded accumulators, lives in a fixed array inside the library's device image
 * (SSLM_B200_RESIDENT_MAX_ROWS rows). Every pointer is a device pointer on the calling
 * thread's current device; x, w and out_folded 16-byte aligned; out_folded is required
 * ([M,N] int32), out_codes / out_scales / row_status may be NULL. The work is enqueued on
 * `stream` (a cudaStream_t, NULL = the default stream) and the call returns without waiting.
 *  - M > SSLM_B200_RESIDENT_MAX_ROWS or K > 16384: SSLM_INVALID_ARGUMENT, nothing is launched.
 *  - The first call on a device also looks up the array's address (set-up): make that call
 *    before any stream capture begins.
 *  - All calls on a device share the array. It reads zero at load time and every call leaves
 *    it zero again; calls whose kernels may overlap in time (other streams or threads) race
 *    on it and must be ordered by the caller.
 * From two rows on it runs on the tensor cores, its tensor maps encoded on the stack of the call. */
#define SSLM_B200_RESIDENT_MAX_ROWS 256
SSLM_API sslm_status sslm_b200_linear_resident(const int8_t* d_x, const int8_t* d_w, const int32_t* d_fold,
                                               int32_t M, int32_t N, int32_t K, const int64_t* d_in_scales,
                                               int64_t site_m, int64_t site_e, int32_t* d_out_folded,
                                               int8_t* d_out_codes, int64_t* d_out_scales,
                                               int32_t* d_row_status, void* stream);

/* ---- operators on a caller's own tensors, besides the linear layer above. As there: every pointer is a
 * device pointer on the calling thread's current device, nothing is allocated, the work is enqueued on
 * `stream` (a cudaStream_t, NULL = the default stream) and the call returns without waiting. They have no
 * scratch: calls may overlap, on any streams, and may be captured into graphs (the first call of a kind
 * on a device sets its kernels up: make it before a capture begins). What a call leaves out, rows of no
 * group or refused rows, is left as it was. `struct_size` is the size of the struct, `reserved` 0.
 *
 * Row statuses (row_status, int32 [rows], may be NULL): 0, or why the row was refused by the kernel: */
#define SSLM_B200_ROW_LENGTH 7       /* a length below zero or above the room the call gave */
#define SSLM_B200_ROW_CONSTANTS 20   /* constants outside their domain */
#define SSLM_B200_ROW_WAIT 100       /* a bounded wait inside the kernel ran out; the row's outputs are not valid */
#define SSLM_B200_ROW_INDEX 101      /* a page id, or a mask's number, that does not exist */

/* Integer attention of rows that share prefixes, each prefix read and multiplied once for all its rows (the
 * attention of sslm_decode_step over P + S positions of the paged pool, src/forward/forward_sites.cpp:1858-1903).
 * Row r is one token; group g is the rows group_start[g] .. group_start[g + 1] (ascending, device memory); its
 * rows see prefix_len[g] positions of prefix_pages[g] and then suffix_len[r] positions of suffix_pages[r]. Either
 * length may be 0 or end inside a page; a row that sees nothing has a context of zeros. Several rows may name
 * the same suffix pages (a draft of several tokens: lengths one apart).
 *   s_k = q . K_k;  x = min(max s - s_k, 30 q_ln2);  z = floor(x / q_ln2);  e_k = ((q_b - x + z q_ln2)^2 + q_c) >> z
 *   p_k = floor(2^15 e_k / sum e);  out = fold(sum p_k V_k)
 * Query head h uses K / V head h / (heads / kv_heads). head_dim 32, 64 or 128; at most 8 query heads per K / V head;
 * at most 32,768 positions a row, 65,535 rows and groups. Constants: 1 <= q_ln2 <= q_b < 2^24, q_c >= 0,
 * peak = q_b^2 + q_c <= 2^47 and peak * width < 2^63, else the row is refused, as is one with a length or page
 * id out of range (all rows of a prefix with a bad id).
 * kv is one layer of a pool: [kv_heads][K, V][num_pages] pages of 16 positions, a K page [16][head_dim], a V page
 * [head_dim][16]. fold (may be NULL: none): per query head (identity, multiplier, shift 0..31). out_codes / out_scales
 * (may be NULL): the context funnel of the row with the site constant, int8 codes [rows][heads * head_dim] and
 * (m, e) pairs, the operands sslm_b200_linear_resident takes; they need row_status.
 * Alignment: kv and out 16 bytes, out_stride a multiple of 4 elements, q 4 bytes and q_stride a multiple of 4. */
typedef struct sslm_b200_prefix_attention {
	uint32_t struct_size;
	int32_t rows, groups, heads, kv_heads, head_dim;
	int32_t max_prefix, max_suffix;   /* no length is above these (each at most 32,768); the launch is sized by them */
	const int8_t* q;                  /* [rows][heads][head_dim] rotated codes */
	int64_t q_stride;                 /* elements between rows, as every stride here */
	const int64_t* consts;            /* [rows][kv_heads][3] q_ln2, q_b, q_c */
	const int8_t* kv;
	int64_t num_pages;
	const int32_t* group_start;       /* [groups + 1] */
	const int32_t* prefix_len;        /* [groups] */
	const int32_t* prefix_pages;      /* [groups][prefix_stride] */
	int64_t prefix_stride;
	const int32_t* suffix_len;        /* [rows] */
	const int32_t* suffix_pages;      /* [rows][suffix_stride] */
	int64_t suffix_stride;
	const int32_t* fold;              /* [heads][3] */
	int32_t* out;                     /* [rows][heads][head_dim] */
	int64_t out_stride;
	int64_t site_m, site_e;
	int8_t* out_codes;
	int64_t* out_scales;
	int32_t* row_status;
	uint64_t reserved;
} sslm_b200_prefix_attention;
SSLM_API sslm_status sslm_b200_attention_prefix_resident(const sslm_b200_prefix_attention* call, void* stream);

/* The greedy token of logit rows that penalties, biases and masks have changed. Per token v of row r:
 *   not allowed where the logit is INT32_MIN, or bit v of mask page mask_page[r] is clear (-1: no mask)
 *   n = how often v is among the row's history_len[r] history ids (at most 65,535); where n > 0:
 *       x = x > 0 ? floor(x 2^15 / repetition) : -floor(-x repetition / 2^15);  x -= presence + frequency n
 *   x += every bias whose token is v (at most 1,024 a row; the same token twice counts twice)
 *   x is held between -(2^31 - 1) and 2^31 - 1, INT32_MIN where v is not allowed
 * out_tokens[r] is the lowest index of the largest x, -2 where nothing is allowed; out_best[r] that x; out_logits the
 * changed row (may be `logits` itself, may not overlap it otherwise). Each may be NULL, not all. Ids outside
 * the vocabulary, in either list, count for nothing. params, history, bias_tokens and mask_page may be NULL: none.
 * A repetition below 1 (Q15: 32,768 is 1.0), a length below 0 or above its maximum or a mask number that does
 * not exist refuses the row. */
typedef struct sslm_b200_pick {
	uint32_t struct_size;
	int32_t rows, vocab, num_masks;
	int32_t max_history, max_bias;    /* no length is above these; every row's lists have room for as many (all of it may be read) */
	uint32_t reserved;
	const int32_t* logits;            /* [rows][logits_stride] */
	int64_t logits_stride;
	const int32_t* params;            /* [rows][3] repetition (Q15), presence, frequency (logit units) */
	const int32_t* history;           /* [rows][history_stride] */
	int64_t history_stride;
	const int32_t* history_len;       /* [rows] */
	const int32_t* bias_tokens;       /* [rows][bias_stride] */
	const int32_t* bias_values;       /* [rows][bias_stride] */
	int64_t bias_stride;
	const int32_t* bias_len;          /* [rows] */
	const uint8_t* masks;             /* [num_masks][mask_stride] bytes, bit v & 7 of byte v / 8 */
	int64_t mask_stride;
	const int32_t* mask_page;         /* [rows] */
	int32_t* out_tokens;              /* [rows] */
	int32_t* out_best;                /* [rows] */
	int32_t* out_logits;              /* [rows][out_stride] */
	int64_t out_stride;
	int32_t* row_status;
} sslm_b200_pick;
SSLM_API sslm_status sslm_b200_pick_resident(const sslm_b200_pick* call, void* stream);

/* The q/k/v site of a layer: what lies between its projections and its attention (src/forward/forward_sites.cpp:1114-1146, :1281-1415,
 * :663-761, :1806-1856), for heads of any number, with norms of the heads and other rotations. Row r is one token at position
 * positions[r]; q, k and v are rows of int32 projections (out_folded of sslm_b200_linear_resident), in_scales the (m, e) of the rows
 * that were projected, 2^30 <= m < 2^31 and |e| <= 4,096.
 *   q    without q_gain: the funnel of the whole row with the site constant q_site, codes and (m, e) as out_codes and out_scales there
 *        with q_gain: each head by itself normed to a mean square of one, times the gains, as codes of the scale q_site
 *   K    without k_gain: landed on its head's scale, round(x m R / 2^(62 - e + e_t)), k_landing = (m_t, e_t, R = round(2^62 / m_t))
 *        with k_gain: normed as q
 *   V    landed as K, with v_landing
 *   norm of a head x:  y = x 2^s, 2^23 <= max |y| <= 2^24;  root = floor(sqrt(64 sum y^2 / head_dim));
 *        u = round(y floor(2^54 / root) / 2^36) (15 bits behind the point);  code = round(u gain / 2^shift);  a head of zeros: zeros
 * Every code is held between -127 and 127; roundings are to the nearest, halves away from zero. The first `rotary` channels of q and K
 * then turn by row positions[r] of the tables (30 bits behind the point), channels (2 i, 2 i + 1) or, with `halves`, (i, i + rotary / 2):
 *   a' = round(a cos - b sin),  b' = round(a sin + b cos), between -127 and 127
 * K and V go to place places[r] (NULL: positions[r]) of page table table_of[r] (NULL: r): page pages[table][place / 16] of kv, which is
 * laid out as for sslm_b200_attention_prefix_resident. consts: the softmax constants of each K / V head from q's scale and khead's (m, e).
 * saturations: the K and V codes of the row that were held. q, or k and v, may be NULL: that part is left out.
 * A position of -1 leaves its row out (a padded batch). Refused, and nothing of it written, is a row with a position outside the tables of
 * angles or a place outside its page table (SSLM_B200_ROW_LENGTH), scales outside their domain (_CONSTANTS), a page or table that does not
 * exist (_INDEX). SSLM_B200_ROW_SOFTMAX: the row is written, but some head has no constants: zeros, which attention refuses.
 * No two rows of a call may name the same place: which of them it holds then is not said.
 * head_dim 32, 64 or 128; (heads + 2 kv_heads) head_dim at most 32,768; rotary a multiple of 8, 0 .. head_dim; shifts 1 .. 62. Alignment: q,
 * k, v, cos and sin 16 bytes and their strides a multiple of 4 elements, q_codes 4 bytes and its stride a multiple of 4, kv 16 bytes. */
#define SSLM_B200_ROW_SOFTMAX 23
typedef struct sslm_b200_qkv_site {
	uint32_t struct_size;
	int32_t rows, heads, kv_heads, head_dim;
	int32_t rotary, halves;
	int32_t num_positions;            /* rows of cos and sin */
	int32_t num_tables, table_pages;  /* page tables, and entries of each */
	int32_t q_shift, k_shift;
	const int32_t *q, *k, *v;         /* [rows][heads, kv_heads, kv_heads][head_dim] */
	int64_t q_stride, k_stride, v_stride;
	const int64_t* in_scales;         /* [rows][2] */
	const int32_t* positions;         /* [rows] */
	const int32_t* places;            /* [rows] */
	const int32_t* table_of;          /* [rows] */
	const int32_t* pages;             /* [num_tables][pages_stride] */
	int64_t pages_stride;
	const int32_t *cos, *sin;         /* [num_positions][rotary / 2] */
	const int16_t *q_gain, *k_gain;   /* [head_dim] */
	int64_t q_site_m, q_site_e;
	const int64_t *k_landing, *v_landing;      /* [kv_heads][3] */
	const int64_t* khead;             /* [kv_heads][2] */
	int8_t* kv;
	int64_t num_pages;
	int8_t* q_codes;                  /* [rows][heads][head_dim] */
	int64_t q_codes_stride;
	int64_t* q_scales;                /* [rows][2], may be NULL */
	int64_t* consts;                  /* [rows][kv_heads][3], may be NULL */
	int32_t* saturations;             /* [rows], may be NULL */
	int32_t* row_status;
	uint64_t reserved;
} sslm_b200_qkv_site;
SSLM_API sslm_status sslm_b200_qkv_site_resident(const sslm_b200_qkv_site* call, void* stream);

/* A token drawn from the logits of each row, in integers. Per row, over the tokens v with a logit x_v other than INT32_MIN (as
 * sslm_b200_pick_resident writes one that is not allowed), with params[r] = slope, cut, top_k, top_p, min_p and d_v = max x - x_v:
 *   t = floor(d slope / 2^cut);  w_v = floor(P(t mod 2^24) / 2^floor(t / 2^24)), 0 from t = 2^29 on: 2^31 2^(-t / 2^24), P 2^31 at 0 and falling,
 *       3.4e-6 off at most: P = c0 - hi(f, c1 - hi(f, c2 - hi(f, c3 - hi(f, c4)))), f = 2^8 (t mod 2^24), hi(f, c) = floor(f c / 2^32),
 *       c = 2147483648, 1488326151, 514119776, 114090822, 14555373
 *   slope / 2^cut is thus 2^24 times the octaves a logit unit is worth: 2^24 scale / (temperature ln 2)
 *   kept are, in the order of falling logits, equal ones by rising index: the first top_k (0: all); of these, with S the sum of their w, those in
 *       front of which less than floor(S top_p / 2^30) lies (2^30: all); of these those with w >= 2 min_p; and never one with w = 0
 *   the token is the lowest v for which the kept w up to and including it, by index, are more than floor(T draws[r] / 2^31), T their sum
 * out_tokens[r] is the token, -2 where every logit is INT32_MIN; out_mass[r] its w and T (the token's probability is their quotient), zeros
 * there; out_kept[r] how many are kept. Each may be NULL, not all. A slope or draw below 0, a cut outside 0 .. 63, a top_k below 0, a top_p outside
 * 1 .. 2^30 or a min_p outside 0 .. 2^30 refuses the row (SSLM_B200_ROW_CONSTANTS). At most 65,535 rows and 2^20 tokens. */
typedef struct sslm_b200_sample {
	uint32_t struct_size;
	int32_t rows, vocab;
	uint32_t reserved;
	const int32_t* logits;            /* [rows][logits_stride] */
	int64_t logits_stride;
	const int32_t* params;            /* [rows][5] */
	const int32_t* draws;             /* [rows] 0 .. 2^31 - 1 */
	int32_t* out_tokens;              /* [rows] */
	int64_t* out_mass;                /* [rows][2] */
	int32_t* out_kept;                /* [rows] */
	int32_t* row_status;
} sslm_b200_sample;
SSLM_API sslm_status sslm_b200_sample_resident(const sslm_b200_sample* call, void* stream);

/* The sequences of a paged cache continue from others, grow or end, all at once: a beam search's step, several answers to one question,
 * room for the next positions. Sequence i has lengths[i] positions in the pages tables[i]; holders[p] says how many tables (or whoever else) hold
 * page p, 0: it is free. All inputs are read as they were before the call:
 *   parents[i] = i    it stays, and takes grow[i] more positions
 *   parents[i] = p    it becomes a copy of p with grow[i] more positions: p's full pages are held in common, a partly filled one is copied
 *   parents[i] = -1   it ends
 * What a sequence held and no longer holds it lets go. Pages that are drawn were free before the call, lowest first, in the order of the
 * sequences: drawn[0 .. counts[1]) (behind these, free pages that were too few for a sequence may follow). moves[0 .. counts[0]) are the pages
 * copied, (from, to), whole, in every plane of kv (NULL: none are copied, for a caller whose planes lie apart). Entries of out_tables behind a
 * sequence's pages, and of moves behind the count, stay as they were. status[i]: 0, or why the sequence stays what it was: a parent that does not exist or
 * a page id of it that does not (SSLM_B200_ROW_INDEX), a length or growth below 0 or together above the table's room (_LENGTH), not enough free pages for it
 * (_PAGES: those in front of it are served). Without sequences holders go to out_holders as they are and counts are zeros. Outputs may not overlap
 * inputs. At most 65,535 sequences and 65,536 pages a table; page_bytes a multiple of 16, kv on a 16-byte boundary, moves on an 8-byte one. Two launches. */
#define SSLM_B200_ROW_PAGES 102
typedef struct sslm_b200_fork {
	uint32_t struct_size;
	int32_t sequences, table_pages, planes, page_bytes;
	uint32_t reserved;
	int64_t num_pages;
	int8_t* kv;                       /* [planes][num_pages][page_bytes]: of the pool of sslm_b200_attention_prefix_resident, 2 kv_heads planes a layer */
	const int32_t* holders;           /* [num_pages] */
	const int32_t* tables;            /* [sequences][tables_stride] */
	int64_t tables_stride;
	const int32_t* lengths;           /* [sequences] */
	const int32_t* parents;           /* [sequences] */
	const int32_t* grow;              /* [sequences], NULL: zeros */
	int32_t* out_holders;             /* [num_pages] */
	int32_t* out_tables;              /* [sequences][out_stride] */
	int64_t out_stride;
	int32_t* out_lengths;             /* [sequences] */
	int32_t* drawn;                   /* [num_pages] */
	int32_t* moves;                   /* [sequences][2] */
	int32_t* counts;                  /* [2] moves, pages drawn */
	int32_t* status;                  /* [sequences] */
} sslm_b200_fork;
SSLM_API sslm_status sslm_b200_fork_resident(const sslm_b200_fork* call, void* stream);

/* The pages in use (holders above or below 0) move to the front of the pool: with `live` of them, those at live and behind go to the free ones
 * in front of it, the lowest to the lowest. new_of[p] is page p's new id, -1 where it is free; moves[0 .. counts[0]) are (from, to), copied in every
 * plane of kv (NULL: not); counts[1] = live. out_holders and out_tables are holders and tables under the new ids; entries behind a sequence's
 * pages, and of moves behind the count, stay as they were. status[i] (may be NULL): 0, or a length below 0 or above the table's room
 * (SSLM_B200_ROW_LENGTH), a page id that does not exist or is free (_INDEX): such a table is not written. out_tables may be tables with
 * the same stride; other outputs may not overlap inputs. Limits and alignment as above. Two launches. */
typedef struct sslm_b200_compact {
	uint32_t struct_size;
	int32_t sequences, table_pages, planes, page_bytes;
	uint32_t reserved;
	int64_t num_pages;
	int8_t* kv;
	const int32_t* holders;           /* [num_pages] */
	const int32_t* tables;            /* [sequences][tables_stride] */
	int64_t tables_stride;
	const int32_t* lengths;           /* [sequences] */
	int32_t* out_holders;             /* [num_pages] */
	int32_t* out_tables;              /* [sequences][out_stride] */
	int64_t out_stride;
	int32_t* new_of;                  /* [num_pages] */
	int32_t* moves;                   /* [num_pages / 2][2] */
	int32_t* counts;                  /* [2] moves, pages in use */
	int32_t* status;                  /* [sequences], may be NULL */
} sslm_b200_compact;
SSLM_API sslm_status sslm_b200_compact_resident(const sslm_b200_compact* call, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SSLM_B200_H */
