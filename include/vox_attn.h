/* libvoxattn: MI355X (gfx950) paged-KV attention for the VoxCPM2 engine, C ABI.
 *
 * The three launch entry points replace the GPU calls that the reference's Attention.forward makes
 * (reference: nanovllm_voxcpm/model/layers.py:326-362). All device buffers are owned by the caller; the library
 * never allocates, frees or synchronizes, so every call is stream-ordered on `stream` (a hipStream_t, NULL = the
 * null stream) and may be captured into a HIP graph. Element types: bf16 tensors are passed as raw pointers to
 * 16-bit words, index tensors are int32. Strides are in elements.
 *
 * Every function returns VOX_OK or an error code; vox_last_error() returns the calling thread's message for the
 * last failure. No function throws.
 */
#ifndef VOX_ATTN_H_
#define VOX_ATTN_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VOX_ABI_VERSION 16

#define VOX_OK 0
#define VOX_EINVAL 1 /* bad argument: shape, stride, alignment or null pointer (reference: the asserts of
                        nanovllm_voxcpm/model/layers.py:299-302 and kernels/prefill_attn.py:107-108) */
#define VOX_EHIP 2   /* the HIP runtime reported an error at launch */

/* Plan modes of the decode calls (the `plan` argument). The decode layout (how the sequences' tokens are dealt to the
 * workgroups, and the block id of every tile) depends only on the lengths, the block tables and, in store mode, the
 * slots, which every layer of one decode step shares. No reference counterpart: the reference likewise builds
 * per-step metadata once per forward context for all layers (nanovllm_voxcpm/engine/utils.py:53-57).
 *   VOX_PLAN_NONE    every workgroup scans the lengths and stages the table itself
 *   VOX_PLAN_RECORD  the same, and the layout is recorded in the workspace
 *   VOX_PLAN_REUSE   the layout is read from the workspace, where the last VOX_PLAN_RECORD call on it recorded it;
 *                    the caller guarantees that call had the same batch, context lengths (varlen: cu_seqlens), block
 *                    tables, slots (store mode: reuse only after a store-mode record) and workgroup count. Parts of
 *                    the layout a record cannot hold are scanned again. Batches above 512 sequences run unplanned.
 * A call that fails records nothing, nor does a varlen call whose one-query rows the decode kernels do not take. */
#define VOX_PLAN_NONE 0
#define VOX_PLAN_RECORD 1
#define VOX_PLAN_REUSE 2

const char* vox_last_error(void);
int vox_abi_version(void);

/* KV slot scatter. Replaces store_kvcache / store_kvcache_kernel (reference: nanovllm_voxcpm/model/layers.py:266-305).
 * For each token i < num_tokens with slot = slot_mapping[i] in [0, num_slots): copies the num_kv_heads*head_dim
 * contiguous elements of key row i (rows key_row_stride apart) to k_cache + slot*num_kv_heads*head_dim, and
 * likewise value -> v_cache. slot -1 (padding) is skipped, as in the reference; other out-of-range slots are skipped
 * too instead of writing outside the cache. Bit-exact. */
int vox_store_kvcache(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride,
                      void* k_cache, void* v_cache, int64_t num_slots, const int32_t* slot_mapping,
                      int64_t num_tokens, int num_kv_heads, int head_dim, void* stream);

/* Paged decode attention, one query token per sequence. Replaces the decode branch's
 * flash_attn_with_kvcache(q.unsqueeze(1), k_cache, v_cache, cache_seqlens=context_lens, block_table=block_tables,
 * softmax_scale, causal=True) (reference: nanovllm_voxcpm/model/layers.py:349-358).
 *   q            bf16 [batch, num_heads, head_dim], sequence rows q_row_stride apart, heads head_dim apart
 *   k/v_cache    bf16 [num_blocks, block_size, num_kv_heads, head_dim], contiguous
 *   block_tables int32 [batch, bt_stride]; the first max_blocks columns of every row must be readable (the
 *                kernel may stage them all), but entries past ceil(context_lens[b] / block_size) are never used;
 *                an entry inside the context outside [0, num_blocks) masks that block's keys (no weight)
 *   context_lens int32 [batch]; 0 = padded row, whose output is written as zeros
 *   plan         VOX_PLAN_NONE, VOX_PLAN_RECORD or VOX_PLAN_REUSE (above)
 *   workspace    >= vox_decode_workspace_bytes(batch) bytes of scratch, 16-byte aligned: the split-KV partials and
 *                the step layout the two kernels of the call (launched in order on `stream`) pass on, and the plan
 *                records. VOX_PLAN_REUSE reads what the recording call left there, so the workspace must be the
 *                same and untouched by other calls in between; no other contents need to survive a call.
 *   out          bf16 [batch, num_heads, head_dim], contiguous
 * Supported: head_dim 128, num_kv_heads 1 or 2, num_heads <= 16, block_size a multiple of 32. */
int vox_decode_attn(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                    int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                    int max_blocks, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                    int head_dim, float softmax_scale, int plan, void* workspace, size_t workspace_bytes,
                    void* out, void* stream);

/* The decode step's KV store and decode attention in one call: vox_store_kvcache(key, value, key_row_stride,
 * value_row_stride, k_cache, v_cache, num_blocks * block_size, slot_mapping, batch, ...) followed by
 * vox_decode_attn(...) (reference: the decode branch of nanovllm_voxcpm/model/layers.py:326-358, store_kvcache then
 * flash_attn_with_kvcache), without the store's own launch: the split kernel reads each sequence's new token from
 * key / value where the tile it loads holds that token's slot, and writes the rows into the caches. Same results as
 * the two calls when no slot_mapping[b] lies inside another sequence's context (the engine's sequences each write
 * only their own last block); slot -1 and slots outside the cache store nothing.
 *   key / value    bf16 [batch, num_kv_heads, head_dim], heads contiguous, rows *_row_stride elements apart
 *                  (multiples of 8), 16-byte aligned
 *   slot_mapping   int32 [batch]
 * Other arguments as vox_decode_attn. */
int vox_decode_attn_store(const void* q, int64_t q_row_stride, const void* key, const void* value,
                          int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                          void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                          const int32_t* block_tables, int64_t bt_stride, int max_blocks, const int32_t* context_lens,
                          int batch, int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int plan,
                          void* workspace, size_t workspace_bytes, void* out, void* stream);

/* vox_decode_attn without the workspace argument: the split-KV scratch is a static device array of 16 MiB
 * (16777216 bytes) that each GPU the library runs on holds until the process ends, so the
 * call allocates nothing (no hipMalloc, no allocator call of any kind). No counterpart in the reference: it is for
 * callers that cannot allocate (code under HIP graph capture that must not touch an allocator, tight serving loops).
 * Returns VOX_EINVAL when vox_decode_workspace_bytes(batch) exceeds the array (not for any batch at the default
 * workgroup count: batches are launched 512 sequences at a time). Every call on one GPU shares that GPU's array:
 * calls that overlap on one GPU (different streams, or host threads) race and must be serialized by the caller.
 * The array needs no clearing: each call writes every scratch value it reads. Runs with VOX_PLAN_NONE. Other
 * arguments as vox_decode_attn. */
int vox_decode_attn_noalloc(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                            int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                            int max_blocks, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                            int head_dim, float softmax_scale, void* out, void* stream);

/* Workspace bytes vox_decode_attn needs for `batch` sequences on the current device. No reference
 * counterpart: flash-attn sizes its split-KV buffers internally (reference call site: nanovllm_voxcpm/model/layers.py:350). */
size_t vox_decode_workspace_bytes(int batch);

/* Workgroups the decode split kernel runs on the current device (one per CU), and a process-wide override for tuning
 * and tests (0 restores the built-in choice; change it only between calls, the workspace size depends on it). No
 * reference counterpart. */
int vox_decode_workgroups(void);
void vox_set_decode_workgroups(int workgroups);

/* Varlen attention for prefill steps. Replaces flash_attn_varlen_func(q, k, v, max_seqlen_q, cu_seqlens_q,
 * max_seqlen_k, cu_seqlens_k, softmax_scale, causal=True, block_table) (reference: nanovllm_voxcpm/model/layers.py:
 * 337-348), the Triton paged_prefill_attention / short_causal_attention in bf16 mode (reference:
 * nanovllm_voxcpm/kernels/prefill_attn.py:98-124, kernels/short_attn.py:156-179), and, with causal = 0 and uniform
 * lengths, flash_attn_func(q, k, v, softmax_scale, causal=False) (reference: nanovllm_voxcpm/model/layers.py:361).
 *   q              bf16 [T, num_heads, head_dim], token rows q_row_stride apart
 *   key/value      packed bf16 [Tk, num_kv_heads, head_dim] rows (used when block_tables is NULL)
 *   k/v_cache      paged bf16 [num_blocks, block_size, num_kv_heads, head_dim] (used when block_tables != NULL)
 *   cu_seqlens_q/k int32 [batch + 1]; both NULL selects uniform lengths uniform_seqlen_q / uniform_seqlen_k
 *   causal         bottom-right aligned: query i of a sequence with nq queries and nk keys sees keys j <= nk-nq+i
 *   out            bf16 [T, num_heads, head_dim], token rows out_row_stride apart
 *   plan, workspace
 *                  NULL, or a decode workspace (>= vox_prefill_workspace_bytes(batch) bytes, under vox_decode_attn's
 *                  contract) and its plan mode: with block tables and cu_seqlens, sequences with exactly one query (the
 *                  decode rows of a mixed prefill + decode step) then run on the split-KV decode kernel, which spreads
 *                  long contexts over every CU (needs num_heads <= 16, num_kv_heads 1 or 2, block_size a multiple of
 *                  32, out 16-byte aligned with out_row_stride a multiple of 8; otherwise, or with NULL, the prefill
 *                  kernel takes every row). Calls of up to 256 sequences over blocks of a multiple of 64 tokens run
 *                  both kinds of rows in one launch, sharing every CU. Results within the same tolerance either way.
 * Supported: head_dim 128, num_heads / num_kv_heads dividing 128. */
int vox_prefill_attn(const void* q, int64_t q_row_stride, const void* key, const void* value,
                     int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                     int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                     int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                     int max_seqlen_q, int uniform_seqlen_q, int uniform_seqlen_k, int num_heads, int num_kv_heads,
                     int head_dim, float softmax_scale, int causal, void* out, int64_t out_row_stride, int plan,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Scratch bytes vox_prefill_attn's one-query rows need for `batch` sequences on the current device. No reference
 * counterpart (flash-attn sizes its buffers internally; reference call site: nanovllm_voxcpm/model/layers.py:337). */
size_t vox_prefill_workspace_bytes(int batch);

/* A packed prefill step's KV store and its attention in one call: vox_store_kvcache(key, value, key_row_stride,
 * value_row_stride, k_cache, v_cache, num_slots, slot_mapping, num_tokens, num_kv_heads, head_dim) followed by
 * vox_prefill_attn over the packed rows key / value (no block table) (reference: the prefill branch of
 * nanovllm_voxcpm/model/layers.py:326-348 without a block table, store_kvcache then flash_attn_varlen_func over the
 * step's own k and v). The attention reads the packed rows, not the cache, so the copy rides in the attention launch
 * (workgroups that have done their own work, or have none, copy the rows) instead of a launch of its own. Outputs and
 * caches are identical to the two calls. Rows the 16-byte copy cannot move (16-byte aligned rows, strides multiples of
 * 8) take the two calls. Arguments as in those two functions; num_tokens = the rows of key / value and slot_mapping. */
int vox_prefill_attn_store(const void* q, int64_t q_row_stride, const void* key, const void* value,
                           int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                           void* k_cache, void* v_cache, int64_t num_slots, int64_t num_tokens,
                           const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                           int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int causal, void* out,
                           int64_t out_row_stride, void* stream);

/* A paged prefill step's KV store and its attention in one call: vox_store_kvcache(key, value, key_row_stride,
 * value_row_stride, k_cache, v_cache, num_blocks * block_size, slot_mapping, num_tokens, num_kv_heads, head_dim)
 * followed by vox_prefill_attn over the caches through block_tables (reference: the prefill branch of
 * nanovllm_voxcpm/model/layers.py:326-348 with a block table, store_kvcache then flash_attn_varlen_func over
 * k_cache / v_cache; the mixed steps of nanovllm_voxcpm/engine/scheduler.py:340 (_ride) take this branch).
 * With blocks of a multiple of 64 tokens and rows 16-byte aligned with strides multiples of 8 (below 2^24 elements),
 * the store rides in the attention launch: each sequence's new keys (its last nq key positions) are read from the
 * rows key / value (row cu_seqlens_q[b] + i for the i-th) instead of the cache, and the rows are written into the
 * caches: after the reads by the merge kernel when the call runs as one mixed launch (vox_prefill_attn's conditions:
 * workspace, up to 256 sequences, some sequence with more than one query), else, when it runs on the prefill kernel
 * alone (no workspace), beside the reads by workgroups of the launch. That equals the two calls when, as the engine's scheduler
 * guarantees, slot_mapping holds for each sequence's new tokens the slots its block table gives their positions, and
 * no sequence's new slots lie inside another sequence's context. Otherwise (a workspace whose call is not one mixed
 * launch, other block sizes, other rows) the two calls run. Outputs and caches are identical to the two calls;
 * num_tokens = the rows of key / value and slot_mapping; plan as vox_prefill_attn's, except that a REUSE call needs a
 * record made by this function (records hold the new tokens' slots). */
int vox_prefill_attn_store_paged(const void* q, int64_t q_row_stride, const void* key, const void* value,
                                 int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                                 int64_t num_tokens, void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                                 const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                 const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                                 int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int causal,
                                 void* out, int64_t out_row_stride, int plan, void* workspace, size_t workspace_bytes,
                                 void* stream);

/* vox_prefill_attn with the int8 output epilogue the W8A8 o_proj consumes. Replaces the quant=True modes of the
 * Triton paged_prefill_attention, short_causal_attention and short_attention (reference:
 * nanovllm_voxcpm/kernels/prefill_attn.py:84-92 and :98-124, kernels/short_attn.py:55-64, :70-90, :137-146, :156-179;
 * caller kernels/fused_layer.py:698-730). Per token t, with o the fp32 attention output over all heads:
 *   x = o * inv_smooth (inv_smooth fp32 [num_heads * head_dim], NULL = 1), amax = max(max_c |x[c]|, 1e-6),
 *   out_scale[t] = amax / 127,   out_q[t, c] = rint(x[c] / out_scale[t])  (round half to even, int8).
 *   out_q      int8 [T, num_heads * head_dim], token rows out_q_row_stride apart (multiple of 4, 4-byte aligned)
 *   out_scale  fp32 [T]
 *   num_tokens T, the query rows (cu_seqlens_q[batch], or batch * uniform_seqlen_q) that out_q, out_scale and
 *              the workspace hold; rows at or past it are neither read nor written, so a cu_seqlens_q reaching past
 *              it truncates the output instead of writing out of bounds (0: nothing to do)
 *   workspace  NULL, or >= vox_prefill_int8_workspace_bytes(...) bytes of scratch (16-byte aligned): where that is
 *              nonzero the call runs as two passes (the bf16 kernel into the workspace, then a per-token
 *              quantization of its rows), which is faster for long sequences whose work items outnumber the CUs;
 *              the codes then come from the bf16-rounded o (as the reference's flash-attn + quantize path computes
 *              them) instead of the fp32 accumulators, within one code step of each other
 * Other arguments as vox_prefill_attn. Supported: num_kv_heads 1 or 2 (one workgroup holds all heads of its tokens). */
int vox_prefill_attn_int8(const void* q, int64_t q_row_stride, const void* key, const void* value,
                          int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                          int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                          int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                          int max_seqlen_q, int uniform_seqlen_q, int uniform_seqlen_k, int num_heads,
                          int num_kv_heads, int head_dim, float softmax_scale, int causal, const float* inv_smooth,
                          void* out_q, int64_t out_q_row_stride, float* out_scale, int64_t num_tokens,
                          void* workspace, size_t workspace_bytes, void* stream);

/* A prefill step's KV store and its int8-output attention in one call: vox_store_kvcache(key, value, key_row_stride,
 * value_row_stride, k_cache, v_cache, num_blocks * block_size, slot_mapping, store_rows, num_kv_heads, head_dim)
 * followed by vox_prefill_attn_int8, over the packed rows key / value (block_tables NULL) or over the caches through
 * block_tables. Replaces the W8A8 layer's store_kvcache + short_causal_attention(quant=True) pair (the head-start step
 * of a burst) and its store_kvcache + paged_prefill_attention(quant=True) pair (eager prefix-cache steps) (reference:
 * nanovllm_voxcpm/kernels/fused_layer.py:643-667 and :619-641). The copy rides in the int8 launch (the last
 * workgroups copy the rows after their own work; in the two-pass form, in the bf16 pass); with block tables the launch
 * reads each sequence's new keys (its last nq key positions) from the rows instead of the cache, which equals the two
 * calls when, as the engine guarantees, slot_mapping holds the slots the tables give those positions and no sequence's
 * new slots lie inside another sequence's context. Outputs and caches identical to the two calls; rows the 16-byte
 * copy cannot move, and block sizes other than multiples of 64 with block tables, take the two calls. Arguments as in
 * those two functions (k_cache / v_cache [num_blocks, block_size, HK, head_dim]; store_rows = the rows of key / value
 * and slot_mapping, num_tokens = the query rows). */
int vox_prefill_attn_int8_store(const void* q, int64_t q_row_stride, const void* key, const void* value,
                                int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                                int64_t store_rows, void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                                const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int max_seqlen_q,
                                int num_heads, int num_kv_heads, int head_dim, float softmax_scale, int causal,
                                const float* inv_smooth, void* out_q, int64_t out_q_row_stride, float* out_scale,
                                int64_t num_tokens, void* workspace, size_t workspace_bytes, void* stream);

/* Scratch bytes for vox_prefill_attn_int8's two-pass form for a call of this shape: num_tokens * num_heads *
 * head_dim * 2 where the two passes are the faster form, 0 where the fused epilogue is (then pass NULL). No
 * reference counterpart (the reference's quant kernels allocate their outputs only). */
size_t vox_prefill_int8_workspace_bytes(int64_t num_tokens, int batch, int max_seqlen_q, int num_heads,
                                        int num_kv_heads, int head_dim, int causal);

/* Copy the first n token slots of KV-cache blocks in every (layer, K/V) plane, in one launch. Replaces
 * copy_kv_block_prefix (reference: nanovllm_voxcpm/kernels/kv_copy.py:17-41; callers model/runner.py:232-248,
 * model/engine.py:383-452).
 *   kv          2-byte elements [num_planes, num_blocks, block_size, per_token], contiguous (the engine's
 *               [layers, 2, blocks, block_size, kv_heads, head_dim] tensor: num_planes = layers * 2,
 *               per_token = kv_heads * head_dim)
 *   entries     device int32 [num_entries, 3]: (src block, dst block, n tokens); n is clipped to block_size and
 *               n <= 0 does nothing; entries with a block outside [0, num_blocks) are skipped
 *   max_tokens  an upper bound of the entries' n (sizes the launch; host-known, as the reference's grid)
 * Bit-exact. Entries that write a block another entry of the same call reads race, as in the reference. */
int vox_copy_kv_block_prefix(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t per_token,
                             int elem_bytes, const int32_t* entries, int num_entries, int max_tokens, void* stream);

/* ---- KV caches held in 4 bits. No reference counterpart (its caches are bf16): a step's bytes and a pool's size are 0.27
 * of the bf16 cache's.
 *
 * The format is OCP MXFP4: every 32 channels of one token and kv head share a scale, a byte b that stands for
 * 2^(b - 127) (255: not a number), and a value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, with a sign (codes 0-7, and
 * 8-15 for the negatives; channel 2i in the low nibble of byte i). A plane is num_blocks blocks of block_size *
 * num_kv_heads * 68 bytes; in a block the codes [block_size][num_kv_heads][64] come first, then the scales [block_size]
 * [num_kv_heads][4]. Caches are 16-byte aligned, block_size a multiple of 64, head_dim 128, num_blocks * block_size
 * below 2^31. */

/* Quantises key / value rows (bf16 [num_tokens, num_kv_heads, head_dim], rows *_row_stride elements apart, heads
 * contiguous) into their slots; slots outside [0, num_blocks * block_size) (-1: padding) store nothing. Of a group whose
 * largest magnitude is amax the scale is the least power of two 2^e >= 2^-126 with amax <= 7 * 2^e, and 2^125 where that is
 * more (6 * 2^125 is the largest that bf16 holds); a value becomes the nearest one of the grid, ties to the even code, at most
 * 6 * 2^e. A group that holds an infinity or NaN gets scale 255.
 * The codes are a function of the row alone. Slots that occur twice in a call hold a mix of their rows. */
int vox_store_kvcache_fp4(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride,
                          void* k_cache, void* v_cache, int64_t num_blocks, int block_size, const int32_t* slot_mapping,
                          int64_t num_tokens, int num_kv_heads, int head_dim, void* stream);

/* The values held at slots as bf16 rows: key / value [num_tokens, num_kv_heads, head_dim], contiguous, 16-byte aligned.
 * Exact; zeros for slots outside the cache, infinities for what bf16 does not hold (no stored row: 4 and 6 times 2^126, 2 to 6
 * times 2^127). */
int vox_load_kvcache_fp4(const void* k_cache, const void* v_cache, int64_t num_blocks, int block_size,
                         const int32_t* slots, int64_t num_tokens, int num_kv_heads, int head_dim, void* key,
                         void* value, void* stream);

/* vox_decode_attn over 4-bit caches: the attention over the values that the caches hold. Where a value row's group of 32 channels
 * is not a number, or has a value past bf16's largest (no stored row), the outputs that see it are NaN in those channels.
 * Arguments, workspace and plans as vox_decode_attn's (records may not be shared with calls of other functions). softmax_scale
 * must be positive. */
int vox_decode_attn_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                        int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                        int max_blocks, const int32_t* context_lens, int batch, int num_heads, int num_kv_heads,
                        int head_dim, float softmax_scale, int plan, void* workspace, size_t workspace_bytes,
                        void* out, void* stream);

/* vox_store_kvcache_fp4 of one row a sequence and vox_decode_attn_fp4 in one call: the new tokens are attended over as the
 * cache will hold them, and their rows stored behind the reads. Same results as the two calls when no slot_mapping[b] lies
 * inside another sequence's context, as vox_decode_attn_store's. Rows that are not 16-byte aligned with strides multiples of 8
 * take the two calls. Plans: calls of either form may follow each other; a record made by one is not used by the other, which
 * scans the layout. */
int vox_decode_attn_store_fp4(const void* q, int64_t q_row_stride, const void* key, const void* value,
                              int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                              void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                              const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                              const int32_t* context_lens, int batch, int num_heads, int num_kv_heads, int head_dim,
                              float softmax_scale, int plan, void* workspace, size_t workspace_bytes, void* out,
                              void* stream);

/* vox_prefill_attn over 4-bit caches through block tables, with cu_seqlens. num_tokens: the rows that q and out hold; rows
 * at or past it are neither read nor written by the prefill kernel. plan, workspace: as vox_prefill_attn's (with the
 * workspace the one-query sequences run on the decode kernels, up to 256 sequences in the same launch). num_heads /
 * num_kv_heads divides 128, softmax_scale is
 * positive. */
int vox_prefill_attn_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                         int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                         int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                         int max_seqlen_q, int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim,
                         float softmax_scale, int causal, void* out, int64_t out_row_stride, int plan, void* workspace,
                         size_t workspace_bytes, void* stream);

/* ---- The care of a paged cache's blocks, in every plane at once. kv is [num_planes][num_blocks] blocks, one behind the
 * other; a block is block_size slots of slot_bytes and behind them block_size slots of scale_bytes (a bf16 cache:
 * num_kv_heads * 256 and 0; a 4-bit cache: num_kv_heads * 64 and num_kv_heads * 4). kv and both runs of a block are
 * 16-byte aligned. */

/* vox_copy_kv_block_prefix for caches of any slot: entries int32 [num_entries, 3] on the device: (src block, dst block, n),
 * the first n slots copied. Entries that write a block another entry of the same call reads race. */
int vox_copy_kv_blocks(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                       int64_t scale_bytes, const int32_t* entries, int num_entries, void* stream);

/* Forks sequences. Row p = parents[i] of block_tables (int32 [batch, bt_stride], the first max_blocks columns) with
 * context_lens[p] tokens gets a child: it shares the parent's full blocks, and where the last block is partly filled its
 * filled slots are copied to block new_blocks[i], which takes that block's place. child_tables int32 [num_forks,
 * max_blocks] (-1 past the context), child_lens int32 [num_forks]. new_blocks must be blocks that no table names, no two
 * the same; one whose parent ends with a full block is left alone. A parent outside [0, batch) gives an empty child; a
 * last block or new block outside the cache copies nothing and leaves -1 in the child's table; a context past what
 * max_blocks blocks hold counts as that. */
int vox_fork_kv_blocks(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                       int64_t scale_bytes, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                       const int32_t* context_lens, int batch, const int32_t* parents, const int32_t* new_blocks,
                       int num_forks, int32_t* child_tables, int32_t* child_lens, void* stream);

/* Moves the live blocks (those that a row of block_tables names within its context) to the front of the cache: with L of
 * them, those at or past L move to the dead blocks below L, the lowest to the lowest. Blocks shared by several rows move
 * once. new_tables int32 [batch, max_blocks]: the tables with the new numbers (-1 past the context, entries outside the
 * cache as they were); remap int32 [num_blocks]: each live block's new number, -1 for the dead; live int32 [1]: L. moves
 * int32 [2 num_blocks + 1]: scratch. Blocks from L on are free afterwards; num_blocks at most 2^18. */
int vox_compact_kv_blocks(void* kv, int64_t num_planes, int64_t num_blocks, int block_size, int64_t slot_bytes,
                          int64_t scale_bytes, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                          const int32_t* context_lens, int batch, int32_t* new_tables, int32_t* remap, int32_t* live,
                          int32_t* moves, void* stream);

/* ---- What each cached token receives of the attention, and its eviction. key_weights fp32 [num_weight_rows, num_kv_heads,
 * weight_width] holds, for the sequence whose row it is (weight_rows int32 [batch] on the device, or NULL: sequence b's is row
 * b; a row outside [0, num_weight_rows): none is kept) and each kv head, the sum of its cached tokens' probabilities over the
 * kv head's query heads and every query so far. No two sequences of a call have the same row. softmax_scale is positive. */

/* Scratch of vox_decode_attn_weights: the scores of every 16-token step that the tables allow. */
size_t vox_decode_scores_bytes(int batch, int max_blocks, int block_size, int num_heads);

/* vox_decode_attn, or with key (not NULL) vox_decode_attn_store, that also adds what every key received: a token before the
 * last one of its context gets it on top of its weight, the last one's weight becomes it. Tokens at or past weight_width are
 * left out. scores: vox_decode_scores_bytes bytes of scratch (16-byte aligned), the call's own. plan, workspace: as
 * vox_decode_attn's. */
int vox_decode_attn_weights(const void* q, int64_t q_row_stride, const void* key, const void* value,
                            int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping, void* k_cache,
                            void* v_cache, int64_t num_blocks, int block_size, const int32_t* block_tables,
                            int64_t bt_stride, int max_blocks, const int32_t* context_lens, int batch, int num_heads,
                            int num_kv_heads, int head_dim, float softmax_scale, float* key_weights,
                            const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width, void* scores,
                            size_t scores_bytes, int plan, void* workspace, size_t workspace_bytes, void* out,
                            void* stream);

/* The same over 4-bit caches, as vox_decode_attn_fp4 and vox_decode_attn_store_fp4: a row's scores are off by at most x =
 * softmax_scale (2^-13 sum |q||k| + 2^-18 max |q| sum |k|), a probability by at most e^(2x) - 1 of it beside the roundings in 32
 * bits. */
int vox_decode_attn_weights_fp4(const void* q, int64_t q_row_stride, const void* key, const void* value,
                                int64_t key_row_stride, int64_t value_row_stride, const int32_t* slot_mapping,
                                void* k_cache, void* v_cache, int64_t num_blocks, int block_size,
                                const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                const int32_t* context_lens, int batch, int num_heads, int num_kv_heads, int head_dim,
                                float softmax_scale, float* key_weights, const int32_t* weight_rows,
                                int64_t num_weight_rows, int64_t weight_width, void* scores, size_t scores_bytes, int plan,
                                void* workspace, size_t workspace_bytes, void* out, void* stream);

/* vox_prefill_attn with cu_seqlens, causal, that also adds what every key received: the last cu_seqlens_q[b + 1] -
 * cu_seqlens_q[b] tokens of a sequence are the step's own, and their weights become it, the earlier ones' grow by it. A
 * sequence without queries keeps its weights. max_seqlen_k: no sequence has more keys (further ones are left out of the
 * weights). num_tokens: the rows that q and out hold. Paged blocks are a multiple of 64 tokens. scratch:
 * vox_prefill_weights_bytes bytes (16-byte aligned), the call's own. plan, workspace: as vox_prefill_attn's; with the workspace
 * (NULL: none) the one-query sequences of a paged call run on the decode kernels, and scores is vox_decode_scores_bytes bytes
 * of scratch. */
size_t vox_prefill_weights_bytes(int64_t num_tokens, int batch, int max_seqlen_q, int max_seqlen_k, int num_heads,
                                 int num_kv_heads);
int vox_prefill_attn_weights(const void* q, int64_t q_row_stride, const void* key, const void* value,
                             int64_t key_row_stride, int64_t value_row_stride, const void* k_cache, const void* v_cache,
                             int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                             int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                             int max_seqlen_q, int max_seqlen_k, int64_t num_tokens, int num_heads, int num_kv_heads,
                             int head_dim, float softmax_scale, float* key_weights, const int32_t* weight_rows,
                             int64_t num_weight_rows, int64_t weight_width, void* scratch,
                             size_t scratch_bytes, void* scores, size_t scores_bytes, int plan, void* workspace,
                             size_t workspace_bytes, void* out, int64_t out_row_stride, void* stream);

/* The same over 4-bit caches through a block table, as vox_prefill_attn_fp4; scores as vox_decode_attn_weights_fp4's, in the
 * sums that a chunk's probabilities are divided by: those of one query add up to 1 within e^x - 1. */
int vox_prefill_attn_weights_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                 int64_t num_blocks, int block_size, const int32_t* block_tables, int64_t bt_stride,
                                 int max_blocks, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                                 int max_seqlen_q, int max_seqlen_k, int64_t num_tokens, int num_heads,
                                 int num_kv_heads, int head_dim, float softmax_scale, float* key_weights,
                                 const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width,
                                 void* scratch, size_t scratch_bytes, void* scores, size_t scores_bytes, int plan,
                                 void* workspace, size_t workspace_bytes, void* out, int64_t out_row_stride,
                                 void* stream);

/* For a step with fewer queries than new tokens, ahead of its vox_prefill_attn_weights (which takes as many tokens of a sequence
 * as it has queries for the step's own): sets the weights of the last cu_seqlens_new[b + 1] - cu_seqlens_new[b] (int32 [batch +
 * 1]) tokens of sequence b's cu_seqlens_k[b + 1] - cu_seqlens_k[b] to 0. max_keys: what the block tables reach (a longer
 * sequence ends there; packed keys: INT32_MAX); tokens at or past max_tokens are left alone. */
int vox_clear_key_weights(float* key_weights, const int32_t* weight_rows, int64_t num_weight_rows, int64_t weight_width,
                          int num_kv_heads, const int32_t* cu_seqlens_new, const int32_t* cu_seqlens_k, int batch,
                          int max_keys, int max_tokens, void* stream);

/* Drops tokens from sequences longer than `budget`: their first `sinks` and last `recent` tokens stay and, in every layer
 * and kv head apart, the budget - sinks - recent heaviest of the others by key_weights (fp32 [num_layers, num_weight_rows,
 * num_kv_heads, weight_width], weight_width >= max_blocks * block_size; of equal ones the earliest, NaN above every number).
 * They move in their order to the first `budget` slots of the sequence, their weights to the first places of its row; what
 * lies behind keeps what it held. A sequence within the budget, or without a row of weights, stays as it is.
 *   kv           [num_layers][2][num_blocks] blocks: block_size slots of num_kv_heads * head_bytes, then block_size slots of
 *                num_kv_heads * scale_bytes; head_bytes a multiple of 16, scale_bytes 0 or 4; num_blocks * block_size < 2^31
 *   into         int32 [batch, into_stride] or NULL: where into[b][c] is not negative, block c of what sequence b keeps is
 *                that one, which no table of the call names, in place of its own (which then stays as it was). Blocks that
 *                several rows name need it in every row that is over the budget.
 *   moves        int32 [num_layers, batch, num_kv_heads, min(budget, max_blocks * block_size) + 1, 2], 8-byte aligned: scratch
 *   new_tables   int32 [batch, max_blocks]: the blocks still in use, -1 behind them; new_lens int32 [batch]
 * A context past what max_blocks blocks hold counts as that. Tokens whose block, or whose new block, is not one of the cache
 * are not moved: their new slots keep what they held. */
int vox_evict_kv_tokens(void* kv, int64_t num_layers, int64_t num_blocks, int block_size, int num_kv_heads, int head_bytes,
                        int scale_bytes, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                        const int32_t* context_lens, int batch, float* key_weights, const int32_t* weight_rows,
                        int64_t num_weight_rows, int64_t weight_width, int budget, int sinks, int recent,
                        const int32_t* into, int64_t into_stride, int32_t* moves, int32_t* new_tables, int32_t* new_lens,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif /* VOX_ATTN_H_ */
