/* C ABI of the MI355X continuous-depth-batching decode-step kernels.
 *
 * Every entry point takes plain device pointers, element counts and an
 * explicit hipStream_t, allocates nothing, and returns CDB_OK (0) or a
 * negative CDB_ERR_* code; no C++ exception crosses this boundary. All
 * buffers are owned by the caller, so every call is capturable into a HIP
 * graph. Tensors are dense and row-major; "dtype" selects fp32 or bf16
 * storage for activations, weights and KV pages (accumulation is fp32).
 *
 * Paged KV layout: cache layer l's keys are the rows of
 *   k_pool + l * layer_stride  viewed as [pool_blocks * block_size, Hkv, D]
 * (values likewise from v_pool), which is the reference's per-layer cache
 * tensor shape (continuous_batching/cache.py:131-144). Token position t of a
 * sequence lives at row block_table[t / block_size] * block_size + t % block_size
 * (continuous_batching/cache_manager.py:190-213).
 */
#ifndef CDB_AMD_H_
#define CDB_AMD_H_

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  CDB_OK = 0,
  CDB_ERR_NULL = -1,        /* a required pointer is null */
  CDB_ERR_SHAPE = -2,       /* an extent or stride is out of range */
  CDB_ERR_UNSUPPORTED = -3, /* dtype / head_dim combination not compiled */
  CDB_ERR_HIP = -4,         /* a HIP launch failed */
  CDB_ERR_CAPACITY = -5     /* a caller buffer is too small */
};

enum { CDB_DTYPE_F32 = 0, CDB_DTYPE_BF16 = 1 };

/* Bytes of decode workspace for num_rows rows whose new-token positions are
 * all < max_seqlen with chunks of split_pages pages: an int32 header of
 * num_rows + 2 entries padded to 256 bytes, 1 KiB of work-queue counters and
 * one int32 arrival counter per (row, head) padded to 256 bytes (all zeroed by
 * the plan), then per chunk a 64-byte descriptor and an
 * fp32 partial of num_heads * (head_dim + 2) floats. A smaller workspace is
 * legal as long as it holds the header and one chunk per row: the plan then
 * lengthens the chunks until they fit. Returns -1 on bad input. */
int64_t cdb_paged_decode_workspace_bytes(int32_t num_rows, int32_t num_heads, int32_t head_dim, int32_t max_seqlen,
                                         int32_t block_size, int32_t split_pages);

/* Mixed-depth paged decode attention with fused RoPE and KV append.
 *
 * Replaces flash_attn_with_kvcache as called by the reference's paged decode
 * branch (transformers integrations/flash_paged.py:100-147, reached from
 * ouro/modeling_ouro.py:407-428 and huginn/modeling_huginn.py:275-300), plus
 * the RoPE applied just before it (ouro/modeling_ouro.py:179-204 split-half,
 * rope_style 1; huginn/modeling_huginn.py:178-196 interleaved, rope_style 2).
 *
 * q [B,H,D], k_new/v_new [B,Hkv,D] are the un-rotated projections of the
 * batch's new tokens. Row b appends its rotated key and its value at position
 * p = seqlens[b] (FA's cache_seqlens) in cache layer cache_layer0 + cache_layer[b]
 * (cache_layer0 alone when cache_layer is null: a row's KV slot offset
 * slot*num_layers goes in cache_layer, the physical layer in cache_layer0) and attends over
 * positions 0..p with softmax scale `scale`. seqlens[b] < 0 marks a padding
 * row (no KV write, zero output). Block table row for batch row b is
 * table_row[b] (or b when null). rope_cos/rope_sin are [max_positions, D/2]
 * fp32 tables holding the values the reference's rotary module produces
 * (rounded to the model dtype for Ouro); rope_style 0 applies no rotation.
 * q_bias [H,D] / k_bias [Hkv,D] are optional pre-rotation biases (Huginn's
 * qk_bias). Rows whose position or cache layer is out of range get a NaN
 * output and no KV write. workspace: cdb_paged_decode_workspace_bytes(...).
 * q_stride / kv_stride: elements between consecutive rows of q and of
 * k_new/v_new (0 = dense), so q, k and v may be column slices of one fused
 * QKV projection output.
 * Each row's context is cut into chunks of split_pages pages (min_split_pages
 * when split_pages <= 0), processed in parallel and merged in chunk order, so a row's output does not
 * depend on which other rows share the launch. Only a workspace too small for
 * the launch's chunks lengthens them.
 * Returns CDB_ERR_CAPACITY when workspace_bytes cannot hold the header and one
 * chunk per row. */
int cdb_paged_decode_attention(const void* q, const void* k_new, const void* v_new, void* k_pool, void* v_pool,
                               int64_t layer_stride, int32_t num_cache_layers, int64_t pool_blocks,
                               const int32_t* cache_layer, int32_t cache_layer0, const int32_t* block_table,
                               const int32_t* table_row, int32_t table_width, const int32_t* seqlens,
                               const float* rope_cos, const float* rope_sin, int32_t rope_style,
                               int32_t max_positions, const void* q_bias, const void* k_bias, void* out,
                               void* workspace, int64_t workspace_bytes, int32_t num_rows, int32_t num_heads,
                               int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t split_pages,
                               int32_t min_split_pages, float scale,
                               int64_t q_stride, int64_t kv_stride, int32_t dtype, hipStream_t stream);

/* Stages of cdb_paged_decode_attention_staged. */
enum { CDB_DECODE_STAGE_PLAN = 1, CDB_DECODE_STAGE_ATTEND = 2 };

/* cdb_paged_decode_attention in two stages, for a batch whose rows run through
 * several layers with the same positions (seqlens), table rows (table_row) and
 * cache-layer offsets (cache_layer), as the reference's recurrent stage runs its
 * rows through every layer of the loop block (continuous_api.py:1171-1183,
 * ouro/modeling_ouro.py:407-428). CDB_DECODE_STAGE_PLAN writes the chunk plan
 * of those rows into the workspace; CDB_DECODE_STAGE_ATTEND runs attention and
 * the merge from the plan last written to this workspace, which must describe
 * the same rows (only cache_layer0, q/k/v, the pools and out may differ).
 * stages = PLAN | ATTEND is cdb_paged_decode_attention. Arguments and errors as
 * cdb_paged_decode_attention; CDB_ERR_SHAPE for any other stages value. */
int cdb_paged_decode_attention_staged(const void* q, const void* k_new, const void* v_new, void* k_pool,
                                      void* v_pool, int64_t layer_stride, int32_t num_cache_layers,
                                      int64_t pool_blocks, const int32_t* cache_layer, int32_t cache_layer0,
                                      const int32_t* block_table, const int32_t* table_row, int32_t table_width,
                                      const int32_t* seqlens, const float* rope_cos, const float* rope_sin,
                                      int32_t rope_style, int32_t max_positions, const void* q_bias,
                                      const void* k_bias, void* out, void* workspace, int64_t workspace_bytes,
                                      int32_t num_rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                      int32_t block_size, int32_t split_pages, int32_t min_split_pages, float scale,
                                      int64_t q_stride, int64_t kv_stride, int32_t dtype, int32_t stages,
                                      hipStream_t stream);

/* No counterpart in the reference. cdb_paged_decode_attention for callers that cannot allocate
 * device memory: code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc. Same arguments and results without the workspace: the split header and partials
 * live in a fixed device array of CDB_DECODE_SCRATCH_BYTES per GPU (resolved once per device,
 * held until the process ends). The call allocates nothing and frees nothing. Nothing in the
 * scratch must start at zero: each call's plan writes its header and zeroes its counters before
 * the decode kernel reads them.
 * Every call on one GPU shares that GPU's array, so calls that overlap on one GPU (two streams,
 * or two threads) race; serialize them. Returns CDB_ERR_CAPACITY when the header plus one
 * chunk per row (a 64-byte descriptor and num_heads * (head_dim + 2) floats) exceeds the
 * scratch after the header, queue counters and arrival counters (at 16 heads x 128: more than
 * 1984 rows); a smaller surplus only lengthens the chunks. */
#define CDB_DECODE_SCRATCH_BYTES ((int64_t)16 << 20)
int cdb_paged_decode_attention_noalloc(const void* q, const void* k_new, const void* v_new, void* k_pool,
                                       void* v_pool, int64_t layer_stride, int32_t num_cache_layers,
                                       int64_t pool_blocks, const int32_t* cache_layer, int32_t cache_layer0,
                                       const int32_t* block_table, const int32_t* table_row, int32_t table_width,
                                       const int32_t* seqlens, const float* rope_cos, const float* rope_sin,
                                       int32_t rope_style, int32_t max_positions, const void* q_bias,
                                       const void* k_bias, void* out, int32_t num_rows, int32_t num_heads,
                                       int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                       int32_t split_pages, int32_t min_split_pages,
                                       float scale, int64_t q_stride, int64_t kv_stride, int32_t dtype,
                                       hipStream_t stream);

/* Fused RMSNorm sandwich over rows of `width` elements.
 *   norm_w(x) = R(w * R(x * rsqrt(mean(x^2) + eps)))  (R rounds to the storage dtype)
 *   mode 0: out_h = norm_a(x)
 *   mode 1: out_h = R(residual + norm_a(x)); out_y = norm_b(out_h)   (Ouro layer,
 *           ouro/modeling_ouro.py:445-450 and :481-502)
 *   mode 2: out_h = norm_a(R(residual + x)); out_y = norm_b(out_h)   (Huginn block,
 *           huginn/modeling_huginn.py:141-146 and :335-338)
 * out_y is written only when w_b is non-null. out_h may alias x or residual. */
int cdb_rmsnorm_fused(const void* x, const void* residual, const void* w_a, const void* w_b, void* out_h,
                      void* out_y, int64_t rows, int32_t width, int32_t mode, float eps_a, float eps_b,
                      int32_t dtype, hipStream_t stream);

/* cdb_rmsnorm_fused with x given as the fp32 split-K partials of the projection
 * that produces it (cdb_linear_parts): x[r, c] = R(sum over s < splits, in
 * order, of x_parts[s, r, c]), the projection's own rounded output, then the
 * same modes as cdb_rmsnorm_fused. bf16 only; x_parts [splits, rows, width]
 * contiguous and 16-byte aligned; 1 <= splits <= 64. Fuses the O and down
 * projections' outputs into the residual norms that follow them
 * (ouro/modeling_ouro.py:168,431 into :445-450 and :481-502). */
int cdb_rmsnorm_fused_parts(const float* x_parts, int32_t splits, const void* residual, const void* w_a,
                            const void* w_b, void* out_h, void* out_y, int64_t rows, int32_t width, int32_t mode,
                            float eps_a, float eps_b, int32_t dtype, hipStream_t stream);

/* out[r, :] = R(R(silu(g)) * u) for gate_up[r] = [g | u] of 2*width elements
 * (ouro/modeling_ouro.py:167-169, huginn/modeling_huginn.py:314-316). */
int cdb_silu_mul(const void* gate_up, void* out, int64_t rows, int32_t width, int32_t dtype, hipStream_t stream);

/* Row gather/scatter: dst[dst_index[i]] = src[src_index[i]] for i < rows, rows of
 * row_bytes bytes (a multiple of 4). A null index means the identity; a negative
 * (or out-of-range) src index writes zeros; a negative dst index skips the row.
 * Replaces the hidden-bank index_select/index_copy_ of cdb/model_runner.py:685-693,
 * :559 and :1101, the embedding lookup of cdb/adapters/ouro.py:199-212 and the
 * device token gather of cdb/model_runner.py:439-457. */
int cdb_copy_rows(const void* src, const int64_t* src_index, int64_t src_rows, void* dst, const int64_t* dst_index,
                  int64_t dst_rows, int64_t rows, int64_t row_bytes, hipStream_t stream);

/* Block-table cell updates with the count in device memory: table[idx[i]] = val[i]
 * for i < min(*count, capacity); cells outside [0, cells) are skipped. It lets a
 * launch's metadata upload carry the table cells its rows' new blocks changed and
 * a captured graph apply them, in place of a separate flush
 * (the block-table refresh of cdb/cache.py:115-144, cache_manager.py:72-90). */
int cdb_table_updates(int32_t* table, int64_t cells, const int64_t* idx, const int32_t* val, const int32_t* count,
                      int32_t capacity, hipStream_t stream);

/* Exit routing of one recurrent launch on the device, in launch order: writes
 * lists = [n_exit, n_stay, the n_exit exiting rows, the n_stay staying rows], the
 * rows being indices into the launch (exit_flags[r] != 0: row r leaves for the coda)
 * and rows with a negative bank slot (padding) in neither list. Replaces the
 * per-row routing pass over the launch's decisions on the synchronous horizon
 * (cdb/continuous_api.py:1171-1183 after cdb/model_runner.py:694-699,796-821):
 * exiting rows go to the coda queue in this order, staying rows back to the head of
 * the depth queue in this order. lists holds 2 + rows ints. */
int cdb_route_compact(const uint8_t* exit_flags, const int64_t* bank_slots, int32_t rows, int32_t* lists,
                      hipStream_t stream);

/* Greedy sampling: out[r] = first index of the maximum of logits[r, :vocab]
 * (torch.argmax semantics incl. NaN; cdb/model_runner.py:1062,1105). */
int cdb_argmax(const void* logits, int64_t* out, int64_t rows, int32_t vocab, int32_t dtype, hipStream_t stream);

/* Early-exit gate and decision for one recurrent launch.
 * kind 0: signal[b] = R(hidden[b] . weight + bias) -- Ouro's Linear(E,1) gate
 *         (cdb/adapters/ouro.py:286-291);
 * kind 1: signal[b] = R(||hidden[b] - prev[b]|| / max(||hidden[b]||, 1e-9)) --
 *         Huginn's latent difference (huginn/exit_gates.py:33-40).
 * The token policy state (fp64 cdf/survival, pending signal) is kept in arrays
 * of state_capacity entries indexed by state_index[b] (< 0: padding row). The
 * decision follows cdb/exit_policy.py:150-169 and cdb/continuous_api.py:1671-1724:
 * forced exit at step max_steps-1; a replayed synthetic_depth[b] >= 0 exits at
 * step >= depth; otherwise, with has_threshold, rule 0 accumulates the sigmoid
 * hazard (rounded to the storage dtype when round_hazard) into the cdf and exits
 * when cdf >= threshold, rule 1 exits when signal < threshold, both only once
 * step+1 >= min_steps. delayed=1 decides on the previous launch's signal
 * (DecisionHorizon.OFFSET_ONE). exit_flags[b] is 1 for an exit. */
int cdb_exit_gate(const void* hidden, const void* prev, const void* weight, const void* bias, void* signal,
                  double* cdf, double* survival, float* pending, int64_t state_capacity, const int64_t* state_index,
                  const int32_t* steps, const int32_t* synthetic_depth, uint8_t* exit_flags, int64_t rows,
                  int32_t width, int32_t kind, int32_t rule, int32_t delayed, int32_t round_hazard,
                  int32_t min_steps, int32_t max_steps, double threshold, int32_t has_threshold, int32_t dtype,
                  hipStream_t stream);

/* Reset the gate state of n fresh tokens: cdf 0, survival 1, no pending signal
 * (TokenExitPolicyState(), cdb/exit_policy.py:43-48). */
int cdb_exit_gate_reset(double* cdf, double* survival, float* pending, int64_t state_capacity,
                        const int64_t* index, int64_t n, hipStream_t stream);

/* Copy-on-exit KV propagation (kv_policy "last_exited"): for token i at pool row
 * rows[i] that exited at KV slot exit_slot[i], copy its K and V rows from cache
 * layer layer_base + exit_slot*core_layers + l to layer_base + s*core_layers + l
 * for every core layer l and every deeper slot s < num_slots
 * (cdb/continuous_api.py:1225-1245, kv_cache_policy.py:235-258, cdb/cache.py:105-113). */
int cdb_exit_kv_copy(void* k_pool, void* v_pool, int64_t layer_stride, int64_t pool_rows, int32_t num_kv_heads,
                     int32_t head_dim, const int64_t* rows, const int32_t* exit_slot, int64_t n, int32_t layer_base,
                     int32_t core_layers, int32_t num_slots, int32_t dtype, hipStream_t stream);

/* Prefill-side RoPE + paged KV write for T tokens: q_out = rotate(q [+ q_bias]);
 * rotate(k [+ k_bias]) and v are written to cache layer `layer` at pool rows
 * rows[t] (negative rows write nothing). Replaces the write half of
 * PagedAttentionCache.update (continuous_batching/cache.py:284-318) and the
 * RoPE before it. q, k and v may be column slices of one fused QKV output:
 * q_stride / kv_stride are the elements between consecutive tokens (0: dense
 * [T, H, D] / [T, Hkv, D]); q_out is dense. */
int cdb_rope_kv_write(const void* q, const void* k, const void* v, void* q_out, void* k_pool, void* v_pool,
                      int64_t layer_stride, int32_t layer, const int64_t* rows, int64_t pool_rows,
                      const int32_t* positions, const float* rope_cos, const float* rope_sin, int32_t rope_style,
                      int32_t max_positions, const void* q_bias, const void* k_bias, int64_t tokens,
                      int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int64_t q_stride, int64_t kv_stride,
                      int32_t dtype, hipStream_t stream);

/* Varlen causal prefill attention over the paged pool on MFMA tiles.
 * Replaces flash_attn_varlen_func as the reference's prefill calls it after
 * the chunk's KV write (continuous_batching/prefill_graph.py:265-309,
 * transformers integrations/flash_paged.py:62-86). Sequence s has query tokens
 * cu_q[s] .. cu_q[s+1]-1 of q [T,H,D] (already rotated) at positions
 * past[s] + i; each attends to positions 0..(its own) of cache layer `layer`
 * through block-table row table_row[s]. The chunk's own K/V must already be in
 * the pool. Work is split into tiles of 128 query tokens: tile n covers
 * sequence tile_seq[n], queries tile_q0[n] .. +127. out is [T,H,D]. scale must
 * be positive and finite (CDB_ERR_SHAPE otherwise). */
int cdb_prefill_attention(const void* q, const void* k_pool, const void* v_pool, int64_t layer_stride, int32_t layer,
                          int32_t num_cache_layers, int64_t pool_blocks, const int32_t* block_table,
                          const int32_t* table_row, int32_t table_width, const int32_t* cu_q, const int32_t* past,
                          int32_t num_seqs, const int32_t* tile_seq, const int32_t* tile_q0, int32_t num_tiles,
                          void* out, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                          float scale, int32_t dtype, hipStream_t stream);

/* Bytes of the partial-result buffer cdb_prefill_attention_split needs for
 * num_slots partial slots (-1 for invalid arguments). No reference counterpart:
 * a sizing helper for the split work list below. */
int64_t cdb_prefill_partial_bytes(int32_t num_slots, int32_t num_heads, int32_t head_dim);

/* cdb_prefill_attention with the key range of long tiles split over several
 * workgroups (bf16 only), so that one long sequence does not set the length of
 * the whole launch; same operation, same outputs up to fp32 rounding of the
 * merge. Replaces the same flash_attn_varlen_func call as cdb_prefill_attention
 * (continuous_batching/prefill_graph.py:265-309).
 *   items  [num_items][4] int32: (sequence, first query of the 128-query tile,
 *          first key block | end key block << 16 (blocks of 32 keys),
 *          partial slot, or -1 for a whole tile written straight to out).
 *          A part must not start past the tile's first query position.
 *   merges [num_merges][4] int32: (sequence, first query, first slot, parts):
 *          the parts of one split tile occupy consecutive slots.
 *   partials: cdb_prefill_partial_bytes(num_slots, ...) bytes of scratch.
 * Two launches on `stream`: the tiles and parts, then the merge. */
int cdb_prefill_attention_split(const void* q, const void* k_pool, const void* v_pool, int64_t layer_stride,
                                int32_t layer, int32_t num_cache_layers, int64_t pool_blocks,
                                const int32_t* block_table, const int32_t* table_row, int32_t table_width,
                                const int32_t* cu_q, const int32_t* past, int32_t num_seqs, const int32_t* items,
                                int32_t num_items, const int32_t* merges, int32_t num_merges, int32_t num_slots,
                                void* partials, int64_t partials_bytes, void* out, int32_t num_heads,
                                int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                int32_t dtype, hipStream_t stream);

/* Repack a bf16 weight w [rows, in_features] (row stride ldw) into the operand
 * order cdb_linear reads: for each tile of 16 rows and each 32-element step of
 * in_features, a contiguous 1 KiB block whose 16-byte unit l holds
 * w[16 t + l % 16][32 s + 8 (l / 16) .. +8]; tiles follow each other, steps
 * within a tile likewise. w_packed holds rows * in_features elements. rows must
 * be a multiple of 16 and in_features of 32. Run once per weight at load time. */
int cdb_linear_pack_weight(const void* w, int64_t ldw, void* w_packed, int64_t rows, int32_t in_features,
                           int32_t dtype, hipStream_t stream);

/* Dense projection of a decode batch: y[r, n] = R(sum_k x[r, k] * w[n, k]) for
 * r < rows, n < out_features, bf16 only (fp32 accumulation, one rounding),
 * with w given packed by cdb_linear_pack_weight. rows <= 64, or up to 256 when
 * in_features is 2048 and out_features a multiple of 128 of at least 4096, or
 * up to 128 when in_features is 5280 and out_features at least 4096 (a
 * streaming kernel); other shapes above 64 rows return CDB_ERR_SHAPE.
 * Replaces the nn.Linear calls of a recurrent step (ouro/modeling_ouro.py:162-168,
 * :371-374,390-392,431; huginn/modeling_huginn.py:239-242,310-316,372).
 * gated != 0: w holds 2*out_features rows, gate rows then up rows (the MLP's
 * concatenated gate/up projection), and y[r, n] = R(R(silu(g)) * u) with
 * g = R(x.w[n]) and u = R(x.w[out_features + n]) (ouro/modeling_ouro.py:168,
 * huginn/modeling_huginn.py:315-316). Row strides ldx, ldy are in elements
 * (multiples of 8 and 4); out_features must be a multiple of 16 and
 * in_features a multiple of 32. */
int cdb_linear(const void* x, int64_t ldx, const void* w_packed, void* y, int64_t ldy, int32_t rows,
               int32_t out_features, int32_t in_features, int32_t gated, int32_t dtype, hipStream_t stream);

/* Number of K ranges cdb_linear_parts splits a projection of this shape into,
 * or 0 when it has no split form for it (then use cdb_linear or a library GEMM).
 * Split forms exist for bf16 with in_features 2048 (up to 128 rows) or 5632 (up
 * to 256 rows) and out_features a multiple of 64 -- the Ouro O and down
 * projections (ouro/modeling_ouro.py:168,431) -- and with in_features 5280 or
 * 17920 (up to 256 rows) and out_features a multiple of 16 -- the Huginn O and
 * down projections (huginn/modeling_huginn.py:242,302,311,316). */
int32_t cdb_linear_parts_splits(int64_t rows, int32_t out_features, int32_t in_features, int32_t dtype);

/* Split-K projection: parts[s, r, n] = fp32 sum over k in the s-th of
 * splits = cdb_linear_parts_splits(...) equal K ranges of x[r, k] * w[n, k],
 * unrounded, for the consumer to add in order and round once
 * (cdb_rmsnorm_fused_parts). w packed by cdb_linear_pack_weight; parts holds
 * parts_elems >= splits * rows * out_features floats, 16-byte aligned; x row
 * stride ldx a multiple of 8 elements. Shapes without a split form return
 * CDB_ERR_SHAPE. Same projections as cdb_linear (ouro/modeling_ouro.py:168,431). */
int cdb_linear_parts(const void* x, int64_t ldx, const void* w_packed, float* parts, int64_t parts_elems,
                     int32_t rows, int32_t out_features, int32_t in_features, int32_t dtype, hipStream_t stream);

/* Workspace bytes cdb_linear_argmax needs: rows * (out_features / 16) * 8
 * (-1 for invalid sizes). */
int64_t cdb_linear_argmax_workspace_bytes(int32_t rows, int32_t out_features);

/* Greedy coda in one call: out[r] = the first n maximizing R(sum_k x[r, k] *
 * w[n, k]) over n < out_features, NaN counting as the maximum (torch.argmax over
 * the bf16 logits). It replaces lm_head followed by argmax
 * (cdb/model_runner.py:1062,1105; ouro/modeling_ouro.py:755-775). The logits
 * are never stored. The projection kernel keeps, per row and 16-column tile,
 * the best rounded value and its column in `workspace`; a second kernel
 * combines them. bf16, w packed by cdb_linear_pack_weight, 1 <= rows <= 64,
 * out_features a multiple of 16, in_features a multiple of 32, ldx a multiple
 * of 8; workspace 16-byte aligned, at least cdb_linear_argmax_workspace_bytes
 * bytes (CDB_ERR_CAPACITY otherwise).
 * With embed non-null ([out_features, width] bf16, the token embedding) the
 * same call also runs the next token's prelude for rows with a successor:
 * bank[bank_slots[r]] = embed[out[r]] when 0 <= bank_slots[r] < bank_rows --
 * the eager re-entry's embedding lookup (cdb/model_runner.py:439-457,
 * cdb/adapters/ouro.py:199-212) fused into the coda. embed and bank 16-byte
 * aligned, width a multiple of 8. */
int cdb_linear_argmax(const void* x, int64_t ldx, const void* w_packed, int64_t* out, void* workspace,
                      int64_t workspace_bytes, int32_t rows, int32_t out_features, int32_t in_features,
                      const void* embed, void* bank, int64_t bank_rows, const int64_t* bank_slots, int32_t width,
                      int32_t dtype, hipStream_t stream);

/* One greedy coda tick in a single call on `stream`, replacing the coda stage's
 * slot upload, hidden-row gather, LM head + argmax, token download and the
 * successors' gate-state reset (cdb/model_runner.py:1036-1125, 439-457,
 * 1359-1363; cdb/exit_policy.py:43-48):
 *   1. dev_upload[:count] = host_upload[:count] (pinned host memory), where the
 *      upload is [coda rows' bank slots (rows) | each row's successor bank slot
 *      or -1 (rows) | the successors' slots (num_successors)] when embed is given
 *      and only the first part otherwise (count = 2*rows + num_successors or rows);
 *   2. hidden[r] = bank[dev_upload[r]]  (hidden: [rows, width] device scratch);
 *   3. cdb_linear_argmax over hidden (ldx = in_features = width) into tokens,
 *      with the successors' embedding rows written when embed is given;
 *   4. host_tokens[:rows] = tokens  (pinned host memory, asynchronous);
 *   5. the gate state of the num_successors successor slots is reset.
 * The same preconditions as cdb_linear_argmax apply (bf16, 1 <= rows <= 64). The
 * host buffers must stay untouched until the stream has passed this call. */
int cdb_coda_greedy(const int64_t* host_upload, int64_t* dev_upload, int32_t rows, int32_t num_successors,
                    void* bank, int64_t bank_rows, int32_t width, void* hidden, const void* w_packed, int32_t vocab,
                    int64_t* tokens, void* workspace, int64_t workspace_bytes, const void* embed,
                    int64_t* host_tokens, double* cdf, double* survival, float* pending, int64_t state_capacity,
                    int32_t dtype, hipStream_t stream);

/* ---- 8-bit KV cache ------------------------------------------------------------------------------------------
 * No counterpart in the reference, whose cache holds the model's type. Keys and values are held in tiles of
 * 16 tokens of one KV head, as e4m3 codes with one power-of-two scale a tile, keys and values apart:
 *   codes  [num_cache_layers, 2, pool_blocks, Hkv, block_size / 16, 16 * D] bytes, 16-byte aligned;
 *   scales [num_cache_layers, 2, pool_blocks, Hkv, block_size / 16] bytes b, the scale being 2^(b - 127); written ones
 *          are 1 to 254. A byte of 0, as in a pool of zeros, is read as 1 and one of 255 as 254.
 * A key tile lies as [D / 16][16 tokens][16], a value tile as [4][D][4 tokens]. block_size is a power of two
 * of at least 16; D is 64, 96 or 128; the codes need no address below 2^63 bytes, and offsets are 64-bit.
 * Position t of a sequence is token t % 16 of tile t % block_size / 16 of block block_table[t / block_size].
 *
 * Writing: a tile's scale is the smallest power of two s with |x| <= 448 s for the finite values written
 * (2^-126 at least). Tokens that join a tile behind earlier ones keep the larger of its scale and theirs, and
 * where it grows the earlier codes are rounded again. A tile written from its first token starts anew. Codes
 * behind the last token written stay as they are, and count for nothing. An infinity or NaN is held as NaN.
 * Rotations are computed in fp32, each product and sum rounded once, and not rounded to the storage type
 * before they are coded. Scores past fp32's range are infinities, or NaN from 2^132 on. */

/* Rotate and append a batch of tokens: q_out = rotate(q [+ q_bias]); rotate(k [+ k_bias]) and v are coded into
 * cache layer `layer` at slots rows[t] = block * block_size + offset. The 8-bit counterpart of
 * cdb_rope_kv_write, with its q/k/v views, strides, rotation styles and biases. The tokens of one tile follow
 * each other in the call at consecutive slots, as a sequence's tokens do; a slot is written once in a call. Tokens
 * with a negative slot are padding: nothing of theirs is read or written, q_out included. A slot past the pool
 * or a position outside the angle tables writes no key or value (and NaN to q_out for such a position). A token left
 * out in one of these ways between others of its tile keeps its place in the call, the next one's slot being two
 * further: its codes stay as they were, and the others share one scale as if they followed each other.
 * num_heads 0 (q and q_out null) writes keys and values alone. q_out is dense and 16-byte aligned. */
int cdb_kv8_write(const void* q, const void* k, const void* v, void* q_out, void* codes, void* scales,
                  int32_t num_cache_layers, int64_t pool_blocks, int32_t layer, const int64_t* rows,
                  const int32_t* positions, const float* rope_cos, const float* rope_sin, int32_t rope_style,
                  int32_t max_positions, const void* q_bias, const void* k_bias, int64_t tokens, int32_t num_heads,
                  int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int64_t q_stride, int64_t kv_stride,
                  int32_t dtype, hipStream_t stream);

/* Workspace bytes of cdb_kv8_decode_attention for positions below max_seqlen (-1 for invalid arguments): per row
 * and chunk of 1024 tokens (64 chunks at most) an fp32 partial of head_dim + 2 values a query head and 8 bytes a
 * KV head. A smaller workspace is legal down to one chunk a row: it has partials for workspace_bytes / num_rows, and
 * rows with more chunks take longer ones. Nothing in it need be set before a call; calls that may overlap need one
 * each. */
int64_t cdb_kv8_decode_workspace_bytes(int32_t num_rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                       int32_t max_seqlen);

/* Mixed-depth paged decode attention over the 8-bit cache, with fused rotation and append: the counterpart of
 * cdb_paged_decode_attention, with its rows, positions (seqlens), per-row cache layers, block table, biases and
 * padding rows. Row b's new key and value are coded into its cache first, and it attends over the codes of
 * positions 0..seqlens[b], its own included. Rows whose position, table row or cache layer is out of range get a
 * NaN output and no write; a row with a block in use outside the pool gets NaN, and writes its token where the
 * token's own block is inside. num_heads is a multiple of num_kv_heads. Two rows of a call never append to the same
 * tile, and none reads a tile that another appends to. A row's context is cut into chunks of 1024 tokens (64 at most,
 * longer ones past that), merged in order, so its output does not depend on the other rows: with a workspace that the
 * function above gives for at least the call's rows and positions. With a smaller one the chunks of rows that it is
 * short for, and so their rounding, depend on num_rows too. */
int cdb_kv8_decode_attention(const void* q, const void* k_new, const void* v_new, void* codes, void* scales,
                             int32_t num_cache_layers, int64_t pool_blocks, const int32_t* cache_layer,
                             int32_t cache_layer0, const int32_t* block_table, const int32_t* table_row,
                             int32_t table_rows, int32_t table_width, const int32_t* seqlens, const float* rope_cos,
                             const float* rope_sin, int32_t rope_style, int32_t max_positions, const void* q_bias,
                             const void* k_bias, void* out, void* workspace, int64_t workspace_bytes,
                             int32_t num_rows, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                             int32_t block_size, float scale, int64_t q_stride, int64_t kv_stride, int32_t dtype,
                             hipStream_t stream);

/* Workspace bytes of cdb_kv8_prefill_attention (0 for splits == 1; -1 for invalid arguments): per tile, split and
 * head an fp32 partial of 128 * (head_dim + 2) values. */
int64_t cdb_kv8_prefill_workspace_bytes(int32_t num_tiles, int32_t splits, int32_t num_heads, int32_t head_dim);

/* Varlen causal prefill attention over the 8-bit cache: the counterpart of cdb_prefill_attention, with its
 * sequences, block table and tiles of 128 query tokens (tile_seq[n] < 0: no tile). q [T, H, D] is rotated; the
 * chunk's own keys and values are already in the cache. splits > 1 cuts every tile's key range into that many
 * parts (at most 64), merged in order by a second launch: for few tiles with long histories. The rounding of a
 * sequence's output depends on splits, and on nothing else of the other sequences. Queries of a sequence
 * whose table row is out of range or too short get NaN, and so do those that see a block outside the pool, with
 * the rest of their 32 in a tile. q and out are dense. */
int cdb_kv8_prefill_attention(const void* q, const void* codes, const void* scales, int32_t num_cache_layers,
                              int64_t pool_blocks, int32_t layer, const int32_t* block_table,
                              const int32_t* table_row, int32_t table_rows, int32_t table_width, const int32_t* cu_q,
                              const int32_t* past, int32_t num_seqs, const int32_t* tile_seq, const int32_t* tile_q0,
                              int32_t num_tiles, void* out, int64_t tokens, int32_t splits, void* workspace,
                              int64_t workspace_bytes, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                              int32_t block_size, float scale, int32_t dtype, hipStream_t stream);

enum {
  CDB_LAYOUT_MAX_SEQS = 4000,  /* requests of one call: their four prefixes fill 64 KB of LDS */
  /* bits of counts[3] */
  CDB_LAYOUT_TOKENS_FULL = 1,  /* more tokens than token_capacity: the rest is left out */
  CDB_LAYOUT_TILES_FULL = 2,   /* more tiles than tile_capacity: the last of the list are left out */
  CDB_LAYOUT_NO_BLOCKS = 4,    /* more new blocks than free ones: -1 in the table, slot -1 for their tokens */
  CDB_LAYOUT_BAD_REQUEST = 8   /* a negative length, one past the table's width, or a table row out of range:
                                  the request counts as one without tokens */
};

/* Block tables, slot map and attention tiles of a batch, on the device, from its requests' lengths: what the
 * engine otherwise assembles on the host for a prefill launch (continuous_batching/cache_manager.py:72-90,
 * :190-213; prefill_tiles). Request s holds past[s] tokens and brings lens[s] >= 0 more. Its
 * blocks ceil(past / block_size).. ceil((past + lens) / block_size) are taken from the front of free_blocks, in
 * request order, and written to row table_row[s] (s when null) of block_table; each request has a row of its own.
 *   cu_q [num_seqs + 1]; positions, rows [token_capacity]: position and slot of each token, -1 behind the last;
 *   tile_seq, tile_q0 [tile_capacity]: tiles of 128 query tokens, longest key range first and in request order
 *   among equals, (-1, 0) behind the last;
 *   counts [4]: tokens, tiles, blocks taken, CDB_LAYOUT_* bits. The caller drops counts[2] ids from its free list.
 * A batch of 2^31 - 1 tokens or more is counted as that many, flagged CDB_LAYOUT_TOKENS_FULL, and not laid out: the
 * table stays, and every entry is that behind the last. */
int cdb_batch_layout(const int32_t* past, const int32_t* lens, int32_t num_seqs, int32_t* block_table,
                     const int32_t* table_row, int32_t table_rows, int32_t table_width, const int32_t* free_blocks,
                     int32_t num_free, int32_t block_size, int32_t* cu_q, int32_t* positions, int64_t* rows,
                     int32_t token_capacity, int32_t* tile_seq, int32_t* tile_q0, int32_t tile_capacity,
                     int32_t* counts, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Rows that share prefixes
 * ------------------------------------------------------------------------ */

enum {
  CDB_PREFIX_QUERIES = 128,  /* queries (row, head) of an item */
  CDB_PREFIX_FEW = 16,       /* of the first num_few items: those of groups with few queries */
  CDB_PREFIX_ITEM = 8,       /* words of an item */
  CDB_PREFIX_MAX_PARTS = 64  /* parts that a prefix is cut into */
};

/* Workspace bytes of cdb_prefix_decode_attention for num_rows rows, num_items items, the first num_few of them of few
 * queries, and rows of up to max_own tokens of their own (-1 for invalid arguments). Rows with more are served too, in
 * fewer and longer chunks, whose number depends on how many rows share the workspace. */
int64_t cdb_prefix_decode_plan_workspace_bytes(int32_t num_rows, int32_t num_few, int32_t num_items, int32_t num_heads,
                                               int32_t num_kv_heads, int32_t head_dim, int32_t max_own);

/* The same where num_few is not known: enough for any. An item of few queries needs CDB_PREFIX_FEW /
 * CDB_PREFIX_QUERIES of what this counts for it. */
int64_t cdb_prefix_decode_workspace_bytes(int32_t num_rows, int32_t num_items, int32_t num_heads, int32_t num_kv_heads,
                                          int32_t head_dim, int32_t max_own);

/* cdb_paged_decode_attention for rows that begin with the same tokens, which are read once for each CDB_PREFIX_FEW or
 * CDB_PREFIX_QUERIES queries of a KV head that share them (128 rows of as many heads as KV heads: once): rotate the
 * row's new query and key, append key and value at position seqlens[b] of the row's cache layer, attend over positions
 * 0..seqlens[b]. Arguments as there, but for the plan; block_size is a power of two of at least 16, and the block table
 * has table_rows rows. Rotations are fp32: the key is rounded once, to the cache's type, and the query is not (that call
 * rounds both, in bf16 after each step, and so appends other bits in bf16).
 *
 * The rows of a group follow each other in listed; they hold the same first tokens, at the same slots of the same cache
 * layer or as copies, which are read through the table row and cache layer of the group's first row that is no padding;
 * the others are read only from there on. Queries of a group are counted row by row, the group's num_heads /
 * num_kv_heads heads of a KV head each. items [num_items][CDB_PREFIX_ITEM] (16-byte aligned) = (the group's first place
 * in listed, its rows, its first row, tokens of its prefix, first query, a multiple of the item's queries, first token,
 * end token, 0): the parts of a group's tokens for one run of queries follow each other, and the runs of a group too; 0
 * rows is no item. The first num_few items have CDB_PREFIX_FEW queries each, the others CDB_PREFIX_QUERIES. row_info
 * [num_rows][4] = (row's first query in its group, tokens of its prefix, its group's first item, parts, negative where
 * the items are of the first num_few), zeros for a row without a group. A row is listed at most once.
 *
 * A row's result depends, in its last bits, on the parts that the plan cuts its prefix into and on which of the two kinds
 * its items are, but not on what else is in the plan or the batch, while the workspace has a chunk for each 1024 of its
 * own tokens.
 *
 * A row of negative position is padding: zeros. NaN for a row, and no append, where its position is out of the table's
 * or the angles' range or inside its prefix, or its cache layer or table row out of range; NaN where its cache layer is
 * not that of the row through which its group's tokens are read, and where a block outside the pool is met, for all rows
 * of the group if it is in the prefix. A value that is infinite makes its element infinite in every row that sees the
 * token (NaN where the token's weight vanishes in fp32), a key whose score is -infinity has no weight. Calls that may
 * overlap need a workspace each. */
int cdb_prefix_decode_attention(const void* q, const void* k_new, const void* v_new, void* k_pool, void* v_pool,
                                int64_t layer_stride, int32_t num_cache_layers, int64_t pool_blocks,
                                const int32_t* cache_layer, int32_t cache_layer0, const int32_t* block_table,
                                const int32_t* table_row, int32_t table_rows, int32_t table_width,
                                const int32_t* seqlens, const float* rope_cos, const float* rope_sin,
                                int32_t rope_style, int32_t max_positions, const void* q_bias, const void* k_bias,
                                const int32_t* listed, int32_t num_listed, const int32_t* items, int32_t num_items,
                                int32_t num_few, const int32_t* row_info, void* out,
                                void* workspace, int64_t workspace_bytes, int32_t num_rows, int32_t num_heads,
                                int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                int64_t q_stride, int64_t kv_stride, int32_t dtype, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Drawing tokens
 * ------------------------------------------------------------------------ */

enum { CDB_SAMPLE_MAX_VOCAB = 1 << 20 };

/* Workspace bytes of cdb_sample (-1 for invalid arguments). */
int64_t cdb_sample_workspace_bytes(int32_t rows, int32_t vocab);

/* One token a row of logits [rows, vocab] (rows row_stride elements apart), drawn with the given numbers uniform
 * [rows] in [0, 1): beside cdb_argmax, which takes the largest. Token i weighs exp((x_i - max x) / temperature);
 * tokens are ordered by logit, the larger first and the lower index among equals.
 *   top_k: the first k of the order are kept (0 and less, or vocab and more: all);
 *   top_p: of those, the shortest beginning that holds top_p of what they weigh together, one token at least
 *   (1 and more: all);
 *   min_p: of those, the ones that weigh at least min_p times the largest (0 and less: all; 1 and more: its equals).
 * Drawn is the first kept token, by index, at which the running weight of the kept ones passes uniform times their
 * total; numbers outside [0, 1) count as the nearest inside. temperature, top_k, top_p and min_p have an entry a row,
 * or are null: 1 and no filter. A temperature not above 0 takes the first token of the order (the index cdb_argmax
 * gives, where no logit is NaN). Logits of -infinity and NaN are never drawn; where one is +infinity only such are.
 * tokens [rows]; logprobs [rows]: the logarithm of the drawn token's share of the kept weight, 0 for a token that is
 * kept alone and never above. A row without a token to draw gets -1 and -infinity. Weights are counted in units of 2^-46
 * of the largest (vocabularies above 65536: of 2^-(62 - ceil(log2 vocab))) and summed exactly, so a row's token depends
 * on nothing but the row; what weighs less than half a unit is never drawn. workspace holds nothing at present, as its
 * size says, and may be null. */
int cdb_sample(const void* logits, int64_t row_stride, const double* uniform, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, int64_t* tokens, float* logprobs,
               void* workspace, int64_t workspace_bytes, int32_t rows, int32_t vocab, int32_t dtype,
               hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* CDB_AMD_H_ */
