/* Entry points of libnvdsa.so beyond the reference's operators: parts of its
 * PyTorch functions that this library runs as kernels of their own.  Same
 * conventions as nvdsa.h (descriptors, status codes, caller-owned workspace,
 * launches on the given stream). */
#ifndef NVDSA_EXT_H
#define NVDSA_EXT_H

#include "nvdsa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The products of hidden_states that the indexer takes for many tokens, in
 * two launches that read it once:
 *   index_weights_out[t] = round16(fp32(hidden_states[t] . weights_proj_weight^T) * score_scale)
 * for fp32 weights_proj_weight (reference nanovllm/models/dsa_indexer_project.py:82-86;
 * with 16-bit weights rounded after the projection and again after a scale
 * other than 1, :74-81), and, unless wk_weight is NULL,
 *   index_k_out[t] = RoPE(layer_norm(round16(hidden_states[t] . wk_weight^T)))
 * (:245-293; eps 1e-6, k_norm_bias may be NULL).  Limits: n_head 16, 32 or
 * 64, hidden_size a multiple of 64, 128-wide keys.  The workspace is sized by
 * nvdsa_dsa_indexer_project_kw_workspace_size and holds no state. */
size_t nvdsa_dsa_indexer_project_kw_workspace_size(int64_t tokens, int64_t n_head, int64_t hidden_size,
                                                   int32_t with_k);
int nvdsa_dsa_indexer_project_kw(const nvdsa_tensor* hidden_states,
                                 const nvdsa_tensor* cos,
                                 const nvdsa_tensor* sin,
                                 const nvdsa_tensor* wk_weight,
                                 const nvdsa_tensor* k_norm_weight,
                                 const nvdsa_tensor* k_norm_bias,
                                 const nvdsa_tensor* weights_proj_weight,
                                 const nvdsa_tensor* index_k_out,
                                 const nvdsa_tensor* index_weights_out,
                                 int64_t rope_dim,
                                 double score_scale,
                                 void* workspace,
                                 size_t workspace_bytes,
                                 void* stream);

/* The tile (64, 128 or 256 tokens by as many outputs) in which
 * nvdsa_dsa_indexer_project_query_only multiplies more than 64 tokens into
 * `outputs` = n_head * head_dim values; 0 for up to 64 tokens, which take no
 * tiled product. */
int nvdsa_dsa_indexer_project_tile(int64_t tokens, int64_t outputs);

/* One row-wise copy of nvdsa_stage_inputs: rows [0, real) of dst (dst_bytes
 * apart) take src_bytes of src's row (src_stride bytes apart) and the 32-bit
 * pattern `fill` after them, rows [real, rows) the pattern alone.  All sizes
 * and addresses are multiples of 2 (of 4 unless the pattern's halves are
 * equal). */
typedef struct nvdsa_stage_item {
  void* dst;
  const void* src;
  int64_t rows;
  int64_t real;
  int64_t dst_bytes;
  int64_t src_bytes;
  int64_t src_stride;
  int64_t fill;
} nvdsa_stage_item;
/* Up to 16 such copies in one launch: the inputs of a decode step into a
 * captured graph's fixed buffers (reference
 * nanovllm/engine/full_decode_graph.py:546-720 copies them one by one).  No
 * item may read what another one writes. */
int nvdsa_stage_inputs(const nvdsa_stage_item* items, int64_t count, void* stream);

/* ---------------------------------------------------------------------- */
/* The 8-bit latent cache: latent_cache [blocks, 128, G, 576] e4m3 (512
 * latent ++ 64 rope values of a token and latent head), cache_scale
 * [blocks, G] fp32 (positive, finite): value = code * scale.  Requests own
 * their pages through block_table [B, cols] (entries that name no block are
 * skipped); token records (positions int32, accumulated attention weights
 * fp32) are pool rows [pool_rows, cols * 128], request b's at
 * req_pool_entries[b], one value per cache slot of the request.  Two requests
 * of a call that write must share neither a written page nor a pool row.
 *
 * Query / new rows are packed: request b's are
 * [actual_seq_lengths_query[b-1], actual_seq_lengths_query[b]), and
 * actual_seq_lengths_kv[b] counts its cached tokens with the new ones.  Ends
 * must not decrease: rows that two requests share hold either's result, their
 * requests' token weights go by that, and where the rows' work counts more than
 * once the call may leave rows and records as they were.  Rows behind the last
 * request are neither read nor written.  No counterpart in
 * the reference, whose caches are 16-bit. */

/* New row i of n goes to slot actual_seq_lengths_kv[b] - n + i.  A page's
 * scale is the least power of two (2^-126 to 2^120) under which its rows'
 * largest finite magnitude is at most 448; a page that holds older rows keeps
 * its scale where that suffices, and otherwise its older codes are rounded to
 * the larger one.  Codes are rounded to nearest even; infinities and NaN
 * become NaN.  kv [T, G, 512], k_rope [T, G, 64] (16-bit).  positions [T] and
 * token_positions go together, either of them or token_weights (set to 0 at
 * new slots) needs req_pool_entries; all four may be NULL.  No workspace. */
int nvdsa_latent8_append(const nvdsa_tensor* kv,
                         const nvdsa_tensor* k_rope,
                         const nvdsa_tensor* actual_seq_lengths_query,
                         const nvdsa_tensor* actual_seq_lengths_kv,
                         const nvdsa_tensor* block_table,
                         const nvdsa_tensor* latent_cache,
                         const nvdsa_tensor* cache_scale,
                         const nvdsa_tensor* positions,
                         const nvdsa_tensor* req_pool_entries,
                         const nvdsa_tensor* token_positions,
                         const nvdsa_tensor* token_weights,
                         void* stream);

/* attention_out[r] = softmax(scale_value * q[r] . k) . k[:512] over the slots
 * that row r sees: row i of a request's n sees the first
 * actual_seq_lengths_kv - (n - 1 - i), or, with topk_ids [T, K], those of its
 * list (entries outside that range are skipped, a slot listed twice counts
 * twice).  A row that sees nothing is zero.  query [T, N, 512], query_rope
 * [T, N, 64], N a multiple of G: head h attends latent head h / (N / G).
 * With token_weights (not with topk_ids), every slot's attention weight,
 * summed over the request's rows and heads, is added to its record. */
size_t nvdsa_latent8_attention_workspace_size(int64_t query_rows, int64_t heads, int32_t with_weights);
int nvdsa_latent8_attention(const nvdsa_tensor* query_rope,
                            const nvdsa_tensor* query,
                            const nvdsa_tensor* actual_seq_lengths_query,
                            const nvdsa_tensor* actual_seq_lengths_kv,
                            const nvdsa_tensor* block_table,
                            const nvdsa_tensor* latent_cache,
                            const nvdsa_tensor* cache_scale,
                            const nvdsa_tensor* topk_ids,
                            const nvdsa_tensor* req_pool_entries,
                            const nvdsa_tensor* token_weights,
                            double scale_value,
                            const nvdsa_tensor* attention_out,
                            void* workspace, size_t workspace_bytes,
                            void* stream);

/* Brings every request with more than budgets[b] cached tokens down to that
 * many.  Kept are tokens at a position below protect_first or among the
 * protect_last latest positions, then those of the largest weight (NaN above
 * all), ties to the lower slot; where more are protected than the budget holds,
 * those at the lower slots stay (of a request that nothing was evicted from, the
 * earliest: a budget below protect_first + protect_last gives up latest ones).
 * The kept tokens at slots >= budget move, in order, into the slots below it that were given up: their rows (to the
 * larger of the pages' scales), positions and weights.  move_src_slots /
 * move_dst_slots [B, cols * 128] list the moves (entries past move_counts[b]
 * are left as they were), kept_lengths[b] is the new length.  A request whose
 * pool entry names no row is left alone.  Of tokens whose page, or whose new
 * slot's page, names no block the records move but no rows, so the pages of a
 * request over its budget should all be there. */
size_t nvdsa_latent8_evict_workspace_size(int64_t batch, int64_t table_cols, int64_t latent_heads);
int nvdsa_latent8_evict(const nvdsa_tensor* actual_seq_lengths_kv,
                        const nvdsa_tensor* budgets,
                        const nvdsa_tensor* block_table,
                        const nvdsa_tensor* req_pool_entries,
                        const nvdsa_tensor* latent_cache,
                        const nvdsa_tensor* cache_scale,
                        const nvdsa_tensor* token_positions,
                        const nvdsa_tensor* token_weights,
                        int64_t protect_first,
                        int64_t protect_last,
                        const nvdsa_tensor* move_src_slots,
                        const nvdsa_tensor* move_dst_slots,
                        const nvdsa_tensor* move_counts,
                        const nvdsa_tensor* kept_lengths,
                        void* workspace, size_t workspace_bytes,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NVDSA_EXT_H */
