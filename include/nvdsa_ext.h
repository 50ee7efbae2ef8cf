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

/* ---------------------------------------------------------------------- */
/* Many continuations of one prefix on the 16-bit latent cache (kv_cache
 * [blocks, 128, 1, 512], k_rope [blocks, 128, 1, 64]); packed rows, ends,
 * lengths and tables as above.  No counterpart in the reference. */

/* The rows between the projections and the attention.  Row i of a request's n
 * goes to slot actual_seq_lengths_kv[b] - n + i (skipped where that names no
 * page):
 *   kv_cache[slot] = kv[t, :512] * rsqrt(mean(kv[t, :512]^2) + eps) * kv_norm_weight
 *   k_rope[slot]   = R_t kv[t, 512:]
 *   query_rope[t]  = R_t query[t, :, D - 64:]
 * and with query_norm_weight [D] and query_nope [T, N, D - 64] (both or
 * neither), the heads' queries, all D dims of them, are normalised in the same
 * way first and the other dims written to query_nope.  R_t turns pairs by
 * cos / sin [T, 64 or more] as dsa_indexer_query_rope_inplace does.  fp32
 * throughout, one rounding at the store.  query [T, N, D], 64 <= D <= 576; all
 * of one 16-bit dtype.  Rows behind the last request are neither read nor
 * written.  No workspace. */
int nvdsa_norm_rope_append(const nvdsa_tensor* query,
                           const nvdsa_tensor* kv,
                           const nvdsa_tensor* cos,
                           const nvdsa_tensor* sin,
                           const nvdsa_tensor* kv_norm_weight,
                           const nvdsa_tensor* actual_seq_lengths_query,
                           const nvdsa_tensor* actual_seq_lengths_kv,
                           const nvdsa_tensor* block_table,
                           const nvdsa_tensor* k_rope,
                           const nvdsa_tensor* kv_cache,
                           const nvdsa_tensor* query_rope,
                           const nvdsa_tensor* query_norm_weight,
                           const nvdsa_tensor* query_nope,
                           double eps,
                           void* stream);

/* attention_out[r] = softmax(scale_value * q[r] . k) . k[:512] over the slots
 * that row r sees: row i of a request's n sees the first
 * actual_seq_lengths_kv - (n - 1 - i); slots whose table entry names no page are
 * skipped, a row that sees nothing is zero.  query [T, N, 512], query_rope
 * [T, N, 64].  Scores and sums are fp32; the weights are rounded to the cache's
 * 16 bits and divided by the sum of what they are rounded to.
 * Groups (both tensors [S], or neither): requests [prefix_request_ends[s-1],
 * prefix_request_ends[s]) hold the same pages for their first prefix_lengths[s]
 * tokens (whole pages: the rest of that length counts as their own).  Where that
 * saves enough time they are read through the table of the first request that has
 * rows, once for the group; requests without rows may hold anything.  Requests behind
 * the last end share nothing.  Values that a row does not
 * see may be anything; a NaN or a score of +inf that it sees makes it NaN; the dims
 * of an infinite value whose score is -inf are NaN or without that key, as the work
 * is cut.  The workspace holds no state. */
size_t nvdsa_shared_prefix_attention_workspace_size(int64_t query_rows, int64_t heads, int64_t batch, int64_t groups);
int nvdsa_shared_prefix_attention(const nvdsa_tensor* query_rope,
                                  const nvdsa_tensor* query,
                                  const nvdsa_tensor* actual_seq_lengths_query,
                                  const nvdsa_tensor* actual_seq_lengths_kv,
                                  const nvdsa_tensor* block_table,
                                  const nvdsa_tensor* k_rope,
                                  const nvdsa_tensor* kv_cache,
                                  double scale_value,
                                  const nvdsa_tensor* attention_out,
                                  const nvdsa_tensor* prefix_request_ends,
                                  const nvdsa_tensor* prefix_lengths,
                                  void* workspace, size_t workspace_bytes,
                                  void* stream);

/* Requests that go on from others, and the pages that they write to next.
 * block_table entries that name no page are -1; page_refs[p] counts the rows
 * that hold page p (and whoever else does), 0: free.
 * With parents [B], row b first takes over what row parents[b] held before the
 * call, table and length, and page_refs follow; a parent that names no row
 * leaves it empty.  Then every row gets the pages that its next new_tokens[b]
 * tokens fall into (those within the table): a new one where it has none, and
 * where others hold its page too, except that a page with older rows stays with
 * the lowest of the rows that write on where only these hold it.  New pages are
 * the lowest free ones, given out by row and column (those that the rows' old
 * tables gave back among them).  copy_src / copy_dst / copy_tokens [B] say which
 * rows the new page of a row has to receive (-1, -1, 0: none).  All rows get
 * their pages or, where too few are free, none does: missing[0] is the number that
 * lacks, or 0.  What the rows took over stays theirs either way: the call is
 * repeated with parents NULL, or with parents that go by the rows as they are
 * now. */
size_t nvdsa_pages_branch_workspace_size(int64_t pages);
int nvdsa_pages_branch(const nvdsa_tensor* seq_lens,
                       const nvdsa_tensor* new_tokens,
                       const nvdsa_tensor* block_table,
                       const nvdsa_tensor* page_refs,
                       const nvdsa_tensor* copy_src,
                       const nvdsa_tensor* copy_dst,
                       const nvdsa_tensor* copy_tokens,
                       const nvdsa_tensor* missing,
                       const nvdsa_tensor* parents,
                       void* workspace, size_t workspace_bytes,
                       void* stream);

/* Brings the held pages together: with L of them, those at or behind L go, in
 * ascending order, to the free ones below L.  Tables and page_refs follow;
 * move_src / move_dst [pages] list the moves (entries past move_count[0] are
 * left as they were). */
size_t nvdsa_pages_compact_workspace_size(int64_t pages);
int nvdsa_pages_compact(const nvdsa_tensor* block_table,
                        const nvdsa_tensor* page_refs,
                        const nvdsa_tensor* move_src,
                        const nvdsa_tensor* move_dst,
                        const nvdsa_tensor* move_count,
                        void* workspace, size_t workspace_bytes,
                        void* stream);

/* Pages src_ids[k] to dst_ids[k] of up to 16 caches [pages, ...] (an array of
 * descriptors).  With tokens [pairs], the first tokens[k] rows of caches
 * [pages, 128, ...] and, where there are any, whole pages of others; with
 * count [1], the first count[0] pairs.  Pairs that name no page are skipped.
 * No page of a call may be a source and a destination, or a destination twice. */
int nvdsa_pages_copy(const nvdsa_tensor* src_ids,
                     const nvdsa_tensor* dst_ids,
                     const nvdsa_tensor* caches,
                     int64_t cache_count,
                     const nvdsa_tensor* tokens,
                     const nvdsa_tensor* count,
                     void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NVDSA_EXT_H */
