// Host-side launch interface between the C ABI layer (nvdsa_abi.hip) and the
// kernel translation units.  Arguments are already validated by the caller.
#pragma once

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nvdsa {

enum class Elem { kBf16, kF16 };

// Kernel ids of the timing instrumentation (nvdsa_profile_*).
enum KernelId : int {
  kKernScatter = 0,
  kKernLimScore = 1,
  kKernLimHist = 2,
  kKernLimMtpPassA = 3,
  kKernSfaSplit = 4,
  kKernSfaSplitFused = 5,
  kKernSfaCombine = 6,
  kKernLiduInit = 7,
  kKernLiduShared = 8,
  kKernLimThreshold = 9,
  kKernLimMtpVictims = 10,
  kKernLimMtpPassB = 11,
  kKernSfaMtpOverlap = 12,
  kKernSfaSplitCopied = 13,
  kKernIdxProject = 14,
  kKernIdxRope = 15,
  kKernPersist = 16,
  kKernLimClassify = 17,
  kKernLimChunks = 18,
  kKernLimResolve = 19,
  kKernIdxKw = 20,
  kKernIdxKwFinish = 21,
  kKernStage = 22,
  kKernLatent8Append = 23,
  kKernLatent8Attention = 24,
  kKernLatent8Join = 25,
  kKernLatent8Weights = 26,
  kKernLatent8Select = 27,
  kKernLatent8Move = 28,
  kKernNormRope = 29,
  kKernPagesTake = 30,
  kKernPagesReserve = 31,
  kKernPagesCount = 32,
  kKernPagesRank = 33,
  kKernPagesRename = 34,
  kKernPagesCopy = 35,
  kKernPrefixPlan = 36,
  kKernPrefixAttention = 37,
  kKernPrefixJoin = 38,
  kKernPagesCompact = 39,
  kKernCount = 40
};
// Timing events for the next launch of `kernel_id` when instrumentation is
// on for the calling thread (nvdsa_profile_begin); both null otherwise.
struct ProfEvents {
  hipEvent_t start = nullptr;
  hipEvent_t stop = nullptr;
};
ProfEvents prof_events(int kernel_id);

// Launch `kernel` on `stream`.  When timed, the events ride on the kernel's
// own dispatch (hipExtLaunchKernelGGL), so the recorded interval is the
// kernel's execution alone, without the gaps of separate event records.
template <typename F, typename... Args>
inline void launch_kernel(int kernel_id, F kernel, dim3 grid, dim3 block, hipStream_t stream, Args... args) {
  const ProfEvents ev = prof_events(kernel_id);
  if (ev.start != nullptr) {
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, ev.start, ev.stop, 0, args...);
  } else {
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, args...);
  }
}

// ---- scatter_copy --------------------------------------------------------
struct ScatterArgs {
  const int32_t* src_ids;      // [B, cap]
  const int32_t* dst_slots;    // [B, cap]
  const int32_t* copy_counts;  // [B]
  const int32_t* hbm_table;    // [B, hbm_cols]
  const int32_t* dram_table;   // [B, dram_cols]
  void* hbm_kpe;               // [hbm_blocks, 128, 64]
  void* hbm_ckv;               // [hbm_blocks, 128, 512]
  const void* dram_kpe;        // [dram_blocks, 128, 64]
  const void* dram_ckv;        // [dram_blocks, 128, 512]
  int64_t batch;
  int64_t cap;
  int64_t hbm_cols;
  int64_t dram_cols;
  int64_t hbm_blocks;
  int64_t dram_blocks;
};
hipError_t launch_scatter_copy(const ScatterArgs& a, hipStream_t stream);

// ---- fused_li_manage (MTP0 and MTP3) ---------------------------------------
struct LimArgs {
  const void* query;            // [B*Q, H, 128]
  const void* weights;          // [B*Q, H]
  const void* key_cache;        // [key_blocks, 128, 1, 128]
  const int32_t* block_table;   // [B, cols]
  const int32_t* num_candidates;  // [B]
  const int32_t* num_cache;     // [B]
  const int32_t* pool_entries;  // [B]
  int32_t* pool;                // [pool_rows, cols*128]
  int32_t* topk_src;            // [B*Q, 1, 2048]
  int32_t* topk_dst;            // [B*Q, 1, 2048]
  int32_t* miss_src;            // [B, 8192]   (MTP only)
  int32_t* miss_dst;            // [B, 8192]   (MTP only)
  int32_t* miss_counts;         // [B]
  int64_t batch;
  int64_t heads;
  int64_t cols;                 // block-table columns
  int64_t key_blocks;
  int64_t pool_rows;
  int64_t source_capacity;      // cols * 128
  Elem elem;
  void* workspace;
  size_t workspace_bytes;
};
size_t lim_workspace_bytes(int64_t batch, int64_t source_capacity, int queries);
hipError_t launch_fused_li_manage(const LimArgs& a, hipStream_t stream);
hipError_t launch_fused_li_manage_mtp(const LimArgs& a, hipStream_t stream);

// ---- first-decode LIDU initialisation -------------------------------------
struct LiduInitArgs {
  const void* query;            // [H, 128] (one request)
  const void* weights;          // [H]
  const void* key_cache;        // [key_blocks, 128, 1, 128]
  const int32_t* index_table;   // [index_cols]
  int64_t index_cols;
  int64_t key_blocks;
  int64_t heads;
  Elem elem;
  int64_t n;                    // candidate tokens (whole blocks)
  int64_t c;                    // cache budget C
  int32_t* pool_row;            // [row_len] token -> slot
  int64_t row_len;
  void* hbm_kpe;                // [hbm_blocks, 128, 64]
  void* hbm_ckv;                // [hbm_blocks, 128, 512]
  const void* dram_kpe;
  const void* dram_ckv;
  const int32_t* hbm_table;     // [hbm_cols]
  int64_t hbm_cols;
  int64_t hbm_blocks;
  const int32_t* dram_table;    // [dram_cols]
  int64_t dram_cols;
  int64_t dram_blocks;
  void* workspace;
  size_t workspace_bytes;
};
size_t lidu_init_workspace_bytes(int64_t source_capacity);
int64_t lidu_list_capacity();
// Scores, top-C selection, pool row and copy list (then launch_lidu_copy).
hipError_t launch_lidu_init(const LiduInitArgs& a, hipStream_t stream);
// Copy list of a shared layer from the owner's pool row; its length is
// written to lidu_list_count(a) on the device.
hipError_t launch_lidu_shared_list(const LiduInitArgs& a, hipStream_t stream);
const int32_t* lidu_list_count(const LiduInitArgs& a);
// DRAM -> HBM copy of the list (scatter_copy kernel).
hipError_t launch_lidu_copy(const LiduInitArgs& a, hipStream_t stream);

// ---- sparse-tail attention (+ fused copy) --------------------------------
struct SfaArgs {
  const void* query_rope;       // [R, N, 64]
  const void* query;            // [R, N, 512]
  const int32_t* seq_kv;        // [B]
  const int32_t* num_cache;     // [B]
  const int32_t* topk_dst;      // [R, 1, 2048]
  const int32_t* hbm_table;     // [B, hbm_cols]
  void* hbm_kpe;                // [hbm_blocks, 128, 1, 64]
  void* hbm_ckv;                // [hbm_blocks, 128, 1, 512]
  void* out;                    // [R, N, 512]
  int64_t batch;
  int64_t rows_per_request;     // 1 or 4
  int64_t heads;
  int64_t hbm_cols;
  int64_t hbm_blocks;
  float scale;
  Elem elem;
  // fused copy (null when not fused)
  const int32_t* copy_src;      // MTP0: topk_src_ids [B, 2048]; MTP3: miss_src_ids [B, 8192]
  const int32_t* copy_dst;      // MTP0: topk_dst_slots; MTP3: miss_dst_slots
  const int32_t* copy_counts;   // [B]
  int64_t copy_cap;             // 2048 or 8192
  const int32_t* dram_table;    // [B, dram_cols]
  const void* dram_kpe;
  const void* dram_ckv;
  int64_t dram_cols;
  int64_t dram_blocks;
  const int32_t* key_src;       // MTP3 fused: topk_src_ids [R, 2048] (>= 0: a key copied by this call)
  void* workspace;
  size_t workspace_bytes;
};
size_t sfa_workspace_bytes(int64_t query_rows, int64_t heads, int64_t max_kv_tokens);
hipError_t launch_sparse_tail_attention(const SfaArgs& a, hipStream_t stream);
hipError_t launch_fused_copy_sfa(const SfaArgs& a, hipStream_t stream);
// Copies the current device's record of the XCDs the MTP3 overlap kernel's
// copy ([0]) and attention ([1]) workgroups ran on; clears it after the read
// when `reset`.  Synchronises the device.
hipError_t sfa_xcd_roles(uint32_t masks[2], bool reset);
// Whether launches made from now on write that record (off by default).
void sfa_xcd_roles_record(bool on);

// ---- indexer projection (decode query rows and head weights) -------------
struct IndexerArgs {
  const void* hidden;   // [tokens, hid]          16-bit
  const void* q_c;      // [tokens, rank]
  const void* cos;      // [tokens, cos_stride]   (first rope_dim used)
  const void* sin;
  const void* wq_b;     // [heads * head_dim, rank]
  const void* w_proj;   // [heads, hid], or null: weights not computed here
  void* q_out;          // [tokens, heads, head_dim]
  void* w_out;          // [tokens, heads]
  int64_t tokens, hid, rank, heads, head_dim, rope_dim, cos_stride;
  float score_scale;
  Elem elem;
};
// K extents (rank, hid) must be multiples of this.
int64_t indexer_k_chunk();
int indexer_gemm_tile(int64_t tokens, int64_t outs);
hipError_t launch_indexer_project(const IndexerArgs& a, hipStream_t stream);

// Products of hidden_states for many tokens: the index key (wk != null) and
// the head weights.
struct IndexerKwArgs {
  const void* hidden;       // [tokens, hid] 16-bit
  const void* wk;           // [128, hid] 16-bit, or null: no key
  const void* norm_weight;  // [128] 16-bit
  const void* norm_bias;    // [128] 16-bit, or null
  const void* w_proj;       // [heads, hid] fp32 (w_fp32) or 16-bit
  const void* cos;          // [tokens, cos_stride]
  const void* sin;
  void* k_out;              // [tokens, 128]
  void* w_out;              // [tokens, heads]
  float* partial;           // workspace
  int64_t tokens, hid, heads, rope_dim, cos_stride;
  float score_scale;
  int w_fp32;
  Elem elem;
};
bool indexer_kw_supported(int64_t heads, int64_t hid);
size_t indexer_kw_workspace_bytes(int64_t tokens, int64_t heads, int64_t hid, bool with_k);
hipError_t launch_indexer_kw(const IndexerKwArgs& a, hipStream_t stream);

struct RopeArgs {
  void* q;              // [rows = tokens * heads, head_dim], rotated in place
  const void* cos;      // [tokens, rope_dim]
  const void* sin;
  int64_t rows, heads, head_dim, rope_dim;
  Elem elem;
};
hipError_t launch_indexer_rope(const RopeArgs& a, hipStream_t stream);

// ---- prefill -> DRAM persistence ------------------------------------------
struct PersistArgs {
  const void* hbm_ckv;      // [hbm_blocks, 128, 512]
  const void* hbm_kpe;      // [hbm_blocks, 128, 64]
  void* dram_ckv;           // [dram_blocks, 128, 512] (host-mapped)
  void* dram_kpe;           // [dram_blocks, 128, 64]
  const int32_t* hbm_ids;   // [count]
  const int32_t* dram_ids;  // [count]
  int64_t count, hbm_blocks, dram_blocks;
};
hipError_t launch_persist_blocks(const PersistArgs& a, hipStream_t stream);

// ---- staging of a captured graph's inputs ---------------------------------
// Rows [0, real) take src_bytes from src (src_stride bytes apart) and `fill`
// (32-bit pattern; its low half for 2-byte units) after them; rows
// [real, rows) take `fill` alone.  Rows of dst lie dst_bytes apart.
struct StageItem {
  void* dst;
  const void* src;
  int64_t rows, real, dst_bytes, src_bytes, src_stride;
  int32_t fill;
  int32_t unit;  // 16, 4 or 2 bytes, set by the launch
};
constexpr int kMaxStageItems = 16;
struct StageArgs {
  StageItem items[kMaxStageItems];
  int32_t first_block[kMaxStageItems];
  int32_t count;
};
hipError_t launch_stage_inputs(StageArgs& a, hipStream_t stream);

// ---- 8-bit latent cache -----------------------------------------------------
struct Latent8AppendArgs {
  const void* kv;               // [rows, G, 512] 16-bit
  const void* k_rope;           // [rows, G, 64]
  const int32_t* positions;     // [rows] (with token_positions)
  const int32_t* seq_q;         // [B] end of each request's rows
  const int32_t* seq_kv;        // [B] cached tokens, the new ones among them
  const int32_t* block_table;   // [B, cols]
  const int32_t* entries;       // [B], or null: no token records
  void* latent_cache;           // [blocks, 128, G, 576] e4m3
  float* cache_scale;           // [blocks, G]
  int32_t* token_positions;     // [pool_rows, cols * 128], or null
  float* token_weights;         // [pool_rows, cols * 128], or null
  int64_t rows, batch, cols, blocks, latent_heads, pool_rows;
  Elem elem;
};
hipError_t launch_latent8_append(const Latent8AppendArgs& a, hipStream_t stream);

struct Latent8Args {
  const void* query;            // [rows, heads, 512] 16-bit
  const void* query_rope;       // [rows, heads, 64]
  const int32_t* seq_q;         // [B] end of each request's rows
  const int32_t* seq_kv;        // [B]
  const int32_t* block_table;   // [B, cols]
  const void* latent_cache;     // [blocks, 128, G, 576] e4m3
  const float* cache_scale;     // [blocks, G]
  const int32_t* topk;          // [rows, list_len], or null: every cached token
  const int32_t* entries;       // [B] (with token_weights)
  float* token_weights;         // [pool_rows, cols * 128], or null
  void* out;                    // [rows, heads, 512]
  int64_t rows, heads, latent_heads, batch, cols, blocks, list_len, pool_rows;
  int64_t parts;                // set by the launch, as are the next three
  int64_t joins;                // entries for the joining kernel:
  bool join_items;              //   one an item, or one a part
  int32_t per;                  // heads / latent_heads
  float scale;
  Elem elem;
  void* workspace;
};
// At most so many items (up to 64 (row, head) pairs of a request and latent
// head; with a list, of a row).
int64_t latent8_items(int64_t rows, int64_t heads, int64_t latent_heads, int64_t batch, bool list);
size_t latent8_attention_workspace_bytes(int64_t rows, int64_t heads, bool weights);
hipError_t launch_latent8_attention(const Latent8Args& a, hipStream_t stream);

struct Latent8EvictArgs {
  const int32_t* seq_kv;        // [B]
  const int32_t* budgets;       // [B]
  const int32_t* block_table;   // [B, cols]
  const int32_t* entries;       // [B]
  void* latent_cache;           // [blocks, 128, G, 576] e4m3
  float* cache_scale;           // [blocks, G]
  int32_t* token_positions;     // [pool_rows, cols * 128]
  float* token_weights;         // [pool_rows, cols * 128]
  int32_t* move_src;            // [B, cols * 128]
  int32_t* move_dst;            // [B, cols * 128]
  int32_t* move_counts;         // [B]
  int32_t* kept_lengths;        // [B]
  int64_t batch, cols, blocks, latent_heads, pool_rows;
  int64_t protect_first, protect_last;
  void* workspace;
  int32_t* hole_start;          // workspace, set by the launch: [B, cols + 1]
  float* border_scale;          // [B, G]
};
size_t latent8_evict_workspace_bytes(int64_t batch, int64_t cols, int64_t latent_heads);
hipError_t launch_latent8_evict(const Latent8EvictArgs& a, hipStream_t stream);

// ---- new rows of the 16-bit latent cache ------------------------------------
struct NormRopeArgs {
  const void* query;            // [rows, heads, query_dim] 16-bit
  const void* kv;               // [rows, 576]
  const void* cos;              // [rows, cos_stride] (first 64 used)
  const void* sin;
  const void* kv_weight;        // [512]
  const void* query_weight;     // [query_dim], or null: queries are only rotated
  const int32_t* seq_q;         // [B] end of each request's rows
  const int32_t* seq_kv;        // [B] cached tokens, the new ones among them
  const int32_t* block_table;   // [B, cols]
  void* k_rope;                 // [blocks, 128, 1, 64]
  void* kv_cache;               // [blocks, 128, 1, 512]
  void* query_rope;             // [rows, heads, 64]
  void* query_nope;             // [rows, heads, query_dim - 64] (with query_weight)
  int64_t rows, heads, query_dim, cos_stride, batch, cols, blocks;
  float eps;
  Elem elem;
};
hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t stream);

// ---- attention of requests that share a prefix ------------------------------
struct PrefixAttentionArgs {
  const void* query;            // [rows, heads, 512] 16-bit
  const void* query_rope;       // [rows, heads, 64]
  const int32_t* seq_q;         // [B] end of each request's rows
  const int32_t* seq_kv;        // [B]
  const int32_t* block_table;   // [B, cols]
  const void* k_rope;           // [blocks, 128, 1, 64]
  const void* kv_cache;         // [blocks, 128, 1, 512]
  const int32_t* group_ends;    // [groups] end of each group's requests
  const int32_t* prefix_lens;   // [groups]
  void* out;                    // [rows, heads, 512]
  int64_t rows, heads, batch, groups, cols, blocks;
  float scale;
  Elem elem;
  void* workspace;
};
size_t prefix_attention_workspace_bytes(int64_t rows, int64_t heads, int64_t batch, int64_t groups);
hipError_t launch_prefix_attention(const PrefixAttentionArgs& a, hipStream_t stream);

// ---- pages of the caches ----------------------------------------------------
constexpr int kMostBranchRows = 16384;
struct PagesBranchArgs {
  int32_t* seq_lens;            // [B]
  const int32_t* new_tokens;    // [B]
  int32_t* block_table;         // [B, cols]
  int32_t* page_refs;           // [pages]
  const int32_t* parents;       // [B], or null: every row goes on as it is
  int32_t* copy_src;            // [B]
  int32_t* copy_dst;            // [B]
  int32_t* copy_tokens;         // [B]
  int32_t* missing;             // [1]
  int64_t batch, cols, pages;
  void* workspace;
  int32_t* fresh;               // workspace, set by the launch: [pages]
  int32_t* given_up;            // [pages]
};
size_t pages_branch_workspace_bytes(int64_t pages);
hipError_t launch_pages_branch(PagesBranchArgs a, hipStream_t stream);

struct PagesCompactArgs {
  int32_t* block_table;         // [B, cols]
  int32_t* page_refs;           // [pages]
  int32_t* move_src;            // [pages]
  int32_t* move_dst;            // [pages]
  int32_t* move_count;          // [1]
  int64_t batch, cols, pages;
  void* workspace;
  int32_t* rank;                // workspace, set by the launch: [pages]
  int32_t* counts;              // [chunks]
};
size_t pages_compact_workspace_bytes(int64_t pages);
hipError_t launch_pages_compact(PagesCompactArgs a, hipStream_t stream);

constexpr int kMostCopyCaches = 16;
struct PagesCopyArgs {
  const int32_t* src;           // [pairs]
  const int32_t* dst;           // [pairs]
  const int32_t* tokens;        // [pairs], or null: whole pages
  const int32_t* count;         // [1], or null: every pair
  int64_t pairs, pages;
  int32_t caches;
  void* cache[kMostCopyCaches];             // [pages, page_bytes]
  int64_t page_bytes[kMostCopyCaches];
  int64_t token_bytes[kMostCopyCaches];     // 0: a page of it has no rows of tokens
  bool wide[kMostCopyCaches];               // everything in units of 16 bytes, else of 4
  int32_t first_piece[kMostCopyCaches + 1]; // set by the launch
};
hipError_t launch_pages_copy(PagesCopyArgs a, hipStream_t stream);

}  // namespace nvdsa
