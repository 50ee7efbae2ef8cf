// The pages of the caches: requests that branch off others, a cache brought
// together at its low pages, and the copies that either asks for.
//
// A page is held by the requests whose table names it (and by whoever else
// counts in page_refs); one with no holder is free.  The free pages are found in
// the counts themselves, lowest first, so no list has to be kept beside them.
//
//   branch    table[b] = table[parents[b]], page_refs follow; then pages for the
//             columns that the next new_tokens[b] tokens fall into: new ones
//             where there is none or where others hold it too, or none at all
//             where too few are free (what was taken over stays).
//   compact   with L pages held, those at or behind L go, in order, to the free
//             ones below L.
//   copy      pages src[k] to dst[k] of several caches, or their first tokens[k].
#include "nvdsa_common.h"
#include "nvdsa_kernels.h"

namespace nvdsa {
namespace {

// ---------------------------------------------------------------- take over
// A workgroup owns some columns of every row, so that rows can take over each
// other's entries in place.  Only entries that change touch the counts: beams
// that swap within a shared prefix leave them alone.
constexpr int kTakeThreads = 256;
constexpr int kTakeEntries = 16384;  // of LDS
// Columns of a workgroup: an entry a thread, as its two counts are what takes the
// time (64 rows of 256 columns that all change: 8.7 us with 16 columns, 5.3 us with
// 4), but 16 bytes of a row at least.
constexpr int kTakeMost = 16, kTakeLeast = 4;

__device__ inline int parent_of(const PagesBranchArgs& a, int b) {
  const int32_t p = a.parents[b];
  return p < 0 || p >= a.batch ? -1 : p;
}
// Columns [col0, col0 + columns) of every row, at most kTakeEntries entries.
template <int THREADS>
__device__ inline void take_over(const PagesBranchArgs& a, int64_t col0, int columns, int32_t* held) {
  const int tid = threadIdx.x;
  const int n = static_cast<int>(a.batch) * columns;
  for (int i = tid; i < n; i += THREADS) {
    const int b = i / columns;
    const int64_t c = col0 + (i - b * columns);
    held[i] = c < a.cols ? a.block_table[b * a.cols + c] : -1;
  }
  __syncthreads();
  for (int i = tid; i < n; i += THREADS) {
    const int b = i / columns, k = i - b * columns;
    const int64_t c = col0 + k;
    if (c >= a.cols) continue;
    const int p = parent_of(a, b);
    const int32_t before = held[i], after = p < 0 ? -1 : held[p * columns + k];
    if (before == after) continue;
    a.block_table[b * a.cols + c] = after;
    if (after >= 0 && after < a.pages) atomicAdd(&a.page_refs[after], 1);
    if (before >= 0 && before < a.pages) atomicAdd(&a.page_refs[before], -1);
  }
}
// And the rows' lengths.
template <int THREADS>
__device__ inline void take_lengths(const PagesBranchArgs& a, int32_t* held) {
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += THREADS) held[b] = a.seq_lens[b];
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += THREADS) {
    const int p = parent_of(a, b);
    a.seq_lens[b] = p < 0 ? 0 : held[p];
  }
}

__global__ __launch_bounds__(kTakeThreads) void pages_take_kernel(PagesBranchArgs a, int columns) {
  __shared__ int32_t held[kTakeEntries];
  take_over<kTakeThreads>(a, static_cast<int64_t>(blockIdx.x) * columns, columns, held);
  if (blockIdx.x == 0) take_lengths<kTakeThreads>(a, held);
}

// ------------------------------------------------------------------ reserve
// One workgroup: what every row needs, the free pages from the lowest on, and
// who gets which.  Rows and columns are served in order, all or none.
constexpr int kReserveThreads = 1024;
constexpr int kScanPer = 8;  // counts of a thread and round
// Entries of a table that this workgroup takes over by itself: 14 us for 256 that all
// change, as much as two kernels, and a launch less; 21 us for 2048, where two take 15.
constexpr int kTakeAlone = 512;

struct Wanted {   // columns [first, stop) of a row receive tokens
  int first, stop;
  int part;       // rows of the first column's page that stay: > 0, a page that is written on
};
__device__ inline Wanted wanted_of(const PagesBranchArgs& a, int b) {
  const int64_t cap = a.cols * kBlock;
  int64_t len = a.seq_lens[b], end = len + static_cast<int64_t>(a.new_tokens[b]);
  len = len < 0 ? 0 : len;
  end = end > cap ? cap : end;
  if (a.new_tokens[b] <= 0 || end <= len) return {0, 0, 0};
  return {static_cast<int>(len >> kBlockShift), static_cast<int>((end + kBlock - 1) >> kBlockShift),
          static_cast<int>(len & (kBlock - 1))};
}

// TAKES: and what the rows take over, first.
template <bool TAKES>
__global__ __launch_bounds__(kReserveThreads) void pages_reserve_kernel(PagesBranchArgs a) {
  __shared__ int32_t writes_on[kMostBranchRows];  // the page that a row's next token falls into, among older rows; -1
  if constexpr (TAKES) {
    __shared__ int32_t held[kTakeAlone];
    take_over<kReserveThreads>(a, 0, static_cast<int>(a.cols), held);
    take_lengths<kReserveThreads>(a, held);
    __threadfence();  // (counts changed in the L2: no older copy is read)
    __syncthreads();
  }
  __shared__ int scratch[kReserveThreads / 64 + 1];
  const int tid = threadIdx.x;
  const int batch = static_cast<int>(a.batch);
  const int per = (batch + kReserveThreads - 1) / kReserveThreads;
  const int b0 = tid * per, b1 = b0 + per < batch ? b0 + per : batch;
  auto named = [&](int32_t page) { return page >= 0 && page < a.pages; };
  for (int b = b0; b < b1; ++b) {
    const Wanted w = wanted_of(a, b);
    writes_on[b] = w.part > 0 ? a.block_table[b * a.cols + w.first] : -1;
  }
  __syncthreads();
  // A page that is written on stays with the lowest of the rows that write on it
  // where nobody else holds it.
  uint32_t keeps = 0;  // a bit a row
  int need = 0;
  auto takes = [&](int b, const Wanted& w, int c, bool keep) -> bool {
    const int32_t page = a.block_table[b * a.cols + c];
    if (!named(page)) return true;
    return a.page_refs[page] > 1 && !(c == w.first && keep);
  };
  for (int b = b0; b < b1; ++b) {
    const Wanted w = wanted_of(a, b);
    bool keep = false;
    const int32_t page = writes_on[b];
    if (named(page)) {
      const int32_t holders = a.page_refs[page];
      if (holders > 1) {
        int writers = 0, lowest = batch;
        for (int o = batch - 1; o >= 0; --o)
          if (writes_on[o] == page) {
            ++writers;
            lowest = o;
          }
        keep = holders == writers && lowest == b;
      }
    }
    keeps |= keep ? 1u << (b - b0) : 0u;
    for (int c = w.first; c < w.stop; ++c) need += takes(b, w, c, keep) ? 1 : 0;
  }
  int total;
  int at = block_exclusive_scan(need, scratch, &total);
  int32_t* const fresh = a.fresh;      // [pages]: the free pages that are given out
  int32_t* const given_up = a.given_up;  // [pages]: and what each takes the place of, or -1
  int found = 0;
  for (int64_t p0 = 0; p0 < a.pages && found < total; p0 += kReserveThreads * kScanPer) {
    uint32_t free = 0;
    const int64_t mine = p0 + tid * kScanPer;
#pragma unroll
    for (int k = 0; k < kScanPer; ++k)
      if (mine + k < a.pages && a.page_refs[mine + k] == 0) free |= 1u << k;
    int here;
    int k_at = found + block_exclusive_scan(__popc(free), scratch, &here);
#pragma unroll
    for (int k = 0; k < kScanPer; ++k)
      if ((free >> k) & 1u) {
        if (k_at < total) fresh[k_at] = static_cast<int32_t>(mine + k);
        ++k_at;
      }
    found += here;
  }
  const bool enough = found >= total;
  if (tid == 0) *a.missing = enough ? 0 : total - found;
  __syncthreads();
  for (int b = b0; b < b1; ++b) {
    int32_t src = -1, dst = -1, tokens = 0;
    if (enough) {
      const Wanted w = wanted_of(a, b);
      const bool keep = (keeps >> (b - b0)) & 1u;
      for (int c = w.first; c < w.stop; ++c) {
        if (!takes(b, w, c, keep)) continue;
        const int32_t old = a.block_table[b * a.cols + c], page = fresh[at];
        given_up[at] = named(old) ? old : -1;
        ++at;
        a.block_table[b * a.cols + c] = page;
        if (c == w.first && w.part > 0 && named(old)) {
          src = old;
          dst = page;
          tokens = w.part;
        }
      }
    }
    a.copy_src[b] = src;
    a.copy_dst[b] = dst;
    a.copy_tokens[b] = tokens;
  }
  if (!enough) return;
  __syncthreads();  // (the counts change when every row has looked at them)
  for (int k = tid; k < total; k += kReserveThreads) {
    a.page_refs[fresh[k]] = 1;
    if (given_up[k] >= 0) atomicAdd(&a.page_refs[given_up[k]], -1);
  }
}

// ------------------------------------------------------------------ compact
// Held pages of every chunk; ranks of holes and of pages to move from the
// chunks before; then counts and tables by those ranks.
constexpr int kCompactThreads = 1024;
constexpr int kCompactChunk = kCompactThreads * 4;

__device__ inline uint32_t live_of(const PagesCompactArgs& a, int64_t p0) {
  uint32_t live = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (p0 + k < a.pages && a.page_refs[p0 + k] > 0) live |= 1u << k;
  return live;
}

__global__ __launch_bounds__(kCompactThreads) void pages_count_kernel(PagesCompactArgs a) {
  __shared__ int scratch[kCompactThreads / 64 + 1];
  int total;
  block_exclusive_scan(__popc(live_of(a, static_cast<int64_t>(blockIdx.x) * kCompactChunk + threadIdx.x * 4)), scratch, &total);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = total;
}

__global__ __launch_bounds__(kCompactThreads) void pages_rank_kernel(PagesCompactArgs a) {
  __shared__ int scratch[kCompactThreads / 64 + 1];
  const int tid = threadIdx.x;
  const int chunks = gridDim.x;
  // Pages held before this chunk and in all, then below the border.
  auto sum_of = [&](int stop) {
    int s = 0, total;
    for (int i = tid; i < stop; i += kCompactThreads) s += a.counts[i];
    block_exclusive_scan(s, scratch, &total);
    return total;
  };
  const int before = sum_of(blockIdx.x), border = sum_of(chunks);
  const int border_chunk = border / kCompactChunk;
  int below = sum_of(border_chunk < chunks ? border_chunk : chunks);
  {
    const int64_t p0 = static_cast<int64_t>(border_chunk) * kCompactChunk + tid * 4;
    uint32_t live = live_of(a, p0);
    const int64_t room = border - p0;
    live &= room >= 4 ? 0xfu : (room <= 0 ? 0u : (1u << room) - 1u);
    int total;
    block_exclusive_scan(__popc(live), scratch, &total);
    below += total;
  }
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * kCompactChunk + tid * 4;
  const uint32_t live = live_of(a, p0);
  int total;
  int at = before + block_exclusive_scan(__popc(live), scratch, &total);  // pages held before p0
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t p = p0 + k;
    if (p >= a.pages) continue;
    const bool held = (live >> k) & 1u;
    int32_t rank = -1;
    if (held && p >= border) {
      rank = at - below;
      a.move_src[rank] = static_cast<int32_t>(p);
    } else if (!held && p < border) {
      a.move_dst[p - at] = static_cast<int32_t>(p);
    }
    a.rank[p] = rank;
    at += held ? 1 : 0;
  }
  if (blockIdx.x == 0 && tid == 0) *a.move_count = border - below;
}

__global__ __launch_bounds__(256) void pages_rename_kernel(PagesCompactArgs a, int64_t entries) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < a.pages) {
    const int32_t k = a.rank[i];
    if (k >= 0) {
      a.page_refs[a.move_dst[k]] = a.page_refs[i];
      a.page_refs[i] = 0;
    }
  }
  if (i < entries) {
    const int32_t page = a.block_table[i];
    if (page >= 0 && page < a.pages) {
      const int32_t k = a.rank[page];
      if (k >= 0) a.block_table[i] = a.move_dst[k];
    }
  }
}

// The same by one workgroup, ranks in LDS.  Up to 8192 pages: 5 us for 1024, 9 for 4096 and 14 for 8192, where three kernels
// take 12, 15 and 16 (16384: 20 and 16).
constexpr int kAlonePages = 8192;
constexpr int kAloneEntries = 8192;   // of the table

__global__ __launch_bounds__(kCompactThreads) void pages_compact_kernel(PagesCompactArgs a, int entries) {
  constexpr int kChunks = kAlonePages / kCompactChunk;
  __shared__ int32_t rank[kAlonePages];
  __shared__ int scratch[kCompactThreads / 64 + 1];
  const int tid = threadIdx.x;
  const int pages = static_cast<int>(a.pages);
  uint32_t live[kChunks];
  int at[kChunks], border = 0;  // pages held before the thread's of a chunk, and in all
#pragma unroll
  for (int i = 0; i < kChunks; ++i) live[i] = i * kCompactChunk < pages ? live_of(a, i * kCompactChunk + tid * 4) : 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    at[i] = border;
    if (i * kCompactChunk < pages) {
      int total;
      at[i] += block_exclusive_scan(__popc(live[i]), scratch, &total);
      border += total;
    }
  }
  int mine = 0, below;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int room = border - (i * kCompactChunk + tid * 4);
    mine += __popc(live[i] & (room >= 4 ? 0xfu : (room <= 0 ? 0u : (1u << room) - 1u)));
  }
  block_exclusive_scan(mine, scratch, &below);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int p = i * kCompactChunk + tid * 4 + k;
      if (p >= pages) continue;
      const bool held = (live[i] >> k) & 1u;
      int32_t r = -1;
      if (held && p >= border) {
        r = at[i] - below;
        a.move_src[r] = p;
      } else if (!held && p < border) {
        a.move_dst[p - at[i]] = p;
      }
      rank[p] = r;
      at[i] += held ? 1 : 0;
    }
  }
  if (tid == 0) *a.move_count = border - below;
  __syncthreads();
  for (int k = tid; k < border - below; k += kCompactThreads) {
    const int32_t from = a.move_src[k];
    a.page_refs[a.move_dst[k]] = a.page_refs[from];
    a.page_refs[from] = 0;
  }
  for (int i = tid; i < entries; i += kCompactThreads) {
    const int32_t page = a.block_table[i];
    if (page >= 0 && page < pages && rank[page] >= 0) a.block_table[i] = a.move_dst[rank[page]];
  }
}

// --------------------------------------------------------------------- copy
// 16 KiB of a page a workgroup and turn, all loads before the first store.
constexpr int kCopyThreads = 256;
constexpr int kCopyPer = 4;
constexpr int kCopyPiece = kCopyThreads * kCopyPer * 16;
constexpr int kCopyBlocks = 2048;

template <typename UNIT>
__device__ inline void copy_piece(const uint8_t* src, uint8_t* dst, int64_t from, int64_t bytes) {
  constexpr int kUnits = 16 / sizeof(UNIT);
  UNIT v[kCopyPer * kUnits];
#pragma unroll
  for (int i = 0; i < kCopyPer * kUnits; ++i) {
    const int64_t at = from + (i * kCopyThreads + threadIdx.x) * static_cast<int64_t>(sizeof(UNIT));
    if (at < bytes) v[i] = *reinterpret_cast<const UNIT*>(src + at);
  }
#pragma unroll
  for (int i = 0; i < kCopyPer * kUnits; ++i) {
    const int64_t at = from + (i * kCopyThreads + threadIdx.x) * static_cast<int64_t>(sizeof(UNIT));
    if (at < bytes) *reinterpret_cast<UNIT*>(dst + at) = v[i];
  }
}

__global__ __launch_bounds__(kCopyThreads) void pages_copy_kernel(PagesCopyArgs a) {
  int64_t pairs = a.pairs;
  if (a.count != nullptr) {
    const int64_t n = *a.count;
    pairs = n < 0 ? 0 : (n < pairs ? n : pairs);
  }
  const int pieces = a.first_piece[a.caches];
  for (int64_t i = blockIdx.x; i < pairs * pieces; i += gridDim.x) {
    const int64_t k = i / pieces;
    const int piece = static_cast<int>(i - k * pieces);
    const int32_t src = a.src[k], dst = a.dst[k];
    if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages || src == dst) continue;
    int c = 0;
    while (piece >= a.first_piece[c + 1]) ++c;
    int64_t bytes = a.page_bytes[c];
    if (a.tokens != nullptr && a.token_bytes[c] > 0) {
      const int32_t n = a.tokens[k];
      bytes = static_cast<int64_t>(n < 0 ? 0 : (n > kBlock ? kBlock : n)) * a.token_bytes[c];
    } else if (a.tokens != nullptr && a.tokens[k] <= 0) {
      bytes = 0;
    }
    const int64_t from = static_cast<int64_t>(piece - a.first_piece[c]) * kCopyPiece;
    if (from >= bytes) continue;
    uint8_t* base = static_cast<uint8_t*>(a.cache[c]);
    const uint8_t* s = base + src * a.page_bytes[c];
    uint8_t* d = base + dst * a.page_bytes[c];
    if (a.wide[c])
      copy_piece<u32x4_t>(s, d, from, bytes);
    else
      copy_piece<uint32_t>(s, d, from, bytes);
  }
}

}  // namespace

size_t pages_branch_workspace_bytes(int64_t pages) { return sizeof(int32_t) * 2 * static_cast<size_t>(pages < 0 ? 0 : pages); }

hipError_t launch_pages_branch(PagesBranchArgs a, hipStream_t stream) {
  a.fresh = static_cast<int32_t*>(a.workspace);
  a.given_up = a.fresh + a.pages;
  if (a.parents != nullptr && a.batch > 0 && a.batch * a.cols <= kTakeAlone) {
    launch_kernel(kKernPagesReserve, pages_reserve_kernel<true>, dim3(1), dim3(kReserveThreads), stream, a);
    return hipGetLastError();
  }
  if (a.parents != nullptr && a.batch > 0) {
    int64_t columns = kTakeThreads / a.batch;
    columns = columns < kTakeLeast ? kTakeLeast : (columns > kTakeMost ? kTakeMost : columns);
    if (columns * a.batch > kTakeEntries) columns = kTakeEntries / a.batch;
    launch_kernel(kKernPagesTake, pages_take_kernel, dim3(static_cast<uint32_t>(ceil_div(a.cols, columns))), dim3(kTakeThreads),
                  stream, a, static_cast<int>(columns));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  launch_kernel(kKernPagesReserve, pages_reserve_kernel<false>, dim3(1), dim3(kReserveThreads), stream, a);
  return hipGetLastError();
}

size_t pages_compact_workspace_bytes(int64_t pages) {
  return pages <= 0 ? 0 : sizeof(int32_t) * static_cast<size_t>(pages + ceil_div(pages, kCompactChunk));
}

hipError_t launch_pages_compact(PagesCompactArgs a, hipStream_t stream) {
  const int64_t entries = a.batch * a.cols;
  if (a.pages <= kAlonePages && entries <= kAloneEntries) {
    launch_kernel(kKernPagesCompact, pages_compact_kernel, dim3(1), dim3(kCompactThreads), stream, a, static_cast<int>(entries));
    return hipGetLastError();
  }
  const uint32_t chunks = static_cast<uint32_t>(ceil_div(a.pages, kCompactChunk));
  a.rank = static_cast<int32_t*>(a.workspace);
  a.counts = a.rank + a.pages;
  launch_kernel(kKernPagesCount, pages_count_kernel, dim3(chunks), dim3(kCompactThreads), stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  launch_kernel(kKernPagesRank, pages_rank_kernel, dim3(chunks), dim3(kCompactThreads), stream, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  launch_kernel(kKernPagesRename, pages_rename_kernel,
                dim3(static_cast<uint32_t>(ceil_div(entries > a.pages ? entries : a.pages, 256))), dim3(256), stream, a, entries);
  return hipGetLastError();
}

hipError_t launch_pages_copy(PagesCopyArgs a, hipStream_t stream) {
  if (a.pairs == 0 || a.caches == 0) return hipSuccess;
  a.first_piece[0] = 0;
  for (int c = 0; c < a.caches; ++c)
    a.first_piece[c + 1] = a.first_piece[c] + static_cast<int32_t>(ceil_div(a.page_bytes[c], kCopyPiece));
  const int64_t pieces = a.pairs * a.first_piece[a.caches];
  launch_kernel(kKernPagesCopy, pages_copy_kernel, dim3(static_cast<uint32_t>(pieces < kCopyBlocks ? pieces : kCopyBlocks)),
                dim3(kCopyThreads), stream, a);
  return hipGetLastError();
}

}  // namespace nvdsa
