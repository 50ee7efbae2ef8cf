// Attention of requests that share a prefix's pages, over the 16-bit latent
// cache:
//
//   o[t, h] = softmax(scale * (q . ckv + q_rope . kpe)) . ckv   over the slots that row t sees
//
// A query (row, head) is a pair; the packed rows of a group's requests are
// neighbours, so that all their pairs make one product with the pages that the
// group shares: items of up to 128 pairs against those pages, read once, and
// items of one request's pairs against the pages behind them.  A plan lays the
// items' tiles of 32 keys in a row and cuts it into equal parts, one per workgroup
// and CU; what lies across parts, and a pair's two items, leave fp32 partial sums
// that a join kernel adds up.
//
// A softmax in one pass: P = 2^(score - reference) per row, with a reference that
// moves only when a score outgrows it, sums of P and P V in fp32, one division at
// the end.  P is rounded to the cache's 16 bits for the second product, and the sum of
// P is that of the rounded values: they are weights that sum to one, and their half
// steps move a row by half a step of sum p |v - o| at most, also where nearly equal
// weights over thousands of keys are all rounded the same way (with the sum of the
// unrounded P such a row was off by half a step of itself: 1.2 times the tests' bound).
// A second product of what the rounding leaves out, as the sparse attention has it,
// would add 32 to the 68 products of a tile that bind items of 128 pairs: 64 requests
// of 64 heads on prefixes of 32768 tokens would take 366 us and not 280 in this kernel,
// 32 on 16384 109 and 89, 24 requests of 8 heads 23.7 and 22.7, and outputs be off by
// 1.7e-3 (bf16, relative to 64 bits; the store's rounding alone) and not 1.8 to 1.9e-3.
// Everything else stays in fp32.
//
// Bounds.  Items of 128 pairs: their products, 68 of 32 x 32 x 16 a wave and tile,
// 2176 clocks; a tile takes 3480 (loads 230 of them, the softmax 380, the wait for
// LDS at either barrier about 90 each), and the clock falls to 1.8 GHz under them:
// 64 rows of 64 heads on four prefixes of 32768 tokens run at 0.98 PFLOP/s, where the
// library's 8192^3 product reaches 1.25.  Items of up to 64: the pages' way, 64
// bytes a clock and CU (64 requests of 100 to 4000 own tokens, 16 heads: 33 us,
// 4.5 TB/s, a large copy 4.8).  Small calls: latency, 12 us of launch, plan, page
// ids, first tiles, last sums, and 5 of the join.
#include <cstddef>
#include <utility>

#include "lds_load.h"
#include "nvdsa_common.h"
#include "nvdsa_kernels.h"

namespace nvdsa {
namespace {

constexpr int kThreads = 256;
constexpr int kPairs = 128;    // of an item: four tiles of 32, one a wave
constexpr int kKeys = 32;      // of a tile
constexpr int kPageTiles = kBlock / kKeys;
constexpr int kBuffers = 4;    // tiles in LDS
constexpr int kCkvBytes = kCkvDim * 2, kKpeBytes = kKpeDim * 2;
constexpr int kTileBytes = kKeys * (kCkvBytes + kKpeBytes);
constexpr int kSteps = kQkDim / 16;   // products of 16 dims: 32 of the latent, 4 of the rope
constexpr int kTileLoads = 9;         // of a wave
constexpr int kParts = 256;           // workgroups, one per CU (LDS)
// What the begin and end of a segment cost, in tiles (measured: 30 to 45 thousand
// clocks).  With 4: a drafting step of 16 x 4 rows 54 us and not 45, a part that
// begins many segments being the last.
constexpr int kBegin = 8;
// Pairs from which a wave joins one, and not four: 4000 pairs 11 us, and 23 by four
// waves each; 192 pairs cut into 180 parts 12.5 and 7.5 us.
constexpr int kJoinByWave = 2048;
// Tiles of a part at least: half of it would double the sums that are written and
// joined, twice takes as long as the tiles do (24 requests in three groups: 24 us, and
// 35 with 8; with 3 the attention 1 us less, the join of one long request 3 more).
constexpr int kLeastTiles = 4;
// Tiles (of items of 128 pairs) up to which items hold 64, whose segments begin and
// end in half the time.  128 heads, in all: 1000 tokens 25 us and not 29, 32 x 1000
// (1024 tiles) 47 and 51; 32 x 2000 (2016 tiles) 59 and 57, 32 x 4000 88 and 73.
constexpr int kNarrow = 5 * kParts;
// What sharing has to save in all, in half tiles of up to 32 pairs (0.4 us of a
// part each): below, more items that every workgroup has a part of end sooner than
// fewer and their join.  In all, read once and by everybody: 16 requests of 64 heads
// on 4096 tokens (8 a part) 45 us and 42, on 8192 (16) 54 and 56; 16 x 4 rows on
// 8192 to 12301 (14) 56 and 60; 64 of 16 heads on 1024 (12) 39 and 33, on 2048 (24)
// 41 and 42; 32 on 16384 tokens (64) 106 and 149.
constexpr int kLeastSaved = 13 * kParts;
// Parts of an item that may hold fewer than kLeastTiles: the join has them all on
// their way at once.  One request of 16 heads and 1000 tokens 13.6 us and not 14.6, 2
// short ones 12.8 and 19.4; with 16 parts 4 requests of 32 heads on 4096 tokens take
// 3 us more.
constexpr int kEasyParts = 8;
constexpr float kLog2e = 1.4426950408889634f;
// P = 2^(score - reference): a reference is set so that the largest P of its
// tile is 2^kRise and kept until one passes 2^kMost.  fp16 holds P from 2^-24
// on, so keys down to 2^-32 of the row's largest count; bf16 has fp32's range.
constexpr float kRise = 8.f;
constexpr float kMost = 15.9f;

// ---------------------------------------------------------------- the plan
struct Span {        // pairs against tiles of one table row's pages
  int64_t unit0;     // first unit of the first item
  int32_t merge;     // first of the group's pairs that two items have (-1: one item only)
  int32_t pair0, pairs;
  int32_t tile0, tiles;
  int32_t table;     // row of the block table
  int32_t group;     // request: its group's span (-1: none)
  int32_t length;    // request: of the tokens (more than the table holds by its rows at most)
};
struct Start {       // where a part begins
  int64_t unit;
  int64_t stop;
  int32_t span;      // groups first, then requests
};
struct Cut {         // of all units into parts: the first `longer` ones hold one more
  int32_t parts;     // (0: no units)
  int32_t longer;
  int64_t units;     // of the others
  int32_t width;     // pairs of an item
};
struct Plan {
  Start* parts;      // [kParts]
  Cut* cut;          // [1]
  Span* spans;       // [groups + batch]
  int32_t* visible;  // [rows]
  int32_t* request;  // [rows], -1: of no request
  float2* refs;      // of the partial sums: reference and sum of P
  float* sums;       // [..][512]
  int64_t stride;    // pairs of a part's slot
};
__host__ __device__ inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
__host__ __device__ inline int64_t slot_pairs(int64_t rows, int64_t heads) {
  const int64_t n = (rows * heads + 31) / 32 * 32;
  return n < kPairs ? n : kPairs;
}
// Pairs that two items may have: a group of n requests that shares has fewer than 128 n.
__host__ __device__ inline int64_t merge_pairs(int64_t rows, int64_t heads, int64_t batch, int64_t groups) {
  const int64_t n = rows * heads;
  return groups == 0 ? 0 : (n < batch * kPairs ? n : batch * kPairs);
}
__host__ __device__ inline size_t carve(void* ws, int64_t rows, int64_t heads, int64_t batch, int64_t groups, Plan* plan) {
  char* p = static_cast<char*>(ws);
  char* const start = p;
  auto take = [&](size_t bytes) {
    char* at = p;
    p += align256(bytes);
    return at;
  };
  Plan w;
  w.parts = reinterpret_cast<Start*>(take(sizeof(Start) * kParts));
  w.cut = reinterpret_cast<Cut*>(take(sizeof(Cut)));
  w.spans = reinterpret_cast<Span*>(take(sizeof(Span) * (groups + batch)));
  w.visible = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * rows));
  w.request = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * rows));
  w.stride = slot_pairs(rows, heads);
  const int64_t partial = 2 * kParts * w.stride + 2 * merge_pairs(rows, heads, batch, groups);
  w.refs = reinterpret_cast<float2*>(take(sizeof(float2) * partial));
  w.sums = reinterpret_cast<float*>(take(sizeof(float) * partial * kCkvDim));
  if (plan) *plan = w;
  return static_cast<size_t>(p - start);
}

__device__ inline int32_t items_of(const Span& s, int width) { return (s.pairs + width - 1) / width; }
__device__ inline int64_t units_of(const Span& s, int width) { return static_cast<int64_t>(items_of(s, width)) * (s.tiles + kBegin); }
__device__ inline int64_t part_start(const Cut& c, int w) { return w * c.units + (w < c.longer ? w : c.longer); }
// The part of a unit.  (At most kParts of them, so that the guess is off by one at most.)
__device__ inline int part_of(const Cut& c, int64_t unit) {
  int w = static_cast<int>(static_cast<float>(unit) / (static_cast<float>(c.units) + static_cast<float>(c.longer) / static_cast<float>(c.parts)));
  w = w < c.parts ? w : c.parts - 1;
  while (w + 1 < c.parts && part_start(c, w + 1) <= unit) ++w;
  while (w > 0 && part_start(c, w) > unit) --w;
  return w;
}
// x / d, of less than 2^21.
__device__ inline int quotient(int64_t x, int32_t d) {
  int q = static_cast<int>(static_cast<float>(x) / static_cast<float>(d));
  while (static_cast<int64_t>(q + 1) * d <= x) ++q;
  while (static_cast<int64_t>(q) * d > x) --q;
  return q;
}
// What a tile of a request's or a group's items takes, in half tiles of up to 32 pairs
// (measured: 2100, 3000 and 3500 clocks for 32, 64 and 128 pairs).
__device__ inline int32_t time_of(int32_t pairs) { return pairs <= 32 ? 2 : (pairs <= 64 ? 3 : (pairs + kPairs - 1) / kPairs * 4); }
// Values that every lane holds, in scalar registers.
__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(x) >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ inline Span uniform(const Span& s) {
  return {uniform(s.unit0), uniform(s.merge), uniform(s.pair0), uniform(s.pairs),
          uniform(s.tile0), uniform(s.tiles), uniform(s.table), uniform(s.group), uniform(s.length)};
}
// (Pairs fit 26 bits.)
__device__ inline uint32_t row_of(int64_t pair, int64_t heads) { return static_cast<uint32_t>(pair) / static_cast<uint32_t>(heads); }
// Row of the partial sums of a segment's first pair.
__device__ inline int64_t part_row(const Plan& w, int part, bool begins) { return (2 * static_cast<int64_t>(part) + (begins ? 1 : 0)) * w.stride; }
__device__ inline int64_t merge_row(const Plan& w, int64_t merged, int pair, bool own) {
  return 2 * kParts * w.stride + 2 * (merged + pair) + (own ? 1 : 0);
}

constexpr int kPlanThreads = 1024;

// Sums of what the threads before hold, of two values at once; *all_..: of everybody's.
template <int THREADS>
__device__ inline void plan_scan(int64_t& x, int64_t& y, int64_t (*scratch)[2], int64_t* all_x, int64_t* all_y) {
  const int wid = threadIdx.x >> 6;
  const int64_t sx = static_cast<int64_t>(wave_inclusive_scan(static_cast<uint64_t>(x)));
  const int64_t sy = static_cast<int64_t>(wave_inclusive_scan(static_cast<uint64_t>(y)));
  __syncthreads();
  if ((threadIdx.x & 63) == 63) {
    scratch[wid][0] = sx;
    scratch[wid][1] = sy;
  }
  __syncthreads();
  int64_t before_x = 0, before_y = 0, sum_x = 0, sum_y = 0;
  for (int k = 0; k < THREADS / 64; ++k) {
    const int64_t u = scratch[k][0], v = scratch[k][1];
    before_x += k < wid ? u : 0;
    before_y += k < wid ? v : 0;
    sum_x += u;
    sum_y += v;
  }
  *all_x = sum_x;
  *all_y = sum_y;
  x = before_x + sx - x;
  y = before_y + sy - y;
}

// What a plan of THREADS threads holds in LDS: of that many requests and groups
// (the others' are read from memory again).
template <int THREADS, bool HERE>
struct LdsPlan {
  int64_t scratch[THREADS / 64][2];
  int64_t unit0[HERE ? 1 : 2 * THREADS];
  Span group[HERE ? 1 : THREADS];
  int32_t q_ends[THREADS], group_ends[THREADS];
};

// Latency all the way: what it reads comes to LDS at once.  HERE: all spans are
// left in `here`, for which there are threads enough; WRITES: in memory.
template <int THREADS, bool HERE>
__device__ __forceinline__ Cut make_plan(const PrefixAttentionArgs& a, const Plan& w, LdsPlan<THREADS, HERE>& lds, Span* here,
                                         bool writes) {
  const int tid = threadIdx.x;
  const int64_t cap = a.cols * kBlock;
  const int batch = static_cast<int>(a.batch), groups = static_cast<int>(a.groups), rows = static_cast<int>(a.rows);
  const int heads = static_cast<int>(a.heads), spans = groups + batch;
  auto clamp = [](int64_t x, int64_t most) { return static_cast<int>(x < 0 ? 0 : (x > most ? most : x)); };
  int64_t own_length = 0, own_prefix = 0;  // of request and group tid
  if (tid < batch) {
    lds.q_ends[tid] = a.seq_q[tid];
    own_length = a.seq_kv[tid];
  }
  if (tid < groups) {
    lds.group_ends[tid] = a.group_ends[tid];
    own_prefix = a.prefix_lens[tid];
  }
  __syncthreads();
  auto row_at = [&](int b) {  // first packed row of request b
    return b > 0 ? clamp(HERE || b <= THREADS ? lds.q_ends[b - 1] : a.seq_q[b - 1], rows) : 0;
  };
  auto group_end = [&](int g) { return clamp(HERE || g < THREADS ? lds.group_ends[g] : a.group_ends[g], batch); };
  int64_t units = 0, merged = 0, items = 0;
  int width = kPairs;
  // Groups: one that shares has its pages read for several requests, whose pairs
  // fit fewer items, and saves more than its items' beginnings cost.
  auto group_span = [&](int g, int64_t* saved) {
    Span s{};
    s.merge = s.group = -1;
    if (g >= groups) return s;
    const int b0 = g > 0 ? group_end(g - 1) : 0, b1 = group_end(g);
    const int r0 = row_at(b0), r1 = row_at(b1);
    if (b1 - b0 < 2 || r1 <= r0) return s;
    const int tokens = clamp(g == tid ? own_prefix : a.prefix_lens[g], cap);
    s.tiles = tokens / kBlock * kPageTiles;
    s.pair0 = r0 * heads;
    s.table = b0;
    const int pairs = (r1 - r0) * heads, n = b1 - b0;
    const int64_t less = s.tiles * (static_cast<int64_t>(n) * time_of(static_cast<uint32_t>(pairs) / static_cast<uint32_t>(n)) - time_of(pairs));
    if (pairs < static_cast<int64_t>(n) * kPairs && less > 2 * kBegin * time_of(pairs)) {
      s.pairs = pairs;
      *saved += less;
    }
    return s;
  };
  int64_t saved = 0;
  const Span own_group = group_span(tid, &saved);
  for (int g = tid + THREADS; g < groups; g += THREADS) group_span(g, &saved);
  bool shares = true;   // until the first sum is there
  for (int g0 = 0; g0 < groups; g0 += THREADS) {
    const int g = g0 + tid;
    Span s = own_group;
    int64_t rest = 0;
    if (g0 > 0) s = group_span(g, &rest);
    int64_t m = s.pairs, sum_m, all_saved;
    if (g0 == 0) rest = saved;
    plan_scan<THREADS>(m, rest, lds.scratch, &sum_m, &all_saved);
    if (g0 == 0) shares = all_saved >= kLeastSaved;
    if (!shares) s.pairs = 0;
    // (Ends that decrease could count a request's pairs for several groups: there
    // is room for each pair once.)
    if (merged + m + s.pairs > merge_pairs(rows, heads, batch, groups)) s.pairs = 0;
    if (s.pairs > 0) {
      s.merge = merged + m;
      // The table of the first request with rows: one that has ended need not hold the
      // pages any more.
      const int r0 = row_at(s.table);
      int last = group_end(g) - 1;
      if (row_at(s.table + 1) > r0) last = s.table;
      while (s.table < last) {
        const int mid = (s.table + last) >> 1;
        if (row_at(mid + 1) <= r0)
          s.table = mid + 1;
        else
          last = mid;
      }
    }
    merged += sum_m;
    int64_t u = units_of(s, kPairs), n = items_of(s, kPairs), sum_u, sum_n;
    plan_scan<THREADS>(u, n, lds.scratch, &sum_u, &sum_n);
    s.unit0 = units + u;
    units += sum_u;
    items += sum_n;
    if (g < groups) {
      if (writes) w.spans[g] = s;
      if constexpr (HERE) {
        here[g] = s;
      } else {
        if (g < THREADS) lds.group[g] = s;
        if (g < 2 * THREADS) lds.unit0[g] = s.unit0;
      }
    }
  }
  __syncthreads();
  for (int b0 = 0; b0 < batch; b0 += THREADS) {
    const int b = b0 + tid;
    Span s{};
    s.merge = s.group = -1;
    if (b < batch) {
      const int r0 = row_at(b), r1 = row_at(b + 1);
      s.pair0 = r0 * heads;
      s.pairs = r1 > r0 ? (r1 - r0) * heads : 0;
      // (Tokens past the table have no slots; the rows before the last see so many less.)
      s.length = clamp(b == tid ? own_length : a.seq_kv[b], cap + (r1 > r0 ? r1 - r0 : 0));
      s.tiles = static_cast<int>(((s.length < cap ? s.length : cap) + kKeys - 1) / kKeys);
      s.table = b;
      // The group: the first whose end lies behind the request.
      int lo = 0, hi = groups;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (group_end(mid) <= b)
          lo = mid + 1;
        else
          hi = mid;
      }
      if (lo < groups && s.pairs > 0) {
        Span g;
        if constexpr (HERE)
          g = here[lo];
        else
          g = lo < THREADS ? lds.group[lo] : w.spans[lo];
        // (Ends that decrease: a request outside the group's rows is its own.)
        if (g.pairs > 0 && b >= g.table && s.pair0 >= g.pair0 && s.pair0 + s.pairs <= g.pair0 + g.pairs) {
          s.group = lo;
          s.merge = g.merge + (s.pair0 - g.pair0);
          s.tile0 = g.tiles;
          s.tiles = s.tiles > g.tiles ? s.tiles - g.tiles : 0;
        }
      }
    }
    int64_t u = units_of(s, kPairs), sum_u, sum_n;
    int64_t n = items_of(s, kPairs) | static_cast<int64_t>(items_of(s, kPairs / 2)) << 32;  // (both fit 31 bits)
    plan_scan<THREADS>(u, n, lds.scratch, &sum_u, &sum_n);
    int sum_items = static_cast<int>(sum_n);
    const int narrow_items = static_cast<int>(sum_n >> 32);
    if (items == 0 && batch <= THREADS && narrow_items > sum_items && sum_u - sum_items * kBegin <= kNarrow) {
      int64_t none = 0;
      width = kPairs / 2;
      u = units_of(s, width);
      plan_scan<THREADS>(u, none, lds.scratch, &sum_u, &sum_n);
      sum_items = narrow_items;
    }
    s.unit0 = units + u;
    units += sum_u;
    items += sum_items;
    if (b < batch) {
      if (writes) w.spans[groups + b] = s;
      if constexpr (HERE)
        here[groups + b] = s;
      else if (groups + b < 2 * THREADS)
        lds.unit0[groups + b] = s.unit0;
    }
  }
  // The rows' requests, and what they see (HERE: every workgroup some of them).
  for (int t = HERE ? blockIdx.x * THREADS + tid : tid; t < rows; t += HERE ? kParts * THREADS : THREADS) {
    int lo = 0, hi = batch;  // the request: an end behind the row, the end before it not
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (row_at(mid + 1) <= t)
        lo = mid + 1;
      else
        hi = mid;
    }
    if constexpr (!HERE) {
      w.visible[t] = lo < batch ? clamp(static_cast<int64_t>(a.seq_kv[lo]) - (row_at(lo + 1) - 1 - t), cap) : 0;
    }
    w.request[t] = lo < batch ? lo : -1;
  }
  int64_t most = (units - items * kBegin) / kLeastTiles;
  const int64_t few = units - items * kBegin;
  if (most < kEasyParts * items) most = few < kEasyParts * items ? few : kEasyParts * items;
  if (most < items) most = items;
  Cut cut;
  cut.parts = static_cast<int32_t>(most > kParts ? kParts : (most < 1 ? 1 : most));
  cut.units = units / cut.parts;
  cut.longer = static_cast<int32_t>(units - cut.units * cut.parts);
  if (units == 0) cut.parts = 0;
  cut.width = width;
  if (writes && tid == 0) *w.cut = cut;
  __syncthreads();
  return cut;
}

// Where a part begins; unit0_at(i): of span i.
template <typename F>
__device__ __forceinline__ Start start_of(const Cut& cut, int part, int spans, F&& unit0_at) {
  Start p;
  p.unit = part_start(cut, part);
  p.stop = part_start(cut, part + 1);
  // The last span that begins at or before the unit (spans without pairs begin
  // where the next does).
  int lo = 0, hi = spans - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (unit0_at(mid) <= p.unit)
      lo = mid;
    else
      hi = mid - 1;
  }
  p.span = lo;
  return p;
}

__global__ __launch_bounds__(kPlanThreads) void prefix_plan_kernel(PrefixAttentionArgs a) {
  __shared__ LdsPlan<kPlanThreads, false> lds;
  Plan w;
  carve(a.workspace, a.rows, a.heads, a.batch, a.groups, &w);
  const Cut cut = make_plan<kPlanThreads, false>(a, w, lds, nullptr, true);
  const int tid = threadIdx.x;
  if (tid < cut.parts)
    w.parts[tid] = start_of(cut, tid, static_cast<int>(a.groups + a.batch),
                            [&](int i) { return i < 2 * kPlanThreads ? lds.unit0[i] : w.spans[i].unit0; });
}

// ------------------------------------------------------------- the attention
struct LdsFew {   // items of up to 64 pairs
  alignas(16) uint8_t keys[kBuffers][kTileBytes];
  alignas(16) uint16_t p[64 * kKeys];
  float factor[64];
  float2 row[64];       // reference and sum of P, at a segment's end
  float top[2][32];     // of 16 keys each
  int32_t moved[4];     // a wave's rows have new references
  int32_t least[4];     // the least that a row of a wave sees
};
struct LdsMany {  // more
  alignas(16) uint8_t rope[kPairs * kKpeBytes];   // the pairs' rope dims (at a segment's end: references and sums)
  uint8_t p[kPairs * kKeys * 2];
  uint8_t half[4][4][64][16];                     // scores of half the dims, to a wave
  uint8_t keys[3][kTileBytes];
  float factor[kPairs];
  int32_t moved[4];     // the tile at which a wave's rows have new references
  int32_t moved_last;   // the last such tile of all
  int32_t least[4];
};
union Lds {
  LdsFew few;
  LdsMany many;
  LdsPlan<kThreads, true> plan;
};
// Spans, at most, of a plan that every workgroup makes: LDS has room for them beside
// the tiles.  Against a plan kernel before (in all): 2 short requests 18 us and not
// 22, 24 requests in three groups 31 and 36, 32 on 16384 tokens 106 and 110.
constexpr int kHere = kThreads;
constexpr int kStage = 16 * 1024;                // 32 pairs in LDS, of a wave before and after the tiles
static_assert(sizeof(Lds) + kHere * sizeof(Span) <= 160 * 1024 && 4 * kStage <= 2 * kTileBytes, "LDS");
static_assert(offsetof(LdsMany, keys) % 4096 == 0 && offsetof(LdsMany, rope) % 8192 == 0, "exclusive ors within");

struct Segment {
  int64_t pair0;      // of all pairs
  int32_t count;
  int32_t length, end;  // request: its tokens, and the row behind its last; else `end` is -1
  int32_t tile0, tile1;
  const int32_t* table;
  bool direct;        // the output itself
  int64_t row;        // of the partial sums
  int64_t row_step;   // between pairs of it
};

// What a row of a segment sees.
template <bool HERE>
struct Seen {
  const int32_t* visible;   // [rows]; HERE: found among the requests' spans
  const Span* requests;
  int32_t batch, heads;
  // (No lane leaves the others' way here: the compiler has put the copy of a register
  // before the point where all lanes are back.)
  __device__ int operator()(const Segment& s, int64_t pair) const {
    const int row = static_cast<int>(row_of(pair, heads));
    int length = s.length, end = s.end;
    if (s.end < 0) {
      if constexpr (!HERE) return visible[row];
      int at = 0;   // requests that end at or before the pair
      for (int step = kHere; step > 0; step >>= 1) {
        const int next = at + step;
        const Span& last = requests[(next < batch ? next : batch) - 1];
        const int32_t last_end = last.pair0 + last.pairs;
        at = (next < batch) & (last_end <= pair) ? next : at;
      }
      const Span& mine = requests[at];
      length = mine.length;
      end = static_cast<int>(row_of(mine.pair0 + mine.pairs, heads));
    }
    length -= end - 1 - row;
    return length > 0 ? length : 0;
  }
};

// The ids of 64 pages, a lane each (-1: none), from a column on.
struct Pages {
  const int32_t* table;
  int32_t last, blocks;   // column
  int32_t first, held;
  __device__ Pages(const Segment& s, const PrefixAttentionArgs& a) : table(s.table), blocks(static_cast<int32_t>(a.blocks)) {
    const int c = column(s.tile1 - 1);
    last = c < a.cols ? c : static_cast<int32_t>(a.cols) - 1;
    hold(s.tile0);
  }
  __device__ void hold(int tile) {
    first = column(tile);
    const int c = first + (threadIdx.x & 63);
    const int32_t page = table[c <= last ? c : last];   // (no lane leaves: see Seen)
    held = (c <= last) & (page >= 0) & (page < blocks) ? page : -1;
  }
  __device__ static int column(int tile) { return static_cast<int>(static_cast<uint32_t>(tile) / kPageTiles); }
  __device__ bool holds(int tile) const { return column(tile) - first < 64; }
  __device__ int of(int tile) const { return __builtin_amdgcn_readlane(held, column(tile) - first); }
};

// o += a b, with o in accumulation registers: 256 of them hold four tiles of
// pairs, and the compiler would share them with the scores.  Who reads or writes o
// otherwise calls settle() first and after.  WAIT: two wait states, for an operand
// that a vector instruction may have written just before (where one is first used:
// operands come from LDS, but the compiler may have copied them).
template <bool WAIT>
__device__ inline void accumulate(Bf16, u32x4_t a, u32x4_t b, f32x16_t& o) {
  if constexpr (WAIT)
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(b));
  else
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(b));
}
template <bool WAIT>
__device__ inline void accumulate(F16, u32x4_t a, u32x4_t b, f32x16_t& o) {
  if constexpr (WAIT)
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(b));
  else
    asm("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(b));
}
// Waits out a product that writes o, or a write of o before a product.
__device__ inline void settle(f32x16_t& o) { asm volatile("s_nop 15\n\ts_nop 7" : "+a"(o)); }
// The same for all of them at once: what is before stays before, and so behind.
template <int TILES>
__device__ __forceinline__ void settle(f32x16_t (&o)[4][TILES]) {
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < TILES; ++r) asm volatile("" : "+a"(o[d][r]));
  asm volatile("s_nop 15\n\ts_nop 7");
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < TILES; ++r) asm volatile("" : "+a"(o[d][r]));
}

// threadIdx.x, anew for every segment: places in LDS that follow from it would
// otherwise be worked out once for all forms of the loop, and spilled.
__device__ inline int own_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}
// f(0), f(1) .. f(N - 1), each with a constant.
template <typename F, int... J>
__device__ __forceinline__ void steps_of(F&& f, std::integer_sequence<int, J...>) {
  (f(std::integral_constant<int, J>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void steps(F&& f) {
  steps_of(f, std::make_integer_sequence<int, N>{});
}
// A copy that stays one: the compiler would let a chain of products change its
// registers halfway, and wait for it.
__device__ inline float moved_here(float x) {
  float r;
  asm volatile("v_mov_b32 %0, %1" : "=v"(r) : "v"(x));
  return r;
}
// By address in LDS.
__device__ inline u32x4_t lds_get(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(at);
}
__device__ inline void lds_put(uint32_t at, u32x4_t v) { *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(at) = v; }
__device__ inline void lds_put(uint32_t at, uint32_t x, uint32_t y) {
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  *reinterpret_cast<__attribute__((address_space(3))) u32x2_t*>(at) = u32x2_t{x, y};
}
// What this wave has written to LDS is there, and what it has asked for.
__device__ inline void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// Nothing is known of x from here on: what follows from it is worked out where it
// is used, and holds no register across the loop.
__device__ inline void forget(uint32_t& x) { asm volatile("" : "+v"(x)); }
// (fmaxf() would first make its operands canonical.)
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The values of a pack2.
template <typename T>
__device__ inline float low_half(uint32_t v) { return T::to_float(static_cast<uint16_t>(v)); }
template <typename T>
__device__ inline float high_half(uint32_t v) { return T::to_float(static_cast<uint16_t>(v >> 16)); }

// Zeros in the place of infinities and NaN.
template <typename T>
__device__ inline u32x4_t finite_or_zero(u32x4_t v) {
  constexpr uint32_t kInf = std::is_same<T, Bf16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = (v[k] & 0x7fffu) >= kInf ? 0u : v[k] & 0xffffu;
    const uint32_t hi = ((v[k] >> 16) & 0x7fffu) >= kInf ? 0u : v[k] & 0xffff0000u;
    v[k] = lo | hi;
  }
  return v;
}

// A segment's outputs, or its partial sums; rows: references and sums of P.  A
// wave's 128 dims of 32 pairs go through 16 KiB of LDS of its own (at `stage`, of
// its wave), so that a store writes 512 neighbouring bytes of a pair and not 32.
// Place c ^ pair of a pair's chunks of 16 bytes: neighbouring pairs' lie in other banks.
template <typename T, int TILES>
__device__ __forceinline__ void finish(const PrefixAttentionArgs& a, const Plan& w, const Segment& s,
                                       const float2* rows, uint32_t stage, f32x16_t (&o)[4][TILES]) {
  const int lane = own_thread() & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  settle(o);
#pragma unroll
  for (int r = 0; r < TILES; ++r) {
    if (r * 32 >= s.count) break;
    const int left = s.count - r * 32;
    if (s.direct) {
      const float sum = rows[r * 32 + l32].y, by = sum == 0.f ? 0.f : 1.f / sum;
      const uint32_t to = stage + static_cast<uint32_t>(l32 * 256 + 8 * hh);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          lds_put(to + (((d * 4 + i) ^ l32) & 15) * 16, T::pack2(o[d][r][4 * i] * by, o[d][r][4 * i + 1] * by),
                  T::pack2(o[d][r][4 * i + 2] * by, o[d][r][4 * i + 3] * by));
      wait_lds();
      uint16_t* out = static_cast<uint16_t*>(a.out) + (s.pair0 + r * 32) * kCkvDim + wave * 128 + (lane & 15) * 8;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int m = 4 * n + (lane >> 4);
        const u32x4_t v = lds_get(stage + static_cast<uint32_t>(m * 256 + ((lane ^ m) & 15) * 16));
        if (m < left) *reinterpret_cast<u32x4_t*>(out + static_cast<int64_t>(m) * kCkvDim) = v;
      }
    } else {
      if (wave == 0 && hh == 0 && l32 < left) w.refs[s.row + (r * 32 + l32) * s.row_step] = rows[r * 32 + l32];
      const uint32_t to = stage + static_cast<uint32_t>(l32 * 512);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          lds_put(to + ((d * 8 + i * 2 + hh) ^ l32) * 16,
                  u32x4_t{__float_as_uint(o[d][r][4 * i]), __float_as_uint(o[d][r][4 * i + 1]),
                          __float_as_uint(o[d][r][4 * i + 2]), __float_as_uint(o[d][r][4 * i + 3])});
      wait_lds();
      float* out = w.sums + (s.row + r * 32 * s.row_step) * kCkvDim + wave * 128 + l32 * 4;
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const int m = 2 * n + hh;
        const u32x4_t v = lds_get(stage + static_cast<uint32_t>(m * 512 + (l32 ^ m) * 16));
        if (m < left) *reinterpret_cast<u32x4_t*>(out + m * s.row_step * kCkvDim) = v;
      }
    }
    if (r + 1 < TILES) wait_lds();
  }
}

// A segment without tiles.
template <typename T>
__device__ __forceinline__ void nothing(const PrefixAttentionArgs& a, const Plan& w, const Segment& s) {
  if (s.direct) {
    u32x4_t* out = static_cast<u32x4_t*>(a.out) + s.pair0 * (kCkvDim / 8);
    for (int i = threadIdx.x; i < s.count * (kCkvDim / 8); i += kThreads) out[i] = u32x4_t{0, 0, 0, 0};
  } else {
    for (int m = threadIdx.x; m < s.count; m += kThreads) w.refs[s.row + m * s.row_step] = make_float2(-INFINITY, 0.f);
  }
}

// Items of up to 32 TILES pairs, bound by the tiles' way from memory.  For the
// scores of a tile a wave takes 16 pairs, with their queries in registers: all 32
// keys of it where there are 64 pairs, 16 keys where there are 32 (two waves then
// meet in LDS for a row's largest score).  For the outputs it takes 128 dims of
// all pairs.  At barrier A everybody is done with tile t - 1, and tile t + 1 and
// the largest scores of tile t have arrived; then tile t + 3 is asked for and tile
// t weighed; at B its P is there, and its outputs and the scores of tile t + 1 follow.
template <typename T, int TILES, typename SEEN>
__device__ __forceinline__ void attend(const PrefixAttentionArgs& a, const Plan& w, const Segment& s, const SEEN& seen, LdsFew& lds) {
  const int tid = own_thread();
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5, l16 = lane & 15, quad = lane >> 4;
  const int m_mine = (TILES == 2 ? wave : wave & 1) * 16 + l16;
  const int half0 = TILES == 2 ? 0 : wave >> 1;   // first 16 keys of the wave's
  const uint32_t lds_keys = lds_address(lds.keys);

  // A row k of a tile holds chunk c (16 bytes) at place c ^ swizzle(k) within its
  // group of 16: 16 keys of one chunk lie in 64 different banks, and so do four
  // neighbouring keys of four neighbouring chunks.  Rope rows likewise, 8 chunks.
  auto swizzle = [](int k) { return ((k & 3) << 2) | ((k >> 2) & 3); };
  uint32_t byte_of[4], rope_byte;   // this lane's place of a wave's loads
#pragma unroll
  for (int j = 0; j < 4; ++j)
    byte_of[j] = static_cast<uint32_t>(wave * kCkvBytes + ((lane & 48) | ((lane ^ ((wave << 2) | j)) & 15)) * 16);
  {
    const int k = wave * 8 + (lane >> 3);
    rope_byte = static_cast<uint32_t>(k * kKpeBytes + ((lane ^ (k >> 1)) & 7) * 16);
  }
  const int k_row = half0 * 16 + l16;
  const uint32_t k_at = lds_keys + static_cast<uint32_t>(k_row * kCkvBytes + ((quad ^ swizzle(l16)) & 15) * 16);
  const uint32_t r_at = lds_keys + static_cast<uint32_t>(kKeys * kCkvBytes + k_row * kKpeBytes + ((quad ^ (l16 >> 1)) & 7) * 16);
  uint32_t v_at[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int key = 8 * hh + 4 * part + ((lane & 15) >> 2);
    const int c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);   // of four neighbours
    v_at[part] = lds_keys + static_cast<uint32_t>(key * kCkvBytes + wave * 256 + ((c ^ swizzle(key)) & 15) * 16 + (lane & 1) * 8);
  }
  const uint32_t p_at = lds_address(lds.p);
  const uint32_t p_read = p_at + static_cast<uint32_t>(l32 * 64), p_swz = (l32 >> 2) & 3;
  const uint32_t p_write = p_at + static_cast<uint32_t>(m_mine * 64 + (quad & 1) * 8);

  Pages pages(s, a);
  auto load_tile = [&](int tile) {
    int page = pages.of(tile);
    page = page < 0 ? 0 : page;
    const int64_t row = static_cast<int64_t>(page) * kBlock + (tile % kPageTiles) * kKeys;
    const uint8_t* base = static_cast<const uint8_t*>(a.kv_cache) + row * kCkvBytes;
    const uint8_t* rope = static_cast<const uint8_t*>(a.k_rope) + row * kKpeBytes;
    const uint32_t to = lds_keys + (tile % kBuffers) * kTileBytes + wave * 1024;
#pragma unroll
    for (int i = 0; i < 8; ++i) load_to_lds(base + i * 4096, byte_of[i & 3], to + i * 4096);
    load_to_lds(rope, rope_byte, to + kKeys * kCkvBytes);
  };

  lds_barrier();  // (the segment before is done with LDS)
  const int t0 = s.tile0, t1 = s.tile1;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (t0 + k < t1) load_tile(t0 + k);

  constexpr int kWide = kQkDim / 32, kWideLatent = kCkvDim / 32;   // products of 32 dims
  u32x4_t q[kWide];
  const int64_t pair = s.pair0 + (m_mine < s.count ? m_mine : 0);
  int vis = seen(s, pair);
  vis = m_mine < s.count ? vis : 0;
  {
    const u32x4_t* qn = static_cast<const u32x4_t*>(a.query) + pair * (kCkvDim / 8) + quad;
    const u32x4_t* qr = static_cast<const u32x4_t*>(a.query_rope) + pair * (kKpeDim / 8) + quad;
#pragma unroll
    for (int j = 0; j < kWide; ++j) q[j] = j < kWideLatent ? qn[4 * j] : qr[4 * (j - kWideLatent)];
#pragma unroll
    for (int j = 0; j < kWide; ++j) asm volatile("" : "+v"(q[j]));
  }
  f32x16_t o[4][TILES];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < TILES; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][r][e] = 0.f;
  settle(o);
  float ref = 0.f, most = -INFINITY, l_run = 0.f;   // most: what a score may reach before the reference moves
  // The least that a row of this wave sees; every wave's meet in LDS.
  int vis_least = m_mine < s.count ? vis : 0x7fffffff;
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) vis_least = min(vis_least, __shfl_xor(vis_least, d));
  vis_least = __builtin_amdgcn_readfirstlane(vis_least);
  if (lane == 0) lds.least[wave] = vis_least;

  f32x4_t x[TILES];   // scores of key 16 (half0 + h) + 4 quad + e
  float top;
  auto score = [&](int tile) {
    const uint32_t at = (tile % kBuffers) * kTileBytes;
#pragma unroll
    for (int h = 0; h < TILES; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h][e] = 0.f;
    constexpr int kOperands = kWide * TILES, kOnTheWay = 6;   // (LDS answers after five products)
    u32x4_t k[kOnTheWay + 1];
    auto fetch = [&](auto n) __attribute__((always_inline)) {
      constexpr int i = decltype(n)::value, j = i / TILES, h = i % TILES;
      if constexpr (i < kOperands)
        k[i % (kOnTheWay + 1)] = j < kWideLatent ? lds_get(((k_at + at) ^ ((j & 3) * 64)) + (j >> 2) * 256 + h * 16 * kCkvBytes)
                                                 : lds_get(((r_at + at) ^ ((j - kWideLatent) * 64)) + h * 16 * kKpeBytes);
    };
    steps<kOnTheWay>(fetch);
    steps<kOperands>([&](auto n) __attribute__((always_inline)) {
      constexpr int i = decltype(n)::value, j = i / TILES, h = i % TILES;
      fetch(std::integral_constant<int, i + kOnTheWay>{});
      x[h] = T::mfma16(__builtin_bit_cast(typename T::vec8, k[i % (kOnTheWay + 1)]), __builtin_bit_cast(typename T::vec8, q[j]), x[h]);
      __builtin_amdgcn_sched_barrier(0);
    });
    const bool none = pages.of(tile) < 0;
#pragma unroll
    for (int h = 0; h < TILES; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h][e] *= a.scale * kLog2e;
    if (none || (tile + 1) * kKeys > vis_least) {
      const int left = none ? 0 : vis - tile * kKeys - 16 * half0 - 4 * quad;   // keys that the row sees, from the lane's first
#pragma unroll
      for (int h = 0; h < TILES; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h][e] = 16 * h + e < left ? x[h][e] : -INFINITY;
    }
    top = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
    if constexpr (TILES == 2) top = fmaxf(top, fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    top = xor32_op(xor16_op(top, MaxOp{}), MaxOp{});
    if constexpr (TILES == 1)
      if (quad == 0) lds.top[half0][m_mine] = top;
  };
  // Scores to P, against the row's reference.
  auto weigh = [&] {
    if constexpr (TILES == 1) top = fmaxf(lds.top[0][m_mine], lds.top[1][m_mine]);
    const bool past = top > most, moved = past && most != -INFINITY;   // (the first time o is zero)
    float f = 1.f;
    if (past) {
      const float now = top - kRise;
      f = moved ? __builtin_amdgcn_exp2f(ref - now) : 1.f;
      most = now + kMost;
      ref = now;
      l_run *= f;
    }
    const bool any = __any(moved);
    if (half0 == 0) {
      if (quad == 0) lds.factor[m_mine] = f;
      if (lane == 0) lds.moved[wave] = any;
    }
#pragma unroll
    for (int h = 0; h < TILES; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h][e] = __builtin_amdgcn_exp2f(x[h][e] - ref);
      const uint32_t p01 = T::pack2(x[h][0], x[h][1]), p23 = T::pack2(x[h][2], x[h][3]);
      l_run += low_half<T>(p01) + high_half<T>(p01) + low_half<T>(p23) + high_half<T>(p23);
      const int chunk = 2 * (half0 + h) + (quad >> 1);
      lds_put(p_write + static_cast<uint32_t>(((chunk ^ (m_mine >> 2)) & 3) * 16), p01, p23);
    }
  };
  // Values of keys that some row must not see: P is zero there, but zero times an
  // infinity or NaN is not.  (A row that does see such a key has them in its scores:
  // NaN, or +inf, which makes its P NaN.  Under a score of -inf P is zero, and the row
  // loses the NaN that an infinite value makes in its dims elsewhere.)
  auto scrub = [&](int tile) {
    uint8_t* v_tile = lds.keys[tile % kBuffers];
    for (int i = tid; i < kKeys * kCkvBytes / 16; i += kThreads) {
      u32x4_t* p = reinterpret_cast<u32x4_t*>(v_tile + i * 16);
      *p = finite_or_zero<T>(*p);
    }
  };
  auto output = [&](int tile) {
    const uint32_t at = (tile % kBuffers) * kTileBytes;
    const int4 moved = *reinterpret_cast<const int4*>(lds.moved);
#pragma unroll
    for (int r = 0; r < TILES; ++r) {
      if (__builtin_amdgcn_readfirstlane(r == 0 ? moved.x | moved.y : moved.z | moved.w) != 0) {
        const float f = lds.factor[r * 32 + l32];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          settle(o[d][r]);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][r][e] *= f;
          settle(o[d][r]);
        }
      }
    }
    u32x4_t p[2][TILES], v[3];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int r = 0; r < TILES; ++r) p[ks][r] = lds_get(p_read + r * 2048 + static_cast<uint32_t>(((2 * ks + hh) ^ p_swz) * 16));
    auto fetch = [&](auto n) __attribute__((always_inline)) {
      constexpr int i = decltype(n)::value, ks = i >> 2, d = i & 3;
      if constexpr (i < 8) {
        const uint2 lo = read_tr16(((v_at[0] + at) ^ (d * 64)) + ks * 16 * kCkvBytes);
        const uint2 hi = read_tr16(((v_at[1] + at) ^ (d * 64)) + ks * 16 * kCkvBytes);
        v[i % 3] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
      }
    };
    steps<2>(fetch);
    steps<8>([&](auto n) __attribute__((always_inline)) {
      constexpr int i = decltype(n)::value;
      fetch(std::integral_constant<int, i + 2>{});
#pragma unroll
      for (int r = 0; r < TILES; ++r) accumulate<true>(T{}, v[i % 3], p[i >> 2][r], o[i & 3][r]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  wait_loads<0>();
  lds_barrier();
  const int vis_all = __builtin_amdgcn_readfirstlane(min(min(lds.least[0], lds.least[1]), min(lds.least[2], lds.least[3])));
  score(t0);
  for (int t = t0; t < t1; ++t) {
    if (t + 2 < t1)
      wait_loads<kTileLoads>();
    else
      wait_loads<0>();
    lds_barrier();  // A
    if (!pages.holds(t + 3)) pages.hold(t);
    if (t + 3 < t1) load_tile(t + 3);
    weigh();
    if ((t + 1) * kKeys > vis_all || pages.of(t) < 0) scrub(t);
    lds_barrier();  // B
    output(t);
    if (t + 1 < t1) score(t + 1);
  }
  // References and sums of the rows, to every wave.
  l_run = xor32_op(xor16_op(l_run, AddOp{}), AddOp{});
  if constexpr (TILES == 1) {
    lds_barrier();
    if (half0 == 1 && quad == 0) lds.top[0][m_mine] = l_run;
    lds_barrier();
    l_run += lds.top[0][m_mine];
  }
  if (half0 == 0 && quad == 0) lds.row[m_mine] = make_float2(most == -INFINITY && l_run == 0.f ? -INFINITY : ref, l_run);
  lds_barrier();
  finish<T, TILES>(a, w, s, lds.row, lds_keys + wave * kStage, o);
}

// Items of more than 64 pairs, bound by their products.  For the scores of a tile
// a wave takes 64 pairs and half of the dims, so that every operand from LDS has
// two products; two waves meet in LDS, and each goes on with 32 pairs.  For the
// outputs it takes 128 dims of all pairs.  The scores of tile t + 1 are multiplied
// while the vector unit weighs tile t between the products, then the outputs of
// tile t.  Two barriers a tile: at A everybody is done with tile t - 1 and its P,
// tile t + 1 has arrived, and so have the halves of tile t's scores; at B P is
// there.  Products go on across either: operands of the last ones are in registers
// by then, and those behind it on the way.
template <typename T, typename SEEN>
__device__ __forceinline__ void attend_many(const PrefixAttentionArgs& a, const Plan& w, const Segment& s, const SEEN& seen, LdsMany& lds) {
  const int tid = own_thread();
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int rg = wave & 1, dh = wave >> 1;  // 64 pairs, half of the dims
  const int tile_mine = 2 * rg + dh;        // of 32 pairs that this wave weighs
  const int m_mine = tile_mine * 32 + l32;
  constexpr int kHalf = kSteps / 2, kLatentHalf = kHalf - 2;

  // Addresses in LDS; a tile's places are attend()'s, but a wave loads eight
  // neighbouring keys.  (Tiles and the rest lie at
  // multiples of 4 KiB, so that places within one are reached by exclusive ors.)
  const uint32_t keys_at = lds_address(lds.keys), half_at = lds_address(lds.half);
  uint32_t lane16 = static_cast<uint32_t>(lane * 16);
  auto swizzle = [](int k) { return ((k & 3) << 2) | ((k >> 2) & 3); };
  uint32_t byte_of = static_cast<uint32_t>(wave * 8 * kCkvBytes + ((lane & 48) | ((lane ^ ((2 * wave) & 3)) & 15)) * 16);
  const int rope_key = wave * 8 + (lane >> 3);
  const uint32_t rope_byte = static_cast<uint32_t>(rope_key * kKpeBytes + ((lane ^ (rope_key >> 1)) & 7) * 16);
  uint32_t k_at = keys_at + static_cast<uint32_t>(l32 * kCkvBytes + dh * 512 + ((hh ^ swizzle(l32)) & 15) * 16);
  uint32_t r_at = keys_at + static_cast<uint32_t>(kKeys * kCkvBytes + l32 * kKpeBytes + (((4 * dh + hh) ^ (l32 >> 1)) & 7) * 16);
  const int v_key = 8 * hh + ((lane & 15) >> 2);  // (and the key four behind it, whose swizzle differs by 1)
  uint32_t v_at = keys_at + static_cast<uint32_t>(v_key * kCkvBytes + wave * 256 + (lane & 1) * 8 +
                                              (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ swizzle(v_key)) & 15) * 16);
  const int p_swz = (l32 >> 2) & 3;
  uint32_t p_read = lds_address(lds.p) + static_cast<uint32_t>(l32 * 64 + ((hh ^ p_swz) & 3) * 16);
  uint32_t p_write = lds_address(lds.p) + static_cast<uint32_t>(m_mine * 64 + p_swz * 16 + hh * 8);

  Pages pages(s, a);
  auto page_of = [&](int tile) { return pages.of(tile); };
  // A tile's loads, nine of a wave: pairs of keys, and the rope dims.
  struct Load {
    const uint8_t* base;
    const uint8_t* rope;
  };
  const uint32_t lds_tile = keys_at + wave * (8 * kCkvBytes), lds_rope = keys_at + kKeys * kCkvBytes + wave * 1024;
  auto load_of = [&](int tile, int page) {
    const uint32_t row = static_cast<uint32_t>(page < 0 ? 0 : page) * kBlock + (static_cast<uint32_t>(tile) % kPageTiles) * kKeys;
    return Load{static_cast<const uint8_t*>(a.kv_cache) + static_cast<uint64_t>(row) * kCkvBytes,
                static_cast<const uint8_t*>(a.k_rope) + static_cast<uint64_t>(row) * kKpeBytes};
  };
  auto issue = [&](const Load& l, uint32_t buffer, auto which) {  // 0 to 7: a key, 8: the rope dims
    constexpr int n = decltype(which)::value;
    if constexpr (n < 8)
      load_to_lds<(n & 3) * 1024>(l.base, byte_of ^ ((n & 3) * 64 + (n >> 2) * (4096 + 16)), lds_tile + (n >> 2) * 4096, buffer);
    else
      load_to_lds<0>(l.rope, rope_byte, lds_rope, buffer);
  };

  lds_barrier();  // (the segment before is done with LDS)
  const int t0 = s.tile0, t1 = s.tile1;
  {
    const Load l = load_of(t0, page_of(t0));
    steps<kTileLoads>([&](auto n) { issue(l, 0, n); });
  }

  // Of the wave's half of the dims, in steps of 16: i = 2 x + g is chunk pair x of
  // 256-byte group g, for two tiles of 32 pairs, first those that the wave weighs.
  // The rope dims, the last two steps, lie in LDS, for which there is room, and not
  // in registers, for which there is none.
  // They come through LDS, 32 pairs at a time in the wave's own 16 KiB of tiles that
  // are not there yet: a load takes two pairs' 512 neighbouring bytes, where loads
  // to the registers would take 32 bytes of 32 pairs.
  int vis = seen(s, s.pair0 + (m_mine < s.count ? m_mine : 0));
  vis = m_mine < s.count ? vis : 0;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int in = wave * 32 + n * 8 + (lane >> 3), m = in < s.count ? in : 0;
    load_to_lds(static_cast<const uint8_t*>(a.query_rope) + s.pair0 * kKpeBytes,
                static_cast<uint32_t>(m * kKpeBytes + ((lane ^ (in >> 1)) & 7) * 16), lds_address(lds.rope) + wave * 4096 + n * 1024);
  }
  u32x4_t q[kLatentHalf][2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int first = rg * 64 + (r ^ dh) * 32;
    const uint32_t stage = keys_at + kTileBytes + wave * kStage;
    const uint8_t* from = static_cast<const uint8_t*>(a.query) + s.pair0 * kCkvBytes + dh * 512;
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const int in = 2 * n + hh, m = first + in < s.count ? first + in : 0;
      load_to_lds(from, static_cast<uint32_t>(m * kCkvBytes + (l32 ^ in) * 16), stage + n * 1024);
    }
    wait_loads<0>();
#pragma unroll
    for (int i = 0; i < kLatentHalf; ++i) q[i][r] = lds_get(stage + static_cast<uint32_t>(l32 * 512 + (((i & 1) * 16 + (i >> 1) * 2 + hh) ^ l32) * 16));
#pragma unroll
    for (int i = 0; i < kLatentHalf; ++i) asm volatile("" : "+v"(q[i][r]));
  }
  // (Rows of pairs 64 rg + (r ^ dh) 32 + l32: the other tile is 32 rows away.)
  uint32_t qr_at = lds_address(lds.rope) + static_cast<uint32_t>((tile_mine * 32 + l32) * kKpeBytes + (((4 * dh + hh) ^ (l32 >> 1)) & 7) * 16);
  f32x16_t o[4][4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][r][e] = 0.f;
  settle(o);
  float ref = 0.f, l_run = 0.f;
  float room = -INFINITY;  // a score above the reference by more moves it (nothing seen yet: any does)
  int vis_least = m_mine < s.count ? vis : 0x7fffffff;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) vis_least = min(vis_least, __shfl_xor(vis_least, d));
  vis_least = __builtin_amdgcn_readfirstlane(vis_least);
  if (lane == 0) lds.least[wave] = vis_least;
  if (tid < 4) lds.moved[tid] = INT32_MIN;
  if (tid == 0) lds.moved_last = INT32_MIN;
  const float factor = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(a.scale * kLog2e)));

  constexpr int kAhead = 3;   // operands of the scores on their way
  constexpr int kLate = 4;    // products of the outputs that are left for behind barrier A
  u32x4_t v[3], p[4];
  f32x16_t mine;              // the wave's half of the scores of its 32 pairs, then their P
#pragma unroll
  for (int e = 0; e < 16; ++e) mine[e] = 0.f;
  auto fetch_v = [&](uint32_t from, int i) {  // operand i = 4 ks + d
    const uint32_t at = from ^ ((i & 3) * 64);
    const uint2 lo = read_tr16(at + (i >> 2) * 16 * kCkvBytes);
    const uint2 hi = read_tr16((at ^ 16) + ((i >> 2) * 16 + 4) * kCkvBytes);
    v[i % 3] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
  };
  auto fetch_p = [&](int ks, int r) { p[r] = lds_get((p_read ^ (ks * 32)) + r * 2048); };
  u32x4_t k[kAhead + 1];
  auto fetch_k = [&](uint32_t k_from, uint32_t r_from, int i) {
    if (i < kHalf)
      k[i % (kAhead + 1)] = lds_get(i < 16 ? (k_from ^ ((i >> 1) * 32)) + (i & 1) * 256 : r_from ^ ((i - 16) * 32));
  };
  // Barrier A before the scores of a tile in that buffer; `other`: half of the scores
  // of the tile before it.
  u32x4_t other[4];
  auto begin_scores = [&](uint32_t buffer) __attribute__((always_inline)) {
    wait_loads<0>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch_k(k_at + buffer, r_at + buffer, i);
#pragma unroll
    for (int e = 0; e < 4; ++e) other[e] = lds_get(half_at + wave * 4096 + lane16 + e * 1024);
  };

  // Tile t, in buffer `now`, is weighed and put out; the scores of tile t + 1, in
  // buffer `ahead`, come first, and of tile t - 1 kLate products are open.  One
  // form for every t, a tile of zeros before the first one among them: the compiler
  // does not find registers for more.
  uint32_t now = 2 * kTileBytes, ahead = 0, beyond = kTileBytes;
  int page_t = -1, page_1 = 0, page_2 = 0;  // of tiles t, t + 1 and t + 2
  int mask_now = -1, scrub_now = 0;         // negative: some row of the wave's, of the item, does not see all of tile t
  Load load{};                              // of tile t + 2
  int seen_all = 0;                         // tiles that every row of the item sees whole
  const int seen_mine = vis_least / kKeys;  // that every row of the wave's does
  auto round = [&](int t) {
    const uint32_t k_slot = k_at + ahead, r_slot = r_at + ahead, v_from = v_at + now;
    forget(p_read);
    forget(p_write);
    forget(qr_at);
    forget(byte_of);
    forget(lane16);
    forget(k_at);
    forget(r_at);
    forget(v_at);
    u32x4_t qr[2][2];
    f32x16_t next[2];
    const int page = page_t;
    Load next_load;
    int page_next = 0;
    float top = 0.f, more = 0.f;
    int32_t moved_last = 0;
    bool any = false;
    __builtin_amdgcn_sched_barrier(0);
    steps<kSteps>([&](auto step) __attribute__((always_inline)) {
      constexpr int j = decltype(step)::value, i = j >> 1, r = j & 1;
      if constexpr (r == 0) fetch_k(k_slot, r_slot, i + kAhead);
      if constexpr (r == 0 && (i == 14 || i == 15)) {
        qr[i & 1][0] = lds_get(qr_at ^ ((i - 14) * 32));
        qr[i & 1][1] = lds_get(qr_at ^ ((i - 14) * 32 + 32 * kKpeBytes));
      }
      {
        if constexpr (i == 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) next[r][e] = 0.f;
        }
        next[r] = T::mfma32(__builtin_bit_cast(typename T::vec8, k[i % (kAhead + 1)]),
                            __builtin_bit_cast(typename T::vec8, i < kLatentHalf ? q[i % kLatentHalf][r] : qr[i & 1][r]), next[r]);
      }
      {
        // (A load of all four waves takes 64 clocks of the way from the L2, two products.)
        if constexpr (j % 2 == 0 && j < 2 * kTileLoads) issue(load, beyond, std::integral_constant<int, j / 2>{});
        if constexpr (j >= 4 && j < 12) {
          constexpr int e = 2 * (j - 4);
          mine[e] = fmaf(mine[e] + __uint_as_float(other[e / 4][e % 4]), factor, -ref);
          mine[e + 1] = fmaf(mine[e + 1] + __uint_as_float(other[e / 4][e % 4 + 1]), factor, -ref);
        }
        if constexpr (j == 12) if (mask_now < 0) {
          const int left = vis - t * kKeys - 4 * (own_thread() >> 5 & 1);  // keys that the row sees, from the lane's first
#pragma unroll
          for (int e = 0; e < 16; ++e) mine[e] = page >= 0 && 8 * (e >> 2) + (e & 3) < left ? mine[e] : -INFINITY;
        }
        if constexpr (j == 12) top = max3(max3(mine[0], mine[1], mine[2]), max3(mine[3], mine[4], mine[5]), max3(mine[6], mine[7], mine[8]));
        if constexpr (j == 13) top = max3(top, max3(mine[9], mine[10], mine[11]), max3(mine[12], mine[13], max3(mine[14], mine[15], mine[15])));
        if constexpr (j == 14) any = __any(top > room);
        if constexpr (j == 15) {
          if (any) {
            const int th = own_thread();
            top = xor32_op(top, MaxOp{});
            const bool past = top > room;
            const float up = past ? top - kRise : 0.f;
            const bool seen = past && room != -INFINITY;
            const float f = seen ? __builtin_amdgcn_exp2f(-up) : 1.f;
            room = past ? kMost : room;
            ref += up;
            l_run *= f;
#pragma unroll
            for (int e = 0; e < 16; ++e) mine[e] -= up;
            if ((th & 32) == 0) lds.factor[tile_mine * 32 + (th & 31)] = f;
            if (__any(seen) && (th & 63) == 0) lds.moved[tile_mine] = lds.moved_last = t;  // (else o is zero)
          }
        }
        if constexpr (j >= 16 && j < 24) {
          constexpr int e = 2 * (j - 16), n = e / 4;
          mine[e] = __builtin_amdgcn_exp2f(mine[e]);
          mine[e + 1] = __builtin_amdgcn_exp2f(mine[e + 1]);
          if constexpr (e % 4 == 2) {
            const uint32_t p01 = T::pack2(mine[e - 2], mine[e - 1]), p23 = T::pack2(mine[e], mine[e + 1]);
            lds_put(p_write ^ (n * 16), p01, p23);
            mine[e - 2] = low_half<T>(p01);
            mine[e - 1] = high_half<T>(p01);
            mine[e] = low_half<T>(p23);
            mine[e + 1] = high_half<T>(p23);
          }
        }
        if constexpr (j >= 18 && j < 26) {
          l_run += mine[2 * (j - 18)];
          more += mine[2 * (j - 18) + 1];
          asm volatile("" : "+v"(l_run), "+v"(more));  // (here, not all of them between the products)
        }
        if constexpr (j == 26) l_run += more;
        if constexpr (j == 29) moved_last = lds.moved_last;
        if constexpr (j >= 29 && j < 33) fetch_p(0, j - 29);
        if constexpr (j == 33) fetch_v(v_from, 0);
        if constexpr (j == 35) fetch_v(v_from, 1);
        if constexpr (j == 28) {
          // Values of keys that some row must not see: see attend().
          if (scrub_now < 0) {
            for (int c = own_thread(); c < kKeys * kCkvBytes / 16; c += kThreads) {
              u32x4_t* at = reinterpret_cast<u32x4_t*>(&lds.keys[0][0] + now + c * 16);
              *at = finite_or_zero<T>(*at);
            }
          }
          lds_barrier();  // B
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    {
      if (__builtin_amdgcn_readfirstlane(moved_last) == t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (__builtin_amdgcn_readfirstlane(lds.moved[r]) == t) {
            const float f = lds.factor[r * 32 + (own_thread() & 31)];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              settle(o[d][r]);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[d][r][e] *= f;
              settle(o[d][r]);
              __builtin_amdgcn_sched_barrier(0);  // (sixteen values in other registers at a time)
            }
          }
        }
      }
      steps<32>([&](auto step) __attribute__((always_inline)) {
        constexpr int n = decltype(step)::value, i = n >> 2, r = n & 3;
        if constexpr (n == 32 - kLate) begin_scores(beyond);
        if constexpr (n == 5) {
          if (!pages.holds(t + 3)) pages.hold(t);
          page_next = page_of(t + 3);
        }
        if constexpr (n == 10) next_load = load_of(t + 3, page_next);
        if constexpr (n == 14) {
          mask_now = (seen_mine - 2 - t) | page_1;
          scrub_now = (seen_all - 2 - t) | page_1;
        }
        if constexpr (r == 0 && i + 2 < 8) fetch_v(v_from, i + 2);
        accumulate<r == 0 || i == 0 || i == 4>(T{}, v[i % 3], p[r], o[i & 3][r]);
        if constexpr (n % 5 == 3 && n < 20) {
          // To the wave with the other half of the dims, the pairs that it weighs.
          // (Everybody has read the last ones since barrier A; B lies between.  One
          // such write keeps LDS busy for two products of all waves.)
          constexpr int e = 4 * (n / 5);
          lds_put(half_at + (wave ^ 2) * 4096 + lane16 + (n / 5) * 1024,
                  u32x4_t{__float_as_uint(next[1][e]), __float_as_uint(next[1][e + 1]), __float_as_uint(next[1][e + 2]),
                          __float_as_uint(next[1][e + 3])});
        }
        // (Read by assembly: the products that made it lie ten or more products back.)
        if constexpr (n >= 8 && n < 24) mine[n - 8] = moved_here(next[0][n - 8]);
        if constexpr (i == 3) fetch_p(1, r);
        __builtin_amdgcn_sched_barrier(0);
      });
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < kLatentHalf; ++i) asm volatile("" : "+v"(q[i][r]));
    page_t = page_1;
    page_1 = page_2;
    page_2 = page_next;
    load = next_load;
    const uint32_t done = now;
    now = ahead;
    ahead = beyond;
    beyond = done;
  };

  lds_barrier();
  seen_all = __builtin_amdgcn_readfirstlane(min(min(lds.least[0], lds.least[1]), min(lds.least[2], lds.least[3]))) / kKeys;
#pragma unroll
  for (int i = 0; i < kKeys * kCkvBytes / 16 / kThreads; ++i) lds_put(keys_at + now + (tid + i * kThreads) * 16, u32x4_t{0, 0, 0, 0});
  begin_scores(0);
  page_1 = page_of(t0);
  page_2 = page_of(t0 + 1);
  load = load_of(t0 + 1, page_2);
  for (int t = t0 - 1; t < t1; ++t) round(t);   // (the last one's scores are of no tile, and nobody reads them)
  wait_loads<0>();
  l_run = xor32_op(l_run, AddOp{});
  lds_barrier();
  float2* const rows = reinterpret_cast<float2*>(&lds.rope[0]);
  if (hh == 0) rows[m_mine] = make_float2(room == -INFINITY && l_run == 0.f ? -INFINITY : ref, l_run);
  lds_barrier();
  finish<T, 4>(a, w, s, rows, keys_at + wave * kStage, o);
}

// HERE: every workgroup makes the plan by itself, of kHere spans at most; the last
// one, which has no part where they are few, writes it down for the join.
template <typename T, bool HERE>
__global__ __launch_bounds__(kThreads, 1) void prefix_attention_kernel(PrefixAttentionArgs a) {
  struct None {};
  __shared__ __align__(16384) Lds lds;
  __shared__ typename std::conditional<HERE, Span[kHere], None>::type here;
  Plan w;
  carve(a.workspace, a.rows, a.heads, a.batch, a.groups, &w);
  const int part = blockIdx.x;
  Start start;
  int width;
  Seen<HERE> seen{w.visible, nullptr, static_cast<int32_t>(a.batch), static_cast<int32_t>(a.heads)};
  if constexpr (HERE) {
    const Cut cut = make_plan<kThreads, true>(a, w, lds.plan, here, part == kParts - 1);
    if (part >= cut.parts) return;
    width = cut.width;
    start = start_of(cut, part, static_cast<int>(a.groups + a.batch), [&](int i) { return here[i].unit0; });
    seen.requests = here + a.groups;
  } else {
    if (part >= w.cut->parts) return;
    start = w.parts[part];
    width = uniform(w.cut->width);
  }
  const int64_t stop = uniform(start.stop);
  int64_t at = uniform(start.unit);
  int at_span = uniform(start.span);
  auto span_at = [&](int i) -> Span {
    if constexpr (HERE)
      return uniform(here[i]);
    else
      return uniform(w.spans[i]);
  };
  while (at < stop) {
    Span s = span_at(at_span);
    int64_t end = s.unit0 + units_of(s, width);
    while (at >= end) {
      s = span_at(++at_span);
      end = s.unit0 + units_of(s, width);
    }
    const int units = s.tiles + kBegin;
    const int item = uniform(quotient(at - s.unit0, units));
    const int64_t item_start = s.unit0 + static_cast<int64_t>(item) * units, item_end = item_start + units;
    const int64_t seg_end = item_end < stop ? item_end : stop;
    auto tile_of = [&](int64_t u) { return u > kBegin ? static_cast<int>(u) - kBegin : 0; };
    Segment g;
    const int first = item * width;
    g.pair0 = static_cast<int64_t>(s.pair0) + first;
    g.count = s.pairs - first < width ? s.pairs - first : width;
    g.tile0 = s.tile0 + tile_of(at - item_start);
    g.tile1 = s.tile0 + tile_of(seg_end - item_start);
    g.table = a.block_table + s.table * a.cols;
    g.length = s.length;
    g.end = at_span >= a.groups ? static_cast<int>(row_of(s.pair0 + s.pairs, a.heads)) : -1;
    const bool whole = at == item_start && seg_end == item_end;
    g.direct = whole && s.merge < 0;
    g.row = whole ? merge_row(w, s.merge, first, at_span >= a.groups) : part_row(w, part, at == item_start);
    g.row_step = whole ? 2 : 1;
    if (at_span >= a.groups) {  // a request's last row of the item sees the most
      const int tiles = (seen(g, g.pair0 + g.count - 1) + kKeys - 1) / kKeys;
      g.tile1 = g.tile1 < tiles ? g.tile1 : tiles;
      g.tile0 = g.tile0 < g.tile1 ? g.tile0 : g.tile1;
    }
    // Up to 32 pairs: 64 requests of 16 heads 42 us, and 50 as 64 pairs.  Up to 64: 32
    // requests of 2 heads on 4096 tokens 25.5 us, and 29.4 as more; there are no
    // registers for more in attend().
    if (g.tile0 >= g.tile1)
      nothing<T>(a, w, g);
    else if (g.count <= 32)
      attend<T, 1>(a, w, g, seen, lds.few);
    else if (g.count <= 64)
      attend<T, 2>(a, w, g, seen, lds.few);
    else
      attend_many<T>(a, w, g, seen, lds.many);
    at = seg_end;
  }
}

// -------------------------------------------------------------------- the join
// WAVES waves a pair: its segments' references, then their sums, four or eight at a
// time on their way, every wave those of its turn.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixAttentionArgs a) {
  __shared__ float4 others[WAVES > 1 ? 4 : 1][2][64];
  Plan w;
  carve(a.workspace, a.rows, a.heads, a.batch, a.groups, &w);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), turn = wave % WAVES;
  const int pair = static_cast<int>(blockIdx.x) * (4 / WAVES) + wave / WAVES;
  const int heads = static_cast<int>(a.heads);
  if (pair >= a.rows * a.heads) return;
  const int b = w.request[pair / heads];
  if (b < 0) return;
  const Cut cut = *w.cut;
  const Span own = w.spans[a.groups + b];
  struct Run {  // segments of one item
    int w0, n;
    int64_t whole;    // row of the sums where there is one segment
    int m;
  };
  auto run_of = [&](const Span& s, bool is_own) {
    Run r;
    const int in = pair - s.pair0, item = in / cut.width;
    const int64_t units = s.tiles + kBegin, u0 = s.unit0 + item * units;
    r.w0 = part_of(cut, u0);
    r.n = part_of(cut, u0 + units - 1) - r.w0 + 1;
    r.m = in - item * cut.width;
    r.whole = r.n == 1 ? merge_row(w, s.merge, in, is_own) : -1;
    return r;
  };
  const Run mine = run_of(own, true);
  if (own.group < 0 && mine.n == 1) return;  // (written by the attention itself)
  Run shared{};
  if (own.group >= 0) shared = run_of(w.spans[own.group], false);
  const int n = mine.n + shared.n;  // (at most 2 kParts)
  auto row_of = [&](int k) -> int64_t {
    const Run& r = k < shared.n ? shared : mine;
    const int j = k < shared.n ? k : k - shared.n;
    return r.n == 1 ? r.whole : part_row(w, r.w0 + j, j == 0) + r.m;
  };
  float top = -INFINITY;
  for (int k0 = 0; k0 < n; k0 += 64) {
    float2 v = make_float2(-INFINITY, 0.f);
    if (k0 + lane < n) v = w.refs[row_of(k0 + lane)];
    top = fmaxf(top, wave_all_op(v.x, MaxOp{}));
  }
  float l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < n; k0 += 64) {
    float2 v = make_float2(-INFINITY, 0.f);
    int64_t row = 0;
    if (k0 + lane < n) {
      row = row_of(k0 + lane);
      v = w.refs[row];
    }
    const float f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - top);
    // (A part whose weight is zero counts for nothing, unless it has seen a NaN; where a
    // score was infinite, f is NaN.)
    l += wave_all_op(f == 0.f && v.y == v.y ? 0.f : v.y * f, AddOp{});
    const int count = n - k0 < 64 ? n - k0 : 64;
    auto add = [&](int k, auto at_once) __attribute__((always_inline)) {
      constexpr int kRows = decltype(at_once)::value;
      float4 x[kRows][2];
      float by[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int at = k + u * WAVES;  // (lanes from `count` on hold row 0 and a factor of zero)
        by[u] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), at & 63));
        by[u] = at < count ? by[u] : 0.f;
        const int64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(row), at & 63));
        const float4* p = reinterpret_cast<const float4*>(w.sums + lo * kCkvDim) + lane;
        x[u][0] = p[0];
        x[u][1] = p[64];
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (by[u] == 0.f) continue;  // (a part without tiles wrote no sums)
        acc[0] = fmaf(x[u][0].x, by[u], acc[0]);
        acc[1] = fmaf(x[u][0].y, by[u], acc[1]);
        acc[2] = fmaf(x[u][0].z, by[u], acc[2]);
        acc[3] = fmaf(x[u][0].w, by[u], acc[3]);
        acc[4] = fmaf(x[u][1].x, by[u], acc[4]);
        acc[5] = fmaf(x[u][1].y, by[u], acc[5]);
        acc[6] = fmaf(x[u][1].z, by[u], acc[6]);
        acc[7] = fmaf(x[u][1].w, by[u], acc[7]);
      }
    };
    int k = turn;
    if constexpr (WAVES > 1)
      for (; count - k > 4 * WAVES; k += 8 * WAVES) add(k, std::integral_constant<int, 8>{});
    for (; k < count; k += 4 * WAVES) add(k, std::integral_constant<int, 4>{});
  }
  if constexpr (WAVES > 1) {  // (every wave of the workgroup is here, or none: they have one pair)
    static_assert(WAVES == 4, "a workgroup a pair");
    others[wave][0][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    others[wave][1][lane] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      const float4 x = others[k][0][lane], y = others[k][1][lane];
      acc[0] += x.x;
      acc[1] += x.y;
      acc[2] += x.z;
      acc[3] += x.w;
      acc[4] += y.x;
      acc[5] += y.y;
      acc[6] += y.z;
      acc[7] += y.w;
    }
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  uint2* out = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + static_cast<int64_t>(pair) * kCkvDim) + lane;
  out[0] = make_uint2(T::pack2(acc[0] * by, acc[1] * by), T::pack2(acc[2] * by, acc[3] * by));
  out[64] = make_uint2(T::pack2(acc[4] * by, acc[5] * by), T::pack2(acc[6] * by, acc[7] * by));
}

template <typename T>
hipError_t launch(const PrefixAttentionArgs& a, hipStream_t stream) {
  hipError_t e;
  if (a.groups + a.batch <= kHere) {
    launch_kernel(kKernPrefixAttention, prefix_attention_kernel<T, true>, dim3(kParts), dim3(kThreads), stream, a);
  } else {
    launch_kernel(kKernPrefixPlan, prefix_plan_kernel, dim3(1), dim3(kPlanThreads), stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    launch_kernel(kKernPrefixAttention, prefix_attention_kernel<T, false>, dim3(kParts), dim3(kThreads), stream, a);
  }
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.rows * a.heads < kJoinByWave)
    launch_kernel(kKernPrefixJoin, prefix_join_kernel<T, 4>, dim3(static_cast<uint32_t>(a.rows * a.heads)), dim3(256), stream, a);
  else
    launch_kernel(kKernPrefixJoin, prefix_join_kernel<T, 1>, dim3(static_cast<uint32_t>(ceil_div(a.rows * a.heads, 4))), dim3(256),
                  stream, a);
  return hipGetLastError();
}

}  // namespace

size_t prefix_attention_workspace_bytes(int64_t rows, int64_t heads, int64_t batch, int64_t groups) {
  return carve(nullptr, rows, heads, batch, groups, nullptr);
}

hipError_t launch_prefix_attention(const PrefixAttentionArgs& a, hipStream_t stream) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  return a.elem == Elem::kBf16 ? launch<Bf16>(a, stream) : launch<F16>(a, stream);
}

}  // namespace nvdsa
