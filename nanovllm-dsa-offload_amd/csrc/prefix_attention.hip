// Attention of requests that share a prefix's pages, over the 16-bit latent
// cache:
//
//   o[t, h] = softmax(scale * (q . ckv + q_rope . kpe)) . ckv   over the slots that row t sees
//
// A query (row, head) is a pair; the packed rows of a group's requests are
// neighbours, so that all their pairs make one product with the pages that the
// group shares: items of up to 128 pairs against those pages, read once, and
// items of one request's pairs against the pages behind them.  A plan kernel
// lays the items' tiles of keys in a row and cuts it into equal parts, one per
// workgroup; what lies across parts, and a pair's two items, leave fp32 partial
// sums that a join kernel adds up.
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
constexpr int kWindow = 1024;         // pages whose ids are held at a time
constexpr int kParts = 256;           // workgroups, one per CU (LDS)
constexpr int kBegin = 4;             // what the start of a segment costs, in tiles
constexpr int kLeastTiles = 4;        // of a part
constexpr int kLeastShared = 8;       // tiles of a prefix that is read once
constexpr float kLog2e = 1.4426950408889634f;
// P = 2^(score - reference): a reference is set so that the largest P of its
// tile is 2^kRise and kept until one passes 2^kMost.  fp16 holds P from 2^-24
// on, so keys down to 2^-32 of the row's largest count; bf16 has fp32's range.
constexpr float kRise = 8.f;
constexpr float kMost = 15.9f;

// ---------------------------------------------------------------- the plan
struct Span {        // pairs against tiles of one table row's pages
  int64_t unit0;     // first unit of the first item
  int64_t merge;     // first of the group's pairs that two items have (-1: one item only)
  int32_t pair0, pairs;
  int32_t tile0, tiles;
  int32_t table;     // row of the block table
  int32_t group;     // request: its group's span (-1: none)
};
struct Start {       // where a part begins
  int64_t unit;
  int64_t stop;
  int32_t span;      // groups first, then requests
};
struct Plan {
  Start* parts;      // [kParts]
  int32_t* used;     // [1]: parts in use
  int64_t* total;    // [1]
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
__host__ __device__ inline int64_t merge_pairs(int64_t rows, int64_t heads, int64_t batch) {
  const int64_t n = rows * heads;
  return n < batch * kPairs ? n : batch * kPairs;
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
  w.used = reinterpret_cast<int32_t*>(take(sizeof(int32_t)));
  w.total = reinterpret_cast<int64_t*>(take(sizeof(int64_t)));
  w.spans = reinterpret_cast<Span*>(take(sizeof(Span) * (groups + batch)));
  w.visible = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * rows));
  w.request = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * rows));
  w.stride = slot_pairs(rows, heads);
  const int64_t partial = 2 * kParts * w.stride + 2 * merge_pairs(rows, heads, batch);
  w.refs = reinterpret_cast<float2*>(take(sizeof(float2) * partial));
  w.sums = reinterpret_cast<float*>(take(sizeof(float) * partial * kCkvDim));
  if (plan) *plan = w;
  return static_cast<size_t>(p - start);
}

__device__ inline int64_t items_of(const Span& s) { return (static_cast<int64_t>(s.pairs) + kPairs - 1) / kPairs; }
__device__ inline int64_t units_of(const Span& s) { return items_of(s) * (s.tiles + kBegin); }
__device__ inline int64_t part_start(int64_t total, int64_t parts, int64_t w) { return total * w / parts; }
// The part of a unit.
__device__ inline int part_of(int64_t total, int64_t parts, int64_t unit) {
  int64_t w = unit * parts / total;
  while (w + 1 < parts && part_start(total, parts, w + 1) <= unit) ++w;
  while (w > 0 && part_start(total, parts, w) > unit) --w;
  return static_cast<int>(w);
}
// Values that every lane holds, in scalar registers.
__device__ inline int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(x) >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ inline Span uniform(const Span& s) {
  return {uniform(s.unit0), uniform(s.merge), uniform(s.pair0), uniform(s.pairs),
          uniform(s.tile0), uniform(s.tiles), uniform(s.table), uniform(s.group)};
}
// Row of the partial sums of a segment's first pair.
__device__ inline int64_t part_row(const Plan& w, int part, bool begins) { return (2 * static_cast<int64_t>(part) + (begins ? 1 : 0)) * w.stride; }
__device__ inline int64_t merge_row(const Plan& w, int64_t merged, int pair, bool own) {
  return 2 * kParts * w.stride + 2 * (merged + pair) + (own ? 1 : 0);
}

constexpr int kPlanThreads = 1024;

__device__ inline int64_t plan_scan(int64_t v, int64_t* scratch, int64_t* total) {
  const int wid = threadIdx.x >> 6;
  const int64_t x = static_cast<int64_t>(wave_inclusive_scan(static_cast<uint64_t>(v)));
  if ((threadIdx.x & 63) == 63) scratch[wid] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kPlanThreads / 64; ++k) {
    before += k < wid ? scratch[k] : 0;
    all += scratch[k];
  }
  *total = all;
  __syncthreads();
  return before + x - v;
}

__global__ __launch_bounds__(kPlanThreads) void prefix_plan_kernel(PrefixAttentionArgs a) {
  __shared__ int64_t scratch[kPlanThreads / 64];
  Plan w;
  carve(a.workspace, a.rows, a.heads, a.batch, a.groups, &w);
  const int tid = threadIdx.x;
  const int64_t cap = a.cols * kBlock;
  auto row_at = [&](int64_t b) -> int64_t {  // first packed row of request b
    const int64_t r = b > 0 ? a.seq_q[b - 1] : 0;
    return r < 0 ? 0 : (r > a.rows ? a.rows : r);
  };
  auto end_at = [&](int64_t g) -> int64_t {  // first request of group g
    const int64_t b = g > 0 ? a.group_ends[g - 1] : 0;
    return b < 0 ? 0 : (b > a.batch ? a.batch : b);
  };
  int64_t units = 0, merged = 0, items = 0;
  // Groups: one that shares has a request's pages read for several of them, and
  // fewer pairs a request than an item holds (else every item is full anyway).
  for (int64_t g0 = 0; g0 < a.groups; g0 += kPlanThreads) {
    const int64_t g = g0 + tid;
    Span s{};
    s.merge = -1;
    if (g < a.groups) {
      const int64_t b0 = end_at(g), b1 = end_at(g + 1);
      if (b1 - b0 >= 2) {
        const int64_t r0 = row_at(b0), r1 = row_at(b1);
        int64_t tokens = a.prefix_lens[g];
        tokens = tokens < 0 ? 0 : (tokens > cap ? cap : tokens);
        const int64_t tiles = tokens / kBlock * kPageTiles, pairs = (r1 - r0) * a.heads;
        if (tiles >= kLeastShared && r1 > r0 && pairs < (b1 - b0) * kPairs) {
          s.pair0 = static_cast<int32_t>(r0 * a.heads);
          s.pairs = static_cast<int32_t>(pairs);
          s.tiles = static_cast<int32_t>(tiles);
          s.table = static_cast<int32_t>(b0);
        }
      }
    }
    int64_t total;
    s.unit0 = units + plan_scan(s.pairs > 0 ? units_of(s) : 0, scratch, &total);
    units += total;
    const int64_t m = plan_scan(s.pairs, scratch, &total);
    if (s.pairs > 0) s.merge = merged + m;
    merged += total;
    plan_scan(s.pairs > 0 ? items_of(s) : 0, scratch, &total);
    items += total;
    s.group = -1;
    if (g < a.groups) w.spans[g] = s;
  }
  __syncthreads();
  for (int64_t at = 0; at < a.batch; at += kPlanThreads) {
    const int64_t b = at + tid;
    Span s{};
    s.merge = -1;
    s.group = -1;
    if (b < a.batch) {
      const int64_t r0 = row_at(b), r1 = row_at(b + 1);
      int64_t len = a.seq_kv[b];
      len = len < 0 ? 0 : (len > cap ? cap : len);
      s.pair0 = static_cast<int32_t>(r0 * a.heads);
      s.pairs = r1 > r0 ? static_cast<int32_t>((r1 - r0) * a.heads) : 0;
      s.tiles = static_cast<int32_t>((len + kKeys - 1) / kKeys);
      s.table = static_cast<int32_t>(b);
      // The group: the first whose end lies behind the request.
      int64_t lo = 0, hi = a.groups;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.group_ends[mid] <= b)
          lo = mid + 1;
        else
          hi = mid;
      }
      if (lo < a.groups && s.pairs > 0) {
        const Span g = w.spans[lo];
        // (Ends that decrease: a request outside the group's rows is its own.)
        if (g.pairs > 0 && b >= g.table && s.pair0 >= g.pair0 && s.pair0 + s.pairs <= g.pair0 + g.pairs) {
          s.group = static_cast<int32_t>(lo);
          s.merge = g.merge + (s.pair0 - g.pair0);
          s.tile0 = g.tiles;
          s.tiles = s.tiles > g.tiles ? s.tiles - g.tiles : 0;
        }
      }
    }
    int64_t total;
    s.unit0 = units + plan_scan(s.pairs > 0 ? units_of(s) : 0, scratch, &total);
    units += total;
    plan_scan(s.pairs > 0 ? items_of(s) : 0, scratch, &total);
    items += total;
    if (b < a.batch) w.spans[a.groups + b] = s;
  }
  // What the rows see, a wave a request.
  for (int64_t t = tid; t < a.rows; t += kPlanThreads)
    if (t >= row_at(a.batch)) w.request[t] = -1;
  for (int64_t b = tid >> 6; b < a.batch; b += kPlanThreads / 64) {
    const int64_t r0 = row_at(b), r1 = row_at(b + 1);
    int64_t len = a.seq_kv[b];
    len = len < 0 ? 0 : (len > cap ? cap : len);
    for (int64_t t = r0 + (tid & 63); t < r1; t += 64) {
      const int64_t v = len - (r1 - 1 - t);
      w.visible[t] = static_cast<int32_t>(v > 0 ? v : 0);
      w.request[t] = static_cast<int32_t>(b);
    }
  }
  int64_t parts = (units - items * kBegin) / kLeastTiles;
  if (parts < items) parts = items;
  if (parts > kParts) parts = kParts;
  if (parts < 1) parts = 1;
  if (tid == 0) {
    *w.used = units > 0 ? static_cast<int32_t>(parts) : 0;
    *w.total = units;
  }
  __syncthreads();
  if (tid < parts && units > 0) {
    Start p;
    p.unit = part_start(units, parts, tid);
    p.stop = part_start(units, parts, tid + 1);
    // The last span that begins at or before the unit (spans without pairs begin
    // where the next does).
    int64_t lo = 0, hi = a.groups + a.batch - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (w.spans[mid].unit0 <= p.unit)
        lo = mid;
      else
        hi = mid - 1;
    }
    p.span = static_cast<int32_t>(lo);
    w.parts[tid] = p;
  }
}

// ------------------------------------------------------------- the attention
struct LdsFew {   // items of up to 64 pairs
  alignas(16) uint8_t keys[kBuffers][kTileBytes];
  alignas(16) uint16_t p[kPairs * kKeys];
  float factor[kPairs];
  float2 row[kPairs];   // reference and sum of P, at a segment's end
  int32_t pages[kWindow];
  int32_t moved[4];     // a wave's rows have new references
  int32_t least[4];     // the least that a row of a wave sees
};
struct LdsMany {  // more
  alignas(16) uint8_t p[kPairs * kKeys * 2];   // (at a segment's end: references and sums)
  uint8_t half[4][4][64][16];                  // scores of half the dims, to a wave
  uint8_t rope[kPairs * kKpeBytes];            // the pairs' rope dims
  uint8_t keys[3][kTileBytes];
  float factor[kPairs];
  int32_t moved[4];     // the tile at which a wave's rows have new references
  int32_t moved_last;   // the last such tile of all
  int32_t least[4];
};
union Lds {
  LdsFew few;
  LdsMany many;
};
static_assert(sizeof(Lds) <= 160 * 1024, "LDS");
static_assert(offsetof(LdsMany, keys) % 4096 == 0 && offsetof(LdsMany, rope) % 8192 == 0, "exclusive ors within");

struct Segment {
  int64_t pair0;      // of all pairs
  int32_t count;
  int32_t tile0, tile1;
  const int32_t* table;
  bool direct;        // the output itself
  int64_t row;        // of the partial sums
  int64_t row_step;   // between pairs of it
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
// Nothing is known of x from here on: what follows from it is worked out where it
// is used, and holds no register across the loop.
__device__ inline void forget(uint32_t& x) { asm volatile("" : "+v"(x)); }
// (fmaxf() would first make its operands canonical.)
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

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

// A segment's outputs, or its partial sums; rows: references and sums of P.
template <typename T, int TILES>
__device__ __forceinline__ void finish(const PrefixAttentionArgs& a, const Plan& w, const Segment& s, bool empty,
                                       const float2* rows, f32x16_t (&o)[4][TILES]) {
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < TILES; ++r) settle(o[d][r]);
#pragma unroll
  for (int r = 0; r < TILES; ++r) {
    const int m = r * 32 + l32;
    if (m >= s.count) continue;
    const float2 row = rows[m];
    if (s.direct) {
      const float by = row.y == 0.f ? 0.f : 1.f / row.y;
      uint16_t* out = static_cast<uint16_t*>(a.out) + (s.pair0 + m) * kCkvDim + wave * 128 + 4 * hh;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint2*>(out + d * 32 + 8 * i) =
              make_uint2(T::pack2(o[d][r][4 * i] * by, o[d][r][4 * i + 1] * by),
                         T::pack2(o[d][r][4 * i + 2] * by, o[d][r][4 * i + 3] * by));
    } else {
      const int64_t at = s.row + m * s.row_step;
      if (wave == 0 && hh == 0) w.refs[at] = row;
      if (!empty) {
        float* out = w.sums + at * kCkvDim + wave * 128 + 4 * hh;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(out + d * 32 + 8 * i) =
                make_float4(o[d][r][4 * i], o[d][r][4 * i + 1], o[d][r][4 * i + 2], o[d][r][4 * i + 3]);
      }
    }
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

template <typename T, int TILES>
__device__ __forceinline__ void attend(const PrefixAttentionArgs& a, const Plan& w, const Segment& s, LdsFew& lds) {
  const int tid = own_thread();
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const bool scores = wave < TILES;   // the wave has pairs of its own
  const int m_mine = wave * 32 + l32;
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
  const uint32_t k_at = static_cast<uint32_t>(l32 * kCkvBytes + ((hh ^ swizzle(l32)) & 15) * 16);
  const uint32_t r_at = static_cast<uint32_t>(kKeys * kCkvBytes + l32 * kKpeBytes + ((hh ^ (l32 >> 1)) & 7) * 16);
  uint32_t v_at[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int key = 8 * hh + 4 * part + ((lane & 15) >> 2);
    const int c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);   // of four neighbours
    v_at[part] = static_cast<uint32_t>(key * kCkvBytes + wave * 256 + ((c ^ swizzle(key)) & 15) * 16 + (lane & 1) * 8);
  }
  const uint32_t p_read = static_cast<uint32_t>(l32 * 64), p_swz = (l32 >> 2) & 3;

  int page0 = s.tile0 / kPageTiles;   // of the window
  auto fill_window = [&] {
    for (int i = tid; i < kWindow; i += kThreads) {
      const int64_t c = page0 + i;
      int32_t page = -1;
      if (c < a.cols && c * kPageTiles < s.tile1) page = s.table[c];
      lds.pages[i] = page >= 0 && page < a.blocks ? page : -1;
    }
  };
  auto page_of = [&](int tile) { return __builtin_amdgcn_readfirstlane(lds.pages[tile / kPageTiles - page0]); };
  auto load_tile = [&](int tile) {
    int page = page_of(tile);
    page = page < 0 ? 0 : page;
    const uint8_t* base = static_cast<const uint8_t*>(a.kv_cache) +
                          (static_cast<int64_t>(page) * kBlock + (tile % kPageTiles) * kKeys) * kCkvBytes;
    const uint8_t* rope = static_cast<const uint8_t*>(a.k_rope) +
                          (static_cast<int64_t>(page) * kBlock + (tile % kPageTiles) * kKeys) * kKpeBytes;
    const uint32_t to = lds_keys + (tile % kBuffers) * kTileBytes + wave * 1024;
#pragma unroll
    for (int i = 0; i < 8; ++i) load_to_lds(base + i * 4096, byte_of[i & 3], to + i * 4096);
    load_to_lds(rope, rope_byte, to + kKeys * kCkvBytes);
  };

  lds_barrier();  // (the segment before is done with LDS)
  fill_window();
  __syncthreads();
  const int t0 = s.tile0, t1 = s.tile1;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (t0 + k < t1) load_tile(t0 + k);

  u32x4_t q[kSteps];
  int vis = 0;
  if (scores) {
    const int64_t pair = s.pair0 + (m_mine < s.count ? m_mine : 0);
    vis = m_mine < s.count ? w.visible[pair / a.heads] : 0;
    const u32x4_t* qn = static_cast<const u32x4_t*>(a.query) + pair * (kCkvDim / 8) + hh;
    const u32x4_t* qr = static_cast<const u32x4_t*>(a.query_rope) + pair * (kKpeDim / 8) + hh;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) q[j] = j < 32 ? qn[2 * j] : qr[2 * (j - 32)];
  }
  f32x16_t o[4][TILES], sc;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < TILES; ++r)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][r][e] = 0.f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < TILES; ++r) settle(o[d][r]);
  float ref = 0.f, most = -INFINITY, l_run = 0.f;   // most: what a score may reach before the reference moves
  // The least that a row of this wave sees; every wave's meet in LDS.
  int vis_least = scores && m_mine < s.count ? vis : 0x7fffffff;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) vis_least = min(vis_least, __shfl_xor(vis_least, d));
  vis_least = __builtin_amdgcn_readfirstlane(vis_least);
  if (lane == 0) lds.least[wave] = vis_least;

  auto multiply = [&](int tile, f32x16_t& to) {
    const uint8_t* k_tile = lds.keys[tile % kBuffers];
#pragma unroll
    for (int e = 0; e < 16; ++e) to[e] = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const uint32_t at = j < 32 ? (k_at ^ ((j & 7) * 32)) + (j >> 3) * 256 : r_at ^ ((j - 32) * 32);
      const u32x4_t k = *reinterpret_cast<const u32x4_t*>(k_tile + at);
      to = T::mfma32(__builtin_bit_cast(typename T::vec8, k), __builtin_bit_cast(typename T::vec8, q[j]), to);
    }
  };
  // Scores of a tile to P, against the row's reference.
  auto weigh = [&](int tile, f32x16_t& x) {
    const bool none = page_of(tile) < 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= a.scale * kLog2e;
    if (none || (tile + 1) * kKeys > vis_least) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = tile * kKeys + 8 * (e >> 2) + 4 * hh + (e & 3);
        x[e] = !none && key < vis ? x[e] : -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
    top = xor32_op(top, MaxOp{});
    const bool past = top > most;
    const bool any = __any(past);
    if (any) {
      const float now = past ? top - kRise : ref;
      const float f = most == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - now);
      if (past) most = now + kMost;
      ref = now;
      l_run *= f;
      if (hh == 0) lds.factor[m_mine] = f;
    }
    if (lane == 0) lds.moved[wave] = any;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      x[e] = __builtin_amdgcn_exp2f(x[e] - ref);
      sum += x[e];
    }
    l_run += sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 u = make_uint2(T::pack2(x[4 * i], x[4 * i + 1]), T::pack2(x[4 * i + 2], x[4 * i + 3]));
      *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(lds.p) + m_mine * 64 + ((i ^ p_swz) * 16) + hh * 8) = u;
    }
  };
  // Values of keys that some row must not see: P is zero there, but zero times an
  // infinity or NaN is not.  (A row that does see such a key has them in its scores.)
  auto scrub = [&](int tile) {
    uint8_t* v_tile = lds.keys[tile % kBuffers];
    for (int i = tid; i < kKeys * kCkvBytes / 16; i += kThreads) {
      u32x4_t* p = reinterpret_cast<u32x4_t*>(v_tile + i * 16);
      *p = finite_or_zero<T>(*p);
    }
  };
  auto output = [&](int tile) {
    const uint8_t* v_tile = lds.keys[tile % kBuffers];
    const int4 moved = *reinterpret_cast<const int4*>(lds.moved);
    const int any = moved.x | (TILES > 1 ? moved.y : 0) | (TILES > 2 ? moved.z | moved.w : 0);
    if (__builtin_amdgcn_readfirstlane(any) != 0) {
#pragma unroll
      for (int r = 0; r < TILES; ++r) {
        const int mine = r == 0 ? moved.x : (r == 1 ? moved.y : (r == 2 ? moved.z : moved.w));
        if (__builtin_amdgcn_readfirstlane(mine) != 0) {
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
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u32x4_t p[TILES];
#pragma unroll
      for (int r = 0; r < TILES; ++r)
        p[r] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(lds.p) + r * 2048 + p_read +
                                                          (((2 * ks + hh) ^ p_swz) * 16));
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint2 lo = read_tr16(v_tile + (v_at[0] ^ (d * 64)) + ks * 16 * kCkvBytes);
        const uint2 hi = read_tr16(v_tile + (v_at[1] ^ (d * 64)) + ks * 16 * kCkvBytes);
        const u32x4_t v{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int r = 0; r < TILES; ++r) accumulate<true>(T{}, v, p[r], o[d][r]);
      }
    }
  };

  if (t0 < t1) {
    if (t0 + 2 < t1)
      wait_loads<kTileLoads>();
    else
      wait_loads<0>();
    lds_barrier();
    const int vis_all = __builtin_amdgcn_readfirstlane(
        min(min(lds.least[0], lds.least[1]), min(lds.least[2], lds.least[3])));
    if (scores) multiply(t0, sc);
    for (int t = t0; t < t1; ++t) {
      f32x16_t next;
      if (scores && t + 1 < t1) multiply(t + 1, next);
      lds_barrier();  // every wave is done with tile t - 1 and its P
      if (t + 3 < t1) {
        if ((t + 3) / kPageTiles >= page0 + kWindow) {
          page0 = t / kPageTiles;
          fill_window();
          __syncthreads();
        }
        load_tile(t + 3);
      }
      if (scores) weigh(t, sc);
      if ((t + 1) * kKeys > vis_all || page_of(t) < 0) scrub(t);
      if (t + 3 < t1)
        wait_loads<kTileLoads>();
      else
        wait_loads<0>();
      lds_barrier();
      output(t);
      sc = next;
    }
  }
  // References and sums of the rows, to every wave.
  if (scores) {
    l_run = xor32_op(l_run, AddOp{});
    if (hh == 0) lds.row[m_mine] = make_float2(most == -INFINITY && l_run == 0.f ? -INFINITY : ref, l_run);
  }
  lds_barrier();
  finish<T, TILES>(a, w, s, t0 >= t1, lds.row, o);
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
template <typename T>
__device__ __forceinline__ void attend_many(const PrefixAttentionArgs& a, const Plan& w, const Segment& s, LdsMany& lds) {
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

  // The ids of 64 pages, a lane each (-1: none), from column `first_held` on.
  const int last_column = (s.tile1 - 1) / kPageTiles < a.cols ? (s.tile1 - 1) / kPageTiles : static_cast<int>(a.cols) - 1;
  int first_held = s.tile0 / kPageTiles, held = -1;
  auto hold_pages = [&] {
    const int c = first_held + (own_thread() & 63);
    const int32_t page = c <= last_column ? s.table[c] : -1;
    held = page >= 0 && page < a.blocks ? page : -1;
  };
  auto page_of = [&](int tile) { return __builtin_amdgcn_readlane(held, tile / kPageTiles - first_held); };
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
      load_to_lds<(n & 3) * 1024>(l.base + (n >> 2) * 4096, byte_of ^ ((n & 3) * 64 + (n >> 2) * 16),
                                  lds_tile + buffer + (n >> 2) * 4096);
    else
      load_to_lds<0>(l.rope, rope_byte, lds_rope + buffer);
  };

  hold_pages();
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
  u32x4_t q[kLatentHalf][2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int m = rg * 64 + (r ^ dh) * 32 + l32;
    const int64_t pair = s.pair0 + (m < s.count ? m : 0);
    const u32x4_t* qn = static_cast<const u32x4_t*>(a.query) + pair * (kCkvDim / 8) + dh * 32 + hh;
#pragma unroll
    for (int i = 0; i < kLatentHalf; ++i) {
      q[i][r] = qn[(i & 1) * 16 + (i >> 1) * 2];
    }
#pragma unroll
    for (int i = 0; i < kLatentHalf; ++i) asm volatile("" : "+v"(q[i][r]));
  }
  for (int i = tid; i < kPairs * (kKpeDim / 8); i += kThreads) {
    const int m = i >> 3;
    const int64_t pair = s.pair0 + (m < s.count ? m : 0);
    *reinterpret_cast<u32x4_t*>(&lds.rope[0] + m * kKpeBytes + ((i ^ (m >> 1)) & 7) * 16) =
        static_cast<const u32x4_t*>(a.query_rope)[pair * (kKpeDim / 8) + (i & 7)];
  }
  // (Rows of pairs 64 rg + (r ^ dh) 32 + l32: the other tile is 32 rows away.)
  uint32_t qr_at = lds_address(lds.rope) + static_cast<uint32_t>((tile_mine * 32 + l32) * kKpeBytes + (((4 * dh + hh) ^ (l32 >> 1)) & 7) * 16);
  const int vis = m_mine < s.count ? w.visible[(s.pair0 + m_mine) / a.heads] : 0;
  f32x16_t o[4][4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][r][e] = 0.f;
      settle(o[d][r]);
    }
  float ref = 0.f, l_run = 0.f;
  float room = -INFINITY;  // a score above the reference by more moves it (nothing seen yet: any does)
  int vis_least = m_mine < s.count ? vis : 0x7fffffff;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) vis_least = min(vis_least, __shfl_xor(vis_least, d));
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
  // Barrier A before the scores of a tile in that buffer.
  auto begin_scores = [&](uint32_t buffer) {
    wait_loads<0>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch_k(k_at + buffer, r_at + buffer, i);
  };

  // Tile t, in buffer `now`, is weighed and put out; the scores of tile t + 1, in
  // buffer `ahead`, come first, and of tile t - 1 kLate products are open.  One
  // form for every t, the one before the first tile, of a page that names nothing,
  // among them: the compiler does not find registers for more.
  uint32_t now = 2 * kTileBytes, ahead = 0, beyond = kTileBytes;
  int page_t = -1, page_1 = 0, page_2 = 0;  // of tiles t, t + 1 and t + 2
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
    u32x4_t qr[2][2], other[4];
    f32x16_t next[2];
    const int page = page_t;
    Load next_load;
    const int page_next = page_of(t + 3);
#pragma unroll
    for (int e = 0; e < 4; ++e) other[e] = lds_get(half_at + wave * 4096 + lane16 + e * 1024);
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
        if constexpr (j == 12) if (((seen_mine - 1 - t) | page) < 0) {
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
          l_run += mine[e];
          more += mine[e + 1];
          if constexpr (e % 4 == 2)
            lds_put(p_write ^ (n * 16), T::pack2(mine[e - 2], mine[e - 1]), T::pack2(mine[e], mine[e + 1]));
        }
        if constexpr (j == 24) l_run += more;
        if constexpr (j == 29) moved_last = lds.moved_last;
        if constexpr (j >= 29 && j < 33) fetch_p(0, j - 29);
        if constexpr (j == 33) fetch_v(v_from, 0);
        if constexpr (j == 35) fetch_v(v_from, 1);
        if constexpr (j == 28) {
          // Values of keys that some row must not see: see attend().
          if (((seen_all - 1 - t) | page) < 0) {
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
        if constexpr (n == 10) next_load = load_of(t + 3, page_next);
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
  begin_scores(0);
  page_1 = page_of(t0);
  page_2 = page_of(t0 + 1);
  load = load_of(t0 + 1, page_2);
  for (int t = t0 - 1; t < t1; ++t) {
    if ((t + 3) / kPageTiles - first_held >= 64) {
      first_held = t / kPageTiles;
      hold_pages();
    }
    round(t);   // (the last one's scores are of no tile, and nobody reads them)
  }
  wait_loads<0>();
  l_run = xor32_op(l_run, AddOp{});
  lds_barrier();
  float2* const rows = reinterpret_cast<float2*>(&lds.p[0]);
  if (hh == 0) rows[m_mine] = make_float2(room == -INFINITY && l_run == 0.f ? -INFINITY : ref, l_run);
  lds_barrier();
  finish<T, 4>(a, w, s, false, rows, o);
}

template <typename T>
__global__ __launch_bounds__(kThreads, 1) void prefix_attention_kernel(PrefixAttentionArgs a) {
  __shared__ __align__(16384) Lds lds;
  Plan w;
  carve(a.workspace, a.rows, a.heads, a.batch, a.groups, &w);
  const int part = blockIdx.x;
  if (part >= *w.used) return;
  const int64_t stop = uniform(w.parts[part].stop);
  int64_t at = uniform(w.parts[part].unit);
  int at_span = uniform(w.parts[part].span);
  while (at < stop) {
    Span s = uniform(w.spans[at_span]);
    int64_t end = s.unit0 + (s.pairs > 0 ? units_of(s) : 0);
    while (at >= end) {
      s = uniform(w.spans[++at_span]);
      end = s.unit0 + (s.pairs > 0 ? units_of(s) : 0);
    }
    const int units = s.tiles + kBegin;
    const int64_t item = uniform((at - s.unit0) / units);
    const int64_t item_start = s.unit0 + item * units, item_end = item_start + units;
    const int64_t seg_end = item_end < stop ? item_end : stop;
    auto tile_of = [&](int64_t u) { return u > kBegin ? static_cast<int>(u) - kBegin : 0; };
    Segment g;
    const int first = static_cast<int>(item) * kPairs;
    g.pair0 = static_cast<int64_t>(s.pair0) + first;
    g.count = s.pairs - first < kPairs ? s.pairs - first : kPairs;
    g.tile0 = s.tile0 + tile_of(at - item_start);
    g.tile1 = s.tile0 + tile_of(seg_end - item_start);
    g.table = a.block_table + s.table * a.cols;
    const bool whole = at == item_start && seg_end == item_end;
    g.direct = whole && s.merge < 0;
    g.row = whole ? merge_row(w, s.merge, first, at_span >= a.groups) : part_row(w, part, at == item_start);
    g.row_step = whole ? 2 : 1;
    if (at_span >= a.groups) {  // a request's last row of the item sees the most
      const int seen = (uniform(w.visible[(g.pair0 + g.count - 1) / a.heads]) + kKeys - 1) / kKeys;
      g.tile1 = g.tile1 < seen ? g.tile1 : seen;
      g.tile0 = g.tile0 < g.tile1 ? g.tile0 : g.tile1;
    }
    if (g.tile0 >= g.tile1)
      nothing<T>(a, w, g);
    else if (g.count <= 32)
      attend<T, 1>(a, w, g, lds.few);
    else if (g.count <= 64)
      attend<T, 2>(a, w, g, lds.few);
    else
      attend_many<T>(a, w, g, lds.many);
    at = seg_end;
  }
}

// -------------------------------------------------------------------- the join
// A wave a pair: its segments' references, then their sums.
template <typename T>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixAttentionArgs a) {
  Plan w;
  carve(a.workspace, a.rows, a.heads, a.batch, a.groups, &w);
  const int lane = threadIdx.x & 63;
  const int pair = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int heads = static_cast<int>(a.heads);
  if (pair >= a.rows * a.heads) return;
  const int b = w.request[pair / heads];
  if (b < 0) return;
  const int64_t total = *w.total, parts = *w.used;
  const Span own = w.spans[a.groups + b];
  struct Run {  // segments of one item
    int w0, n;
    bool begins;      // the item begins in part w0
    int64_t whole;    // row of the sums where there is one segment
    int m;
  };
  auto run_of = [&](const Span& s, bool is_own) {
    Run r;
    const int in = pair - s.pair0, item = in / kPairs;
    const int64_t units = s.tiles + kBegin, u0 = s.unit0 + item * units;
    r.w0 = part_of(total, parts, u0);
    r.n = part_of(total, parts, u0 + units - 1) - r.w0 + 1;
    r.m = in - item * kPairs;
    r.whole = r.n == 1 ? merge_row(w, s.merge, in, is_own) : -1;
    return r;
  };
  const Run mine = run_of(own, true);
  if (own.group < 0 && mine.n == 1) return;  // (written by the attention itself)
  Run shared{};
  if (own.group >= 0) shared = run_of(w.spans[own.group], false);
  const int n = mine.n + shared.n;
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
    l += wave_all_op(f == 0.f ? 0.f : v.y * f, AddOp{});
    const int count = n - k0 < 64 ? n - k0 : 64;
    for (int k = 0; k < count; ++k) {
      const float fk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), k));
      if (fk == 0.f) continue;  // (a part without tiles wrote no sums)
      const int64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(row), k));
      const float4* p = reinterpret_cast<const float4*>(w.sums + lo * kCkvDim) + lane;
      const float4 x = p[0], y = p[64];
      acc[0] = fmaf(x.x, fk, acc[0]);
      acc[1] = fmaf(x.y, fk, acc[1]);
      acc[2] = fmaf(x.z, fk, acc[2]);
      acc[3] = fmaf(x.w, fk, acc[3]);
      acc[4] = fmaf(y.x, fk, acc[4]);
      acc[5] = fmaf(y.y, fk, acc[5]);
      acc[6] = fmaf(y.z, fk, acc[6]);
      acc[7] = fmaf(y.w, fk, acc[7]);
    }
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  uint2* out = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + static_cast<int64_t>(pair) * kCkvDim) + lane;
  out[0] = make_uint2(T::pack2(acc[0] * by, acc[1] * by), T::pack2(acc[2] * by, acc[3] * by));
  out[64] = make_uint2(T::pack2(acc[4] * by, acc[5] * by), T::pack2(acc[6] * by, acc[7] * by));
}

template <typename T>
hipError_t launch(const PrefixAttentionArgs& a, hipStream_t stream) {
  launch_kernel(kKernPrefixPlan, prefix_plan_kernel, dim3(1), dim3(kPlanThreads), stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  launch_kernel(kKernPrefixAttention, prefix_attention_kernel<T>, dim3(kParts), dim3(kThreads), stream, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  launch_kernel(kKernPrefixJoin, prefix_join_kernel<T>, dim3(static_cast<uint32_t>(ceil_div(a.rows * a.heads, 4))), dim3(256),
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
