// The 8-bit latent cache: append, attention and eviction.
//
// A token's row is 576 e4m3 values per latent head (512 latent, 64 rope) in
// pages of 128 tokens, [blocks, 128, G, 576], with one fp32 scale per page and
// latent head: value = code * scale.  The codes are exact in bf16 and fp16, so
// products run on the 16-bit MFMAs with the scale taken outside the sum.
//
//   append    scale = least power of two >= amax / 448 over a page's rows; a
//             page that grows its scale shifts its older rows.
//   attention s = scale * c_page * (q . k), p = softmax(s), o = sum p c_page v
//   weights   token_weights[slot] += sum over rows and heads of p
//   evict     keeps a request's most attended tokens and moves the kept ones
//             beyond the budget into the holes below it.
#include <algorithm>
#include <cfloat>

#include "lds_load.h"
#include "nvdsa_common.h"
#include "nvdsa_kernels.h"

namespace nvdsa {
namespace {

constexpr int kRow = kQkDim;              // bytes of a token's row and latent head
constexpr int kRowChunks = kRow / 16;     // 36 chunks of 16 bytes
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126
constexpr float kLog2e = 1.4426950408889634f;

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------- e4m3 helpers
__device__ inline uint32_t cvt2(Bf16, uint32_t v, std::integral_constant<bool, false>) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, false));
}
__device__ inline uint32_t cvt2(Bf16, uint32_t v, std::integral_constant<bool, true>) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, true));
}
__device__ inline uint32_t cvt2(F16, uint32_t v, std::integral_constant<bool, false>) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, false));
}
__device__ inline uint32_t cvt2(F16, uint32_t v, std::integral_constant<bool, true>) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, true));
}
// Eight codes to eight 16-bit values (exact).
template <typename T>
__device__ inline typename T::vec8 widen8(uint32_t lo, uint32_t hi) {
  u32x4_t r;
  r[0] = cvt2(T{}, lo, std::integral_constant<bool, false>{});
  r[1] = cvt2(T{}, lo, std::integral_constant<bool, true>{});
  r[2] = cvt2(T{}, hi, std::integral_constant<bool, false>{});
  r[3] = cvt2(T{}, hi, std::integral_constant<bool, true>{});
  return __builtin_bit_cast(typename T::vec8, r);
}
// Four fp32 values (at most 448, or NaN) to four codes, round to nearest even.
__device__ inline uint32_t encode4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true));
}
__device__ inline uint32_t rescale4(uint32_t v, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v), false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v), true);
  return encode4(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}
__device__ inline uint4 rescale16(uint4 v, float ratio) {
  return make_uint4(rescale4(v.x, ratio), rescale4(v.y, ratio), rescale4(v.z, ratio), rescale4(v.w, ratio));
}
// Zero in the place of NaN codes (0x7f, 0xff): the byte's low seven bits all
// set carry into bit 7 when one is added.
__device__ inline uint32_t nan_to_zero4(uint32_t v) {
  const uint32_t bad = (((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return v & ~(bad * 0xffu);
}

// Least power of two s in [2^-126, 2^120] with amax / s <= 448 = 1.75 * 2^8.
__device__ inline float least_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int k = static_cast<int>(u >> 23) - 126 - ((u & 0x7fffffu) > 0x600000u ? 8 : 9);
  k = k < -126 ? -126 : (k > 120 ? 120 : k);
  return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

// -------------------------------------------------------------------- append
// One workgroup per (page that receives rows, latent head).  It reads the
// page's new rows once into registers (at most 128 * 72 chunks of 8 values
// over 512 threads), takes their largest magnitude, and writes the codes.
// Bound by the rows' bytes (3 per value); a decode step's by latency.
constexpr int kAppendThreads = 512;
constexpr int kAppendChunks = kBlock * (kRow / 8) / kAppendThreads;  // 18 a thread

struct Span {  // a request's new rows: row0 + i goes to slot first + i, i < count
  int64_t row0;
  int first;
  int count;
};
__device__ inline Span append_span(const Latent8AppendArgs& a, int64_t b) {
  int64_t lo = b > 0 ? a.seq_q[b - 1] : 0, hi = a.seq_q[b];
  lo = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
  hi = hi < lo ? lo : (hi > a.rows ? a.rows : hi);
  const int64_t cap = a.cols * kBlock;
  int64_t s0 = static_cast<int64_t>(a.seq_kv[b]) - (hi - lo), s1 = a.seq_kv[b];
  if (s1 > cap) s1 = cap;
  int64_t skip = 0;
  if (s0 < 0) {
    skip = -s0;
    s0 = 0;
  }
  return {lo + skip, static_cast<int>(s0), static_cast<int>(s1 > s0 ? s1 - s0 : 0)};
}
__device__ inline int pages_of(const Span& s) {
  return s.count > 0 ? ((s.first + s.count - 1) >> kBlockShift) - (s.first >> kBlockShift) + 1 : 0;
}

template <typename T>
__global__ __launch_bounds__(kAppendThreads) void latent8_append_kernel(Latent8AppendArgs a) {
  __shared__ int scratch[kAppendThreads / 64 + 1];
  __shared__ int found_page;
  __shared__ int64_t found_b;
  __shared__ uint32_t wave_max[kAppendThreads / 64];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int g = blockIdx.y;
  // The workgroup's request and page, counted over the requests in order.
  if (tid == 0) found_b = -1;
  int before = 0;
  for (int64_t b0 = 0; b0 < a.batch; b0 += kAppendThreads) {
    const int64_t b = b0 + tid;
    const int n = b < a.batch ? pages_of(append_span(a, b)) : 0;
    int total;
    const int at = before + block_exclusive_scan(n, scratch, &total);
    const int64_t want = blockIdx.x;
    if (want >= at && want < at + n) {
      found_b = b;
      found_page = static_cast<int>(want) - at;
    }
    before += total;
    if (want < before) break;
  }
  __syncthreads();
  const int64_t b = found_b;
  if (b < 0) return;
  const Span span = append_span(a, b);
  const int page = (span.first >> kBlockShift) + found_page;
  const int32_t block = a.block_table[b * a.cols + page];
  const int lo = span.first > page * kBlock ? span.first - page * kBlock : 0;  // first new row of the page
  const int end = span.first + span.count - page * kBlock;
  const int n = (end < kBlock ? end : kBlock) - lo;
  const int64_t row0 = span.row0 + (page * kBlock + lo - span.first);
  if (g == 0 && a.entries != nullptr) {
    const int64_t e = a.entries[b];
    if (e >= 0 && e < a.pool_rows && tid < n) {
      const int64_t at = e * a.cols * kBlock + page * kBlock + lo + tid;
      if (a.token_positions != nullptr) a.token_positions[at] = a.positions[row0 + tid];
      if (a.token_weights != nullptr) a.token_weights[at] = 0.f;
    }
  }
  if (block < 0 || block >= a.blocks) return;

  const int chunks = n * (kRow / 8);
  u32x4_t v[kAppendChunks];
  uint32_t most = 0;
  constexpr uint32_t kInf = std::is_same<T, Bf16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int i = 0; i < kAppendChunks; ++i) {
    const int q = i * kAppendThreads + tid;
    v[i] = u32x4_t{0, 0, 0, 0};
    if (q < chunks) {
      const int r = q / (kRow / 8), c = q - r * (kRow / 8);
      const int64_t at = (row0 + r) * a.latent_heads + g;
      v[i] = *(c < kCkvDim / 8 ? static_cast<const u32x4_t*>(a.kv) + at * (kCkvDim / 8) + c
                               : static_cast<const u32x4_t*>(a.k_rope) + at * (kKpeDim / 8) + c - kCkvDim / 8);
    }
  }
#pragma unroll
  for (int i = 0; i < kAppendChunks; ++i) {
    if (i * kAppendThreads < chunks) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = v[i][k] & 0x7fffu, y = (v[i][k] >> 16) & 0x7fffu;
        if (x < kInf && x > most) most = x;
        if (y < kInf && y > most) most = y;
      }
    }
  }
  most = wave_reduce_to_lane63(most, MaxU32Op{});
  if (lane == 63) wave_max[wave] = most;
  float* scale_at = a.cache_scale + static_cast<int64_t>(block) * a.latent_heads + g;
  const float old = *scale_at;  // (before the barrier: thread 0 writes it at the end)
  __syncthreads();
  most = wave_max[0];
#pragma unroll
  for (int w = 1; w < kAppendThreads / 64; ++w) most = most < wave_max[w] ? wave_max[w] : most;
  const float need = least_scale(T::to_float(static_cast<uint16_t>(most)));
  const bool keeps = lo > 0 && old >= need;
  const float now = keeps ? old : need;
  uint8_t* base = static_cast<uint8_t*>(a.latent_cache) + static_cast<int64_t>(block) * kBlock * a.latent_heads * kRow +
                  static_cast<int64_t>(g) * kRow;
  const int64_t stride = a.latent_heads * kRow;
  if (lo > 0 && !keeps) {  // the older rows under the larger scale
    const float ratio = old / now;
    for (int q = tid; q < lo * kRowChunks; q += kAppendThreads) {
      const int r = q / kRowChunks, c = q - r * kRowChunks;
      uint4* p = reinterpret_cast<uint4*>(base + r * stride) + c;
      *p = rescale16(*p, ratio);
    }
  }
  // Division by a power of two is the product with its reciprocal, exactly.
  const uint32_t bits = __float_as_uint(now);
  const bool pow2 = (bits & 0x807fffffu) == 0 && (bits >> 23) >= 1 && (bits >> 23) <= 253;
  const float inverse = pow2 ? __uint_as_float((254u - (bits >> 23)) << 23) : 0.f;
#pragma unroll
  for (int i = 0; i < kAppendChunks; ++i) {
    const int q = i * kAppendThreads + tid;
    if (q < chunks) {
      const int r = q / (kRow / 8), c = q - r * (kRow / 8);
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint16_t h = static_cast<uint16_t>(v[i][k >> 1] >> (16 * (k & 1)));
        const float x = T::to_float(h);
        const float y = pow2 ? x * inverse : x / now;
        f[k] = (h & 0x7fffu) < kInf ? y : __uint_as_float(0x7fc00000u);  // infinities have no code: NaN
      }
      *(reinterpret_cast<uint2*>(base + (lo + r) * stride) + c) =
          make_uint2(encode4(f[0], f[1], f[2], f[3]), encode4(f[4], f[5], f[6], f[7]));
    }
  }
  if (tid == 0 && !keeps) *scale_at = now;
}

// ----------------------------------------------------------------- attention
// Split attention over a list of units.  A unit is one tile of 64 keys of one
// item; an item is up to 64 (query row, head) pairs of one request and latent
// head (with a list: heads of one query row).  The units of all items lie in a
// row, and workgroup w takes the w-th of equal parts, so a ragged batch loads
// every CU alike; an item that lies across parts leaves fp32 partials that a
// second kernel joins.
constexpr int kAttnThreads = 512;
constexpr int kRows = 64;       // (query row, head) pairs of an item
constexpr int kKeys = 64;       // keys of a tile
constexpr int kWindow = 512;    // resolved pages (or list entries) held at a time
constexpr int kLoads = kKeys * kRowChunks / (kAttnThreads / 2);  // of a thread (group 1) for a tile
constexpr int kPStride = kKeys + 8;  // fp16 row of P in LDS: 144 bytes
constexpr float kNoMax = -3.0e38f;
constexpr float kUnseen = 1.0e30f;
// P is fp16: each off by at most 2^-11 of itself, beside outputs of 8 or 11 bits;
// the normaliser is summed in fp32 from values that are not rounded.  Where
// scores set a row's reference anew its largest P is 2^kRise, and it may grow to
// 2^kMost before the next time: keys down to 2^-22 of the largest p * c keep all
// bits, and smaller ones are off by 2^-33 of it, so that a page of a large scale
// that holds the maximum leaves the others theirs (a reference at the maximum
// itself had them off by 2^-25).  Every bit more makes tiles be weighed again
// more often: calls of 24 x 8,192 tokens with weights take 84.2 us with 2^8 and
// 83.6 with the maximum itself, of 16 x 4 rows over up to 16,387 130.1 and 129.0.
// fp16 outputs are 2.5e-4 (relative, all together) from the 64-bit ones, with a
// P of 32 bits 2.1e-4; bf16 outputs 1.7e-3 either way.  A second fp16 for what P's
// first leaves would add 16 products to a tile's 34.
constexpr float kRise = 8.f;
constexpr float kMost = 15.9f;
// A tile is weighed again where its largest P passes 2^kMost, or where p, P times
// 2^up, might leave fp32's range: with a largest P of 2^top, where top passes
// kMostSum - 4 up.  Up to up = 20 that is kMost; p stays below 2^36 of its
// reference, and a P below 2^-126, which becomes zero, counts only where up
// passes 55, that is where any top from -126 on passes the limit.  In a list,
// where keys have scales of their own, up is that of the least one, and 1 / c and
// 2^lift, which multiply P one after the other, have to be in range too.
constexpr float kMostSum = 95.9f;
constexpr float kMostUp = 55.f;
constexpr float kLeast = -60.f;    // log2 of a list's scales
constexpr float kMostLift = 100.f;
constexpr int kBegin = 6;       // what the start of a segment costs, in tiles
constexpr float kJoinCost = 0.0375f;  // what joining one part more costs, in tiles
constexpr int64_t kParts = 256; // one workgroup per CU (LDS)
constexpr int kPartFloats = kRows * kCkvDim;

struct Plan {
  int64_t total;  // units
  int64_t parts;  // workgroups that share them
  int begin;      // units of an item before its first tile
  int share;      // > 0: a part is a unit, up to so many tiles of one item
};
constexpr int64_t kMostItems = int64_t{1} << 24;  // with tiles below 2^15 an item: see divide

// x / y for 0 <= x < 2^53, y > 0 (a 64-bit division is a microsecond of
// instructions; units stay below 2^40, their product with a part below 2^48).
__device__ inline int64_t divide(int64_t x, int64_t y) {
  int64_t q = static_cast<int64_t>(static_cast<double>(x) / static_cast<double>(y));
  const int64_t rest = x - q * y;
  q += rest < 0 ? -1 : (rest >= y ? 1 : 0);
  return q;
}
__device__ inline int64_t part_start(const Plan& p, int64_t w) { return p.share > 0 ? w : divide(p.total * w, p.parts); }
// The part of an item's last unit.
__device__ inline int64_t part_of_end(const Plan& p, int64_t end) {
  return p.share > 0 ? end - 1 : divide(end * p.parts + p.total - 1, p.total) - 1;
}
// Units of an item of so many tiles, and the tile at which unit u of it begins.
__device__ inline int units_of(const Plan& p, int tiles) {
  return p.share > 0 ? (tiles + p.share - 1) / p.share : tiles + p.begin;
}
__device__ inline int tile_of(const Plan& p, int tiles, int u) {
  if (p.share > 0) return tiles * u / units_of(p, tiles);
  return u > p.begin ? u - p.begin : 0;
}

// Equal parts of the units.  A part that lies across two items begins anew,
// which costs the time of `cost` tiles, so an item counts that much more than
// its tiles (at most an eighth of a part more: a part that lies in the first
// units only has nothing to do).  What the eighth leaves out costs a part that
// many tiles; where shares of single items, of up to total / (parts - items)
// tiles, are shorter than that, they are the parts (`tiles`: what every item
// has, or 0).  24 items of 32 tiles (lists) take 30 us in 8 shares of 4 tiles
// each and 37 in 256 parts of 3; 24 of about 129 tiles 46 in shares of 14 and 50
// in 256 parts of 12; 24 of 512 stay in 256 parts of 48.
// Partial sums have to be joined, at about kJoinCost tiles' time a part of an
// item: beyond sqrt(tiles / kJoinCost) parts of an item, more of them cost more
// than they save (1 x 32,768 tokens, 512 tiles: 28 + 11 us in 117 parts, 25 + 20
// in 256).
__device__ inline Plan make_plan(int64_t items, int64_t tiles_all, int64_t parts, bool joins, int cost, int tiles) {
  Plan p{tiles_all, tiles_all, 0, 0};
  if (joins && items > 0) {
    const float most = static_cast<float>(tiles_all) * static_cast<float>(items) * (1.f / kJoinCost);
    if (most < static_cast<float>(parts * parts)) parts = static_cast<int64_t>(__builtin_amdgcn_sqrtf(most));
  }
  if (p.parts > parts) p.parts = parts;
  if (p.parts < 1) p.parts = 1;
  if (items <= 1) return p;
  const int64_t eighth = divide(tiles_all, 8 * p.parts);
  p.begin = eighth < cost ? static_cast<int>(eighth) : cost;
  if (items < parts) {
    int64_t share = tiles > 0 ? divide(tiles - 1, divide(parts, items)) + 1 : divide(tiles_all - 1, parts - items) + 1;
    if ((share + p.begin - cost) * p.parts < tiles_all + items * p.begin) {
      p.share = static_cast<int>(share);
      return p;  // (total and parts: counted over the requests next)
    }
  }
  p.total += items * p.begin;
  return p;
}

struct Request {
  int64_t row0;   // first query row
  int n;          // query rows
  int len;        // cached tokens, clipped to the table
  int items_g;    // items of one latent head
  int64_t items;
  int tiles;      // units of an item
};
__device__ inline Request make_request(const Latent8Args& a, int64_t row0, int n, int len) {
  Request r;
  r.row0 = row0;
  r.n = n;
  r.len = len;
  r.items_g = a.topk != nullptr ? n * ((a.per + kRows - 1) / kRows) : (n * a.per + kRows - 1) / kRows;
  r.items = static_cast<int64_t>(r.items_g) * a.latent_heads;
  r.tiles = ((a.topk != nullptr ? static_cast<int>(a.list_len) : len) + kKeys - 1) / kKeys;
  if (r.tiles < 1) r.tiles = 1;
  return r;
}
struct Ends {  // as they lie in memory
  int32_t lo, hi, len;
};
__device__ inline Ends ends_of(const Latent8Args& a, int64_t b) {
  return {a.seq_q[b > 0 ? b - 1 : 0], a.seq_q[b], a.seq_kv[b]};
}
__device__ inline Request request_of(const Latent8Args& a, int64_t b, const Ends& e) {
  int64_t lo = b > 0 ? e.lo : 0, hi = e.hi;
  lo = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
  hi = hi < lo ? lo : (hi > a.rows ? a.rows : hi);
  const int64_t cap = a.cols * kBlock, len = e.len;
  return make_request(a, lo, static_cast<int>(hi - lo), static_cast<int>(len < 0 ? 0 : (len > cap ? cap : len)));
}
__device__ inline Request request_of(const Latent8Args& a, int64_t b) { return request_of(a, b, ends_of(a, b)); }

// Work of a request, or of several.
struct Units {
  int64_t items;
  int64_t tiles;
};
// Exclusive prefix over the workgroup's threads.
template <int THREADS>
__device__ inline Units scan_units(const Units& v, Units* scratch, Units* total) {
  const int wid = threadIdx.x >> 6;
  const Units x{static_cast<int64_t>(wave_inclusive_scan(static_cast<uint64_t>(v.items))),
                static_cast<int64_t>(wave_inclusive_scan(static_cast<uint64_t>(v.tiles)))};
  if ((threadIdx.x & 63) == 63) scratch[wid] = x;
  __syncthreads();
  Units before{0, 0}, all{0, 0};
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const Units t = scratch[w];
    before.items += w < wid ? t.items : 0;
    before.tiles += w < wid ? t.tiles : 0;
    all.items += t.items;
    all.tiles += t.tiles;
  }
  *total = all;
  __syncthreads();
  return {before.items + x.items - v.items, before.tiles + x.tiles - v.tiles};
}

// A value that every lane holds, in scalar registers.
__device__ inline int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(x) >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// Where a workgroup's part begins: the request, and its first unit.
struct Start {
  Plan plan;
  int64_t items;  // of all requests
  int64_t b;
  int64_t base;   // first unit of the request
  int64_t item;   // its first item
  Request r;
};
// EACH(request): the tiles of each of its items, ITEMS(request): their number;
// COST, JOINS: see make_plan; `ends`: of request threadIdx.x (of request 0 where there
// is none), on its way.
template <int THREADS, int COST, bool JOINS, typename ITEMS, typename EACH>
__device__ inline Start find_start(const Latent8Args& a, const Ends& ends, int64_t part, int64_t parts, int tiles,
                                   ITEMS items, EACH each) {
  __shared__ Units scratch[THREADS / 64];
  __shared__ int64_t found[6];
  Start s;
  const int tid = threadIdx.x;
  auto units = [&](const Request& q) -> Units { return {items(q), items(q) * each(q)}; };
  Request r{};
  Units mine{0, 0}, sum{0, 0};
  if (tid < a.batch) {
    r = request_of(a, tid, ends);
    sum = mine = units(r);
  }
  for (int64_t b = tid + THREADS; b < a.batch; b += THREADS) {
    const Units u = units(request_of(a, b));
    sum.items += u.items;
    sum.tiles += u.tiles;
  }
  Units total;
  if (tid == 0) found[0] = -1;
  Units at = scan_units<THREADS>(sum, scratch, &total);
  total = {uniform64(total.items), uniform64(total.tiles)};
  s.plan = make_plan(total.items, total.tiles, parts, JOINS, COST, tiles);
  s.items = total.items;
  // (More items than the rows can have: requests whose ends decrease share
  // rows.  Nothing is done.)
  if (total.items > kMostItems) s.plan.parts = 0;
  // Shares: parts are counted in the place of tiles; where all items have as
  // many, the items say it.
  const bool shares = s.plan.share > 0, alike = shares && tiles > 0;
  auto counted = [&](const Request& q) -> Units {
    if (shares && !alike) return {items(q), items(q) * units_of(s.plan, each(q))};
    return units(q);
  };
  if (alike) {
    s.plan.total = s.plan.parts = total.items * units_of(s.plan, tiles);
  } else if (shares) {
    if (tid < a.batch) sum = mine = counted(r);
    for (int64_t b = tid + THREADS; b < a.batch; b += THREADS) {
      const Units u = counted(request_of(a, b));
      sum.items += u.items;
      sum.tiles += u.tiles;
    }
    at = scan_units<THREADS>(sum, scratch, &total);
    s.plan.total = s.plan.parts = uniform64(total.tiles);
  }
  if (part < s.plan.parts && total.tiles > 0) {
    const int64_t u = part_start(s.plan, part);
    auto place = [&](const Units& x) {
      if (alike) return x.items * units_of(s.plan, tiles);
      return shares ? x.tiles : x.tiles + x.items * s.plan.begin;
    };
    Units before{0, 0};
    for (int64_t b0 = 0; b0 < a.batch; b0 += THREADS) {
      const int64_t b = b0 + tid;
      if (a.batch > THREADS) {  // (the first scans were over strided sums)
        r = Request{};
        mine = {0, 0};
        if (b < a.batch) {
          r = request_of(a, b);
          mine = counted(r);
        }
        Units chunk;
        at = scan_units<THREADS>(mine, scratch, &chunk);
        at = {at.items + before.items, at.tiles + before.tiles};
        before = {before.items + chunk.items, before.tiles + chunk.tiles};
      }
      if (u >= place(at) && u < place({at.items + mine.items, at.tiles + mine.tiles})) {
        found[0] = b;
        found[1] = place(at);
        found[2] = r.row0;
        found[3] = r.n;
        found[4] = r.len;
        found[5] = at.items;
      }
      if (a.batch > THREADS && u < place(before)) break;
    }
  }
  __syncthreads();
  s.b = uniform64(found[0]);
  s.base = uniform64(found[1]);
  s.item = uniform64(found[5]);
  s.r = make_request(a, uniform64(found[2]), static_cast<int>(uniform64(found[3])), static_cast<int>(uniform64(found[4])));
  return s;
}

// The item's rows: pair f = first + m (m < count) is query row f / per, head
// f % per of the latent head's; it sees `vis` keys.
struct Item {
  int g;
  int first;
  int count;
  int lead;  // list: the item's query row
};
__device__ inline Item item_of(const Latent8Args& a, const Request& r, int64_t it) {
  Item x;
  const int per = a.per;
  x.g = a.latent_heads == 1 ? 0 : static_cast<int>(it) / r.items_g;
  int j = static_cast<int>(it) - x.g * r.items_g;
  if (a.topk != nullptr) {
    const int groups = (per + kRows - 1) / kRows;
    x.lead = j / groups;
    j -= x.lead * groups;
    x.first = x.lead * per + j * kRows;
    const int left = per - j * kRows;
    x.count = left < kRows ? left : kRows;
  } else {
    // Early and late rows in turn: under the causal bound they cost little and
    // much, and neighbours share a workgroup's part.
    j = (j & 1) ? r.items_g - 1 - (j >> 1) : (j >> 1);
    x.lead = 0;
    x.first = j * kRows;
    const int left = r.n * per - j * kRows;
    x.count = left < kRows ? left : kRows;
  }
  return x;
}
__device__ inline int visible(const Request& r, int i) {
  const int64_t v = static_cast<int64_t>(r.len) - (r.n - 1 - i);
  return v > 0 ? static_cast<int>(v) : 0;
}

// What the joining kernel needs of an item that lies across parts.
struct JoinEntry {
  int64_t row0;
  int32_t first, count, g;
  int32_t slot0;   // slot of the first part's partial
  int32_t w0, w1;  // parts w0 .. w1 (w0's partial in slot0, w's in 2 w)
};

struct Work {
  float* part;      // [2 parts][64 * 512], in the accumulators' order
  float4* refs;     // [2 parts][64]: reference of the sums, of the normaliser, the normaliser
  JoinEntry* join;  // [parts], of an item each or named by a part; row0 < 0: nothing
  int32_t* idle;    // [1]: the attention did nothing (ends that decrease)
  float* lse;       // [rows, heads], base 2 (with weights)
};
constexpr size_t round256(size_t x) { return (x + 255) & ~size_t(255); }
__host__ __device__ inline Work carve_work(void* ws, int64_t parts) {
  Work w;
  char* p = static_cast<char*>(ws);
  w.part = reinterpret_cast<float*>(p);
  p += sizeof(float) * 2 * parts * kPartFloats;
  w.refs = reinterpret_cast<float4*>(p);
  p += sizeof(float4) * 2 * parts * kRows;
  w.join = reinterpret_cast<JoinEntry*>(p);
  p += round256(sizeof(JoinEntry) * parts);
  w.idle = reinterpret_cast<int32_t*>(p);
  p += round256(sizeof(int32_t));
  w.lse = reinterpret_cast<float*>(p);
  return w;
}

__device__ inline uint2 read_tr8(const uint8_t* p) {
  typedef int v2i __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) v2i lds_v2i;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(const_cast<uint8_t*>(p))));
}

__device__ inline float first_lane(float x) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

// What a page's (or list entry's) scale c enters: scores take it as a factor,
// P its logarithm into the exponent (p * c multiplies V's codes; exact for a
// power of two, else off by the logarithm's rounding).
struct alignas(16) Window {
  int32_t row;    // first cache row of the page, or the entry's row; -1: none
  float score;    // softmax scale * log2(e) * c
  float log2c;
  float inverse;  // 1 / c (of a list's entry)
};
__device__ inline int32_t row_of_slot(const Latent8Args& a, int64_t b, int64_t slot, bool ok) {
  if (!ok) return -1;
  const int32_t block = a.block_table[b * a.cols + (slot >> kBlockShift)];
  return block < 0 || block >= a.blocks ? -1 : block * kBlock + static_cast<int32_t>(slot & (kBlock - 1));
}
__device__ inline void add_scale(const Latent8Args& a, int g, Window& w) {  // the fields but row
  const int32_t block = w.row >> kBlockShift;
  float c = w.row < 0 ? 1.f : a.cache_scale[static_cast<int64_t>(block) * a.latent_heads + g];
  c = fminf(fmaxf(c, kMinScale), FLT_MAX);
  const uint32_t u = __float_as_uint(c);
  w.score = a.scale * kLog2e * c;
  const float exponent = static_cast<float>(static_cast<int>(u >> 23) - 127);
  w.log2c = exponent + __builtin_amdgcn_logf(__uint_as_float((u & 0x7fffffu) | 0x3f800000u));
  w.inverse = 1.f / c;
}

// base * 2^x / l where l > 0, else 0: in two factors, since 2^x alone may pass
// fp32's range on either side.
struct Quotient {
  float a, b;
  __device__ inline Quotient(float x, float l) {
    const float root = __builtin_amdgcn_exp2f(0.5f * x);
    a = l == 0.f ? 0.f : root / l;
    b = l == 0.f ? 0.f : root;
  }
  __device__ inline float of(float base) const { return base * a * b; }
};

// Eight waves in two groups of four: group g owns rows 32 g .. 32 g + 31 of the
// item.  For a tile, a group's wave takes S^T = K Q^T of 32 keys over half of
// the 576 dims (the halves meet through LDS, so that every lane holds 8 keys
// of one row), and O^T += V^T P^T of 128 latent dims, V^T by transposing 8-bit
// LDS reads, P in fp16.
//
// The groups run in opposite phases, one barrier a phase: while one multiplies
// (the scores of tile t and the output product of tile t - 1, two independent
// streams of MFMAs), the other takes its softmax, and each SIMD holds one wave
// of either.  P(t) is taken against a reference, the running maximum at some
// tile before; where a tile outgrows that by more than fp16 holds, or is the
// first that a row sees, the group weighs it again against its own maximum.
//
// The normaliser sums p without the scale, in fp32, against a reference of its
// own: p * c and p have their maxima in different pages where scales differ, by
// up to 2^246 (a page of zero rows has scale 2^-126 and weighs exp(0) a key all
// the same), and one reference would overflow or lose one of the two.
//
// Bound by the phases, of about 2,050 clocks each: a wave's 34 MFMAs of 32
// clocks (1,088) take 1,600 alone on their SIMD and 1,900 next to the other
// group's softmax, group 1's softmax with the loads 1,500.  In the loop that is
// 1.0 PFLOP/s, of the 1.27 that a large product reaches.  A part's start (10
// us) and its partial sums (3 us) come to that: 24 requests of 32,768 tokens
// and 64 heads in 138 us (110 GFLOP, 453 MB), 40 ragged ones with 8 heads in
// 99 us (4.8 TB/s), 2 x 515 rows over up to 8,197 tokens, 2 x 16 heads, in
// 454 us.  One phase for all waves took 175, 166 and 565.  Weighed against it:
// the same products on the 8-bit MFMAs, with bf16 queries split into two codes
// and P into three, took 164 us for the first and twice as long for lists.
template <typename T, bool LIST>
__global__ __launch_bounds__(kAttnThreads, 2) void latent8_attention_kernel(Latent8Args a) {
  __shared__ __align__(16) uint8_t keys[3][kKeys * kRow];
  __shared__ __align__(16) float4 half_s[8 * 2 * 64];
  __shared__ __align__(16) uint16_t p_tile[2][32 * kPStride];
  __shared__ __align__(16) float row_max[2][2][32][4];  // group, tile parity, row, wave
  __shared__ __align__(16) float row_top[LIST ? 2 : 1][2][32][4];  // likewise, without the scales
  __shared__ float2 row_ref[2][32];                     // group, row: see lift and the normaliser's reference
  __shared__ int outgrown[2][2];                        // group, tile parity
  __shared__ int bad_entries[2][LIST ? kWindow / kKeys : 1];  // tiles of a window with entries that name nothing
  __shared__ Window windows[LIST ? 2 : 1][kWindow];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hh = lane >> 5;
  const int grp = wave >> 2, kg = wave & 1, dh = (wave >> 1) & 1, wg = wave & 3;
  const int64_t part = blockIdx.x;
  const Ends ends = ends_of(a, tid < a.batch ? tid : 0);
  const int per = a.per;
  const int64_t row_bytes = a.latent_heads * kRow;

  // A tile's row k in LDS holds chunk c (16 bytes) at place c ^ ((k >> 2) & 3)
  // within its group of four: 16 keys of one chunk then lie in 64 different
  // banks.  Rows go straight to LDS, 64 places a wave (of group 1) and load;
  // this lane's places of a tile, the byte that belongs there: of the page, or,
  // with a list, of its row in the low 16 bits and the key above them.
  uint32_t byte_of[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int q = i * (kAttnThreads / 2) + wg * 64 + lane;
    const int k = q / kRowChunks, c = q - k * kRowChunks;
    byte_of[i] = static_cast<uint32_t>(((c & ~3) | ((c ^ (k >> 2)) & 3)) * 16 + (LIST ? k << 16 : k * row_bytes));
  }
  const uint32_t lds_keys = lds_address(keys) + wg * 1024;
  // LDS addresses of the score operand (chunks 18 dh + 2 j + hh) and of V.
  int k_at[2], v_at[2];
  {
    // The second half's waves take their 32 keys with the halves swapped, so
    // that accumulators 0-7 are the keys that a wave finishes itself.
    const int k = kg * 32 + (l32 ^ (dh * 16));
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const int c = 18 * dh + hh + 2 * odd;
      k_at[odd] = k * kRow + ((c & ~3) | ((c ^ (k >> 2)) & 3)) * 16;
    }
    const int i = lane & 15, sixteen = (lane >> 4) & 1;
    const int vk = 8 * hh + (i >> 1);
#pragma unroll
    for (int odd = 0; odd < 2; ++odd)
      v_at[odd] = vk * kRow + (wg * 8 + ((2 * odd + sixteen) ^ ((vk >> 2) & 3))) * 16 + 8 * (i & 1);
  }
  const int key_mine = kg * 32 + dh * 16 + 4 * hh;  // keys key_mine + 8 e + 0..3, e < 2, of a tile
  const int m_mine = grp * 32 + l32;
  uint16_t* const p_mine = p_tile[grp];

  const Start start = find_start<kAttnThreads, kBegin, true>(
      a, ends, part, a.parts, LIST ? (static_cast<int>(a.list_len) + kKeys - 1) / kKeys : 0,
      [](const Request& r) { return r.items; }, [](const Request& r) { return r.tiles; });
  const Work work = carve_work(a.workspace, a.parts);
  // Entries that no item writes below: all of the parts', or those behind the
  // last item's.  (More items than entries: ends that decrease.)
  const bool many = a.join_items && start.items > a.joins;
  if (tid == 0 && part == 0) *work.idle = many || start.items > kMostItems;
  if (tid == 0)
    for (int64_t k = a.join_items && !many ? start.items + part : part; k < a.joins; k += a.parts) work.join[k].row0 = -1;
  if (many || part >= start.plan.parts || start.b < 0) return;
  const int64_t stop = part_start(start.plan, part + 1);
  int64_t at = part_start(start.plan, part);
  int64_t b = start.b;
  int64_t base = start.base;
  int64_t item_base = start.item;
  Request r = start.r;

  while (at < stop) {
    // The next segment: units [u0, u1) of one item.
    int units = units_of(start.plan, r.tiles);
    while (at >= base + r.items * units) {
      base += r.items * units;
      item_base += r.items;
      ++b;
      r = request_of(a, b);
      units = units_of(start.plan, r.tiles);
    }
    const int64_t it = divide(at - base, units);
    const int64_t item_start = base + it * units;
    const int64_t item_end = item_start + units;
    const int64_t seg_end = item_end < stop ? item_end : stop;
    const Item x = item_of(a, r, it);
    const int i_last = LIST ? x.lead : (x.first + x.count - 1) / per;
    const int i_first = LIST ? x.lead : x.first / per;
    const int vis_most = visible(r, i_last), vis_least = visible(r, i_first);
    const int list_len = LIST ? static_cast<int>(a.list_len) : vis_most;
    int t0 = tile_of(start.plan, r.tiles, static_cast<int>(at - item_start));
    int t1 = tile_of(start.plan, r.tiles, static_cast<int>(seg_end - item_start));
    const int tiles_seen = (list_len + kKeys - 1) / kKeys;
    if (t1 > tiles_seen) t1 = tiles_seen;
    if (t0 > t1) t0 = t1;
    const bool busy = grp == 0 || x.count > 32;  // the group has rows

    const int32_t* list = LIST ? a.topk + (r.row0 + x.lead) * a.list_len : nullptr;
    // Tiles [c0, c1) run together: their pages are resolved before them, or,
    // with a list, windows of entries as the tiles pass, two at a time.
    constexpr int kWindowTiles = LIST ? kWindow / kKeys : 2 * kWindow;
    int c0 = t0, c1 = t1, w0 = t0;
    // This thread's entry of the window that begins with a tile: its row, and
    // the rest, for which nobody waits before the rows themselves are on the way.
    auto window_at = [&](int tile) -> Window& { return windows[LIST ? ((tile - w0) / kWindowTiles) & 1 : 0][tid]; };
    auto window_rows = [&](int tile) {
      if (LIST) {
        const int e = tile * kKeys + tid;
        const int id = e < list_len ? list[e] : -1;
        const int32_t row = row_of_slot(a, b, id, id >= 0 && id < vis_most);
        window_at(tile).row = row;
        const bool bad = __any(row < 0);
        if (lane == 0) bad_entries[((tile - w0) / kWindowTiles) & 1][LIST ? wave : 0] = bad;
      } else {
        const int64_t slot = (static_cast<int64_t>(tile >> 1) + tid) * kBlock;
        window_at(tile).row = row_of_slot(a, b, slot, slot < vis_most);
      }
    };
    auto window_scales = [&](int tile) { add_scale(a, x.g, window_at(tile)); };
    int vis_row;
    u32x4_t q[9][2];
    {
      const int f = x.first + (m_mine < x.count ? m_mine : 0);
      const int i = f / per, h = f - i * per;
      vis_row = m_mine < x.count ? visible(r, i) : 0;
      const int64_t row = (r.row0 + i) * a.heads + x.g * per + h;
      const u32x4_t* qn = static_cast<const u32x4_t*>(a.query) + row * (kCkvDim / 8);
      const u32x4_t* qr = static_cast<const u32x4_t*>(a.query_rope) + row * (kKpeDim / 8);
#pragma unroll
      for (int j = 0; j < 9; ++j) {
        const int c = dh * 36 + 4 * j + 2 * hh;  // chunk of 8 values
        const u32x4_t* p = (dh == 1 && j >= 7) ? qr + (c - kCkvDim / 8) : qn + c;
        q[j][0] = p[0];
        q[j][1] = p[1];
      }
    }
    f32x16_t o[4], s;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    // ref: the reference of P and o.  l_run, l_tile: sums of p against the
    // normaliser's, row_ref.y; it lies row_ref.x below ref ("lift": kUnseen, and
    // ref is 0, before the row's first key).
    float ref = 0.f, l_run = 0.f, l_tile = 0.f;
    float2* const my_row_ref = &row_ref[grp][l32];
    float sc[8];

    auto window_of = [&](int tile) -> const Window* {
      const unsigned i = tile - w0;
      if (LIST) return &windows[LIST ? (i / kWindowTiles) & 1 : 0][(i % kWindowTiles) * kKeys];
      return &windows[0][(i >> 1) & (kWindow - 1)];
    };
    // Without a list: the pages of the tiles in the three buffers and of the
    // one after them, in scalar registers.
    Window page_before{}, page_now{}, page_next{}, page_far{};
    auto scalar = [&](const Window& v) {
      return Window{__builtin_amdgcn_readfirstlane(v.row), first_lane(v.score), first_lane(v.log2c), 0.f};
    };
    // A tile's loads, by the waves of group 1, issued a few at a time.
    struct TileLoad {
      const uint8_t* base;
      uint32_t to;
      int32_t row[LIST ? kLoads : 1];
      bool on;
    };
    auto begin_load = [&](int tile, int buf, int32_t page_row) {
      TileLoad l;
      l.on = tile < c1;
      l.to = lds_keys + buf * (kKeys * kRow);
      if (LIST) {
        l.base = static_cast<const uint8_t*>(a.latent_cache) + x.g * kRow;
        if (l.on) {
          const Window* w = window_of(tile);
#pragma unroll
          for (int i = 0; i < kLoads; ++i) l.row[LIST ? i : 0] = w[byte_of[i] >> 16].row;
        }
      } else {
        l.base = static_cast<const uint8_t*>(a.latent_cache) +
                 (static_cast<int64_t>(page_row < 0 ? 0 : page_row) + (tile & 1) * kKeys) * row_bytes + x.g * kRow;
      }
      return l;
    };
    auto issue_load = [&](const TileLoad& l, int i0, int i1) {
      if (!l.on) return;
#pragma unroll
      for (int i = i0; i < i1; ++i) {
        if (LIST) {
          const int32_t row = l.row[LIST ? i : 0];
          load_to_lds(l.base + static_cast<int64_t>(row < 0 ? 0 : row) * row_bytes + (byte_of[i] & 0xffffu), l.to + i * 4096);
        } else {
          load_to_lds(l.base, byte_of[i], l.to + i * 4096);
        }
      }
    };
    auto load_tile = [&](int tile, int buf, int32_t page_row) {
      const TileLoad l = begin_load(tile, buf, page_row);
      issue_load(l, 0, kLoads);
    };
    // Scale fields of this lane's keys of the tile before: one page's (uniform), or each entry's.
    auto fields = [&](int tile, Window(&w)[LIST ? 8 : 1]) {
      if (LIST) {
        const Window* from = window_of(tile);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[LIST ? e : 0] = from[key_mine + 8 * (e >> 2) + (e & 3)];
      } else {
        w[0] = page_before;
      }
    };
    // Whether some row must not see some key of the tile before.
    auto ragged_tile = [&](int tile) -> bool {
      if (LIST) {
        const unsigned i = tile - w0;
        return __builtin_amdgcn_readfirstlane(bad_entries[(i / kWindowTiles) & 1][LIST ? i % kWindowTiles : 0]) != 0;
      }
      return (tile + 1) * kKeys > vis_least || page_before.row < 0;
    };
    // P of the tile's scores against the row's reference, into LDS; l_tile: the
    // sum of p, which is P times 2^(lift - log2c) as long as the row's limit keeps
    // that in range; ALONE: by exponents of its own.
    auto weigh = [&](const Window(&w)[LIST ? 8 : 1], float lift, auto alone) {
      constexpr bool ALONE = decltype(alone)::value;
      l_tile = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float pw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          pw[k] = __builtin_amdgcn_exp2f(sc[4 * e + k]);
          l_tile += ALONE ? __builtin_amdgcn_exp2f(sc[4 * e + k] + (lift - w[LIST ? 4 * e + k : 0].log2c))
                          : (LIST ? pw[k] * w[LIST ? 4 * e + k : 0].inverse : pw[k]);
        }
        const uint2 packed = make_uint2(F16::pack2(pw[0], pw[1]), F16::pack2(pw[2], pw[3]));
        *reinterpret_cast<uint2*>(&p_mine[l32 * kPStride + key_mine + 8 * e]) = packed;
      }
      if (!ALONE) l_tile *= __builtin_amdgcn_exp2f(fminf(LIST ? lift : lift - w[0].log2c, kMostLift));
    };
    auto most_of = [&](const float(&of)[4]) {
      const float4 v = *reinterpret_cast<const float4*>(of);
      return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
    };
    // A tile that outgrew a reference: both follow their maxima, the sums so far
    // follow them, and the tile is weighed again.  Returns the row's new
    // row_ref, to be stored when every wave has read the old one.
    auto weigh_again = [&](int tile) {
      const float2 old = *my_row_ref;
      const bool unseen = old.x == kUnseen;
      const float most = most_of(row_max[grp][tile & 1][l32]) - kRise;
      const float most_sum = LIST ? most_of(row_top[LIST ? grp : 0][tile & 1][l32]) : most + (kRise - page_before.log2c);
      const bool past = most > (unseen ? -INFINITY : ref), past_sum = most_sum > (unseen ? -INFINITY : old.y);
      const float down = past ? ref - most : 0.f;
      const float grow = unseen ? 1.f : __builtin_amdgcn_exp2f(down);
      ref = past ? most : ref;
      const float sum_ref = past_sum ? most_sum : old.y;
      l_run *= unseen || !past_sum ? 1.f : __builtin_amdgcn_exp2f(old.y - most_sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) sc[e] += down;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= grow;
      Window w[LIST ? 8 : 1];
      fields(tile, w);
      const float lift = unseen && !past ? kUnseen : ref - sum_ref;
      // (Exponents of their own for a list only where they have to be: they are
      // most of what 24 lists of 2,048 gain, 39.5 -> 38.4 us; without a list they
      // cost nothing.)
      if (LIST) {
        weigh(w, lift, std::false_type{});
        float low = w[0].log2c;
#pragma unroll
        for (int e = 1; e < 8; ++e) low = fminf(low, w[LIST ? e : 0].log2c);
        if (__any(low < kLeast || lift > kMostLift || lift - low > kMostUp)) {
          l_tile = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) l_tile += __builtin_amdgcn_exp2f(sc[e] + (lift - w[LIST ? e : 0].log2c));
        }
      } else {
        weigh(w, lift, std::true_type{});
      }
      return make_float2(lift, sum_ref);
    };
    // S^T of tile t in nine steps of 32 dims, and O^T of tile t - 1 in eight
    // steps of 16 keys and two of the wave's four tiles of dims (OUTPUT), step
    // by step together: two independent streams of MFMAs, each step's operands
    // read two steps ahead.
    auto multiply = [&](int t, const uint8_t* k_tile, const uint8_t* v_tile, auto with_output) {
      constexpr bool OUTPUT = decltype(with_output)::value;
      constexpr int kAhead = 2;
      u32x4_t k[kAhead + 1];
      uint2 v[kAhead + 1][2];
      f16x8_t p[2];
      auto fetch_p = [&](int ks) {
        p[ks & 1] = *reinterpret_cast<const f16x8_t*>(&p_mine[l32 * kPStride + ks * 16 + 8 * hh]);
      };
      auto fetch = [&](int j) {
        const int at = j % (kAhead + 1);
        if (j < 9) k[at] = *reinterpret_cast<const u32x4_t*>(&k_tile[k_at[j & 1] + (j >> 1) * 64]);
        if (OUTPUT && j < 8) {
          const int ks = j >> 1;
          if ((j & 1) == 0) fetch_p(ks);
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) v[at][odd] = read_tr8(&v_tile[v_at[odd] + (j & 1) * 64 + ks * 16 * kRow]);
        }
      };
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      int again = 0;
      if (OUTPUT) again = outgrown[grp][(t - 1) & 1];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) fetch(j);
      if (OUTPUT) {
        if (__builtin_amdgcn_readfirstlane(again) != 0) {  // (every wave waits for it)
          const float2 now = weigh_again(t - 1);
          lds_barrier();
          if (wg == 0 && hh == 0) *my_row_ref = now;
          fetch_p(0);
        }
        l_run += l_tile;
        // Values with one use each: the first product of a tile then adds to
        // the accumulators in place (the compiler keeps a second set otherwise).
        asm volatile("" : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]));
      }
#pragma unroll
      for (int j = 0; j < 9; ++j) {
        fetch(j + kAhead);
        const int at = j % (kAhead + 1);
        const u32x4_t kj = k[at];
        s = T::mfma32(widen8<T>(kj[0], kj[1]), __builtin_bit_cast(typename T::vec8, q[j][0]), s);
        if (OUTPUT && j < 8)
          o[2 * (j & 1)] = F16::mfma32(widen8<F16>(v[at][0].x, v[at][0].y), p[(j >> 1) & 1], o[2 * (j & 1)]);
        s = T::mfma32(widen8<T>(kj[2], kj[3]), __builtin_bit_cast(typename T::vec8, q[j][1]), s);
        if (OUTPUT && j < 8)
          o[2 * (j & 1) + 1] = F16::mfma32(widen8<F16>(v[at][1].x, v[at][1].y), p[(j >> 1) & 1], o[2 * (j & 1) + 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      // Keys 0-15 of a wave's 32 are finished by the first half of the
      // dims' waves, 16-31 by the second: each hands the other eight over.
#pragma unroll
      for (int e = 0; e < 2; ++e)
        half_s[(wave * 2 + e) * 64 + lane] = make_float4(s[8 + 4 * e], s[9 + 4 * e], s[10 + 4 * e], s[11 + 4 * e]);
    };
    // Phase 2: P of tile t, and (group 1) the loads of tile t + 2 into buffer
    // `to`, spread over it.  Returns whether the other group weighs again in
    // this phase.
    auto softmax = [&](int t, int to, auto with_rows) -> bool {
      constexpr bool ROWS = decltype(with_rows)::value;
      const int other_tile = t + grp - 1;  // weighed last by the other group
      int past = 0;
      if (other_tile >= c0) past = outgrown[grp ^ 1][other_tile & 1];
      Window far{};
      if (!LIST) far = *window_of(t + 3);
      if constexpr (ROWS) {
        float4 other[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) other[e] = half_s[((wave ^ 2) * 2 + e) * 64 + lane];
        Window w[LIST ? 8 : 1];
        fields(t, w);
        if (wg == 0 && lane == 0) outgrown[grp][(t + 1) & 1] = 0;
        TileLoad load;
        load.on = false;
        if (!LIST && grp == 1) load = begin_load(t + 2, to, page_next.row);
        issue_load(load, 0, 3);
        const float lift = my_row_ref->x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float4& x4 = other[e >> 2];
          const float half = (e & 3) == 0 ? x4.x : (e & 3) == 1 ? x4.y : (e & 3) == 2 ? x4.z : x4.w;
          sc[e] = fmaf(s[e] + half, w[LIST ? e : 0].score, w[LIST ? e : 0].log2c - ref);
        }
        if (ragged_tile(t)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool ok = w[LIST ? e : 0].row >= 0 && (LIST || t * kKeys + key_mine + 8 * (e >> 2) + (e & 3) < vis_row);
            sc[e] = ok ? sc[e] : -INFINITY;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        // (A list's rows come when its scale fields have been used: both at
        // once do not fit the registers.)
        if (LIST && grp == 1) load = begin_load(t + 2, to, 0);
        issue_load(load, LIST ? 0 : 3, 6);
        float top = sc[0], top_sum = sc[0] - w[0].log2c, low = w[0].log2c;
#pragma unroll
        for (int e = 1; e < 8; ++e) {
          top = fmaxf(top, sc[e]);
          if (LIST) top_sum = fmaxf(top_sum, sc[e] - w[LIST ? e : 0].log2c);
          if (LIST) low = fminf(low, w[LIST ? e : 0].log2c);
        }
        top = xor32_op(top, MaxOp{});
        if (LIST) top_sum = xor32_op(top_sum, MaxOp{});
        if (hh == 0) {
          row_max[grp][t & 1][l32][wg] = top + ref;
          if (LIST) row_top[LIST ? grp : 0][t & 1][l32][wg] = top_sum + ref;
        }
        float limit = fminf(kMost, kMostSum - 4.f * (lift - low));
        if (LIST) limit = low < kLeast || lift > kMostLift ? -kUnseen : limit;
        const bool past_most = top > limit;
        if (__any(past_most) && lane == 0) outgrown[grp][t & 1] = 1;
        __builtin_amdgcn_sched_barrier(0);
        issue_load(load, 6, kLoads);
        weigh(w, lift, std::false_type{});
      } else {
        if (grp == 1) load_tile(t + 2, to, page_next.row);
      }
      if (!LIST) page_far = scalar(far);
      return __builtin_amdgcn_readfirstlane(past) != 0;
    };
    // Group 0 multiplies tile t in phase 2 (t - c0) and weighs it in the next,
    // group 1 a phase later.  Tile t is in buffer (t - c0) % 3, loaded during
    // the two phases before 2 (t - c0): the last reader of what was there,
    // group 1's product of tile t - 3, ran in phase 2 (t - c0) - 3.
    int buf = 0, before = 2, next = 1;
    auto rotate = [&] {
      page_before = page_now;
      page_now = page_next;
      page_next = page_far;
      before = buf;
      buf = next;
      next = next == 2 ? 0 : next + 1;
    };
    // What every wave does at the start of the phase in which group 0
    // multiplies tile t: with a list, the next window of entries; and, before
    // anyone's output product of tile t - 1, zeros for its NaN codes if some
    // row must not see some key of it (P is zero there, but zero times NaN is
    // not; a row that does see such a key has NaN scores, hence NaN sums).
    auto even_phase = [&](int t) {
      if (LIST && t + 1 < c1 && (t + 1 - w0) % kWindowTiles == 0) {
        window_rows(t + 1);
        window_scales(t + 1);
        __syncthreads();
      }
      if (t > c0 && ragged_tile(t - 1)) {
        for (int c = tid; c < kKeys * kRowChunks; c += kAttnThreads) {
          u32x4_t* v = reinterpret_cast<u32x4_t*>(&keys[before][c * 16]);
          const u32x4_t u = *v;
          *v = u32x4_t{nan_to_zero4(u[0]), nan_to_zero4(u[1]), nan_to_zero4(u[2]), nan_to_zero4(u[3])};
        }
        lds_barrier();
      }
    };
    const std::true_type yes;
    const std::false_type no;
    // The phases of a group (ROWS: it has rows; one without keeps step with
    // the loads and barriers).
    auto phases = [&](auto with_rows) {
      constexpr bool ROWS = decltype(with_rows)::value;
      even_phase(c0);
      if (grp == 1) {
        load_tile(c0 + 1, 1, page_next.row);
        lds_barrier();
      }
      if constexpr (ROWS) multiply(c0, keys[0], keys[0], no);
      if (grp == 1) wait_loads<0>();
      lds_barrier();
      rotate();
      for (int t = c0;; ++t) {
        // Phase 2 of tile t.
        if (grp == 1) even_phase(t + 1);
        const bool past = softmax(t, next, with_rows);
        if (past) lds_barrier();
        lds_barrier();
        // Phase 1 of tile t + 1.  (After the last tile its scores are those of
        // no tile, and nobody reads them: with a second form of the product the
        // compiler keeps a copy of the accumulators, 64 registers that spill.)
        if (grp == 0) even_phase(t + 1);
        if constexpr (ROWS) {
          multiply(t + 1, keys[buf], keys[before], yes);
        }
        if (grp == 1) wait_loads<0>();
        lds_barrier();
        if (t + 1 >= c1) break;
        rotate();
      }
      if (grp == 0) {
        if (__builtin_amdgcn_readfirstlane(outgrown[1][(c1 - 1) & 1]) != 0) lds_barrier();
        lds_barrier();
      }
    };
    for (; c0 < t1; c0 = c1) {
      lds_barrier();  // the tiles before are done with LDS
      if (!LIST) c1 = t1 - (c0 & ~1) < kWindowTiles ? t1 : (c0 & ~1) + kWindowTiles;
      w0 = LIST ? c0 : c0 & ~1;
      if (tid < kRows && c0 == t0) row_ref[tid >> 5][tid & 31] = make_float2(kUnseen, kNoMax);
      window_rows(w0);
      if (tid < 4) outgrown[tid >> 1][tid & 1] = 0;
      lds_barrier();
      buf = 0;
      before = 2;
      next = 1;
      if (grp == 1) load_tile(c0, 0, LIST ? 0 : __builtin_amdgcn_readfirstlane(window_of(c0)->row));
      window_scales(w0);
      wait_loads<0>();
      lds_barrier();
      if (!LIST) {
        page_now = scalar(*window_of(c0));
        page_next = scalar(*window_of(c0 + 1));
        page_far = scalar(*window_of(c0 + 2));
      }
      if (busy)
        phases(yes);
      else
        phases(no);
    }
    lds_barrier();

    // Sum of p of every row: over the lane halves and the group's four waves.
    l_run = xor32_op(l_run, AddOp{});
    if (hh == 0) row_max[grp][0][l32][wg] = l_run;
    lds_barrier();
    float l_all;
    const float2 refs = *my_row_ref;
    {
      const float4 v = *reinterpret_cast<const float4*>(row_max[grp][0][l32]);
      l_all = (v.x + v.y) + (v.z + v.w);
    }
    const bool whole = at == item_start && seg_end == item_end;
    if (whole) {
      uint16_t* out = static_cast<uint16_t*>(a.out);
      if (m_mine < x.count) {
        const int f = x.first + m_mine, i = f / per, h = f - i * per;
        const int64_t row = (r.row0 + i) * a.heads + x.g * per + h;
        const Quotient by(refs.x, l_all);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = wg * 128 + dt * 32 + 8 * e + 4 * hh;
            const uint2 u = make_uint2(T::pack2(by.of(o[dt][4 * e]), by.of(o[dt][4 * e + 1])),
                                       T::pack2(by.of(o[dt][4 * e + 2]), by.of(o[dt][4 * e + 3])));
            *reinterpret_cast<uint2*>(&out[row * kCkvDim + d]) = u;
          }
        if (a.token_weights != nullptr && wg == 0 && hh == 0)
          work.lse[row] = l_all == 0.f ? -INFINITY : refs.y + __builtin_amdgcn_logf(l_all);
      }
      if (a.join_items && tid == 0) work.join[item_base + it].row0 = -1;
    } else {
      const bool first_seg = at == part_start(start.plan, part);
      const int64_t slot = 2 * part + (first_seg ? 0 : 1);
      float4* p = reinterpret_cast<float4*>(work.part) + slot * (kPartFloats / 4);
      const bool empty = t0 >= t1;
      if (!empty && m_mine < x.count) {
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            p[((wave * 4 + dt) * 4 + e) * 64 + lane] =
                make_float4(o[dt][4 * e], o[dt][4 * e + 1], o[dt][4 * e + 2], o[dt][4 * e + 3]);
      }
      if (wg == 0 && hh == 0)
        work.refs[slot * kRows + m_mine] = make_float4(empty ? -INFINITY : (refs.x == kUnseen ? kNoMax : ref),
                                                       empty ? -INFINITY : refs.y, l_all, 0.f);
      // The first border of parts inside an item names it to the joining kernel.
      if (first_seg && at > item_start && tid == 0 && part_start(start.plan, part - 1) <= item_start) {
        JoinEntry j;
        j.row0 = r.row0;
        j.first = x.first;
        j.count = x.count;
        j.g = x.g;
        j.w0 = static_cast<int32_t>(part - 1);
        j.slot0 = static_cast<int32_t>(2 * (part - 1) + (part_start(start.plan, part - 1) == item_start ? 0 : 1));
        j.w1 = static_cast<int32_t>(part_of_end(start.plan, item_end));
        work.join[a.join_items ? item_base + it : part] = j;
      }
    }
    at = seg_end;
  }
}

// Joins the partials of items that lie across parts: block (y, k) takes the k-th
// entry, the y-th 4 of the 128 groups of 64 x 4 values that the accumulators'
// order consists of.  The parts' factors go through LDS first, so that the loads
// of the partials depend on nothing.  Entries belong to items where these are no
// more than the parts, so that few blocks find nothing to do; y counts fastest,
// so that each item's blocks lie on all XCDs.  Bound by the partials' bytes and
// the launch: 24 items over 256 parts, 34 MB, in 9 us (30 with the entries of
// parts, counting fastest).  Where few items have many parts, four groups of
// waves take every fourth part each, and their sums meet in LDS.  us with four
// groups / one:
//
//     items       1          2         4         8        12        16        24        80
//   32,768   11.8/21.6  11.1/20.5  9.2/12.0  9.6/10.4  11.1/8.7  11.9/9.1  14.2/8.7  34.5/11.9
//    8,192    8.2/12.2   6.9/10.0  7.7/10.2   7.8/8.2  10.8/8.1  10.8/8.2  13.0/7.6  31.5/10.6
//    2,048     6.4/8.2    5.4/4.7   5.8/5.1   6.7/6.2  10.6/7.2   9.7/6.6  12.1/6.6   31.1/8.8
constexpr int kJoinGroups = 4;
constexpr int kFewJoins = 8;
constexpr int kJoinBlocks = 32;
constexpr int kJoinParts = 64;  // parts whose factors are held at a time
template <typename T, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS) void latent8_join_kernel(Latent8Args a) {
  constexpr int kSlices = 8 * GROUPS;
  __shared__ float factor[kJoinParts][32];  // of a part and row
  __shared__ float2 row_part[kSlices][32];
  __shared__ float4 sums[GROUPS > 1 ? GROUPS - 1 : 1][256];
  const Work work = carve_work(a.workspace, a.parts);
  const JoinEntry j = work.join[blockIdx.y];
  if (j.row0 < 0) return;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int e = (tid >> 6) & 3, group = tid >> 8;
  // The wave whose accumulators these are, and its tile of dims.
  const int grp = blockIdx.x >> 4, wg = (blockIdx.x >> 2) & 3, dt = blockIdx.x & 3;
  if (grp * 32 >= j.count) return;
  const int n = j.w1 - j.w0 + 1;
  const int per = a.per;
  const int m = tid & 31, s = tid >> 5;  // thread (s, m): parts s, s + kSlices, ... of row m
  auto slot_of = [&](int w) -> int64_t { return w == 0 ? j.slot0 : 2 * static_cast<int64_t>(j.w0 + w); };
  auto refs_of = [&](int w) { return work.refs[slot_of(w) * kRows + grp * 32 + m]; };
  float2 most = make_float2(-INFINITY, -INFINITY);  // references of the sums and of the normaliser
  for (int w = s; w < n; w += kSlices) {
    const float4 v = refs_of(w);
    most = make_float2(fmaxf(most.x, v.x), fmaxf(most.y, v.y));
  }
  row_part[s][m] = most;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSlices; ++k) most = make_float2(fmaxf(most.x, row_part[k][m].x), fmaxf(most.y, row_part[k][m].y));
  float l = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const bool mine = grp * 32 + m < j.count;  // (m == lane & 31; the parts hold no other rows)
  const u32x4_t* parts = reinterpret_cast<const u32x4_t*>(work.part) + (blockIdx.x * 4 + e) * 64 + lane;
  for (int c0 = 0; c0 < n; c0 += kJoinParts) {
    const int c1 = c0 + kJoinParts < n ? c0 + kJoinParts : n;
    __syncthreads();
    for (int w = c0 + s; w < c1; w += kSlices) {
      const float4 v = refs_of(w);
      factor[w - c0][m] = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - most.x);
      if (v.x != -INFINITY) l = fmaf(v.z, __builtin_amdgcn_exp2f(v.y - most.y), l);
    }
    __syncthreads();
#pragma unroll 8
    for (int w = c0 + group; w < c1; w += GROUPS) {
      u32x4_t v{0, 0, 0, 0};
      if (mine) v = parts[slot_of(w) * (kPartFloats / 4)];
      const float f = factor[w - c0][lane & 31];
      // (A part without tiles wrote no sums: its factor is zero, its memory anything.)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = fmaf(f == 0.f ? 0.f : __uint_as_float(v[k]), f, acc[k]);
    }
  }
  row_part[s][m].x = l;
  if (group > 0) sums[group - 1][tid & 255] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (group > 0 || !mine) return;
  l = 0.f;
#pragma unroll
  for (int k = 0; k < kSlices; ++k) l += row_part[k][m].x;
#pragma unroll
  for (int k = 0; k < GROUPS - 1; ++k) {
    const float4 v = sums[k][tid];
    acc[0] += v.x;
    acc[1] += v.y;
    acc[2] += v.z;
    acc[3] += v.w;
  }
  const int f = j.first + grp * 32 + m, i = f / per, h = f - i * per;
  const int64_t row = (j.row0 + i) * a.heads + j.g * per + h;
  if (a.token_weights != nullptr && wg == 0 && dt == 0 && s == 0) work.lse[row] = most.y + __builtin_amdgcn_logf(l);
  const Quotient by(most.x - most.y, l);
  const int d = wg * 128 + dt * 32 + 8 * e + 4 * (lane >> 5);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * kCkvDim + d) =
      make_uint2(T::pack2(by.of(acc[0]), by.of(acc[1])), T::pack2(by.of(acc[2]), by.of(acc[3])));
}

// -------------------------------------------------------- attention weights
// token_weights[slot] += sum over the request's (row, head) pairs of p, from
// the scores once more and the rows' known log-sums.  S^T = K Q^T has keys in
// registers and pairs in lanes, so that the sum over pairs stays in registers.
// A wave takes slices of 32 keys, their codes in its registers; 128 pairs lie
// in LDS, and the waves go through the slices of the workgroup's run without a
// barrier, each next slice loaded into the registers that the last product
// leaves.  Every slot has one owner: no atomics, one order of summation.
//
// Bound by the cache's bytes and the products alike: 24 requests of 8,192
// tokens and 64 heads, 113 MB and 14 GFLOP, in 33 us, of which 13 pass before the
// first product (the part's place 4, the pairs' rows and the first codes 9).
// Parts that lie across requests, which bring other pairs, made it 39; one
// workgroup a page, its codes and 32 pairs at a time in LDS, took 111.
constexpr int kSumThreads = 512;
constexpr int kSumWaves = kSumThreads / 64;
constexpr int kSumPairs = 128;
constexpr int kSumKeys = 32;   // keys of a slice
constexpr int kSumBegin = 12;  // what the pairs of a request cost, in slices
constexpr int kSumRun = 96;    // slices whose sums over the blocks of pairs are held at a time
constexpr int kSumParts = 256; // one workgroup per CU (LDS)
template <typename T>
__global__ __launch_bounds__(kSumThreads, 2) void latent8_weights_kernel(Latent8Args a) {
  __shared__ __align__(16) uint8_t q_tile[kSumPairs * kRow * 2];
  __shared__ float sums[kSumRun * kSumKeys];
  __shared__ float pair_lse[kSumPairs];
  __shared__ int pair_vis[kSumPairs];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hh = lane >> 5;
  const Work work = carve_work(a.workspace, a.parts);
  const int32_t idle = *work.idle;  // (then nobody wrote the log-sums)
  const int per = a.per;
  const int64_t row_bytes = a.latent_heads * kRow;
  auto slices = [](const Request& r) -> int { return r.n > 0 ? (r.len + kSumKeys - 1) / kSumKeys : 0; };
  const Start start = find_start<kSumThreads, kSumBegin, false>(
      a, ends_of(a, tid < a.batch ? tid : 0), blockIdx.x, kSumParts, 0,
      [&](const Request& r) -> int64_t { return slices(r) > 0; }, slices);
  if (idle != 0 || static_cast<int64_t>(blockIdx.x) >= start.plan.parts || start.b < 0) return;
  const int64_t stop = part_start(start.plan, blockIdx.x + 1);
  int64_t b = start.b, base = start.base;
  Request r = start.r;

  // A pair's row in LDS holds chunk c (16 bytes) at place c ^ ((row >> 1) & 7)
  // within its group of eight: 16 rows of one chunk lie in 64 different banks.
  int q_at[2][2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      q_at[odd][half] = l32 * (kRow * 2) + ((4 * odd + 2 * hh + half) ^ ((l32 >> 1) & 7)) * 16;
  const uint32_t q_lds = lds_address(q_tile);
  // Where a lane's share of a slice's sums ends up: see below.
  const int e_mine = l32 >> 1;
  const int key_mine = 8 * (e_mine >> 2) + 4 * hh + (e_mine & 3);

  for (int64_t at = part_start(start.plan, blockIdx.x); at < stop;) {
    int n_units = slices(r) > 0 ? units_of(start.plan, slices(r)) : 0;
    while (at >= base + n_units) {
      base += n_units;
      ++b;
      r = request_of(a, b);
      n_units = slices(r) > 0 ? units_of(start.plan, slices(r)) : 0;
    }
    const int64_t end = base + n_units < stop ? base + n_units : stop;
    const int first_slice = tile_of(start.plan, slices(r), static_cast<int>(at - base));
    const int stop_slice = tile_of(start.plan, slices(r), static_cast<int>(end - base));
    at = end;
    const int64_t entry = a.entries[b];
    if (entry < 0 || entry >= a.pool_rows) continue;
    float* const record = a.token_weights + entry * a.cols * kBlock;
    const int32_t* const table = a.block_table + b * a.cols;
    auto block_of = [&](int slice) { return __builtin_amdgcn_readfirstlane(table[slice >> 2]); };
    const int pairs = r.n * per;
    for (int s0 = first_slice; s0 < stop_slice; s0 += kSumRun) {
      const int s1 = stop_slice < s0 + kSumRun ? stop_slice : s0 + kSumRun;
      auto row_of = [&](int f, int g) -> int64_t {  // of pair f in query, out and lse
        const int64_t row = r.row0 * a.heads + g * per + f;
        return a.latent_heads == 1 ? row : row + (f / per) * (a.heads - per);
      };
      for (int g = 0; g < a.latent_heads; ++g) {
        for (int f0 = 0; f0 < pairs; f0 += kSumPairs) {
          const bool first = g == 0 && f0 == 0, last = g == a.latent_heads - 1 && f0 + kSumPairs >= pairs;
          const int count = pairs - f0 < kSumPairs ? pairs - f0 : kSumPairs;
          const int tiles = count <= 32 ? 1 : (count <= 64 ? 2 : 4);  // of 32 pairs
          const int vis_most = visible(r, (f0 + count - 1) / per), vis_least = visible(r, f0 / per);
          u32x4_t k[18];
          // The codes of a slice: chunks 2 j + hh of the lane's key.
          const uint32_t lane_at = static_cast<uint32_t>(l32 * row_bytes + hh * 16);
          auto slice_at = [&](int slice) -> const uint8_t* {
            const int32_t block = block_of(slice < s1 ? slice : s0);
            const int64_t row =
                static_cast<int64_t>(block < 0 || block >= a.blocks ? 0 : block) * kBlock + (slice & 3) * kSumKeys;
            return static_cast<const uint8_t*>(a.latent_cache) + row * row_bytes + g * kRow;
          };
          __syncthreads();  // (the last block's pairs are done with)
          // The pairs' rows, straight to LDS, 64 places a wave and load, and
          // behind them the first slice's codes.
          const uint8_t* const qn = static_cast<const uint8_t*>(a.query);
          const uint8_t* const qr = static_cast<const uint8_t*>(a.query_rope);
#pragma unroll 1
          for (int q0 = wave * 64; q0 < tiles * 32 * (kRow / 8); q0 += kSumThreads) {
            const int q = q0 + lane;
            const int m = q / (kRow / 8), c = (q - m * (kRow / 8)) ^ ((m >> 1) & 7);
            const int64_t row = row_of(f0 + (m < count ? m : 0), g);
            load_to_lds(c < kCkvDim / 8 ? qn + row * (kCkvDim * 2) + c * 16 : qr + row * (kKpeDim * 2) + c * 16 - kCkvDim * 2,
                        q_lds + q0 * 16);
          }
          {
            const uint8_t* p = slice_at(s0 + wave);
#pragma unroll
            for (int j = 0; j < 18; ++j) k[j] = *reinterpret_cast<const u32x4_t*>(p + lane_at + 32 * j);
          }
          if (tid < kSumPairs) {
            const int f = f0 + (tid < count ? tid : 0);
            pair_vis[tid] = tid < count ? visible(r, f / per) : 0;
            pair_lse[tid] = tid < count ? work.lse[row_of(f, g)] : INFINITY;
          }
          wait_loads<0>();
          lds_barrier();
          for (int slice = s0 + wave; slice < s1; slice += kSumWaves) {
            const int32_t block = block_of(slice);
            const bool known = block >= 0 && block < a.blocks;
            const int slot = slice * kSumKeys + key_mine;
            const bool mine = (l32 & 1) == 0;
            float* const held = &sums[(slice - s0) * kSumKeys + key_mine];
            const float before = !first ? *held : 0.f;
            const float total = last && known && slot < r.len ? record[slot] : 0.f;
            float sum[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[e] = 0.f;
            if (slice * kSumKeys < vis_most) {
              const float c = known ? a.cache_scale[static_cast<int64_t>(block) * a.latent_heads + g] : 1.f;
              const float score = a.scale * kLog2e * fminf(fmaxf(c, kMinScale), FLT_MAX);
              const bool ragged = (slice + 1) * kSumKeys > vis_least;
              const uint8_t* const next = slice_at(slice + kSumWaves);
              // The scores of all tiles of pairs in 36 steps of 16 dims, each
              // step's operands read a step ahead.
              auto add_pairs = [&](auto tiles_n) {
                constexpr int N = decltype(tiles_n)::value;
                f32x16_t s[N];
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                  for (int e = 0; e < 16; ++e) s[n][e] = 0.f;
                u32x4_t q[2][N];
                auto fetch = [&](int j) {
#pragma unroll
                  for (int n = 0; n < N; ++n)
                    q[j & 1][n] = *reinterpret_cast<const u32x4_t*>(
                        &q_tile[n * 32 * kRow * 2 + (j >> 2) * 128 + q_at[(j >> 1) & 1][j & 1]]);
                };
                fetch(0);
#pragma unroll
                for (int j = 0; j < 36; ++j) {
                  if (j < 35) fetch(j + 1);
                  // (Widened here: the compiler would do it ahead for all forms at
                  // once, and spill.)
                  if ((j & 1) == 0) asm volatile("" : "+v"(k[j >> 1]));
                  const auto kj = widen8<T>(k[j >> 1][2 * (j & 1)], k[j >> 1][2 * (j & 1) + 1]);
                  if (j & 1) k[j >> 1] = *reinterpret_cast<const u32x4_t*>(next + lane_at + 16 * (j & ~1));
#pragma unroll
                  for (int n = 0; n < N; ++n)
                    s[n] = T::mfma32(kj, __builtin_bit_cast(typename T::vec8, q[j & 1][n]), s[n]);
                  __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                  const float lse = pair_lse[n * 32 + l32];
                  if (ragged) {
                    const int vis = pair_vis[n * 32 + l32] - slice * kSumKeys - 4 * hh;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                      const float p = __builtin_amdgcn_exp2f(fmaf(s[n][e], score, -lse));
                      sum[e] += 8 * (e >> 2) + (e & 3) < vis ? p : 0.f;
                    }
                  } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum[e] += __builtin_amdgcn_exp2f(fmaf(s[n][e], score, -lse));
                  }
                }
              };
              if (tiles == 1)
                add_pairs(std::integral_constant<int, 1>{});
              else if (tiles == 2)
                add_pairs(std::integral_constant<int, 2>{});
              else
                add_pairs(std::integral_constant<int, 4>{});
              // Over the 32 pairs: a lane keeps half of its values each time and
              // hands its neighbour the others, until it holds value e_mine.
#pragma unroll
              for (int x = 16; x >= 2; x >>= 1) {
                const bool up = (l32 & x) != 0;
#pragma unroll
                for (int e = 0; e < x / 2; ++e) {
                  const float keep = up ? sum[e + x / 2] : sum[e], give = up ? sum[e] : sum[e + x / 2];
                  sum[e] = keep + __shfl_xor(give, x, 64);
                }
              }
              sum[0] += __shfl_xor(sum[0], 1, 64);
            }
            const float now = before + sum[0];
            if (!last) {
              if (mine) *held = now;
            } else if (mine && known && slot < r.len) {
              record[slot] = total + now;
            }
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------ eviction
// Selection: one workgroup per request finds the K-th largest key by three
// digit counts, then lists holes and sources in slot order.  Bound by the
// passes: with the keys in registers (32,768 slots) and lanes that count for
// themselves 1 x 2,176 slots take 10 us, 48 x 8,320 17 us and 16 x 32,768 29 us,
// against 13, 32 and 97 with every pass reading them anew, and 10, 20 and 35
// with lane masks in the one scalar unit of a CU.  About 6 us of it are the
// digits' barriers and scans.  Slots beyond the registers are read anew by every
// pass: 4 x 65,536 take 71 us, 2 x 1,048,576 1.9 ms.
constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kDigitBins = 2048;
constexpr int kHeld = 32;  // keys of a thread in registers: 32,768 slots a request
constexpr int kAhead = 4;  // rounds loaded and walked at a time

// Set bits of a ballot below the lane.
__device__ inline int before_lane(uint64_t ballot) {
  return static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(ballot >> 32),
                                                    __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(ballot), 0u)));
}

// Protected tokens first, then NaN, then by weight; no token has key 0.
__device__ inline uint32_t evict_key(const Latent8EvictArgs& a, float w, int32_t pos, int64_t latest) {
  if (pos < a.protect_first || pos > latest - a.protect_last) return 0xffffffffu;
  return w == w ? float_key(w + 0.f) : 0xfffffffeu;  // (-0 counts as 0)
}

struct SelectLds {
  uint4 bins[kDigitBins];  // four counts a digit, one for every fourth lane
  int scratch[kEvictWaves + 1];
  int wave_latest[kEvictWaves];
  int bin, above;
  int wave_a[kEvictWaves], wave_b[kEvictWaves];
};

__device__ inline void select_slots(const Latent8EvictArgs& a, SelectLds& l, int64_t b, int64_t entry, int len, int keep) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t cap = a.cols * kBlock;
  const float* weights = a.token_weights + entry * cap;
  const int32_t* positions = a.token_positions + entry * cap;
  // Wave w's slots: [w seg, w seg + seg), 64 a round.
  const int seg = static_cast<int>(ceil_div(ceil_div(len, kEvictWaves), 64)) * 64;
  const int s0 = wave * seg, s1 = s0 + seg < len ? s0 + seg : len;
  auto at = [&](int s) { return s < s1 ? s : 0; };  // (slot 0 in the place of one behind the end)
  for (int i = tid; i < kDigitBins; i += kEvictThreads) l.bins[i] = make_uint4(0, 0, 0, 0);
  int latest = INT32_MIN;
  // kHeld rounds of 64 keys stay in registers; what lies beyond is read anew
  // by every pass.
  uint32_t held[kHeld];
  {
    float w[kHeld];
    int32_t p[kHeld];
#pragma unroll
    for (int r = 0; r < kHeld; r += kAhead)
      if (s0 + 64 * r < s1) {
#pragma unroll
        for (int i = r; i < r + kAhead; ++i) {
          w[i] = weights[at(s0 + 64 * i + lane)];
          p[i] = positions[at(s0 + 64 * i + lane)];
        }
      }
#pragma unroll
    for (int r = 0; r < kHeld; r += kAhead)
      if (s0 + 64 * r < s1) {
#pragma unroll
        for (int i = r; i < r + kAhead; ++i) latest = p[i] > latest ? p[i] : latest;
      }
    for (int r0 = s0 + 64 * kHeld; r0 < s1; r0 += 64 * kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int x = positions[at(r0 + 64 * i + lane)];
        latest = x > latest ? x : latest;
      }
    }
    latest = static_cast<int>(wave_reduce_to_lane63(static_cast<uint32_t>(latest) ^ 0x80000000u, MaxU32Op{}) ^ 0x80000000u);
    if (lane == 63) l.wave_latest[wave] = latest;
    __syncthreads();
    latest = l.wave_latest[0];
    for (int k = 1; k < kEvictWaves; ++k) latest = l.wave_latest[k] > latest ? l.wave_latest[k] : latest;
#pragma unroll
    for (int r = 0; r < kHeld; r += kAhead)
      if (s0 + 64 * r < s1) {
#pragma unroll
        for (int i = r; i < r + kAhead; ++i) held[i] = s0 + 64 * i + lane < s1 ? evict_key(a, w[i], p[i], latest) : 0u;
      }
  }
  // f(first slot, key) of every round of 64 slots that the wave owns, and of
  // some behind them; a slot that is not the wave's has key 0.
  auto rounds = [&](auto f) {
#pragma unroll
    for (int r = 0; r < kHeld; r += kAhead)
      if (s0 + 64 * r < s1) {
#pragma unroll
        for (int i = r; i < r + kAhead; ++i) f(s0 + 64 * i, held[i]);
      }
    for (int r0 = s0 + 64 * kHeld; r0 < s1; r0 += 64 * kAhead) {
      float w[kAhead];
      int32_t p[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        w[i] = weights[at(r0 + 64 * i + lane)];
        p[i] = positions[at(r0 + 64 * i + lane)];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        f(r0 + 64 * i, r0 + 64 * i + lane < s1 ? evict_key(a, w[i], p[i], latest) : 0u);
    }
  };

  // The keep-th largest key: digits of 11, 11 and 10 bits from the top.
  uint32_t prefix = 0;
  int want = keep;  // rank among the keys that share the prefix
  int shift = 32;
  for (int round = 0; round < 3; ++round) {
    const int bits = round < 2 ? 11 : 10;
    shift -= bits;
    rounds([&](int, uint32_t k) {
      if (k != 0 && (round == 0 || (k >> (shift + bits)) == prefix))
        atomicAdd(reinterpret_cast<uint32_t*>(&l.bins[(k >> shift) & ((1u << bits) - 1)]) + (lane & 3), 1u);
    });
    __syncthreads();
    // Thread t owns bins top - 2t and top - 2t - 1 (from the largest digit
    // down), and leaves them empty for the next digit.
    const int top = (1 << bits) - 1;
    const int hi = top - 2 * tid, lo = hi - 1;
    auto take = [&](int digit) -> int {
      if (digit < 0) return 0;
      const uint4 v = l.bins[digit];
      l.bins[digit] = make_uint4(0, 0, 0, 0);
      return static_cast<int>(v.x + v.y + v.z + v.w);
    };
    const int c_hi = take(hi), c_lo = take(lo);
    int total;
    const int before = block_exclusive_scan(c_hi + c_lo, l.scratch, &total);
    if (before < want && want <= before + c_hi) {
      l.bin = hi;
      l.above = before;
    } else if (before + c_hi < want && want <= before + c_hi + c_lo) {
      l.bin = lo;
      l.above = before + c_hi;
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<uint32_t>(l.bin);
    want -= l.above;
  }
  const uint32_t threshold = prefix;  // `want` of the keys equal to it are kept, the lower slots first

  // Larger keys and ties of the wave below the budget (low half) and above it,
  // counted by lanes: one scalar unit serves all waves, and masks keep it busy.
  uint32_t larger = 0, ties = 0;
  rounds([&](int r0, uint32_t k) {
    const uint32_t one = r0 + lane < keep ? 1u : 0x10000u;
    larger += k > threshold ? one : 0u;
    ties += k == threshold ? one : 0u;
  });
  auto over_wave = [](uint32_t v) { return static_cast<int>(__builtin_amdgcn_readlane(wave_inclusive_scan(v), 63)); };
  const int larger_below = over_wave(larger & 0xffffu), larger_above = over_wave(larger >> 16);
  const int ties_below = over_wave(ties & 0xffffu), ties_above = over_wave(ties >> 16);
  const int equal = ties_below + ties_above;
  if (lane == 0) l.wave_a[wave] = equal;
  __syncthreads();
  int equal_before = 0;
  for (int w = 0; w < wave; ++w) equal_before += l.wave_a[w];
  __syncthreads();
  const int room = want - equal_before;  // for the wave's ties
  const bool partly = room > 0 && room < equal;
  const int below_all = (s1 < keep ? s1 : keep) - s0;
  int holes = (below_all > 0 ? below_all : 0) - larger_below, sources = larger_above;
  if (room >= equal) {
    holes -= ties_below;
    sources += ties_above;
  }
  // A wave that keeps some of its ties (there is one at most): each(first slot,
  // its holes, its sources) of every round, as lane masks.
  auto walk_ties = [&](auto each) {
    int left = room;
    rounds([&](int r0, uint32_t k) {
      const uint64_t owned = __ballot(k != 0), same = __ballot(k == threshold), below = __ballot(r0 + lane < keep);
      const uint64_t kept = __ballot(k > threshold || (k == threshold && before_lane(same) < left));
      left -= __popcll(same);
      each(r0, owned & below & ~kept, kept & ~below);
    });
  };
  if (partly) {
    holes = sources = 0;
    walk_ties([&](int, uint64_t hole, uint64_t source) {
      holes += __popcll(hole);
      sources += __popcll(source);
    });
  }
  if (lane == 0) {
    l.wave_a[wave] = holes;
    l.wave_b[wave] = sources;
  }
  __syncthreads();
  int hole_at = 0, source_at = 0, count = 0;
  for (int w = 0; w < kEvictWaves; ++w) {
    if (w < wave) {
      hole_at += l.wave_a[w];
      source_at += l.wave_b[w];
    }
    count += l.wave_a[w];
  }
  int32_t* hole_start = a.hole_start + b * (a.cols + 1);
  int32_t* dst = a.move_dst + b * cap;
  int32_t* src = a.move_src + b * cap;
  auto page_start = [&](int r0) {
    if ((r0 & (kBlock - 1)) == 0 && r0 < s1 && lane == 0) hole_start[r0 >> kBlockShift] = hole_at;
  };
  auto list = [&](int32_t* to, int& at_slot, int r0, bool mine) {
    const uint64_t all = __ballot(mine);
    if (mine) to[at_slot + before_lane(all)] = r0 + lane;
    at_slot += __popcll(all);
  };
  if (partly) {
    const uint64_t me = 1ull << lane;
    walk_ties([&](int r0, uint64_t hole, uint64_t source) {
      page_start(r0);
      list(dst, hole_at, r0, (hole & me) != 0);
      list(src, source_at, r0, (source & me) != 0);
    });
  } else {
    const uint32_t last_out = room >= equal ? threshold - 1 : threshold;  // the largest key that goes (0: no token's)
    rounds([&](int r0, uint32_t k) {
      page_start(r0);
      if (r0 < keep) list(dst, hole_at, r0, k - 1u < last_out && r0 + lane < keep);
      if (r0 + 64 > keep) list(src, source_at, r0, k > last_out && r0 + lane >= keep);
    });
  }
  if (tid == 0) {
    a.move_counts[b] = count;
    a.kept_lengths[b] = keep;
  }
  // The page that holds both kept slots and slots beyond the budget may grow
  // its scale while other pages still read rows from it: its scale as it was.
  if ((keep & (kBlock - 1)) != 0 && tid < a.latent_heads) {
    const int32_t block = a.block_table[b * a.cols + (keep >> kBlockShift)];
    a.border_scale[b * a.latent_heads + tid] =
        block >= 0 && block < a.blocks ? a.cache_scale[static_cast<int64_t>(block) * a.latent_heads + tid] : 0.f;
  }
}

__global__ __launch_bounds__(kEvictThreads) void latent8_select_kernel(Latent8EvictArgs a) {
  __shared__ SelectLds l;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t cap = a.cols * kBlock;
  int64_t len64 = a.seq_kv[b];
  const int len = static_cast<int>(len64 < 0 ? 0 : (len64 > cap ? cap : len64));
  const int budget = a.budgets[b] < 0 ? 0 : a.budgets[b];
  const int64_t entry = a.entries[b];
  const bool known = entry >= 0 && entry < a.pool_rows;
  const int keep = known && budget < len ? budget : len;
  if (keep == len || keep == 0) {
    if (tid == 0) {
      a.move_counts[b] = 0;
      a.kept_lengths[b] = keep;
    }
    return;
  }
  select_slots(a, l, b, entry, len, keep);
}

// Moves: one workgroup per (request, page that has holes).  Bound by the bytes
// of the moved rows: 16 x 8,200 rows of 576, read and written once, in 28 us
// (5.4 TB/s, part of it from cache).  With a load and a store in turn it took 51.
// That is without pages that grow their scales, whose other rows are rounded
// again with a load and a store in turn: where 748 of them do, 39 us.
constexpr int kMoveThreads = 256;
constexpr int kMovePages = 256;  // workgroups of a request at most
constexpr int kMoveAhead = 6;  // chunks of a thread in flight
__global__ __launch_bounds__(kMoveThreads) void latent8_move_kernel(Latent8EvictArgs a) {
  __shared__ int64_t from[kBlock];  // cache row of the n-th source, -1: none
  __shared__ int to[kBlock];        // row of the page that it moves to
  __shared__ float factor[kBlock];
  __shared__ uint8_t moved[kBlock];
  __shared__ float wave_top[kMoveThreads / 64];
  const int64_t b = blockIdx.y;
  const int tid = threadIdx.x;
  const int64_t cap = a.cols * kBlock;
  const int keep = a.kept_lengths[b], count = a.move_counts[b];
  if (count <= 0) return;
  const int64_t entry = a.entries[b];
  const int32_t* table = a.block_table + b * a.cols;
  const int32_t* hole_start = a.hole_start + b * (a.cols + 1);
  const int border = (keep & (kBlock - 1)) != 0 ? keep >> kBlockShift : -1;
  const int pages = static_cast<int>(ceil_div(keep, kBlock));
  const int64_t stride = a.latent_heads * kRow;
  uint8_t* const cache = static_cast<uint8_t*>(a.latent_cache);
  for (int page = blockIdx.x; page < pages; page += gridDim.x) {
    const int h0 = hole_start[page], h1 = page + 1 < pages ? hole_start[page + 1] : count;
    const int n = h1 - h0;
    const int32_t block = table[page];
    if (n <= 0) continue;
    const int rows = keep - page * kBlock < kBlock ? keep - page * kBlock : kBlock;
    __syncthreads();
    if (tid < kBlock) moved[tid] = 0;
    __syncthreads();
    int source_page = -1;  // that thread tid's source lies in
    int32_t source_block = -1;
    if (tid < n) {
      const int src = a.move_src[b * cap + h0 + tid];
      const int dst = a.move_dst[b * cap + h0 + tid] - page * kBlock;
      source_page = src >> kBlockShift;
      const int32_t sb = table[source_page];
      if (sb >= 0 && sb < a.blocks) source_block = sb;
      from[tid] = source_block < 0 ? -1 : static_cast<int64_t>(source_block) * kBlock + (src & (kBlock - 1));
      to[tid] = dst;
      moved[dst] = 1;
      float* w = a.token_weights + entry * cap;
      int32_t* p = a.token_positions + entry * cap;
      w[page * kBlock + dst] = w[src];
      p[page * kBlock + dst] = p[src];
    }
    if (block < 0 || block >= a.blocks) continue;
    for (int g = 0; g < a.latent_heads; ++g) {
      float* scale_at = a.cache_scale + static_cast<int64_t>(block) * a.latent_heads + g;
      const float old = *scale_at;
      float mine = 0.f;
      if (source_page == border && source_page >= 0)
        mine = a.border_scale[b * a.latent_heads + g];
      else if (source_block >= 0)
        mine = a.cache_scale[static_cast<int64_t>(source_block) * a.latent_heads + g];
      const float top = wave_all_op(mine, MaxOp{});
      if ((tid & 63) == 0) wave_top[tid >> 6] = top;
      __syncthreads();  // (every thread has read the old scale and is done with the last head's factors)
      float now = old;
      for (int w = 0; w < kMoveThreads / 64; ++w) now = fmaxf(now, wave_top[w]);
      if (tid < n) factor[tid] = mine / now;
      __syncthreads();
      uint8_t* base = cache + static_cast<int64_t>(block) * kBlock * stride + g * kRow;
      if (now != old) {
        const float stay = old / now;
        for (int q = tid; q < rows * kRowChunks; q += kMoveThreads) {
          const int r = q / kRowChunks, c = q - r * kRowChunks;
          if (moved[r]) continue;
          uint4* at = reinterpret_cast<uint4*>(base + r * stride) + c;
          *at = rescale16(*at, stay);
        }
      }
      for (int q0 = tid; q0 < n * kRowChunks; q0 += kMoveAhead * kMoveThreads) {
        uint4 v[kMoveAhead];
#pragma unroll
        for (int i = 0; i < kMoveAhead; ++i) {
          const int q = q0 + i * kMoveThreads < n * kRowChunks ? q0 + i * kMoveThreads : q0;
          const int m = q / kRowChunks, c = q - m * kRowChunks;
          const int64_t row = from[m] < 0 ? 0 : from[m];
          v[i] = *(reinterpret_cast<const uint4*>(cache + row * stride + g * kRow) + c);
        }
#pragma unroll
        for (int i = 0; i < kMoveAhead; ++i) {
          const int q = q0 + i * kMoveThreads;
          if (q >= n * kRowChunks) break;
          const int m = q / kRowChunks, c = q - m * kRowChunks;
          if (from[m] < 0) continue;
          const float f = factor[m];
          *(reinterpret_cast<uint4*>(base + to[m] * stride) + c) = f == 1.f ? v[i] : rescale16(v[i], f);
        }
      }
      if (tid == 0 && now != old) *scale_at = now;
    }
  }
}

}  // namespace

// ------------------------------------------------------------------- launches
hipError_t launch_latent8_append(const Latent8AppendArgs& a, hipStream_t stream) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  // A request of n rows touches at most n pages and at most n / 128 + 2.
  const int64_t pages = std::min(a.rows, a.rows / kBlock + 2 * std::min(a.batch, a.rows));
  const dim3 grid(static_cast<unsigned>(pages), static_cast<unsigned>(a.latent_heads));
  if (a.elem == Elem::kBf16)
    launch_kernel(kKernLatent8Append, latent8_append_kernel<Bf16>, grid, dim3(kAppendThreads), stream, a);
  else
    launch_kernel(kKernLatent8Append, latent8_append_kernel<F16>, grid, dim3(kAppendThreads), stream, a);
  return hipGetLastError();
}

int64_t latent8_items(int64_t rows, int64_t heads, int64_t latent_heads, int64_t batch, bool list) {
  if (latent_heads <= 0) return 0;
  if (list) return rows * ceil_div(heads / latent_heads, kRows) * latent_heads;
  return ceil_div(rows * heads, kRows) + std::min(batch, rows) * latent_heads;
}

size_t latent8_attention_workspace_bytes(int64_t rows, int64_t heads, bool weights) {
  return sizeof(float) * 2 * kParts * (kPartFloats + kRows * 4) + round256(sizeof(JoinEntry) * kParts) +
         round256(sizeof(int32_t)) +
         (weights ? sizeof(float) * rows * heads : 0);
}

template <typename T>
static void attend(const Latent8Args& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.parts));
  if (a.topk != nullptr)
    launch_kernel(kKernLatent8Attention, latent8_attention_kernel<T, true>, grid, dim3(kAttnThreads), stream, a);
  else
    launch_kernel(kKernLatent8Attention, latent8_attention_kernel<T, false>, grid, dim3(kAttnThreads), stream, a);
  const dim3 join(kJoinBlocks, static_cast<unsigned>(a.joins));
  if (a.join_items && a.joins <= kFewJoins)
    launch_kernel(kKernLatent8Join, latent8_join_kernel<T, kJoinGroups>, join, dim3(256 * kJoinGroups), stream, a);
  else
    launch_kernel(kKernLatent8Join, latent8_join_kernel<T, 1>, join, dim3(256), stream, a);
  if (a.token_weights != nullptr)
    launch_kernel(kKernLatent8Weights, latent8_weights_kernel<T>, dim3(kSumParts), dim3(kSumThreads), stream, a);
}

hipError_t launch_latent8_attention(const Latent8Args& args, hipStream_t stream) {
  if (args.rows == 0 || args.batch == 0) return hipSuccess;
  Latent8Args a = args;
  a.parts = kParts;
  a.per = static_cast<int32_t>(a.heads / a.latent_heads);
  const int64_t items = latent8_items(a.rows, a.heads, a.latent_heads, a.batch, a.topk != nullptr);
  a.join_items = items <= kParts;
  a.joins = a.join_items ? items : kParts;
  if (a.elem == Elem::kBf16)
    attend<Bf16>(a, stream);
  else
    attend<F16>(a, stream);
  return hipGetLastError();
}

size_t latent8_evict_workspace_bytes(int64_t batch, int64_t cols, int64_t latent_heads) {
  return round256(sizeof(int32_t) * batch * (cols + 1)) + sizeof(float) * batch * latent_heads;
}

hipError_t launch_latent8_evict(const Latent8EvictArgs& args, hipStream_t stream) {
  if (args.batch == 0) return hipSuccess;
  Latent8EvictArgs a = args;
  a.hole_start = static_cast<int32_t*>(a.workspace);
  a.border_scale = reinterpret_cast<float*>(static_cast<char*>(a.workspace) +
                                            round256(sizeof(int32_t) * a.batch * (a.cols + 1)));
  launch_kernel(kKernLatent8Select, latent8_select_kernel, dim3(static_cast<unsigned>(a.batch)), dim3(kEvictThreads),
                stream, a);
  launch_kernel(kKernLatent8Move, latent8_move_kernel,
                dim3(static_cast<unsigned>(std::min<int64_t>(a.cols, kMovePages)), static_cast<unsigned>(a.batch)),
                dim3(kMoveThreads), stream, a);
  return hipGetLastError();
}

}  // namespace nvdsa
