// norm_rope_append: the new rows of the 16-bit latent cache and the queries
// beside them, between the projections and the attention.
//
//   kv_cache[slot] = kv[t, :512] * rsqrt(mean(kv[t, :512]^2) + eps) * kv_norm_weight
//   k_rope[slot]   = R_t kv[t, 512:]
//   query          = query * rsqrt(mean(query^2) + eps) * query_norm_weight   (per head; with weights only)
//   query_nope     = query[:, :D - 64]                                        (likewise)
//   query_rope     = R_t query[:, D - 64:]
//
// R_t turns pairs: (x0, x1) -> (x0 c0 - x1 s0, x1 c1 + x0 s1).  Everything is
// computed in fp32 and rounded once, at the store.
//
// One pass: a row is held by its lanes, 16 bytes each, from the load over the
// sum of squares (a butterfly of the row's lanes) to the store.  A wave takes a
// cache row, or as many query rows as its lanes hold times kUnroll, whose loads
// are all issued before the first is used.  Bound by the rows' bytes: a prompt of
// 8190 rows whose 64 heads turn 64 dims takes 25.3 us (155 MB, 6.1 TB/s, partly from
// the caches), six prompts of 16 heads of 256 dims, normalised, 42 us with kUnroll 4
// (250 MB, 6.0 TB/s), 45 with 2 and 49 with 8.  A decode step's call, 4.1 us, is bound by its launch.
#include "nvdsa_common.h"
#include "nvdsa_kernels.h"

namespace nvdsa {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / 64;
constexpr int kChunk = 8;                        // values of a lane's 16 bytes
constexpr int kRopeChunks = kKpeDim / kChunk;    // 8
constexpr int kUnroll = 4;

template <typename T>
__device__ inline void unpack8(const u32x4_t& v, float (&x)[kChunk]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[2 * k] = T::to_float(static_cast<uint16_t>(v[k]));
    x[2 * k + 1] = T::to_float(static_cast<uint16_t>(v[k] >> 16));
  }
}
template <typename T>
__device__ inline u32x4_t pack8(const float (&x)[kChunk]) {
  u32x4_t v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = T::pack2(x[2 * k], x[2 * k + 1]);
  return v;
}
__device__ inline float squares(const float (&x)[kChunk]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < kChunk; ++k) s = fmaf(x[k], x[k], s);
  return s;
}
// Sum over the LANES lanes of a row (8 to 64, aligned), in every one of them.
template <int LANES>
__device__ inline float row_sum(float x) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) x += __shfl_xor(x, d);
  return x;
}
template <typename T>
__device__ inline void rotate8(const u32x4_t& cos, const u32x4_t& sin, float (&x)[kChunk]) {
  float c[kChunk], s[kChunk];
  unpack8<T>(cos, c);
  unpack8<T>(sin, s);
#pragma unroll
  for (int k = 0; k < kChunk; k += 2) {
    const float x0 = x[k], x1 = x[k + 1];
    x[k] = x0 * c[k] - x1 * s[k];
    x[k + 1] = x1 * c[k + 1] + x0 * s[k + 1];
  }
}

// The request of packed row t: the first whose end lies behind it.  64 ends at a
// time, after one look at every (B / 64)-th.
__device__ inline int64_t request_of_row(const NormRopeArgs& a, int64_t t) {
  const int lane = threadIdx.x & 63;
  const int64_t step = (a.batch + 63) / 64;
  const int64_t probe = (lane + 1) * step - 1;
  int64_t first = 0;
  if (step > 1) first = step * __popcll(__ballot(probe < a.batch && a.seq_q[probe] <= t));
  int64_t b = first;
  const int64_t stop = step > 1 ? (first + step < a.batch ? first + step : a.batch) : a.batch;
  for (int64_t at = first; at < stop; at += 64) {
    const int64_t i = at + lane;
    const int passed = __popcll(__ballot(i < stop && a.seq_q[i] <= t));
    b += passed;
    if (passed < 64) break;
  }
  return b;
}

template <typename T>
__device__ inline void cache_row(const NormRopeArgs& a, int64_t t) {
  const int lane = threadIdx.x & 63;
  const u32x4_t* row = static_cast<const u32x4_t*>(a.kv) + t * (kQkDim / kChunk);
  const u32x4_t latent = row[lane], weight = static_cast<const u32x4_t*>(a.kv_weight)[lane];
  u32x4_t rope{0, 0, 0, 0}, cos = rope, sin = rope;
  if (lane < kRopeChunks) {
    rope = row[kCkvDim / kChunk + lane];
    cos = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.cos) + t * a.cos_stride + lane * kChunk);
    sin = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.sin) + t * a.cos_stride + lane * kChunk);
  }
  const int64_t b = request_of_row(a, t);
  if (b >= a.batch) return;
  const int64_t end = a.seq_q[b] < a.rows ? a.seq_q[b] : a.rows;   // (as the attention counts a request's rows)
  const int64_t slot = a.seq_kv[b] - (end - t);
  if (slot < 0 || slot >= a.cols * kBlock) return;
  const int32_t page = a.block_table[b * a.cols + (slot >> kBlockShift)];
  if (page < 0 || page >= a.blocks) return;
  const int64_t at = static_cast<int64_t>(page) * kBlock + (slot & (kBlock - 1));
  float x[kChunk], w[kChunk];
  unpack8<T>(latent, x);
  unpack8<T>(weight, w);
  const float r = rsqrtf(row_sum<64>(squares(x)) * (1.f / kCkvDim) + a.eps);
#pragma unroll
  for (int k = 0; k < kChunk; ++k) x[k] = x[k] * r * w[k];
  static_cast<u32x4_t*>(a.kv_cache)[at * (kCkvDim / kChunk) + lane] = pack8<T>(x);
  if (lane < kRopeChunks) {
    unpack8<T>(rope, x);
    rotate8<T>(cos, sin, x);
    static_cast<u32x4_t*>(a.k_rope)[at * kRopeChunks + lane] = pack8<T>(x);
  }
}

// LANES lanes a row of `chunks` chunks, PER of them a lane (chunk lane + i LANES);
// without norms only the rope part's chunks.
template <typename T, int LANES, int PER, bool NORM>
__device__ inline void query_rows(const NormRopeArgs& a, int64_t first, int64_t stop) {
  const int lane = threadIdx.x & 63;
  constexpr int kTogether = 64 / LANES;
  const int in_row = lane & (LANES - 1), which = lane / LANES;
  const int all = static_cast<int>(a.query_dim / kChunk), nope = all - kRopeChunks;
  const int chunks = NORM ? all : kRopeChunks, skip = NORM ? 0 : nope;
  u32x4_t v[kUnroll][PER], cos[kUnroll][PER], sin[kUnroll][PER];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t r = first + u * kTogether + which;
    const int64_t t = r / a.heads;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = in_row + i * LANES;
      v[u][i] = cos[u][i] = sin[u][i] = u32x4_t{0, 0, 0, 0};
      if (r < stop && c < chunks) {
        v[u][i] = static_cast<const u32x4_t*>(a.query)[r * all + skip + c];
        const int turn = c + skip - nope;
        if (turn >= 0) {
          cos[u][i] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.cos) + t * a.cos_stride + turn * kChunk);
          sin[u][i] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.sin) + t * a.cos_stride + turn * kChunk);
        }
      }
    }
  }
  float w[PER][kChunk];
  if (NORM) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = in_row + i * LANES;
      u32x4_t g{0, 0, 0, 0};
      if (c < chunks) g = static_cast<const u32x4_t*>(a.query_weight)[c];
      unpack8<T>(g, w[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t r = first + u * kTogether + which;
    float x[PER][kChunk], sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      unpack8<T>(v[u][i], x[i]);
      if (NORM) sum += squares(x[i]);
    }
    if (NORM) {
      const float scale = rsqrtf(row_sum<LANES>(sum) / static_cast<float>(a.query_dim) + a.eps);
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < kChunk; ++k) x[i][k] = x[i][k] * scale * w[i][k];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = in_row + i * LANES, turn = c + skip - nope;
      if (r >= stop || c >= chunks) continue;
      if (turn >= 0) {
        rotate8<T>(cos[u][i], sin[u][i], x[i]);
        static_cast<u32x4_t*>(a.query_rope)[r * kRopeChunks + turn] = pack8<T>(x[i]);
      } else {
        static_cast<u32x4_t*>(a.query_nope)[r * nope + c] = pack8<T>(x[i]);
      }
    }
  }
}

// Waves of the launch: a.rows take a cache row each, the others the query rows.
template <typename T, int LANES, int PER, bool NORM>
__global__ __launch_bounds__(kNormThreads) void norm_rope_kernel(NormRopeArgs a) {
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * kNormWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave < a.rows) {
    cache_row<T>(a, wave);
    return;
  }
  constexpr int64_t kRowsOfWave = 64 / LANES * kUnroll;
  const int64_t first = (wave - a.rows) * kRowsOfWave;
  // (Rows behind the last request are left as they were.)
  int64_t stop = a.seq_q[a.batch - 1];
  stop = (stop < 0 ? 0 : (stop > a.rows ? a.rows : stop)) * a.heads;
  if (first < stop) query_rows<T, LANES, PER, NORM>(a, first, stop);
}

template <typename T, int LANES, int PER, bool NORM>
hipError_t launch(const NormRopeArgs& a, hipStream_t stream) {
  constexpr int64_t kRowsOfWave = 64 / LANES * kUnroll;
  const int64_t waves = a.rows + ceil_div(a.rows * a.heads, kRowsOfWave);
  launch_kernel(kKernNormRope, norm_rope_kernel<T, LANES, PER, NORM>, dim3(static_cast<uint32_t>(ceil_div(waves, kNormWaves))),
                dim3(kNormThreads), stream, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_for(const NormRopeArgs& a, hipStream_t stream) {
  if (a.query_weight == nullptr) return launch<T, kRopeChunks, 1, false>(a, stream);
  const int64_t chunks = a.query_dim / kChunk;
  if (chunks <= 8) return launch<T, 8, 1, true>(a, stream);
  if (chunks <= 16) return launch<T, 16, 1, true>(a, stream);
  if (chunks <= 32) return launch<T, 32, 1, true>(a, stream);
  if (chunks <= 64) return launch<T, 64, 1, true>(a, stream);
  return launch<T, 64, 2, true>(a, stream);
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t stream) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  return a.elem == Elem::kBf16 ? launch_for<Bf16>(a, stream) : launch_for<F16>(a, stream);
}

}  // namespace nvdsa
