// Causal attention over a sliding window and the first keys (lm_ops.cuh),
// forward and backward.
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "lm_ops.cuh"
#include "tcgen05.cuh"

namespace tysor {
namespace {

void check_launch() {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  TYSOR_CUDA(cudaGetLastError());
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kTile = 128;  // rows of a tile
__host__ __device__ inline int tiles_of(int rows) { return (rows + kTile - 1) / kTile; }

// First value of row `r` of head `h` of sequence `b`.
__device__ __forceinline__ int64_t row_at(const AttentionShape& s, int b, int h, int r, int heads, int len) {
  return (s.seq_major ? ((int64_t)b * len + r) * heads + h : ((int64_t)b * heads + h) * len + r) * s.head_dim;
}

// A sequence's keys [0, n) and its first query's position, both whole numbers.
struct __align__(8) Sequence {
  int start, n;
};

__device__ __forceinline__ Sequence sequence_of(const AttentionShape& s, int b, int* err) {
  Sequence q{s.k_len - s.q_len, s.k_len};
  if (s.lengths != nullptr) {
    const float v = s.lengths[b];
    const int n = (int)fminf(v, 536870912.0f);  // NaN: that; k_len is at most that
    if (v >= 0.0f && n <= s.k_len && (float)n == v) {
      q.n = n;
    } else {
      q.n = 0;
      atomicCAS(err, 0, (int)kErrSequence);
    }
  }
  if (s.starts != nullptr) {
    const float v = s.starts[b];
    const int start = (int)v;  // out of range: the end of it
    if (fabsf(v) < 536870912.0f && (float)start == v) {  // positions stay below 2^30
      q.start = start;
    } else {
      q.n = 0;
      q.start = 0;
      atomicCAS(err, 0, (int)kErrSequence);
    }
  }
  return q;
}

// The keys a query at position p sees: [0, first) and [low, high).
struct Seen {
  int first, low, high;
};

__device__ __forceinline__ Seen seen_by(const AttentionShape& s, const Sequence& q, int p) {
  if (p < 0 || p >= q.n) return {0, 0, 0};
  Seen v{0, 0, p + 1};
  if (s.window > 0 && p + 1 > s.window) {
    v.low = p + 1 - s.window;
    v.first = min(s.sinks, v.low);
  }
  return v;
}

// Whether the row at position p sees one key, and so a score without a gradient: its
// probability is 1 (NaN if the score is).  (dP and delta, formed in different orders,
// would leave the rounding of their terms.)
__device__ __forceinline__ bool sees_one(const AttentionShape& s, int p) {
  return p == 0 || (s.window == 1 && s.sinks == 0);
}

// ---- every value: one warp per row -------------------------------------------------

// What is not finite would spoil the hidden places of a matrix product (0 times
// it is not 0), so rows and keys that meet such values go one by one, taking in
// only what they see; so do those that see nothing, and those whose scores may be
// so large that a gradient has to form them as the softmax did, bit for bit, for
// its probabilities to be any (kFarScore).

// A row's values over a warp's lanes: lane l holds columns l, l + 32, ...
constexpr int kLaneDims = kMaxHeadDim / 32;

__device__ __forceinline__ void lane_load(const float* __restrict__ p, int dim, float (&v)[kLaneDims]) {
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) {
    const int c = (threadIdx.x & 31) + 32 * i;
    v[i] = c < dim ? p[c] : 0.0f;
  }
}

__device__ __forceinline__ void lane_store(float* __restrict__ p, int dim, const float (&v)[kLaneDims],
                                           int accumulate) {
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) {
    const int c = (threadIdx.x & 31) + 32 * i;
    if (c < dim) p[c] = accumulate ? p[c] + v[i] : v[i];
  }
}

__device__ __forceinline__ float lane_dot(const float (&a)[kLaneDims], const float (&b)[kLaneDims]) {
  float d = 0.0f;
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) d += a[i] * b[i];
  return warp_sum(d);
}

// A score, rounded (a multiplication and subtraction in one would not be).
__device__ __forceinline__ float lane_score(const AttentionShape& s, const float (&q)[kLaneDims],
                                            const float (&k)[kLaneDims]) {
  return __fmul_rn(lane_dot(q, k), s.scale);
}

// The greatest score and the sum of exp(score - greatest) with one more score.
__device__ __forceinline__ float2 with_score(float2 st, float x) {
  const float top = x > st.x || x != x ? x : st.x;
  const float keep = st.x == top ? 1.0f : expf(st.x - top);
  return make_float2(top, st.y * keep + (x == top && x == -INFINITY ? 0.0f : expf(x - top)));
}

__device__ void simple_forward_row(const AttentionShape& s, const Sequence& sq, const float* q, const float* k,
                                   const float* v, float* out, float* stats, int b, int h, int r) {
  const int g = h / (s.heads / s.kv_heads);
  const Seen seen = seen_by(s, sq, sq.start + r);
  float qv[kLaneDims] = {}, acc[kLaneDims] = {};
  if (seen.high > 0) lane_load(q + row_at(s, b, h, r, s.heads, s.q_len), s.head_dim, qv);
  float m = -INFINITY, l = 0.0f;
#pragma unroll 1
  for (int j = 0; j < seen.high; ++j) {
    if (j == seen.first && j < seen.low) j = seen.low;
    float kv[kLaneDims];
    lane_load(k + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
    const float x = lane_score(s, qv, kv);
    const float top = x > m || x != x ? x : m;
    const float keep = m == top ? 1.0f : expf(m - top);
    const float p = x == top && x == -INFINITY ? 0.0f : expf(x - top);
    lane_load(v + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
    // acc stays a mean, so that values near fp32's greatest do not overflow.
    l = l * keep + p;
    const float take = l == 0.0f ? p : p / l;
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) acc[i] = acc[i] * (1.0f - take) + take * kv[i];
    m = top;
  }
  lane_store(out + row_at(s, b, h, r, s.heads, s.q_len), s.head_dim, acc, 0);
  if (stats != nullptr && (threadIdx.x & 31) == 0)
    *(float2*)(stats + 2 * (((int64_t)b * s.heads + h) * s.q_len + r)) = make_float2(m, l);
}

// Leaves the row's greatest score and sum at `own`: those of the scores as formed
// here and in simple_dkv_row, which the forward's may have formed in another order.
__device__ void simple_dq_row(const AttentionShape& s, const Sequence& sq, const float* q, const float* k,
                              const float* v, const float* out, const float* dout, float* dq, float2* own,
                              int accumulate, int b, int h, int r) {
  const int g = h / (s.heads / s.kv_heads);
  const Seen seen = seen_by(s, sq, sq.start + r);
  const int64_t at = row_at(s, b, h, r, s.heads, s.q_len);
  float qv[kLaneDims], gv[kLaneDims], kv[kLaneDims], vv[kLaneDims], acc[kLaneDims] = {};
  if (seen.high == 0) {
    if (!accumulate) lane_store(dq + at, s.head_dim, acc, 0);
    return;
  }
  lane_load(out + at, s.head_dim, kv);
  lane_load(dout + at, s.head_dim, gv);
  lane_load(q + at, s.head_dim, qv);
  const float delta = lane_dot(kv, gv);
  float2 st = make_float2(-INFINITY, 0.0f);
#pragma unroll 1
  for (int j = 0; j < seen.high; ++j) {
    if (j == seen.first && j < seen.low) j = seen.low;
    lane_load(k + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
    st = with_score(st, lane_score(s, qv, kv));
  }
  if ((threadIdx.x & 31) == 0) *own = st;
#pragma unroll 1
  for (int j = 0; j < seen.high; ++j) {
    if (j == seen.first && j < seen.low) j = seen.low;
    lane_load(k + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
    lane_load(v + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, vv);
    const float p = expf(lane_score(s, qv, kv) - st.x) / st.y;
    const float ds = p * (sees_one(s, sq.start + r) ? 0.0f : lane_dot(gv, vv) - delta);
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) acc[i] += ds * (kv[i] * s.scale);  // see `down` in grad_kernel
  }
  lane_store(dq + at, s.head_dim, acc, accumulate);
}

// The query rows that see key j: those at positions [j, end).
__device__ __forceinline__ void rows_seeing(const AttentionShape& s, const Sequence& sq, int j, int* r0, int* r1) {
  int end = sq.n;
  if (s.window > 0 && j >= s.sinks && end - j > s.window) end = j + s.window;
  *r0 = min(max(j - sq.start, 0), s.q_len);
  *r1 = j >= sq.n ? *r0 : min(max(end - sq.start, 0), s.q_len);
}

__device__ void simple_dkv_row(const AttentionShape& s, const Sequence& sq, const float* q, const float* k,
                               const float* v, const float* out, const float2* stats, const float* dout, float* dk,
                               float* dv, int accumulate_k, int accumulate_v, int b, int g, int j) {
  const int group = s.heads / s.kv_heads;
  const int64_t at = row_at(s, b, g, j, s.kv_heads, s.k_len);
  float kv[kLaneDims], vv[kLaneDims], ak[kLaneDims] = {}, av[kLaneDims] = {};
  int r0, r1;
  rows_seeing(s, sq, j, &r0, &r1);
  if (r0 >= r1 && accumulate_k && accumulate_v) return;
  if (r0 < r1) {
    lane_load(k + at, s.head_dim, kv);
    lane_load(v + at, s.head_dim, vv);
    for (int h = g * group; h < (g + 1) * group; ++h)
#pragma unroll 1
      for (int r = r0; r < r1; ++r) {
        const int64_t row = row_at(s, b, h, r, s.heads, s.q_len);
        float qv[kLaneDims], gv[kLaneDims], ov[kLaneDims];
        lane_load(q + row, s.head_dim, qv);
        lane_load(dout + row, s.head_dim, gv);
        lane_load(out + row, s.head_dim, ov);
        const float2 st = stats[((int64_t)b * s.heads + h) * tiles_of(s.q_len) * kTile + r];
        const float p = expf(lane_score(s, qv, kv) - st.x) / st.y;
        const float ds = p * (sees_one(s, sq.start + r) ? 0.0f : lane_dot(gv, vv) - lane_dot(gv, ov));
#pragma unroll
        for (int i = 0; i < kLaneDims; ++i) {
          av[i] += p * gv[i];
          ak[i] += ds * (qv[i] * s.scale);
        }
      }
  }
  lane_store(dk + at, s.head_dim, ak, accumulate_k);
  lane_store(dv + at, s.head_dim, av, accumulate_v);
}

// ---- operands of the tensor-core kernels ---------------------------------------------

// fp32 accuracy out of fp16 matrix instructions: an operand is multiplied by a
// power of two that brings its tile's largest magnitude into [2^14, 2^15) and
// split into hi = fp16(x) and lo = fp16(x - hi), 22 bits together; a product
// is lo.hi + hi.lo + hi.hi, its factors' powers of two undone afterwards.  The
// lowest bit of lo stands for 2^-39 of the tile's largest value, so a row much
// smaller than its neighbours loses bits only where they hardly count.
//
// A packed tile holds 128 rows (queries or keys) of one head, `DP` columns
// (head_dim rounded up to 64 or 128, zeros behind it): [hi | lo][DP / 64] boxes
// of 128 rows x 64 columns, each row 128 bytes, its 16-byte pieces exchanged
// as the matrix unit's 128-byte swizzle wants them.  A copy of whole boxes, or
// of 64 of their rows, is then one untiled bulk copy, and the same box serves
// as an operand summed over its columns (scores) or over its rows (values).
//
// Packing reads 4 bytes a value and writes 4, and HBM bounds it: a forward's q, k
// and v, 201 MB both ways, 34 us = 5.9 TB/s; a gradient's operands with the output
// and the rows' statistics, 403 MB, 88 us = 4.6 TB/s (8192 tokens, 16 heads over 4,
// 128 wide).  Splitting keys and values inside the attention kernels instead would do
// it once per query tile that reads a key tile; a query tile is read by one item (or
// a few segments of it), and its packing is a trip through memory that the forward
// could do without.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kBox = kTile * 128;  // bytes
constexpr uint32_t kLayoutSW128 = 2;

template <int DP>
constexpr int kTileBytes = 2 * (DP / 64) * kBox;

// Row and key tiles whose scores may reach this many powers of two (by their norms)
// go key by key: a tile's score is off by up to 28 steps of 2^-23 of them (measured,
// 2^-22), and a gradient forms it again in another order, so that beside a row's
// greatest score a probability of 1 comes out as 2^(2^-6) here, and as infinity
// in fp16 from 2^19 on.
constexpr float kFarScore = 65536.0f;

// One operand to pack: `heads` heads of `len` rows; rows are keys (valid below
// the sequence's n) or queries (valid where they stand in the sequence).
struct PackJob {
  const float* x;
  uint8_t* tiles;   // [batch][heads][tiles_of(len)] packed tiles
  float* factors;   // the power of two that undoes each tile's scale; NaN: not for the matrix unit (far_exponent)
  int heads, len, queries;
  // Null where not wanted: the tile's greatest 2-norm of a row (queries and keys, for
  // what their scores may come to: at least that, and NaN where the factor is).  For
  // the gradients, rows counted in whole tiles: the rows' norms as well; or, with
  // the output and statistics (x is the output's gradient), each row's (greatest score in powers
  // of two, 1 / sum or 0 for a row that sees one key, delta = sum of x * out, norm),
  // zeros for rows that see nothing, and each tile's greatest |delta| (NaN if a row's values are not finite).
  // Norms and deltas of the output's gradient are in its tile's units, as the packed
  // values are: however small it is, dP and delta are then of ordinary size.
  float *tile_norm, *norm;
  const float *out, *stats;
  float4* info;
  float2* own;  // the statistics as they are
  float2* col;  // (greatest score + log2 of the sum - 14, delta); a row that sees nothing: a score no exponent reaches
  float* tile_delta;
};
// Tiles with values of 2^100 or more, or that are not finite, go key by key: sums
// of such values times probabilities of up to 2^14 would leave fp32, from 2^13 keys
// on (which is where a sum of them reaches 2^128) those of fewer powers too.
constexpr int kFarExponent = 100;
inline int far_exponent(int keys) {
  int powers = 0;
  while (powers < 30 && 1 << powers < keys) ++powers;
  return std::min(kFarExponent, kFarExponent + 13 - powers);
}
struct PackJobs {
  AttentionShape s;
  PackJob job[4];
  int first[5];  // first block of each job
  int far;       // far_exponent of the call
  Sequence* seqs;  // [batch] of the call, for the kernels after this one
};

template <int DP>
__global__ void __launch_bounds__(256) pack_kernel(PackJobs p, int* err) {
  constexpr int kChunks = DP / 8;                  // 8-column pieces of a row
  constexpr int kPer = kTile * kChunks / 256;      // pieces a thread holds
  __shared__ uint32_t warp_max[8];
  int which = 0;
#pragma unroll
  for (int i = 1; i < 4; ++i) which += (int)blockIdx.x >= p.first[i];
  const PackJob& j = p.job[which];
  const AttentionShape& s = p.s;
  const int tiles = tiles_of(j.len);
  const int index = (int)blockIdx.x - p.first[which];
  const int t = index % tiles, h = index / tiles % j.heads, b = index / tiles / j.heads;
  const Sequence sq = sequence_of(s, b, err);
  if (t == 0 && h == 0 && threadIdx.x == 0) p.seqs[b] = sq;
  // Valid rows of the whole operand: [v0, v1).
  int v0 = 0, v1 = sq.n;
  if (j.queries) v0 = -sq.start, v1 = sq.n - sq.start;
  const int r0 = max(t * kTile, v0), r1 = min(min(j.len, (t + 1) * kTile), v1);
  if (r0 >= r1) {  // nothing reads this tile's values
    if (threadIdx.x == 0) {
      j.factors[index] = 1.0f;
      if (j.tile_norm != nullptr) j.tile_norm[index] = 0.0f;
      if (j.tile_delta != nullptr) j.tile_delta[index] = 0.0f;
    }
    if (j.info != nullptr && threadIdx.x < kTile) {
      j.info[(int64_t)index * kTile + threadIdx.x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      j.own[(int64_t)index * kTile + threadIdx.x] = make_float2(0.0f, 0.0f);
      j.col[(int64_t)index * kTile + threadIdx.x] = make_float2(1e30f, 0.0f);
    }
    if (j.norm != nullptr && threadIdx.x < kTile) j.norm[(int64_t)index * kTile + threadIdx.x] = 0.0f;
    return;
  }
  const bool vec = s.head_dim % 4 == 0 && (((uintptr_t)j.x | (uintptr_t)j.out) & 15) == 0;
  // All of a thread's loads come first, so that their latencies overlap.
  __shared__ float2 row_stats[kTile];
  if (j.out != nullptr && threadIdx.x < kTile) {
    const int row = t * kTile + threadIdx.x;
    row_stats[threadIdx.x] = row >= r0 && row < r1
                                 ? *(const float2*)(j.stats + 2 * (((int64_t)b * j.heads + h) * j.len + row))
                                 : make_float2(0.0f, 0.0f);
  }
  float v[kPer][8], dot[kPer];  // dot: of the piece with the output's
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int item = threadIdx.x + 256 * i;
    const int r = t * kTile + item / kChunks, c = item % kChunks * 8;
    const int64_t from = row_at(s, b, h, r, j.heads, j.len) + c;
    const float* src = j.x + from;
    const bool live = r >= r0 && r < r1;
    if (vec) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 f = live && c + e < s.head_dim ? *(const float4*)(src + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[i][e] = f.x, v[i][e + 1] = f.y, v[i][e + 2] = f.z, v[i][e + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = live && c + e < s.head_dim ? src[e] : 0.0f;
    }
    dot[i] = 0.0f;
    if (j.out != nullptr) {
      const float* o = j.out + from;
      if (vec) {
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          if (live && c + e < s.head_dim) {
            const float4 f = *(const float4*)(o + e);
            dot[i] += v[i][e] * f.x, dot[i] += v[i][e + 1] * f.y;
            dot[i] += v[i][e + 2] * f.z, dot[i] += v[i][e + 3] * f.w;
          }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (live && c + e < s.head_dim) dot[i] += v[i][e] * o[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, warp_max[w]);
  const int exponent = (int)(top >> 23) - 127;  // of the largest magnitude; 128: not finite
  const int up = top == 0 ? 0 : min(14 - exponent, 126);
  const float scale = __uint_as_float((uint32_t)(up + 127) << 23);
  const float factor = exponent >= p.far ? NAN : __uint_as_float((uint32_t)(127 - up) << 23);
  // Of queries and keys a bound does unless it, with another tile like this one, comes
  // near kFarScore: the norms take a sixth of the kernel's time, and few tiles need them.
  const float bound = exponent >= p.far ? NAN : __uint_as_float((uint32_t)max(exponent + 128, 1) << 23) * sqrtf((float)s.head_dim);
  const bool for_scores = j.norm == nullptr && j.out == nullptr;
  const bool norms = j.tile_norm != nullptr && !(for_scores && bound * s.scale * bound * kLog2e < kFarScore / 16.0f);
  if (threadIdx.x == 0) {
    j.factors[index] = factor;
    if (!norms && j.tile_norm != nullptr) j.tile_norm[index] = bound;
  }
  uint8_t* dst = j.tiles + (int64_t)index * kTileBytes<DP>;
  float most_norm = 0.0f;
  uint32_t most_delta = 0;  // as bits: NaN is the greatest
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int item = threadIdx.x + 256 * i;
    const int r = item / kChunks, chunk = item % kChunks;
    if (norms) {
      const float back = j.out != nullptr ? 1.0f : __uint_as_float((uint32_t)(127 - up) << 23);
      float q = 0.0f, d = dot[i] * scale;
#pragma unroll
      for (int e = 0; e < 8; ++e) q += v[i][e] * scale * (v[i][e] * scale);
#pragma unroll
      for (int w = kChunks / 2; w > 0; w >>= 1) {
        q += __shfl_xor_sync(0xffffffffu, q, w);
        d += __shfl_xor_sync(0xffffffffu, d, w);
      }
      q = sqrtf(q) * back;
      most_norm = fmaxf(most_norm, q);
      if (chunk == 0) {
        if (j.norm != nullptr) j.norm[(int64_t)index * kTile + r] = q;
        if (j.info != nullptr) {
          const float2 st = row_stats[r];
          j.own[(int64_t)index * kTile + r] = st;
          const float4 f =
              st.y == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                           : make_float4(st.x * kLog2e, sees_one(s, sq.start + t * kTile + r) ? 0.0f : 1.0f / st.y, d, q);
          j.info[(int64_t)index * kTile + r] = f;
          j.col[(int64_t)index * kTile + r] =
              st.y == 0.0f ? make_float2(1e30f, 0.0f) : make_float2(f.x + (log2f(st.y) - 14.0f), d);
          const float all = f.x * 0.0f + f.y * 0.0f + f.z * 0.0f;  // 0, or NaN if one is not finite
          most_delta = max(most_delta, __float_as_uint(fabsf(f.z) + all) & 0x7fffffffu);
        }
      }
    }
    uint4 hi, lo;
    uint32_t* hw = &hi.x;
    uint32_t* lw = &lo.x;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float a = v[i][e] * scale, c = v[i][e + 1] * scale;
      const __half2 h2 = __floats2half2_rn(a, c);
      const float2 back = __half22float2(h2);
      const __half2 l2 = __floats2half2_rn(a - back.x, c - back.y);
      hw[e / 2] = *(const uint32_t*)&h2;
      lw[e / 2] = *(const uint32_t*)&l2;
    }
    uint8_t* at = dst + (chunk / 8) * kBox + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
    *(uint4*)at = hi;
    *(uint4*)(at + (DP / 64) * kBox) = lo;
  }
  if (!norms) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    most_norm = fmaxf(most_norm, __shfl_xor_sync(0xffffffffu, most_norm, o));
    most_delta = max(most_delta, __shfl_xor_sync(0xffffffffu, most_delta, o));
  }
  __shared__ uint32_t tops[2][8];  // both as bits of numbers that are not negative
  if ((threadIdx.x & 31) == 0) tops[0][threadIdx.x >> 5] = __float_as_uint(most_norm), tops[1][threadIdx.x >> 5] = most_delta;
  __syncthreads();
  if (threadIdx.x < 2 && (threadIdx.x == 0 || j.tile_delta != nullptr)) {
    uint32_t m = 0;
    for (int w = 0; w < 8; ++w) m = max(m, tops[threadIdx.x][w]);
    (threadIdx.x == 0 ? j.tile_norm : j.tile_delta)[index] = __uint_as_float(m) + (for_scores ? 0.0f * factor : 0.0f);
  }
}

// ---- pieces of the tensor-core kernels ---------------------------------------------------

__device__ __forceinline__ void bulk_load(uint32_t dst, const uint8_t* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// A bounded wait whose outcome a whole warp shares.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// One lane of a converged warp.  The issuing warps run their loops with all
// lanes and issue from this one: addresses and descriptors then stay in the
// warp's uniform registers, which the matrix instructions take them from.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(yes));
  return yes != 0;
}

// D (+)= A . B over 16 terms, fp16 operands, fp32 accumulator; A (a row per
// lane, two terms per column) and D in tensor memory, B in shared memory.  B's
// descriptor comes as its low word (see column_word and row_word): the high one
// is the same for all, and the words of an operand's steps lie constants apart.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (kLayoutSW128 << 29);  // 1024 bytes between 8-row groups
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "n"(kDescHigh), "r"(idesc), "r"(add));
}
// fp16 x fp16 -> fp32, M = 128; `b_rows`: B is summed over its rows.
__host__ __device__ constexpr uint32_t umma_idesc(int n, bool b_rows) {
  return (1u << 4) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// A box as an operand summed over its columns: 16 columns are 32 bytes.
constexpr uint32_t kColumnStep = 32 >> 4;
__device__ __forceinline__ uint32_t column_word(uint32_t box) { return box >> 4 | 1u << 16; }
// Boxes `stride` bytes apart as an operand summed over their rows: 16 rows are 2048 bytes.
constexpr uint32_t kRowStep = 2048 >> 4;
__device__ __forceinline__ uint32_t row_word(uint32_t box, uint32_t stride) { return box >> 4 | stride >> 4 << 16; }

// A load and the wait for it in one statement: nothing reads the registers in between.
__device__ __forceinline__ void tmem_ld8(uint32_t at, float (&v)[8]) {
  uint32_t r[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(at)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld64(uint32_t at, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(at), "r"(at + 32)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]));
}

// 2^x to about 2^-22, subnormal results as 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Stores 16 neighbouring values as an A operand's 16 columns: 8 with hi (two
// values each), 8 with lo.  Step by step over all of them, here and in the
// kernels: value by value, the chain of dependent instructions takes 40 cycles
// each.
__device__ __forceinline__ void store_split16(uint32_t at, const float* v) {
  uint32_t r[16];
  float rest[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 x = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    r[i] = *(const uint32_t*)&x;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 back = __half22float2(*(const __half2*)&r[i]);
    rest[2 * i] = v[2 * i] - back.x;
    rest[2 * i + 1] = v[2 * i + 1] - back.y;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 y = __floats2half2_rn(rest[2 * i], rest[2 * i + 1]);
    r[8 + i] = *(const uint32_t*)&y;
  }
  tmem_st16(at, r);
}
// Columns of such an operand per 16 terms, and from their hi to their lo part.
constexpr uint32_t kSplitStep = 16, kSplitLo = 8;

// A resident packed tile from shared memory into tensor memory, where it is the
// A operand of every score product: one read instead of one per instruction
// (measured for 128 x 64 x 16 with both operands in shared memory 90 cycles an
// instruction, with A here 41 to 60; 32 would be the products').  Row r is lane r; its hi
// columns are DP / 2 columns of tensor memory, its lo columns the DP / 2 after
// them.  Called by the eight score warps; `half` is the warp's.
template <int DP>
__device__ __forceinline__ void rows_to_tmem(uint32_t tmem_rows, uint32_t tile, int row, int half) {
#pragma unroll
  for (int u = 0; u < DP / 64; ++u) {
    const int unit = 2 * u + half;  // box of the tile: [hi | lo][DP / 64]
    uint32_t r[32];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r[4 * c]), "=r"(r[4 * c + 1]), "=r"(r[4 * c + 2]), "=r"(r[4 * c + 3])
                   : "r"(tile + unit * kBox + row * 128 + ((c ^ (row & 7)) << 4)));
    tmem_st32(tmem_rows + unit * 32, r);
  }
}

// Bits e with lo <= first + e < hi.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi, int first) {
  const int a = min(max(lo - first, 0), 32), z = min(max(hi - first, 0), 32);
  if (a >= z) return 0;
  return (0xffffffffu >> (32 - (z - a))) << a;
}

// A row's statistics in natural units from its reference exponent (in powers
// of two) and sum.  The sum takes up what rounding the exponent loses, so that
// exp(score - greatest) / sum stays consistent (past kFarScore no gradient uses it).
__device__ __forceinline__ float2 natural_stats(float top, float sum) {
  if (!(fabsf(top) < kFarScore)) return make_float2(top == -INFINITY ? top : top * kLn2, sum);
  const float m = top * kLn2;
  return make_float2(m, sum * exp2f(top - m * kLog2e));
}

// What a score in a tile's units is multiplied by.  Kept normal: a hidden
// score's -inf times 0, or a score of 0 times infinity, would be NaN, and past
// either end no score differs from 0, or none but 0 from infinity, any more.
__device__ __forceinline__ float unit_of(double f) {
  return fminf(fmaxf((float)f, 1.17549435e-38f), 3.40282347e38f);
}

// The key tiles that a tile of query rows needs: [0, sinks) and then `low` on.
struct TileRange {
  int sinks, low, count;
  int width;  // of the last of the first `sinks` tiles: the columns that hold sinks, in whole 16s
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : low + i - sinks; }
};
struct RowRange {
  int p0, p1;  // positions of the first and last row that exist
  bool all;    // 128 rows, each standing in the sequence
};

__device__ __forceinline__ RowRange rows_of(const AttentionShape& s, const Sequence& q, int r0) {
  RowRange r;
  r.p0 = q.start + r0;
  r.p1 = q.start + min(r0 + kTile, s.q_len) - 1;
  r.all = r.p0 >= 0 && r.p1 < q.n && r0 + kTile <= s.q_len;
  return r;
}

__device__ __forceinline__ TileRange keys_for(const AttentionShape& s, const Sequence& q, const RowRange& r) {
  const int a = max(r.p0, 0), z = min(r.p1, q.n - 1);
  if (a > z) return {0, 0, 0, kTile};
  const int low = s.window > 0 ? max(a + 1 - s.window, 0) : 0;
  TileRange t;
  t.low = low / kTile;
  t.sinks = min(tiles_of(min(s.sinks, low)), t.low);
  t.count = t.sinks + z / kTile - t.low + 1;
  t.width = min(kTile, (min(s.sinks, low) - (t.sinks - 1) * kTile + 15) / 16 * 16);
  return t;
}

// Whether every row of the tile sees every key of tile t.
__device__ __forceinline__ bool sees_all(const AttentionShape& s, const RowRange& r, int t) {
  const int j0 = t * kTile, j1 = j0 + kTile - 1;
  return r.all && j1 <= r.p0 && (s.window == 0 || r.p1 - j0 < s.window || j1 < s.sinks);
}

// ---- forward ----------------------------------------------------------------------------

// One block per SM walks work items (128 query rows of a head) and, for each,
// the key tiles of 128 that its rows see; the tiles of all items form one
// stream, so that an item's start and end overlap its neighbours' arithmetic.
//   warps 0-7    probabilities: two threads share a row, 64 columns each.  A
//                tile's probabilities are taken relative to the row's greatest
//                score in that tile alone, so that no state goes from tile to
//                tile here: p = 2^(s - m + 14), split into fp16 halves over
//                the scores in tensor memory.
//   warps 8-15   output: each tile's P.V is added to fp32 registers, both
//                brought to the greater of the two reference scores.  (An
//                accumulator that stayed in tensor memory would lose up to a
//                step per matrix instruction, always toward zero.)
//   warp 16      copies packed tiles: the next item's queries, and the keys and
//                values into a ring of 32 KB slots,
//   warp 17      issues the matrix instructions: the scores of a tile before
//                the values of the one before it, so that the two overlap,
//   warps 18-19  rows that take no part in that.
// The query tile is kept in tensor memory (rows_to_tmem).
//
// Three fp16 products bound it at 557 TFLOP/s of fp32-accurate work, all keys of a
// tile counted.  Measured, 128 wide: 8192 causal tokens without a window 400
// TFLOP/s; with a window of 1024 and 4 sinks 215 us = 301 TFLOP/s of the visible
// pairs, tensor pipe 52% (the tiles at both ends of a window are half hidden, and
// a sink tile costs a step for a few columns); 2048 tokens of 8 sequences with a
// window of 512 260 us = 233 TFLOP/s, 44%.  An instruction of 128 x 128 x 16 takes
// about 87 cycles of the issuing warp's chain where 64 would be the products':
// what bounds it is the turn from scores to probabilities and back.
constexpr int kThreads = 20 * 32;
constexpr int kSlotBytes = 2 * kBox;

// Registers per thread: launched with 96 (640 threads), 480 for the five warps
// of each quarter of an SM; after the split 2 x 120 + 2 x 88 + 64 = 480.
constexpr int kScoreRegs = 120, kOutputRegs = 88, kFewRegs = 64;
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int DP>
struct ForwardPlan {
  static constexpr int kHalves = DP / 64;
  static constexpr int kSlots = DP == 64 ? 5 : 4;
  static constexpr int kSmem = 1024 + kTileBytes<DP> + kSlots * kSlotBytes + 9216;
};

struct ForwardArgs {
  AttentionShape s;
  const float *q, *k, *v;
  const uint8_t *pq, *pk, *pv;
  const float *fq, *fk, *fv;
  const float *tnq, *tnk;  // greatest norms of the query and key tiles' rows
  const Sequence* seqs;
  float *out, *stats;
  int segs;         // segments of each item's key tiles
  int* steps;       // segs > 1: key tiles of each unit
  float* part;      // segs > 1: [item][segment][128][DP] sums of P.V, relative to 2^exponent
  float2* part_ml;  // and [item][segment][128] (exponent, sum of P)
};

// Work item `index`: 128 rows of a head, those that see the most keys first.
struct QueryItem {
  int b, h, g, r0, n;  // n: key tiles to walk; 0: none, or not for the matrix unit
  int f0, f1;          // the unit's segment of them
  bool first;          // the first segment
  Sequence sq;
  RowRange rows;
  TileRange range;
  int q_index, k_index;  // of the item's query tile and its head's first key tile
};

// Where item `index` lies: heads, sequence, first row.
__device__ __forceinline__ int query_place(const AttentionShape& s, int index, int* h, int* b) {
  *h = index % s.heads;
  *b = index / s.heads % s.batch;
  return (tiles_of(s.q_len) - 1 - index / (s.heads * s.batch)) * kTile;
}

// Unit `unit`: segment unit % segs of item unit / segs.  Called by whole warps.
__device__ __forceinline__ QueryItem query_item(const ForwardArgs& a, int unit, int* err) {
  const AttentionShape& s = a.s;
  QueryItem t;
  const int index = unit / a.segs, seg = unit - index * a.segs;
  t.r0 = query_place(s, index, &t.h, &t.b);
  t.g = t.h / (s.heads / s.kv_heads);
  t.sq = a.seqs[t.b];
  t.rows = rows_of(s, t.sq, t.r0);
  t.range = keys_for(s, t.sq, t.rows);
  t.q_index = (t.b * s.heads + t.h) * tiles_of(s.q_len) + t.r0 / kTile;
  t.k_index = (t.b * s.kv_heads + t.g) * tiles_of(s.k_len);
  const float norm = a.tnq[t.q_index] * s.scale * kLog2e;
  bool far = false;
  for (int i = threadIdx.x & 31; i < t.range.count; i += 32) {
    const int k = t.k_index + t.range.at(i);
    far |= !(norm * a.tnk[k] + 0.0f * a.fv[k] < kFarScore);
  }
  // A product with a hidden value that is not finite would not be 0: such
  // rows go key by key instead.
  t.n = __any_sync(0xffffffffu, far) ? 0 : t.range.count;
  const int each = (t.n + a.segs - 1) / a.segs;
  t.f0 = min(t.n, seg * each);
  t.f1 = min(t.n, t.f0 + each);
  t.first = seg == 0;
  return t;
}

// The block's item of a round (-1: none in this one); false after the last
// round.  Items come heaviest first, and every other round runs backwards over
// the blocks, so that the rounds' differences even out.
__device__ __forceinline__ bool item_of(int round, int items, int* w) {
  const int blocks = gridDim.x, x = blockIdx.x;
  const int at = round * blocks + (round & 1 ? blocks - 1 - x : x);
  *w = at < items ? at : -1;
  return round * blocks < items;
}

// What a row of an item sees, for the masks of tiles that not all rows see whole.
struct RowMask {
  int low, high, sinks;  // [low, high) and [0, sinks)
};
__device__ __forceinline__ RowMask mask_of(const AttentionShape& s, const QueryItem& t, int row) {
  const int p = t.rows.p0 + row;
  RowMask m;
  m.high = t.r0 + row < s.q_len && p >= 0 && p < t.sq.n ? p + 1 : 0;
  m.low = s.window > 0 ? max(p + 1 - s.window, 0) : 0;
  m.sinks = min(m.high, s.sinks);
  return m;
}
__device__ __forceinline__ uint32_t seen_bits(const RowMask& m, int first) {
  return bits_between(m.low, m.high, first) | bits_between(0, m.sinks, first);
}

// A thread's columns of a row, stored or added.
template <int N>
__device__ __forceinline__ void store_row(float* __restrict__ dst, const float (&v)[N], float by, int cols, bool vec,
                                          int add) {
  if (vec) {
#pragma unroll
    for (int c = 0; c < N; c += 4)
      if (c < cols) {
        float4 o = make_float4(v[c] * by, v[c + 1] * by, v[c + 2] * by, v[c + 3] * by);
        if (add) {
          const float4 p = *(const float4*)(dst + c);
          o.x += p.x, o.y += p.y, o.z += p.z, o.w += p.w;
        }
        *(float4*)(dst + c) = o;
      }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < cols) dst[c] = add ? dst[c] + v[c] * by : v[c] * by;
  }
}

// A row's statistics where p was 2^(s - top), top 14 below the greatest score.
__device__ __forceinline__ float2 tile_stats(float top, float l) {
  return natural_stats(top == -INFINITY ? top : top + 14.0f, l * 0x1p-14f);
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 1) forward_kernel(ForwardArgs a, int items, int* err) {
  using Plan = ForwardPlan<DP>;
  constexpr int kHalves = Plan::kHalves;
  const AttentionShape& s = a.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t q_smem = smem_u32(smem);
  const uint32_t slots = q_smem + kTileBytes<DP>;
  uint8_t* misc = smem + kTileBytes<DP> + Plan::kSlots * kSlotBytes;
  float* ref = (float*)misc;            // [4][128] reference exponents of a tile's rows
  float* sum = ref + 4 * kTile;         // [4][2][128] sums of each half of the tile's columns
  float* most = sum + 8 * kTile;        // [2][2][128] greatest scores of each half
  uint64_t* bars = (uint64_t*)(most + 4 * kTile);
  const uint32_t q_full = smem_u32(bars), q_empty = q_full + 8, slot_full = q_empty + 8;
  const uint32_t slot_empty = slot_full + 8 * Plan::kSlots, s_full = slot_empty + 8 * Plan::kSlots;
  const uint32_t p_full = s_full + 16, o_full = p_full + 16, o_empty = o_full + 16;
  const uint32_t pair_full = o_empty + 16, stats_full = pair_full + 32, q_ready = stats_full + 32, drained = q_ready + 8;
  uint32_t* tmem_slot = (uint32_t*)(bars + 2 * Plan::kSlots + 20);
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 8);
    mbar_init(q_ready, 8);
    for (int i = 0; i < Plan::kSlots; ++i) mbar_init(slot_full + 8 * i, 1), mbar_init(slot_empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 8);
      mbar_init(o_full + 8 * i, 1);
      mbar_init(o_empty + 8 * i, 8);
    }
    for (int i = 0; i < 4; ++i) mbar_init(pair_full + 8 * i, 2), mbar_init(stats_full + 8 * i, 8);
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Tensor memory: the query tile (DP columns), two buffers of scores (128 each) and of values (DP; one if DP is 128).
  constexpr int kOut = DP == 64 ? 2 : 1;
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_s = tmem + DP, tmem_o = tmem_s + 2 * kTile;

  if (warp >= 18) {
    fewer_registers<kFewRegs>();
    // Items that see nothing or meet values that are not finite, key by key.
    // No wait of the pipeline depends on these warps, however long they take.
    for (int round = 0, w; item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const QueryItem t = query_item(a, w, err);
      if (t.n == 0 && t.first)
        for (int r = t.r0 + warp - 18; r < min(t.r0 + kTile, s.q_len); r += 2)
          simple_forward_row(s, t.sq, a.q, a.k, a.v, a.out, a.stats, t.b, t.h, r);
    }
  } else if (warp == 16) {
    fewer_registers<kFewRegs>();
    uint32_t it = 0, loaded = 0;      // slots filled, query tiles loaded
    bool ok = true;
    auto fill = [&](const uint8_t* src, bool is_values) {
      for (int d = 0; d < kHalves && ok; ++d, ++it) {
        const uint32_t slot = it % Plan::kSlots, use = it / Plan::kSlots;
        if (use > 0) ok = mbar_wait(slot_empty + 8 * slot, (use - 1) & 1, err);
        if (!ok) break;
        const uint32_t full = slot_full + 8 * slot, dst = slots + slot * kSlotBytes;
        mbar_expect_tx(full, kSlotBytes);
        if (!is_values || kHalves == 1) {
          // 128 rows of one box, hi and lo.
          bulk_load(dst, src + d * kBox, kBox, full);
          bulk_load(dst + kBox, src + (kHalves + d) * kBox, kBox, full);
        } else {
          // 64 rows (keys) of every box: hi boxes, then lo boxes.
#pragma unroll
          for (int x = 0; x < 2 * kHalves; ++x)
            bulk_load(dst + x * (kBox / 2), src + x * kBox + d * (kBox / 2), kBox / 2, full);
        }
      }
    };
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const QueryItem t = query_item(a, w, err);
      if (lane == 0 && t.f0 < t.f1) {
        if (loaded > 0) ok = mbar_wait(q_empty, (loaded - 1) & 1, err);
        if (ok) {
          mbar_expect_tx(q_full, kTileBytes<DP>);
          bulk_load(q_smem, a.pq + (int64_t)t.q_index * kTileBytes<DP>, kTileBytes<DP>, q_full);
          ++loaded;
        }
        for (int i = t.f0; i <= t.f1 && ok; ++i) {  // a tile's keys, then the values of the one before
          if (i < t.f1) fill(a.pk + (int64_t)(t.k_index + t.range.at(i)) * kTileBytes<DP>, false);
          if (ok && i > t.f0) fill(a.pv + (int64_t)(t.k_index + t.range.at(i - 1)) * kTileBytes<DP>, true);
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
    if (lane == 0 && !ok) {  // copies in flight end before the block does
      if (loaded > 0) mbar_wait(q_full, (loaded - 1) & 1, err);
      for (uint32_t f = it > Plan::kSlots ? it - Plan::kSlots : 0; f < it; ++f)
        mbar_wait(slot_full + 8 * (f % Plan::kSlots), (f / Plan::kSlots) & 1, err);
    }
  } else if (warp == 17) {
    fewer_registers<kFewRegs>();
    constexpr uint32_t kValue = umma_idesc(DP, true);
    const bool leader = elect_one();
    uint32_t it = 0, gi = 0, item = 0;  // slots, tiles and items issued so far
    bool ok = true;
    auto values = [&](uint32_t t, int width) {  // of tile t of the stream, its first `width` keys
      const uint32_t p = tmem_s + (t & 1) * kTile, out = t % kOut, d = tmem_o + out * DP;
      ok = warp_wait(p_full + 8 * (t & 1), (t >> 1) & 1, err);
      if (ok && t >= kOut) ok = warp_wait(o_empty + 8 * out, (t / kOut - 1) & 1, err);
      for (int x = 0; x < kHalves && ok; ++x, ++it) {
        const uint32_t slot = it % Plan::kSlots;
        ok = warp_wait(slot_full + 8 * slot, (it / Plan::kSlots) & 1, err);
        if (!ok) break;
        tc_fence_after();
        constexpr int kSteps = kTile / 16 / kHalves;
        constexpr uint32_t kStride = kBox / kHalves;  // between the slot's boxes
        const uint32_t v = row_word(slots + slot * kSlotBytes, kStride);
        const uint32_t px = p + x * kSteps * kSplitStep;
        if (leader) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            if ((x * kSteps + k) * 16 >= width) break;
            const uint32_t ph = px + k * kSplitStep, vh = v + k * kRowStep, vl = vh + (kBox >> 4);
            umma_ts(d, ph + kSplitLo, vh, kValue, x != 0 || k != 0);
            umma_ts(d, ph, vl, kValue, 1u);
            umma_ts(d, ph, vh, kValue, 1u);
          }
          umma_commit(slot_empty + 8 * slot);
          if (x == kHalves - 1) umma_commit(o_full + 8 * out);
        }
        __syncwarp();
      }
    };
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const QueryItem t = query_item(a, w, err);
      const int n = __shfl_sync(0xffffffffu, t.f1 - t.f0, 0);
      const int sinks = __shfl_sync(0xffffffffu, t.range.sinks - t.f0, 0);
      const int sink_width = __shfl_sync(0xffffffffu, t.range.width, 0);
      if (n <= 0) continue;
      ok = warp_wait(q_ready, item & 1, err);
      ++item;
      for (int i = 0; i <= n && ok; ++i) {
        if (i < n) {
          const uint32_t d = tmem_s + (gi & 1) * kTile;
          const uint32_t score = umma_idesc(i == sinks - 1 ? sink_width : kTile, false);
          for (int x = 0; x < kHalves && ok; ++x, ++it) {
            const uint32_t slot = it % Plan::kSlots;
            ok = warp_wait(slot_full + 8 * slot, (it / Plan::kSlots) & 1, err);
            if (!ok) break;
            tc_fence_after();
            const uint32_t q = tmem + 32 * x, key = column_word(slots + slot * kSlotBytes);
            if (leader) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t qh = q + 8 * k, ql = qh + DP / 2, kh = key + k * kColumnStep, kl = kh + (kBox >> 4);
                umma_ts(d, ql, kh, score, x != 0 || k != 0);
                umma_ts(d, qh, kl, score, 1u);
                umma_ts(d, qh, kh, score, 1u);
              }
              umma_commit(slot_empty + 8 * slot);
              if (x == kHalves - 1) umma_commit(s_full + 8 * (gi & 1));
            }
            __syncwarp();
          }
          if (!ok) break;
          ++gi;
        }
        // The values of the tile before (gi now counts the scores issued).
        if (i > 0) values(gi - (i < n ? 2 : 1), i == sinks ? sink_width : kTile);
      }
    }
    if (!ok && leader) {  // instructions in flight end before the block does
      umma_commit(drained);
      mbar_wait(drained, 0, err);
    }
  } else if (warp < 8) {
    more_registers<kScoreRegs>();
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, at = tmem_s + lanes + half * 64;
    uint32_t gi = 0, item = 0;
    bool ok = true;
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const QueryItem t = query_item(a, w, err);
      if (t.f0 >= t.f1) continue;
      // The products with the query tile before are done: their scores have been read.
      ok = warp_wait(q_full, item & 1, err);
      if (!ok) break;
      rows_to_tmem<DP>(tmem + lanes, q_smem, row, half);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready), mbar_arrive(q_empty);
      ++item;
      const RowMask mask = mask_of(s, t, row);
      const double to_log2 = (double)a.fq[t.q_index] * (double)s.scale * 1.4426950408889634;
      for (int i = t.f0; i < t.f1; ++i, ++gi) {
        const int buf = gi & 1, tile = t.range.at(i);
        const float f = unit_of(to_log2 * (double)a.fk[t.k_index + tile]);
        const bool whole = sees_all(s, t.rows, tile);
        ok = warp_wait(s_full + 8 * buf, (gi >> 1) & 1, err);
        if (!ok) break;
        tc_fence_after();
        // Columns past a narrow tile's width hold what was there before.
        const int width = (i == t.range.sinks - 1 ? t.range.width : kTile) - half * 64;
        float v[64];
        float m0 = -INFINITY;
        if (width > 0) {
          tmem_ld64(at + buf * kTile, v);
          if (!whole) {
            const int j0 = tile * kTile + half * 64;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t seen = 32 * c < width ? seen_bits(mask, j0 + 32 * c) & bits_between(0, width, 32 * c) : 0u;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen >> e & 1u)) v[32 * c + e] = -INFINITY;
            }
          }
          float m1 = v[1], m2 = v[2], m3 = v[3];
          m0 = v[0];
#pragma unroll
          for (int e = 4; e < 64; e += 4) {
            m0 = fmaxf(m0, v[e]);
            m1 = fmaxf(m1, v[e + 1]);
            m2 = fmaxf(m2, v[e + 2]);
            m3 = fmaxf(m3, v[e + 3]);
          }
          m0 = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        }
        // The row's other half is in the warp four further.
        most[(buf * 2 + half) * kTile + row] = m0;
        __syncwarp();
        if (lane == 0) mbar_arrive(pair_full + 8 * (warp & 3));
        ok = warp_wait(pair_full + 8 * (warp & 3), gi & 1, err);
        if (!ok) break;
        m0 = fmaxf(m0, most[(buf * 2 + 1 - half) * kTile + row]);
        const float c0 = m0 == -INFINITY ? 0.0f : fmaf(m0, f, -14.0f);
        float l[4] = {};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (32 * c >= width) break;
#pragma unroll
          for (int e = 0; e < 32; ++e) v[32 * c + e] = fmaf(v[32 * c + e], f, -c0);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[32 * c + e] = exp2_fast(v[32 * c + e]);
#pragma unroll
          for (int e = 0; e < 32; ++e) l[e & 3] += v[32 * c + e];
          store_split16(at + buf * kTile + 32 * c, v + 32 * c);
          store_split16(at + buf * kTile + 32 * c + 16, v + 32 * c + 16);
        }
        // Four buffers, each with its own barrier (stats_full): the scores of
        // tile gi come after the values of gi - 2 were issued, which waited until
        // the output warps had taken gi - 4, its statistics and phase with it.
        sum[((gi & 3) * 2 + half) * kTile + row] = (l[0] + l[1]) + (l[2] + l[3]);
        if (half == 0) ref[(gi & 3) * kTile + row] = m0 == -INFINITY ? -INFINITY : c0;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * buf), mbar_arrive(stats_full + 8 * (gi & 3));
      }
    }
  } else {
    fewer_registers<kOutputRegs>();
    constexpr int kCols = DP / 2;  // output columns of a thread
    const int quad = warp & 3, half = (warp - 8) >> 2, row = quad * 32 + lane;
    const uint32_t at = tmem_o + ((uint32_t)(quad * 32) << 16) + half * kCols;
    uint32_t gi = 0;
    bool ok = true;
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const QueryItem t = query_item(a, w, err);
      if (a.segs > 1 && threadIdx.x == 8 * 32) a.steps[w] = t.f1 - t.f0;
      if (t.f0 >= t.f1) continue;
      float acc[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[c] = 0.0f;
      float top = -INFINITY, l = 0.0f;
      for (int i = t.f0; i < t.f1; ++i, ++gi) {
        const float fv = a.fv[t.k_index + t.range.at(i)];
        const uint32_t ob = gi % kOut;
        ok = warp_wait(stats_full + 8 * (gi & 3), (gi >> 2) & 1, err);
        if (!ok) break;
        const float c0 = ref[(gi & 3) * kTile + row];
        const float parts = sum[(gi & 3) * 2 * kTile + row] + sum[((gi & 3) * 2 + 1) * kTile + row];
        ok = warp_wait(o_full + 8 * ob, (gi / kOut) & 1, err);
        if (!ok) break;
        tc_fence_after();
        const float next = fmaxf(top, c0);
        const float keep = top == -INFINITY ? 0.0f : exp2_fast(top - next);
        const float take = c0 == -INFINITY ? 0.0f : exp2_fast(c0 - next);
        l = l * keep + parts * take;
        top = next;
        const float tv = take * fv;
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          float v[16];
          tmem_ld16(at + ob * DP + c, v);
          if (c == kCols - 16) {  // the last values are out: the buffer is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty + 8 * ob);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(acc[c + e], keep, v[e] * tv);
        }
      }
      const int r = t.r0 + row;
      if (ok && a.segs > 1) {
        const int64_t at_part = (int64_t)w * kTile + row;
        store_row(a.part + at_part * DP + half * kCols, acc, 1.0f, kCols, true, 0);
        if (half == 0) a.part_ml[at_part] = make_float2(top, l);
      } else if (ok && r < s.q_len) {
        store_row(a.out + row_at(s, t.b, t.h, r, s.heads, s.q_len) + half * kCols, acc, l > 0.0f ? 1.0f / l : 0.0f,
                  s.head_dim - half * kCols, s.head_dim % 4 == 0 && ((uintptr_t)a.out & 15) == 0, 0);
        if (a.stats != nullptr && half == 0)
          *(float2*)(a.stats + 2 * (((int64_t)t.b * s.heads + t.h) * s.q_len + r)) = tile_stats(top, l);
      }
      __syncwarp();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Segments that hold a part: the first ones, as each but the last of them is full.
__device__ __forceinline__ int segments_used(const int* steps, int segs, int stride) {
  int used = 0;
  for (int k = threadIdx.x & 31; k < segs; k += 32) used += steps[(int64_t)k * stride] > 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) used += __shfl_xor_sync(0xffffffffu, used, o);
  return used;
}

// Joins an item's segments in order, a few rows per block.
constexpr int kJoinRows = 8;
template <int DP>
__global__ void __launch_bounds__(256) forward_join_kernel(ForwardArgs a) {
  const AttentionShape& s = a.s;
  const int item = blockIdx.x / (kTile / kJoinRows), row0 = blockIdx.x % (kTile / kJoinRows) * kJoinRows;
  int h, b;
  const int r0 = query_place(s, item, &h, &b);
  const int used = segments_used(a.steps + (int64_t)item * a.segs, a.segs, 1);  // 0: written key by key
  if (used == 0) return;
  for (int i = threadIdx.x; i < kJoinRows * DP / 4; i += 256) {
    const int row = row0 + i / (DP / 4), c = i % (DP / 4) * 4, r = r0 + row;
    if (r >= s.q_len || c >= s.head_dim) continue;
    const int64_t first = (int64_t)item * a.segs * kTile + row;
    float top = -INFINITY, l = 0.0f, v[4] = {};
#pragma unroll 4
    for (int k = 0; k < used; ++k) {
      const float2 ml = a.part_ml[first + (int64_t)k * kTile];
      const float4 p = *(const float4*)(a.part + (first + (int64_t)k * kTile) * DP + c);
      const float next = fmaxf(top, ml.x);
      const float keep = top == next ? 1.0f : exp2_fast(top - next);
      const float take = ml.x == next ? 1.0f : exp2_fast(ml.x - next);
      l = l * keep + ml.y * take;
      v[0] = v[0] * keep + p.x * take;
      v[1] = v[1] * keep + p.y * take;
      v[2] = v[2] * keep + p.z * take;
      v[3] = v[3] * keep + p.w * take;
      top = next;
    }
    store_row(a.out + row_at(s, b, h, r, s.heads, s.q_len) + c, v, l > 0.0f ? 1.0f / l : 0.0f, s.head_dim - c,
              s.head_dim % 4 == 0 && ((uintptr_t)a.out & 15) == 0, 0);
    if (a.stats != nullptr && c == 0)
      *(float2*)(a.stats + 2 * (((int64_t)b * s.heads + h) * s.q_len + r)) = tile_stats(top, l);
  }
}

// ---- gradients ------------------------------------------------------------------------------

// Two passes of one pipeline, each summing its own gradients in a fixed order
// (one pass for all three would have to add into dq from many blocks):
//
//   pass      rows (resident)    columns (streamed)   summed
//   queries   queries: Q, dO     keys: K, V           dq += dS.K
//   keys      keys: K, V         queries: Q, dO       dv += P^T.dO, dk += dS^T.Q
//
// A work item is 128 rows; its columns come in steps of 64.  A step forms the
// scores Q.K^T and dP = dO.V^T (or their transposes); P = 2^(score - max) / sum
// and dS = P (dP - delta) become fp16 halves in tensor memory, operands of the
// step's sums, which are added to fp32 registers.  P is at most 1; dS is
// brought near 2^15 by a power of two from |dS| <= |dO_i| |V_j| + |delta_i|, with
// the norms of single rows on the resident side and a tile's greatest on the
// streamed one, all in the units of dO's packed tile (its factor, which may be as
// small as a gradient, only enters where the sums leave tensor memory).
//   warps 0-7    P and dS: two threads share a row, 32 columns each,
//   warps 8-15   sums into registers, half of the columns each,
//   warp 16      copies: resident tiles of the next item, rings of half steps (a
//                step's lo boxes, then its hi ones),
//   warp 17      matrix instructions.  Of a step g: dv of g, the scores of g + 1,
//                dq or dk of g, dP of g + 1.  P of a step is formed while the
//                last step's dS is summed, and its dS while the next scores are.
// Resident tiles are in tensor memory (rows_to_tmem), with one buffer each of
// scores (keys: then P) and of dP (then dS), and two of 64 columns of sums: with
// 256 columns for the resident tiles no wider step fits the 512.
//
// The products, five per visible pair and 128 columns and two of them done twice,
// bound it.  Measured for 8192 tokens, 16 heads over 4, window 1024, 128 wide: 306
// us for dq (tensor pipe 57%), 430 for dk and dv (56%), together 220 TFLOP/s of the
// formulas' work.  An instruction of 128 x 64 x 16 takes 41 to 60 cycles instead of
// 32, and the tiles at a window's ends are half hidden.
// A key tile's queries may be many (a sink's are all that follow), and tiles may
// be few: their steps are cut into segments that go to different blocks, each
// leaving its part in the workspace, joined in order by grad_join_kernel.
// Registers after the split, as in the forward: the keys' pass keeps sums of two
// gradients, 2 x 64 + 2 x 152 + 48 = 480; the queries' 2 x 112 + 2 x 88 + 64 = 464.
template <bool KEYS>
constexpr int kProbRegs = KEYS ? 64 : 112;
template <bool KEYS>
constexpr int kSumRegs = KEYS ? 152 : 88;
template <bool KEYS>
constexpr int kGradFewRegs = KEYS ? 48 : 64;
template <int N>
__device__ __forceinline__ void set_registers() {  // from the 96 of the launch
  if constexpr (N < 96) fewer_registers<N>();
  else more_registers<N>();
}
constexpr int kStep = 64;
constexpr int kStepBox = kStep * 128;  // bytes of 64 rows of a box

// How the key tiles' steps are cut: the first `long_tiles` of each head into
// long_segs segments, the others into short_segs.  A unit is a segment of a
// tile of a head, counted tile by tile.  The query tiles' steps are cut into
// query_segs, a tile's segments counted one after the other.
struct Segments {
  int long_tiles, long_segs, short_segs, query_segs;
};

struct GradArgs {
  AttentionShape s;
  const float *q, *k, *v, *out, *dout;
  const uint8_t *pq, *pk, *pv, *po;
  const float *fq, *fk, *fv, *fo;      // factors
  const float *tnq, *tnk;              // greatest norms of Q's and K's tiles' rows
  const Sequence* seqs;
  const float *nv, *tnv, *tno, *tdo;   // norms of V's rows; greatest norm of V's and dO's tiles, greatest |delta|
  const float4* info;                  // of query rows
  const float2* col;                   // the same for rows that are streamed
  float2* own;                         // statistics for what goes key by key
  float *dq, *dk, *dv;
  int add_q, add_k, add_v;
  double scale_power;                  // s.scale as a power of two times a number from 1 to 2: the
  float scale_rest;                    // power keeps `down` exact below fp32's normal numbers
  Segments seg;
  int* steps;                          // of each unit
  float* part;                         // queries: [unit][128][DP]; keys: [unit][dk, dv][128][DP]
};

template <int DP, bool KEYS>
struct GradPlan {
  static constexpr int kHalves = DP / 64;
  static constexpr int kPart = kHalves * kStepBox;  // a step's hi or lo half
  static constexpr int kEntries1 = 4;               // ring of the scores' operand, used twice: two steps
  static constexpr int kEntries2 = 2;               // ring of dP's operand: one step
  static constexpr int kResident = 2 * kTileBytes<DP>;
  static constexpr int kInfo = KEYS ? 2 * kStep * 8 : 0;
  static constexpr int kSmem = kResident + (kEntries1 + kEntries2) * kPart + kInfo + 512;
  static_assert(kSmem <= 227 * 1024, "shared memory of one block");
  static_assert(2 * DP + 4 * kStep <= 512, "tensor memory");
};

// 128 rows of one head and the steps of 64 columns they need.
struct GradItem {
  int b, h, g, r0, n;  // h: the queries' head, or the first of the keys'; n: steps (keys: per head); 0: none, or not for the matrix unit
  Sequence sq;
  RowRange rows;       // queries
  TileRange range;     // in steps of 64
  int row_tile;        // index of the resident tile
  int f0, f1;          // the unit's part of the heads' steps, counted head by head
  int segs;            // segments of the tile's steps
  bool first;          // the first of them
};

// Where unit `index` lies: heads, sequence, first row, and its segment.
template <bool KEYS>
__device__ __forceinline__ GradItem grad_place(const GradArgs& a, int index, int* segment) {
  const AttentionShape& s = a.s;
  GradItem t;
  if (!KEYS) {
    t.segs = a.seg.query_segs;
    *segment = index % t.segs;
    t.r0 = query_place(s, index / t.segs, &t.h, &t.b);
    t.g = t.h / (s.heads / s.kv_heads);
  } else {
    // The first keys are seen by the most queries.
    const int of_long = a.seg.long_tiles * a.seg.long_segs * s.kv_heads * s.batch;
    const bool is_long = index < of_long;
    t.segs = is_long ? a.seg.long_segs : a.seg.short_segs;
    if (!is_long) index -= of_long;
    const int tk = index / (t.segs * s.kv_heads * s.batch) + (is_long ? 0 : a.seg.long_tiles);
    *segment = index / (s.kv_heads * s.batch) % t.segs;
    t.g = index % s.kv_heads;
    t.b = index / s.kv_heads % s.batch;
    t.h = t.g * (s.heads / s.kv_heads);
    t.r0 = tk * kTile;
  }
  return t;
}

template <bool KEYS>
__device__ __forceinline__ GradItem grad_item(const GradArgs& a, int index, int* err) {
  const AttentionShape& s = a.s;
  const int group = s.heads / s.kv_heads, lane = threadIdx.x & 31;
  const int tiles_q = tiles_of(s.q_len), tiles_k = tiles_of(s.k_len);
  int seg;
  GradItem t = grad_place<KEYS>(a, index, &seg);
  bool far = false;  // or not finite
  if (!KEYS) {
    t.sq = a.seqs[t.b];
    t.rows = rows_of(s, t.sq, t.r0);
    t.row_tile = (t.b * s.heads + t.h) * tiles_q + t.r0 / kTile;
    const int x = max(t.rows.p0, 0), z = min(t.rows.p1, t.sq.n - 1);
    const int low = s.window > 0 ? max(x + 1 - s.window, 0) : 0;
    t.range.low = low / kStep;
    t.range.sinks = min((min(s.sinks, low) + kStep - 1) / kStep, t.range.low);
    t.range.count = x > z ? 0 : t.range.sinks + z / kStep - t.range.low + 1;
    const float norm = a.tnq[t.row_tile] * s.scale * kLog2e + 0.0f * a.fo[t.row_tile];
    const int first = (t.b * s.kv_heads + t.g) * tiles_k;
#pragma unroll 1
    for (int i = lane; i < t.range.count; i += 32) {
      const int k = first + t.range.at(i) / 2;
      far |= !(norm * a.tnk[k] + 0.0f * a.fv[k] < kFarScore);
    }
  } else {
    t.sq = a.seqs[t.b];
    t.rows = {0, 0, false};
    t.row_tile = (t.b * s.kv_heads + t.g) * tiles_k + t.r0 / kTile;
    // Rows that see some key of the tile: positions from the first key on, up
    // to where the last key leaves the window (none leaves it among the sinks).
    const int last = min(t.r0 + kTile, t.sq.n) - 1;
    int end = t.sq.n;
    if (s.window > 0 && t.r0 >= s.sinks && end - last > s.window) end = last + s.window;
    const int x = max(t.r0 - t.sq.start, 0), z = min(end - t.sq.start, s.q_len) - 1;
    t.range.sinks = 0;
    t.range.low = x / kStep;
    t.range.count = t.r0 >= t.sq.n || x > z ? 0 : z / kStep - t.range.low + 1;
    const float norm = a.tnk[t.row_tile] * s.scale * kLog2e + 0.0f * a.fv[t.row_tile];
#pragma unroll 1
    for (int i = lane; i < t.range.count * group; i += 32) {
      const int q = (t.b * s.heads + t.h + i / t.range.count) * tiles_q + t.range.at(i % t.range.count) / 2;
      far |= !(norm * a.tnq[q] + 0.0f * (a.fo[q] + a.tdo[q]) < kFarScore);
    }
  }
  t.n = __any_sync(0xffffffffu, far) ? 0 : t.range.count;
  const int total = (KEYS ? group : 1) * t.n, each = (total + t.segs - 1) / t.segs;
  t.f0 = min(total, seg * each);
  t.f1 = min(total, t.f0 + each);
  t.first = seg == 0;
  return t;
}

// The power of two (its exponent) that brings values up to `bound` below 2^15.
__device__ __forceinline__ int scale_exponent(float bound) {
  const int e = (int)(__float_as_uint(bound) >> 23 & 255u) - 127;
  return bound == 0.0f ? 0 : min(max(14 - e, -126), 126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <int DP, bool KEYS>
__global__ void __launch_bounds__(kThreads, 1) grad_kernel(GradArgs a, int items, int* err) {
  using Plan = GradPlan<DP, KEYS>;
  constexpr int kHalves = Plan::kHalves, kPart = Plan::kPart;
  constexpr uint32_t kEntries1 = Plan::kEntries1, kEntries2 = Plan::kEntries2;
  const AttentionShape& s = a.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_q = tiles_of(s.q_len), tiles_k = tiles_of(s.k_len);
  extern __shared__ __align__(1024) uint8_t smem[];  // at the start of shared memory, as there is no other
  const uint32_t base = smem_u32(smem);
  const uint32_t ring1 = base + Plan::kResident, ring2 = ring1 + kEntries1 * kPart;
  uint8_t* info_smem = smem + Plan::kResident + (kEntries1 + kEntries2) * kPart;
  uint64_t* bars = (uint64_t*)(info_smem + Plan::kInfo);
  const uint32_t a_full = smem_u32(bars), a_empty = a_full + 8, a_ready = a_empty + 8;
  const uint32_t full1 = a_ready + 8, empty1 = full1 + 8 * kEntries1, full2 = empty1 + 8 * kEntries1;
  const uint32_t empty2 = full2 + 8 * kEntries2, s_full = empty2 + 8 * kEntries2, d_full = s_full + 8;
  const uint32_t s_done = d_full + 8, ds_full = s_done + 8, o_full = ds_full + 8, o_empty = o_full + 16;
  const uint32_t drained = o_empty + 16;
  uint32_t* tmem_slot = (uint32_t*)(bars + 3 + 2 * kEntries1 + 2 * kEntries2 + 9);
  if ((base & 1023u) != 0) {  // the swizzle needs it
    if (threadIdx.x == 0) atomicCAS(err, 0, (int)kErrTmemAlloc);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(a_full, 1);
    mbar_init(a_empty, 8);
    mbar_init(a_ready, 8);
    for (int i = 0; i < (int)kEntries1; ++i) mbar_init(full1 + 8 * i, 1), mbar_init(empty1 + 8 * i, 1);
    for (int i = 0; i < (int)kEntries2; ++i) mbar_init(full2 + 8 * i, 1), mbar_init(empty2 + 8 * i, 1);
    mbar_init(s_full, 1);
    mbar_init(d_full, 1);
    mbar_init(s_done, 8);
    mbar_init(ds_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(o_full + 8 * i, 1);
      mbar_init(o_empty + 8 * i, kHalves == 2 ? 4 : 8);
    }
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Tensor memory: resident tiles, scores, dP, two buffers of sums.
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t tmem_s = tmem + 2 * DP, tmem_d = tmem_s + kStep, tmem_o = tmem_d + kStep;

  // Index of the streamed tile of step n of an item's heads' steps.
  auto column_tile = [&](const GradItem& t, int n, int* step) {
    const int x = KEYS ? n / t.n : 0;
    *step = t.range.at(n - x * t.n);
    return KEYS ? (t.b * s.heads + t.h + x) * tiles_q + *step / 2 : (t.b * s.kv_heads + t.g) * tiles_k + *step / 2;
  };

  if (warp >= 18) {
    set_registers<kGradFewRegs<KEYS>>();
    // As in the forward: items for which the matrix unit is of no use.
    for (int round = 0, w; item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const GradItem t = grad_item<KEYS>(a, w, err);
      if (t.n != 0 || !t.first) continue;
      for (int r = t.r0 + warp - 18; r < min(t.r0 + kTile, KEYS ? s.k_len : s.q_len); r += 2) {
        if (!KEYS)
          simple_dq_row(s, t.sq, a.q, a.k, a.v, a.out, a.dout, a.dq,
                        a.own + (int64_t)t.row_tile * kTile + (r - t.r0), a.add_q, t.b, t.h, r);
        else simple_dkv_row(s, t.sq, a.q, a.k, a.v, a.out, a.own, a.dout, a.dk, a.dv, a.add_k, a.add_v, t.b, t.g, r);
      }
    }
  } else if (warp == 16) {
    set_registers<kGradFewRegs<KEYS>>();
    uint32_t gi = 0, loaded = 0;  // steps, items
    bool ok = true;
    // Half a step of a ring: `part` 0 the lo boxes, 1 the hi ones; with the
    // latter the rows' statistics where `with_info`.
    auto fill = [&](uint32_t ring, uint32_t full, uint32_t empty, uint32_t entries, const uint8_t* packed, int tile,
                    int step, uint32_t part, bool with_info) {
      const uint32_t entry = 2 * gi + part, slot = entry % entries, use = entry / entries, bar = full + 8 * slot;
      if (use > 0) ok = mbar_wait(empty + 8 * slot, (use - 1) & 1, err);
      if (!ok) return;
      mbar_expect_tx(bar, kPart + (with_info ? kStep * 8 : 0));
      const uint8_t* src = packed + (int64_t)tile * kTileBytes<DP> + (1 - part) * kHalves * kBox + (step & 1) * kStepBox;
#pragma unroll
      for (int x = 0; x < kHalves; ++x)
        bulk_load(ring + slot * kPart + x * kStepBox, src + x * kBox, kStepBox, bar);
      if (with_info)
        bulk_load(smem_u32(info_smem) + (gi & 1) * (kStep * 8),
                  (const uint8_t*)(a.col + (int64_t)tile * kTile + (step & 1) * kStep), kStep * 8, bar);
    };
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const GradItem t = grad_item<KEYS>(a, w, err);
      if (lane == 0 && t.f0 < t.f1) {
        if (loaded > 0) ok = mbar_wait(a_empty, (loaded - 1) & 1, err);
        if (ok) {
          mbar_expect_tx(a_full, Plan::kResident);
          const int64_t at = (int64_t)t.row_tile * kTileBytes<DP>;
          bulk_load(base, (KEYS ? a.pk : a.pq) + at, kTileBytes<DP>, a_full);
          bulk_load(base + kTileBytes<DP>, (KEYS ? a.pv : a.po) + at, kTileBytes<DP>, a_full);
          ++loaded;
        }
        for (int n = t.f0; n < t.f1 && ok; ++n, ++gi) {
          int step;
          const int tile = column_tile(t, n, &step);
          // The statistics come with the operand that stays until they have been used.
          fill(ring1, full1, empty1, kEntries1, KEYS ? a.pq : a.pk, tile, step, 0, false);
          if (ok) fill(ring1, full1, empty1, kEntries1, KEYS ? a.pq : a.pk, tile, step, 1, KEYS);
          if (ok) fill(ring2, full2, empty2, kEntries2, KEYS ? a.po : a.pv, tile, step, 0, false);
          if (ok) fill(ring2, full2, empty2, kEntries2, KEYS ? a.po : a.pv, tile, step, 1, false);
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    }
    if (lane == 0 && !ok) {
      // Copies in flight end before the block does.  The last step may have
      // been begun only in part: a wait for a fill that never came runs out.
      if (loaded > 0) mbar_wait_limit(a_full, (loaded - 1) & 1, err, kWaitCycles / 8);
      for (uint32_t f = gi > 1 ? 2 * gi - 2 : 0; f < 2 * gi + 2; ++f) {
        mbar_wait_limit(full1 + 8 * (f % kEntries1), (f / kEntries1) & 1, err, kWaitCycles / 8);
        mbar_wait_limit(full2 + 8 * (f % kEntries2), (f / kEntries2) & 1, err, kWaitCycles / 8);
      }
    }
  } else if (warp == 17) {
    set_registers<kGradFewRegs<KEYS>>();
    constexpr uint32_t kProduct = umma_idesc(kStep, false), kSum = umma_idesc(64, true);
    const bool leader = elect_one();
    uint32_t gi = 0, item = 0;           // steps whose scores, items that were issued
    uint32_t sums0 = 0, sums1 = 0;       // sums issued into each buffer
    bool ok = true;
    // D = resident rows (tensor memory) times the 64 streamed ones of step g, then `done`.
    auto product = [&](uint32_t g, uint32_t d, uint32_t rows, uint32_t ring, uint32_t full, uint32_t entries,
                       uint32_t done) {
      for (uint32_t part = 0; part < 2 && ok; ++part) {
        const uint32_t entry = 2 * g + part, slot = entry % entries;
        ok = warp_wait(full + 8 * slot, (entry / entries) & 1, err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t c0 = column_word(ring + slot * kPart);
        if (leader) {
#pragma unroll
          for (int x = 0; x < kHalves; ++x) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t rh = rows + 32 * x + 8 * k, rl = rh + DP / 2, ch = c0 + x * (kStepBox >> 4) + k * kColumnStep;
              if (part == 0) {
                umma_ts(d, rh, ch, kProduct, x != 0 || k != 0);
              } else {
                umma_ts(d, rl, ch, kProduct, 1u);
                umma_ts(d, rh, ch, kProduct, 1u);
              }
            }
          }
          if (part == 1) umma_commit(done);
        }
        __syncwarp();
      }
    };
    // A buffer of sums = P or dS (tensor memory) times 64 columns (x) of step g's 64 rows.
    auto sum_half = [&](uint32_t g, uint32_t p, uint32_t ring, uint32_t entries, int x, uint32_t buf, uint32_t& count) {
      if (count > 0) ok = warp_wait(o_empty + 8 * buf, (count - 1) & 1, err);
      ++count;
      if (!ok) return;
      tc_fence_after();
      const uint32_t lo = (2 * g) % entries, hi = (2 * g + 1) % entries, d = tmem_o + 64 * buf;
      const uint32_t cl = row_word(ring + lo * kPart + x * kStepBox, kStepBox);
      const uint32_t chi = row_word(ring + hi * kPart + x * kStepBox, kStepBox);
      if (leader) {
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k) {
          umma_ts(d, p + k * kSplitStep, cl + k * kRowStep, kSum, k != 0);
          umma_ts(d, p + k * kSplitStep + kSplitLo, chi + k * kRowStep, kSum, 1u);
          umma_ts(d, p + k * kSplitStep, chi + k * kRowStep, kSum, 1u);
        }
        umma_commit(o_full + 8 * buf);
      }
      __syncwarp();
    };
    auto free_step = [&](uint32_t g, uint32_t empty, uint32_t entries) {
      if (leader) {
        umma_commit(empty + 8 * ((2 * g) % entries));
        umma_commit(empty + 8 * ((2 * g + 1) % entries));
      }
      __syncwarp();
    };
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const GradItem t = grad_item<KEYS>(a, w, err);
      const int steps = __shfl_sync(0xffffffffu, t.f1 - t.f0, 0);
      if (steps <= 0) continue;
      ok = warp_wait(a_ready, item & 1, err);
      ++item;
      if (ok) product(gi, tmem_s, tmem, ring1, full1, kEntries1, s_full);
      if (ok) product(gi, tmem_d, tmem + DP, ring2, full2, kEntries2, d_full);
      if (ok && !KEYS) free_step(gi, empty2, kEntries2);
      for (int i = 0; i < steps && ok; ++i, ++gi) {
        const bool more = i + 1 < steps;
        ok = warp_wait(s_done, gi & 1, err);  // the scores have been read; keys: P is there
        if (!ok) break;
        tc_fence_after();
        if (KEYS) {
          sum_half(gi, tmem_s, ring2, kEntries2, 0, 0, sums0);
          if (kHalves == 2 && ok) sum_half(gi, tmem_s, ring2, kEntries2, 1, 1, sums1);
          if (ok) free_step(gi, empty2, kEntries2);
        }
        if (ok && more) product(gi + 1, tmem_s, tmem, ring1, full1, kEntries1, s_full);
        if (ok) ok = warp_wait(ds_full, gi & 1, err);
        if (!ok) break;
        tc_fence_after();
        if (kHalves == 2) {
          sum_half(gi, tmem_d, ring1, kEntries1, 0, 0, sums0);
          if (ok) sum_half(gi, tmem_d, ring1, kEntries1, 1, 1, sums1);
        } else {
          sum_half(gi, tmem_d, ring1, kEntries1, 0, 1, sums1);
        }
        if (ok) free_step(gi, empty1, kEntries1);
        if (ok && more) {
          product(gi + 1, tmem_d, tmem + DP, ring2, full2, kEntries2, d_full);
          if (ok && !KEYS) free_step(gi + 1, empty2, kEntries2);
        }
      }
    }
    if (!ok && leader) {  // instructions in flight end before the block does
      umma_commit(drained);
      mbar_wait(drained, 0, err);
    }
  } else if (warp < 8) {
    set_registers<kProbRegs<KEYS>>();
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, at_s = tmem_s + lanes + 32 * half, at_d = tmem_d + lanes + 32 * half;
    uint32_t gi = 0, item = 0;
    bool ok = true;
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const GradItem t = grad_item<KEYS>(a, w, err);
      if (t.f0 >= t.f1) continue;
      // The products with the resident tiles before are done: they have been read.
      ok = warp_wait(a_full, item & 1, err);
      if (!ok) break;
      rows_to_tmem<DP>(tmem + lanes, base, row, half);
      rows_to_tmem<DP>(tmem + DP + lanes, base + kTileBytes<DP>, row, half);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(a_ready), mbar_arrive(a_empty);
      ++item;
      // Queries: what the row sees and its statistics; keys: the rows [s0, s1)
      // that see the key, and its norm.
      RowMask mask = {0, 0, 0};
      float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      int s0 = 0, s1 = 0;
      float norm;
      if (!KEYS) {
        QueryItem q;
        q.rows = t.rows, q.sq = t.sq, q.r0 = t.r0;
        mask = mask_of(s, q, row);
        st = a.info[(int64_t)t.row_tile * kTile + row];
        norm = st.w;
      } else {
        if (t.r0 + row < t.sq.n) rows_seeing(s, t.sq, t.r0 + row, &s0, &s1);
        norm = a.nv[(int64_t)t.row_tile * kTile + row];
      }
      const double to_log2 = (double)(KEYS ? a.fk : a.fq)[t.row_tile] * (double)s.scale * 1.4426950408889634;
      const float f_row = KEYS ? a.fv[t.row_tile] : 0.0f;
      const bool one = t.sq.n == 1 || sees_one(s, 1);  // each row sees one key: no dS
      for (int n = t.f0; n < t.f1; ++n, ++gi) {
        int step;
        const int tile = column_tile(t, n, &step), c0 = step * kStep;
        const float f = unit_of(to_log2 * (double)(KEYS ? a.fq : a.fk)[tile]);
        const float f2 = KEYS ? f_row : a.fv[tile];  // of dP and delta in dO's units
        const float bound = norm * (KEYS ? a.tno : a.tnv)[tile] + (KEYS ? a.tdo[tile] : fabsf(st.z));
        const float up = KEYS && one ? 0.0f : power_of_two(scale_exponent(bound));
        bool whole;
        uint32_t seen;
        if (!KEYS) {
          whole = t.rows.all && c0 + kStep - 1 <= t.rows.p0 &&
                  (s.window == 0 || t.rows.p1 - c0 < s.window || c0 + kStep <= s.sinks);
          seen = seen_bits(mask, c0 + 32 * half);
        } else {
          const int first = t.sq.start + c0, last = first + kStep - 1, k1 = t.r0 + kTile - 1;
          whole = k1 <= first && last < t.sq.n && c0 + kStep <= s.q_len &&
                  (s.window == 0 || last - t.r0 < s.window || k1 < s.sinks);
          seen = bits_between(s0, s1, c0 + 32 * half);
        }
        ok = warp_wait(s_full, gi & 1, err);
        if (KEYS && ok) {  // the statistics' copy, with the second half of its step
          const uint32_t entry = 2 * gi + 1;
          ok = warp_wait(full1 + 8 * (entry % kEntries1), (entry / kEntries1) & 1, err);
        }
        if (!ok) break;
        tc_fence_after();
        const float2* col = (const float2*)(info_smem + (gi & 1) * (kStep * 8)) + 32 * half;
        float v[32];
        tmem_ld32(at_s, v);
        if (!KEYS) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_done);
        }
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(seen >> e & 1u)) v[e] = -INFINITY;
        }
        // Keys: 2^14 P, the 2^14 / sum and the greatest score in one exponent.
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = fmaf(v[e], f, KEYS ? -col[e].x : -st.x);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = exp2_fast(v[e]);
        if (KEYS) {
          store_split16(at_s, v);
          store_split16(at_s + 16, v + 16);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_done);
        }
        const float rescale = KEYS ? up * 0x1p-14f : up * st.y;
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] *= rescale;
        ok = warp_wait(d_full, gi & 1, err);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
          float d[16];
          tmem_ld16(at_d + c, d);
#pragma unroll
          for (int e = 0; e < 16; ++e) d[e] = fmaf(d[e], f2, KEYS ? -col[c + e].y : -st.z);
#pragma unroll
          for (int e = 0; e < 16; ++e) d[e] *= v[c + e];
          store_split16(at_d + c, d);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_full);
      }
    }
  } else {
    set_registers<kSumRegs<KEYS>>();
    constexpr int kCols = DP / 2;  // columns of a thread
    const int half = (warp - 8) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t taken0 = 0, taken1 = 0;  // sums taken from each buffer
    bool ok = true;
    // acc += by * the next sums of buffer `buf`.
    auto take = [&](float (&acc)[kCols], float by, uint32_t buf, uint32_t& taken) {
      ok = warp_wait(o_full + 8 * buf, taken & 1, err);
      ++taken;
      if (!ok) return;
      tc_fence_after();
      const uint32_t at = tmem_o + lanes + 64 * buf + (kHalves == 2 ? 0 : half * kCols);
#pragma unroll
      for (int c = 0; c < kCols; c += 8) {
        float v[8];
        tmem_ld8(at + c, v);
        if (c == kCols - 8) {  // the last values are out: the buffer is free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(o_empty + 8 * buf);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[c + e] = fmaf(v[e], by, acc[c + e]);
      }
    };
    for (int round = 0, w; ok && item_of(round, items, &w); ++round) {
      if (w < 0) continue;
      const GradItem t = grad_item<KEYS>(a, w, err);
      if (t.segs > 1 && threadIdx.x == 8 * 32) a.steps[w] = t.f1 - t.f0;
      if (t.f0 >= t.f1) continue;
      const float4 st = KEYS ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : a.info[(int64_t)t.row_tile * kTile + row];
      const float norm = KEYS ? a.nv[(int64_t)t.row_tile * kTile + row] : st.w;
      const double unit = a.scale_power * (KEYS ? 1.0 : (double)a.fo[t.row_tile]);
      float acc[kCols], acc_v[kCols];  // acc_v: keys only
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[c] = acc_v[c] = 0.0f;
      for (int n = t.f0; n < t.f1 && ok; ++n) {
        int step;
        const int tile = column_tile(t, n, &step);
        const float bound = norm * (KEYS ? a.tno : a.tnv)[tile] + (KEYS ? a.tdo[tile] : fabsf(st.z));
        // The call's scale goes here: k (or q) times the scale is of a size that fits,
        // as the scores are, where dS times k alone may not be.
        const float down = (float)((double)power_of_two(-scale_exponent(bound)) * unit *
                                   ((double)(KEYS ? a.fq : a.fk)[tile] * (KEYS ? (double)a.fo[tile] : 1.0)));
        if (KEYS) {
          const float down_v = 0x1p-14f * a.fo[tile];
          if (kHalves == 1 || half == 0) take(acc_v, down_v, 0, taken0);
          else take(acc_v, down_v, 1, taken1);
          if (!ok) break;
        }
        if (kHalves == 2 && half == 0) take(acc, down, 0, taken0);
        else take(acc, down, 1, taken1);
      }
      const int r = t.r0 + row, cols = s.head_dim - half * kCols;
      if (ok && t.segs > 1) {
        float* dst = a.part + ((int64_t)w * (KEYS ? 2 : 1) * kTile + row) * DP + half * kCols;
        store_row(dst, acc, a.scale_rest, kCols, true, 0);
        if (KEYS) store_row(dst + kTile * DP, acc_v, 1.0f, kCols, true, 0);
      } else if (ok && KEYS && r < s.k_len) {
        const int64_t at = row_at(s, t.b, t.g, r, s.kv_heads, s.k_len) + half * kCols;
        store_row(a.dk + at, acc, a.scale_rest, cols, s.head_dim % 4 == 0 && ((uintptr_t)a.dk & 15) == 0, a.add_k);
        store_row(a.dv + at, acc_v, 1.0f, cols, s.head_dim % 4 == 0 && ((uintptr_t)a.dv & 15) == 0, a.add_v);
      } else if (ok && !KEYS && r < s.q_len) {
        store_row(a.dq + row_at(s, t.b, t.h, r, s.heads, s.q_len) + half * kCols, acc, a.scale_rest, cols,
                  s.head_dim % 4 == 0 && ((uintptr_t)a.dq & 15) == 0, a.add_q);
      }
      __syncwarp();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Tiles whose segments are joined: `tiles` of them, the first with unit `first`,
// a tile's next segment `stride` units on; `rows` rows per block.
struct JoinSet {
  int tiles, first, segs, stride, rows;
  __host__ __device__ int blocks() const { return segs > 1 ? tiles * (kTile / rows) : 0; }
};

// Adds the segments of one tile in a fixed order, few rows per block: very few
// for a sink tile, whose many segments few blocks would read one after the other.
// Threads that a block's rows leave over share the segments.
template <int DP, bool KEYS>
__global__ void __launch_bounds__(256) grad_join_kernel(GradArgs a, JoinSet one, JoinSet two) {
  constexpr int kGrads = KEYS ? 2 : 1;
  __shared__ float4 slices[256];
  const AttentionShape& s = a.s;
  const bool is_two = (int)blockIdx.x >= one.blocks();
  const JoinSet set = is_two ? two : one;
  const int block = (int)blockIdx.x - (is_two ? one.blocks() : 0), rows = set.rows, segs = set.segs, stride = set.stride;
  const int tile = block / (kTile / rows), row0 = block % (kTile / rows) * rows;
  const int unit = set.first + tile / stride * segs * stride + tile % stride;
  int seg;
  const GradItem t = grad_place<KEYS>(a, unit, &seg);
  const int used = segments_used(a.steps + unit, segs, stride);
  if (used == 0) return;  // written key by key
  const int items = kGrads * rows * DP / 4, count = items < 256 ? 256 / items : 1;  // slices of the segments
  for (int i0 = 0; i0 < items; i0 += 256) {
    // items is a power of two from 32 to 512.
    const int i = i0 + (items < 256 ? threadIdx.x % items : threadIdx.x), slice = items < 256 ? threadIdx.x / items : 0;
    const int which = i / (rows * DP / 4), r = row0 + i / (DP / 4) % rows, c = i % (DP / 4) * 4;
    float v[4] = {};
#pragma unroll 8
    for (int k = slice; k < used; k += count) {
      const float4 p =
          *(const float4*)(a.part + (((int64_t)(unit + k * stride) * kGrads + which) * kTile + r) * DP + c);
      v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
    }
    if (count > 1) {
      slices[threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
      __syncthreads();
      if (slice != 0) return;
      for (int k = 1; k < count; ++k) {
        const float4 p = slices[threadIdx.x + k * items];
        v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
      }
    }
    if (t.r0 + r >= (KEYS ? s.k_len : s.q_len) || c >= s.head_dim) continue;
    float* grad = !KEYS ? a.dq : which ? a.dv : a.dk;
    const int64_t at = KEYS ? row_at(s, t.b, t.g, t.r0 + r, s.kv_heads, s.k_len)
                            : row_at(s, t.b, t.h, t.r0 + r, s.heads, s.q_len);
    store_row(grad + at + c, v, 1.0f, s.head_dim - c, s.head_dim % 4 == 0 && ((uintptr_t)grad & 15) == 0,
              !KEYS ? a.add_q : which ? a.add_v : a.add_k);
  }
}

// ---- a few query rows over a long cache ----------------------------------------------------

// The rows that share a key head, R at a time, go over its keys straight from the
// fp32 cache: with so few rows the reads bound it, not the products.  The keys
// are split over `splits` blocks; each warp takes 8 keys at a time, eight lanes
// per key with 4 NI columns each, and each group of eight lanes keeps a running
// maximum, sum and output of its own, so that only the dot products cross lanes.
// Groups, warps and splits are joined at the end in a fixed order.  `sets` blocks
// of R rows each read the same keys side by side, all but the first from L2.
//
// HBM bounds it up to four rows: 4 heads over each of 4, 128 wide, four sequences of
// up to 32768 keys, 416 MB in 77 to 88 us = 4.7 to 5.4 TB/s of 6.5 (the longest
// sequence's blocks end last); 32 sequences with a window of 1024, 122 MB in 33 us:
// a wave of 256 blocks, each a start, 17 steps and an end.  Eight rows take 131 us
// where four take 98: two blocks of four warps per SM wait for their own arithmetic.
constexpr int kDecodeThreads = 128;
constexpr int kDecodeRows = 8;
constexpr int kDecodeStages = 3;

__device__ __forceinline__ void copy16(float* to, const float* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}

// Two fp32 values in one 64-bit register: one instruction multiplies and adds both.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float first_of(uint64_t p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float second_of(uint64_t p) { return __uint_as_float((uint32_t)(p >> 32)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
constexpr int kMostSplits = 512;

// The keys that some row of a sequence sees: [0, first) and `count` - first
// more from `low` on.
struct SeenKeys {
  int first, low, count;
};
__device__ __forceinline__ SeenKeys keys_of(const AttentionShape& s, const Sequence& q) {
  const int a = max(q.start, 0), z = min(q.start + s.q_len, q.n);  // live positions [a, z)
  if (a >= z) return {0, 0, 0};
  const int low = s.window > 0 ? max(a + 1 - s.window, 0) : 0;
  const int first = s.window > 0 ? min(s.sinks, low) : 0;
  return {first, low, first + z - low};
}

// A row whose output came out infinite or NaN, key by key: a sum of values near
// fp32's greatest passes it where their mean does not.
// (Not inlined: its registers would be the loops'.)
__device__ __noinline__ void one_row_again(const AttentionShape& s, int start, int n, const float* q, const float* k,
                                           const float* v, float* out, float* stats, int b, int h, int r) {
  simple_forward_row(s, {start, n}, q, k, v, out, stats, b, h, r);
}

// Blocks per SM that the compiler keeps registers for (0: as it likes), where that was
// faster: four rows, four sequences of 32768 keys, 128 wide 98 us (100 without), 127
// wide 138 (160); one row, 127 wide, 101 (108).
template <int R>
constexpr int kDecodeBlocks = R == 1 ? 4 : R == 4 ? 2 : 0;

// WHOLE: the keys are in one part, and this kernel writes the output.  (A kernel of
// its own: with a call of one_row_again in it the loops of the others take longer,
// 87 us instead of 85 for four sequences of up to 32768 keys.)
template <int NI, int R, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(kDecodeThreads, kDecodeBlocks<R>) decode_kernel(const __grid_constant__ AttentionShape s, const float* __restrict__ q,
                                                                const float* __restrict__ k,
                                                                const float* __restrict__ v, float* __restrict__ out,
                                                                float* __restrict__ stats, float* __restrict__ part,
                                                                int sets, int splits, int per, int* err) {
  constexpr int kDims = 32 * NI, kWarps = kDecodeThreads / 32;
  __shared__ __align__(16) float qs[R][kDims];
  __shared__ uint32_t again;  // WHOLE: rows whose sums have left fp32
  if (WHOLE && threadIdx.x == 0) again = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, key_of = warp * 4 + (lane >> 3);
  int64_t index = blockIdx.x;
  const int row0 = (int)(index % sets) * R;
  index /= sets;
  const int split = (int)(index % splits);
  index /= splits;
  const int g = (int)(index % s.kv_heads), b = (int)(index / s.kv_heads);
  const int group = s.heads / s.kv_heads, total = group * s.q_len;
  const Sequence sq = sequence_of(s, b, err);
  const SeenKeys seen = keys_of(s, sq);
  const int first = seen.first, low = seen.low, keys = seen.count;
  const int u0 = min(keys, split * per), u1 = min(keys, u0 + per);
  if (!WHOLE && u0 == u1 && split > 0) return;  // the join knows how many splits hold keys
  const float to_log2 = s.scale * kLog2e;
  for (int i = threadIdx.x; i < R * kDims; i += kDecodeThreads) {
    const int r = row0 + i / kDims, c = i % kDims;
    qs[i / kDims][c] = r < total && c < s.head_dim
                           ? q[row_at(s, b, g * group + r / s.q_len, r % s.q_len, s.heads, s.q_len) + c]
                           : 0.0f;
  }
  int at[R];  // position of each row; below 0: not a row, or not in the sequence
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = sq.start + (row0 + r) % s.q_len;
    at[r] = row0 + r < total && p < sq.n ? p : -1;
  }
  __syncthreads();
  float m[R], l[R];
  uint64_t acc[R][2 * NI];  // pairs of values
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < 2 * NI; ++c) acc[r][c] = 0;
  }
  const int64_t step = s.seq_major ? (int64_t)s.kv_heads * s.head_dim : s.head_dim;
  const int64_t base = row_at(s, b, g, 0, s.kv_heads, s.k_len);
  // A lane's 4 NI values of two keys and values per step of the loop, VEC: from
  // a ring that the lane fills for itself two steps ahead, so that loads stay in
  // flight while it computes; otherwise straight from memory.
  // Two blocks per SM fit only because the warps' results take the ring's place.
  extern __shared__ __align__(16) float ring[];  // [warps][kDecodeStages][K, V][2][4][kDims]
  auto joined = (float(*)[R][kDims + 2])ring;    // [warps]
  float* mine = ring + ((size_t)warp * kDecodeStages * 16 + (lane >> 3)) * kDims + 4 * l8;
  auto key_at = [&](int u) { return u < first ? u : low + u - first; };
  auto copy = [&](int it) {
    if (VEC) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int u = u0 + key_of + it * 8 * kWarps + w * 4 * kWarps;
        if (u >= u1) continue;
        const int64_t from = base + key_at(u) * step + 4 * l8;
        float* to = mine + (it % kDecodeStages * 16 + w * 4) * kDims;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (4 * l8 + 32 * i < s.head_dim) {
            copy16(to + 32 * i, k + from + 32 * i);
            copy16(to + 8 * kDims + 32 * i, v + from + 32 * i);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  auto load = [&](const float* __restrict__ x, int it, int which, int w, uint64_t (&d)[2 * NI]) {
    const int u = u0 + key_of + it * 8 * kWarps + w * 4 * kWarps;
    const float* src = VEC ? mine + (it % kDecodeStages * 16 + which * 8 + w * 4) * kDims
                           : x + base + key_at(min(u, u1 - 1)) * step + 4 * l8;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = 4 * l8 + 32 * i;
      if (VEC) {
        const ulonglong2 f = u < u1 && c < s.head_dim ? *(const ulonglong2*)(src + 32 * i) : make_ulonglong2(0, 0);
        d[2 * i] = f.x, d[2 * i + 1] = f.y;
      } else {
        float e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = u < u1 && c + k < s.head_dim ? __ldg(src + 32 * i + k) : 0.0f;
        d[2 * i] = pair_of(e[0], e[1]), d[2 * i + 1] = pair_of(e[2], e[3]);
      }
    }
  };
  const int steps = u1 > u0 ? (u1 - u0 + 8 * kWarps - 1) / (8 * kWarps) : 0;
  for (int it = 0; it < kDecodeStages - 1; ++it) copy(it);
  for (int it = 0; it < steps; ++it) {
    copy(it + kDecodeStages - 1);
    if (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(kDecodeStages - 1) : "memory");
    const int u = u0 + key_of + it * 8 * kWarps;
    const bool one = u < u1, two = u + 4 * kWarps < u1;
    const int j[2] = {key_at(u), key_at(u + 4 * kWarps)};
    uint64_t kd[2][2 * NI], vd[2][2 * NI];
    load(k, it, 0, 0, kd[0]);
    load(k, it, 0, 1, kd[1]);
    float d[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t x[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const ulonglong2 f = *(const ulonglong2*)&qs[r][4 * l8 + 32 * i];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          x[w] = fma_pair(f.x, kd[w][2 * i], x[w]);
          x[w] = fma_pair(f.y, kd[w][2 * i + 1], x[w]);
        }
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) d[r][w] = first_of(x[w]) + second_of(x[w]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        d[r][0] += __shfl_xor_sync(0xffffffffu, d[r][0], o);
        d[r][1] += __shfl_xor_sync(0xffffffffu, d[r][1], o);
      }
    }
    load(v, it, 1, 0, vd[0]);
    load(v, it, 1, 1, vd[1]);
    uint32_t seen_rows = 0;  // two bits per row
    float top[R];
    bool up = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      bool sees[2] = {one, two};
      if (s.q_len > 1)
#pragma unroll
        for (int w = 0; w < 2; ++w)
          sees[w] = sees[w] && j[w] <= at[r] && (s.window == 0 || at[r] - j[w] < s.window || j[w] < s.sinks);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        d[r][w] = sees[w] ? d[r][w] * to_log2 : -INFINITY;
        seen_rows |= (uint32_t)sees[w] << (2 * r + w);
      }
      top[r] = fmaxf(m[r], fmaxf(d[r][0], d[r][1]));
      up |= top[r] > m[r];
    }
    if (up) {  // seldom after the first keys; one branch for all rows
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float keep = top[r] == m[r] ? 1.0f : exp2_fast(m[r] - top[r]);
        m[r] = top[r];
        l[r] *= keep;
        const uint64_t both = pair_of(keep, keep);
#pragma unroll
        for (int c = 0; c < 2 * NI; ++c) acc[r][c] = fma_pair(acc[r][c], both, 0);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float ref = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
      for (int w = 0; w < 2; ++w) d[r][w] = exp2_fast(d[r][w] - ref);  // 0 where hidden
      l[r] += d[r][0] + d[r][1];
    }
    if (s.q_len == 1) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint64_t both = pair_of(d[r][w], d[r][w]);
#pragma unroll
          for (int c = 0; c < 2 * NI; ++c) acc[r][c] = fma_pair(both, vd[w][c], acc[r][c]);
        }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int w = 0; w < 2; ++w)
          if (seen_rows >> (2 * r + w) & 1u) {  // a hidden value takes no part, not even times 0
            const uint64_t both = pair_of(d[r][w], d[r][w]);
#pragma unroll
            for (int c = 0; c < 2 * NI; ++c) acc[r][c] = fma_pair(both, vd[w][c], acc[r][c]);
          }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = m[r];
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float w = m[r] == -INFINITY ? (l[r] == 0.0f ? 0.0f : 1.0f) : exp2_fast(m[r] - top);
    float sum = l[r] * w;
    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
    for (int c = 0; c < 4 * NI; ++c) {
      float x = (c & 1 ? second_of(acc[r][c / 2]) : first_of(acc[r][c / 2])) * w;
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (lane < 8) joined[warp][r][4 * l8 + 32 * (c / 4) + c % 4] = x;
    }
    if (lane == 0) joined[warp][r][kDims] = top, joined[warp][r][kDims + 1] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * kDims; i += kDecodeThreads) {
    const int r = i / kDims, c = i % kDims;
    if (row0 + r >= total || c >= s.head_dim) continue;
    const int h = g * group + (row0 + r) / s.q_len, qr = (row0 + r) % s.q_len;
    float top = -INFINITY, sum = 0.0f, x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, joined[w][r][kDims]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float one = joined[w][r][kDims] == top ? 1.0f : exp2_fast(joined[w][r][kDims] - top);
      sum += joined[w][r][kDims + 1] * one;
      x += joined[w][r][c] * one;
    }
    const int64_t line = ((int64_t)b * s.heads + h) * s.q_len + qr;
    if (WHOLE) {
      const float o = sum == 0.0f ? 0.0f : x / sum;
      if (!isfinite(o)) atomicOr(&again, 1u << r);
      out[row_at(s, b, h, qr, s.heads, s.q_len) + c] = o;
      if (stats != nullptr && c == 0) *(float2*)(stats + 2 * line) = natural_stats(top, sum);
    } else {
      float* dst = part + (line * splits + split) * (s.head_dim + 2);
      dst[2 + c] = x;
      if (c == 0) dst[0] = top, dst[1] = sum;
    }
  }
  if (!WHOLE) return;
  __syncthreads();
  for (int r = warp; r < R; r += kWarps)
    if (WHOLE && again >> r & 1u)
      one_row_again(s, sq.start, sq.n, q, k, v, out, stats, b, g * group + (row0 + r) / s.q_len, (row0 + r) % s.q_len);
}

// One block per row joins its splits: each warp takes every fourth, the warps'
// parts are added in order.
__global__ void __launch_bounds__(128) decode_join_kernel(AttentionShape s, const float* __restrict__ q,
                                                          const float* __restrict__ k, const float* __restrict__ v,
                                                          const float* __restrict__ part, float* __restrict__ out,
                                                          float* __restrict__ stats, int splits, int per, int* err) {
  __shared__ float weight[kMostSplits], joined[4][kMaxHeadDim], tops[4], sums[4];
  const int64_t line = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = (int)(line % s.q_len), h = (int)(line / s.q_len % s.heads), b = (int)(line / s.q_len / s.heads);
  const Sequence sq = sequence_of(s, b, err);
  const int used = max(1, (keys_of(s, sq).count + per - 1) / per);
  const float* src = part + line * splits * (s.head_dim + 2);
  float top = -INFINITY;
  for (int i = threadIdx.x; i < used; i += 128) top = fmaxf(top, weight[i] = src[(int64_t)i * (s.head_dim + 2)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  float sum = 0.0f, x[kLaneDims] = {};
#pragma unroll 4
  for (int i = warp; i < used; i += 4) {
    const float* p = src + (int64_t)i * (s.head_dim + 2);
    const float one = weight[i] == top ? 1.0f : exp2_fast(weight[i] - top);
    sum += p[1] * one;
#pragma unroll
    for (int d = 0; d < kLaneDims; ++d)
      if (lane + 32 * d < s.head_dim) x[d] += p[2 + lane + 32 * d] * one;
  }
#pragma unroll
  for (int d = 0; d < kLaneDims; ++d) joined[warp][lane + 32 * d] = x[d];
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const int c = threadIdx.x;
  float o = 0.0f;
  if (c < s.head_dim) {
    o = (joined[0][c] + joined[1][c]) + (joined[2][c] + joined[3][c]);
    o = sum == 0.0f ? 0.0f : o / sum;
    out[row_at(s, b, h, r, s.heads, s.q_len) + c] = o;
  }
  if (stats != nullptr && c == 0) *(float2*)(stats + 2 * line) = natural_stats(top, sum);
  if (__syncthreads_or(!isfinite(o)) && warp == 0) simple_forward_row(s, sq, q, k, v, out, stats, b, h, r);
}

}  // namespace

namespace {

// Sections of the workspace, in floats, each on a 256-byte boundary.
struct Carver {
  float* base;
  int64_t used = 0;
  float* take(int64_t floats) {
    float* p = base ? base + used : nullptr;
    used += (floats + 63) / 64 * 64;
    return p;
  }
};

constexpr int64_t kSms = 148;

// Lets a kernel take `bytes` of dynamic shared memory, once per device.
template <typename K>
void allow_shared(K* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  TYSOR_CUDA(cudaGetDevice(&device));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return;
  TYSOR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_release);
}

int padded_dim(const AttentionShape& s) { return s.head_dim <= 64 ? 64 : 128; }

struct ForwardWork {
  uint8_t *pq, *pk, *pv;
  float *fq, *fk, *fv, *tnq, *tnk, *part;
  float2* part_ml;
  Sequence* seqs;
  int *steps, segs;
  int64_t floats;
};
// Segments of a query tile's key tiles, of at least `least` tiles each: one unit
// per SM where the items are about alike (a window, or few queries over a long
// cache), two where the first queries see few keys and the last ones all.
// Measured, 128 wide, whole / one per SM / two: 5 queries of 5 heads over 65536
// keys of one 1074 / 98 / 116 us, 128 queries of 8 heads over as many 1179 / 279
// / 299; 8192 over themselves, one head, 148 / 96 / 73, 4096 of four 88 / 88 / 74.
// At least four: 4000 keys, 5 queries of 20 heads, 40 us (two 51, eight 44); of
// the gradients' pass two, as a tile is two steps: 2000 tokens, window 512, two
// heads, forward and backward 112 us (four 116, one 128).
int segments_of_queries(const AttentionShape& s, int least) {
  const int64_t items = (int64_t)s.batch * s.heads * tiles_of(s.q_len);
  int64_t most = tiles_of(s.k_len);
  if (s.window > 0)
    most = std::min<int64_t>(most, ((int64_t)s.window + kTile - 2) / kTile + 1 + tiles_of(std::min(s.sinks, s.k_len)));
  if (items == 0) return 1;
  const int per_sm = s.window > 0 || s.q_len <= s.k_len / 2 ? 1 : 2;
  return (int)std::max<int64_t>(1, std::min(most / least, kSms * per_sm / items));
}
ForwardWork forward_work(const AttentionShape& s, float* base) {
  Carver c{base};
  const int64_t tile = padded_dim(s) == 64 ? kTileBytes<64> / 4 : kTileBytes<128> / 4;
  const int64_t nq = (int64_t)s.batch * s.heads * tiles_of(s.q_len), nk = (int64_t)s.batch * s.kv_heads * tiles_of(s.k_len);
  ForwardWork w;
  w.pq = (uint8_t*)c.take(nq * tile);
  w.pk = (uint8_t*)c.take(nk * tile);
  w.pv = (uint8_t*)c.take(nk * tile);
  w.fq = c.take(nq);
  w.fk = c.take(nk);
  w.fv = c.take(nk);
  w.tnq = c.take(nq);
  w.tnk = c.take(nk);
  w.seqs = (Sequence*)c.take(2 * (int64_t)s.batch);
  w.segs = segments_of_queries(s, 4);
  w.part = c.take(w.segs > 1 ? nq * w.segs * kTile * padded_dim(s) : 0);
  w.part_ml = (float2*)c.take(w.segs > 1 ? nq * w.segs * kTile * 2 : 0);
  w.steps = (int*)c.take(w.segs > 1 ? nq * w.segs : 0);
  w.floats = c.used;
  return w;
}

// decode_kernel or the tiles: the first reads a key head's keys once per eight of
// its rows, the second packs them once and walks them once per 128 rows of a
// query head.  Measured, decode / tiles, 128 wide: one query of 9 heads over one,
// four such groups and sequences of 32768 keys, 267 / 705 us, of 16 heads 280 /
// 1272; 5 queries of 2 heads over one, 80 wide, four such and 8000 keys, 79 / 97,
// of 4 heads, eight such and 8192 keys, 253 / 228 (the rule has these go through
// decode, 11% slower; one that sent them to the tiles would send 5 of 2 heads there
// too, 23% slower); 9 queries and more of one head take the tiles (16 over 8000 keys
// of 6 heads 54).
bool uses_tiles(const AttentionShape& s) {
  const int64_t group = s.heads / s.kv_heads;
  return 2 * ceil_div(group * s.q_len, kDecodeRows) > 2 + group * tiles_of(s.q_len);
}

struct DecodePlan {
  int rows, sets, splits, per;
};
DecodePlan decode_plan(const AttentionShape& s) {
  DecodePlan p;
  const int64_t total = (int64_t)s.q_len * (s.heads / s.kv_heads);
  p.rows = total == 1 ? 1 : total <= 4 ? 4 : kDecodeRows;
  p.sets = (int)ceil_div(total, p.rows);
  // Each split takes the same number of keys, whatever its sequence's length:
  // about four blocks per SM at full length, at least 384 keys each.  Measured
  // for one token, 16 heads over 4, 128 wide: four sequences of up to 32768 keys
  // 83 us (two blocks per SM 89, six 88, twelve 93), 32 sequences with a window
  // of 1024 41 us (at least 512 keys 41, 256 keys 47 to 49).
  int64_t most = s.k_len;
  if (s.window > 0) most = std::min<int64_t>(most, (int64_t)s.window + s.sinks + s.q_len - 1);
  const int64_t blocks = (int64_t)s.batch * s.kv_heads * p.sets;
  const int64_t want = std::max<int64_t>(1, std::min(ceil_div(kSms * 4, blocks > 0 ? blocks : 1), most / 384));
  p.per = (int)(ceil_div(std::max<int64_t>(1, ceil_div(most, std::min<int64_t>(want, kMostSplits))), 32) * 32);
  p.splits = (int)std::max<int64_t>(1, ceil_div(most, p.per));
  return p;
}
int64_t decode_work_elems(const AttentionShape& s) {
  const DecodePlan p = decode_plan(s);
  if (p.splits == 1) return 1;
  return (int64_t)s.batch * s.heads * s.q_len * p.splits * (s.head_dim + 2);
}

template <int NI, int R, bool WHOLE>
void run_decode(const AttentionShape& s, const DecodePlan& p, const float* q, const float* k, const float* v, float* out,
                float* stats, float* part, int* err, cudaStream_t st) {
  const int64_t blocks = (int64_t)s.batch * s.kv_heads * p.sets * p.splits;
  if (blocks > INT_MAX) throw CudaError("window_attention: too many rows");
  const bool vec = s.head_dim % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  constexpr int kRing = kDecodeThreads / 32 * kDecodeStages * 16 * 32 * NI * (int)sizeof(float);
  constexpr int kJoined = kDecodeThreads / 32 * R * (32 * NI + 2) * (int)sizeof(float);  // below 48 KB
  static_assert(kJoined <= kRing, "the ring holds the results");
  static std::atomic<uint64_t> done{0};
  if (vec) allow_shared(decode_kernel<NI, R, true, WHOLE>, kRing, done);
  if (vec)
    decode_kernel<NI, R, true, WHOLE><<<(unsigned)blocks, kDecodeThreads, kRing, st>>>(s, q, k, v, out, stats, part, p.sets, p.splits, p.per, err);
  else
    decode_kernel<NI, R, false, WHOLE><<<(unsigned)blocks, kDecodeThreads, kJoined, st>>>(s, q, k, v, out, stats, part, p.sets, p.splits, p.per, err);
  check_launch();
}
template <int NI>
void run_decode_rows(const AttentionShape& s, const DecodePlan& p, const float* q, const float* k, const float* v,
                     float* out, float* stats, float* part, int* err, cudaStream_t st) {
  auto run = [&](auto whole) {
    if (p.rows == 1) run_decode<NI, 1, whole.value>(s, p, q, k, v, out, stats, part, err, st);
    else if (p.rows == 4) run_decode<NI, 4, whole.value>(s, p, q, k, v, out, stats, part, err, st);
    else run_decode<NI, kDecodeRows, whole.value>(s, p, q, k, v, out, stats, part, err, st);
  };
  if (p.splits == 1) run(std::true_type{});
  else run(std::false_type{});
}

void run_pack(const AttentionShape& s, PackJob (&jobs)[4], int count, Sequence* seqs, int* err, cudaStream_t st) {
  PackJobs p{};
  p.s = s;
  p.far = far_exponent(std::max(s.q_len, s.k_len));
  p.seqs = seqs;
  int64_t at = 0;
  for (int i = 0; i < 4; ++i) {
    p.first[i] = i < count ? (int)at : INT_MAX;
    if (i >= count) continue;
    p.job[i] = jobs[i];
    at += (int64_t)s.batch * jobs[i].heads * tiles_of(jobs[i].len);
  }
  if (at > INT_MAX) throw CudaError("window_attention: too many rows");
  if (padded_dim(s) == 64) pack_kernel<64><<<(unsigned)at, 256, 0, st>>>(p, err);
  else pack_kernel<128><<<(unsigned)at, 256, 0, st>>>(p, err);
  check_launch();
}

struct GradWork {
  uint8_t *pq, *pk, *pv, *po;
  float *fq, *fk, *fv, *fo, *tnq, *tnk, *nv, *tnv, *tno, *tdo;
  float4* info;
  float2 *col, *own;
  Sequence* seqs;
  int* steps;
  float* part;
  int64_t floats;
};

// Segments of a key tile's steps: sixteen steps each, more where that would make
// over three units per SM (each unit's part is written and read once more), and
// fewer, down to four, where it would leave SMs idle.  Measured, forward and
// backward, 128 wide: eight units per SM instead of three, 2048 tokens of 8
// sequences, 16 heads over 4, 2323 / 2023 us, the same of 4096 tokens and 2
// sequences with a window of 512 852 / 803 (two 799, four 765); always sixteen
// steps instead of four, 600 tokens of 8 heads over 2 138 / 109, 128 queries of 2
// heads over 4096 keys of one 191 / 97.
Segments segments_of(const AttentionShape& s) {
  const int64_t group = s.heads / s.kv_heads, all = ceil_div(s.q_len, kStep);
  const int64_t some = s.window > 0 ? std::min<int64_t>(all, ((int64_t)s.window + kTile + 2 * kStep - 3) / kStep) : all;
  Segments g;
  const int tiles = tiles_of(s.k_len);
  g.long_tiles = s.window > 0 ? std::min(tiles, tiles_of(std::min(s.sinks, s.k_len))) : tiles;
  // Without a window a tile's steps are half of all on average.
  const int64_t steps = (s.window > 0 ? g.long_tiles * all : tiles * all / 2) + (tiles - g.long_tiles) * some;
  const int64_t work = steps * group * s.batch * s.kv_heads;
  const int64_t each = std::max(std::min<int64_t>(16, std::max<int64_t>(4, work / kSms)), work / (kSms * 3));
  g.long_segs = (int)std::min<int64_t>(64, std::max<int64_t>(1, group * all / each));
  g.short_segs = (int)std::min<int64_t>(64, std::max<int64_t>(1, group * some / each));
  g.query_segs = segments_of_queries(s, 2);
  return g;
}
int64_t grad_units(const AttentionShape& s, const Segments& g) {
  const int64_t tiles = tiles_of(s.k_len);
  return (g.long_tiles * (int64_t)g.long_segs + (tiles - g.long_tiles) * g.short_segs) * s.kv_heads * s.batch;
}

GradWork grad_work(const AttentionShape& s, float* base) {
  Carver c{base};
  const int64_t tile = padded_dim(s) == 64 ? kTileBytes<64> / 4 : kTileBytes<128> / 4;
  const int64_t nq = (int64_t)s.batch * s.heads * tiles_of(s.q_len), nk = (int64_t)s.batch * s.kv_heads * tiles_of(s.k_len);
  GradWork w;
  w.pq = (uint8_t*)c.take(nq * tile);
  w.po = (uint8_t*)c.take(nq * tile);
  w.pk = (uint8_t*)c.take(nk * tile);
  w.pv = (uint8_t*)c.take(nk * tile);
  w.fq = c.take(nq);
  w.fo = c.take(nq);
  w.fk = c.take(nk);
  w.fv = c.take(nk);
  w.tnq = c.take(nq);
  w.tnk = c.take(nk);
  w.nv = c.take(nk * kTile);
  w.tnv = c.take(nk);
  w.tno = c.take(nq);
  w.tdo = c.take(nq);
  w.info = (float4*)c.take(nq * kTile * 4);
  w.col = (float2*)c.take(nq * kTile * 2);
  w.own = (float2*)c.take(nq * kTile * 2);
  w.seqs = (Sequence*)c.take(2 * (int64_t)s.batch);
  const Segments g = segments_of(s);
  // The queries' pass has joined its segments when the keys' begins.
  const int64_t for_keys = g.long_segs > 1 || g.short_segs > 1 ? grad_units(s, g) * 2 : 0;
  const int64_t for_queries = g.query_segs > 1 ? nq * g.query_segs : 0;
  w.steps = (int*)c.take(std::max<int64_t>(for_keys > 0 ? grad_units(s, g) : 0, for_queries));
  w.part = c.take(std::max(for_keys, for_queries) * kTile * padded_dim(s));
  w.floats = c.used;
  return w;
}

template <int DP, bool KEYS>
void run_grad(const GradArgs& a, int* err, cudaStream_t st) {
  constexpr int kSmem = GradPlan<DP, KEYS>::kSmem;
  static std::atomic<uint64_t> done{0};
  allow_shared(grad_kernel<DP, KEYS>, kSmem, done);
  const AttentionShape& s = a.s;
  const int64_t items = KEYS ? grad_units(s, a.seg) : (int64_t)tiles_of(s.q_len) * s.heads * s.batch * a.seg.query_segs;
  if (items == 0) return;
  if (items > INT_MAX / 64) throw CudaError("window_attention: too many rows");
  grad_kernel<DP, KEYS><<<(unsigned)(items < kSms ? items : kSms), kThreads, kSmem, st>>>(a, (int)items, err);
  check_launch();
  JoinSet one{0, 0, 1, 1, 8}, two{0, 0, 1, 1, 8};
  if (!KEYS) {
    one = {(int)(items / a.seg.query_segs), 0, a.seg.query_segs, 1, 8};
  } else {
    const int stride = s.kv_heads * s.batch, long_tiles = a.seg.long_tiles * stride;
    one = {long_tiles, 0, a.seg.long_segs, stride, s.window > 0 ? 2 : 8};
    two = {tiles_of(s.k_len) * stride - long_tiles, long_tiles * a.seg.long_segs, a.seg.short_segs, stride, 8};
  }
  if (one.blocks() + two.blocks() == 0) return;
  grad_join_kernel<DP, KEYS><<<one.blocks() + two.blocks(), 256, 0, st>>>(a, one, two);
  check_launch();
}

template <int DP>
void run_forward(const ForwardArgs& a, int* err, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  allow_shared(forward_kernel<DP>, ForwardPlan<DP>::kSmem, done);
  const int64_t items = (int64_t)tiles_of(a.s.q_len) * a.s.heads * a.s.batch;  // at most what run_pack took
  const int64_t units = items * a.segs;  // segs > 1: at most two per SM
  forward_kernel<DP><<<(unsigned)(units < kSms ? units : kSms), kThreads, ForwardPlan<DP>::kSmem, st>>>(
      a, (int)units, err);
  check_launch();
  if (a.segs == 1) return;
  forward_join_kernel<DP><<<(unsigned)(items * (kTile / kJoinRows)), 256, 0, st>>>(a);
  check_launch();
}

}  // namespace

int64_t window_attention_work_elems(const AttentionShape& s) {
  return uses_tiles(s) ? forward_work(s, nullptr).floats : decode_work_elems(s);
}
int64_t window_attention_backward_work_elems(const AttentionShape& s) {
  return grad_work(s, nullptr).floats;
}

void launch_window_attention(const AttentionShape& s, const float* q, const float* k, const float* v, float* out,
                             float* stats, float* work, int* err, cudaStream_t st) {
  const int64_t rows = (int64_t)s.batch * s.heads * s.q_len;
  if (rows <= 0) return;
  if (uses_tiles(s)) {
    const ForwardWork w = forward_work(s, work);
    PackJob jobs[4] = {{q, w.pq, w.fq, s.heads, s.q_len, 1, w.tnq},
                       {k, w.pk, w.fk, s.kv_heads, s.k_len, 0, w.tnk},
                       {v, w.pv, w.fv, s.kv_heads, s.k_len, 0}};
    run_pack(s, jobs, 3, w.seqs, err, st);
    const ForwardArgs a{s, q, k, v, w.pq, w.pk, w.pv, w.fq, w.fk, w.fv, w.tnq, w.tnk, w.seqs, out, stats, w.segs, w.steps, w.part, w.part_ml};
    if (padded_dim(s) == 64) run_forward<64>(a, err, st);
    else run_forward<128>(a, err, st);
    return;
  }
  const DecodePlan p = decode_plan(s);
  switch ((s.head_dim + 31) / 32) {
    case 1: run_decode_rows<1>(s, p, q, k, v, out, stats, work, err, st); break;
    case 2: run_decode_rows<2>(s, p, q, k, v, out, stats, work, err, st); break;
    case 3: run_decode_rows<3>(s, p, q, k, v, out, stats, work, err, st); break;
    default: run_decode_rows<4>(s, p, q, k, v, out, stats, work, err, st); break;
  }
  if (p.splits > 1) {
    if (rows > INT_MAX) throw CudaError("window_attention: too many rows");
    decode_join_kernel<<<(unsigned)rows, 128, 0, st>>>(s, q, k, v, work, out, stats, p.splits, p.per, err);
    check_launch();
  }
}

void launch_window_attention_backward(const AttentionShape& s, const float* q, const float* k, const float* v,
                                      const float* out, const float* stats, const float* dout, float* dq, float* dk,
                                      float* dv, float* work, int accumulate_q, int accumulate_k, int accumulate_v,
                                      int* err, cudaStream_t st) {
  if (s.batch == 0 || (s.q_len == 0 && s.k_len == 0)) return;
  const GradWork w = grad_work(s, work);
  PackJob jobs[4] = {{q, w.pq, w.fq, s.heads, s.q_len, 1, w.tnq},
                     {dout, w.po, w.fo, s.heads, s.q_len, 1, w.tno, nullptr, out, stats, w.info, w.own, w.col, w.tdo},
                     {k, w.pk, w.fk, s.kv_heads, s.k_len, 0, w.tnk},
                     {v, w.pv, w.fv, s.kv_heads, s.k_len, 0, w.tnv, w.nv}};
  run_pack(s, jobs, 4, w.seqs, err, st);
  int scale_exponent;
  const float scale_rest = 2.0f * frexpf(s.scale, &scale_exponent);
  const GradArgs a{s,     q,     k,      v,     out,   dout,  w.pq,  w.pk,  w.pv,  w.po,   w.fq,  w.fk, w.fv, w.fo,
                   w.tnq, w.tnk, w.seqs, w.nv,   w.tnv, w.tno, w.tdo, w.info, w.col, w.own, dq,     dk,    dv,   accumulate_q,
                   accumulate_k, accumulate_v, ldexp(1.0, scale_exponent - 1), scale_rest, segments_of(s), w.steps, w.part};
  if (padded_dim(s) == 64) {
    run_grad<64, false>(a, err, st);
    run_grad<64, true>(a, err, st);
  } else {
    run_grad<128, false>(a, err, st);
    run_grad<128, true>(a, err, st);
  }
}

}  // namespace tysor
