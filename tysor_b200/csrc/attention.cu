// Causal attention over a sliding window and the first keys (lm_ops.cuh),
// forward and backward.
#include <limits.h>
#include <math.h>

#include "lm_ops.cuh"

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

// First value of row `r` of head `h` of sequence `b`.
__device__ __forceinline__ int64_t row_at(const AttentionShape& s, int b, int h, int r, int heads, int len) {
  return (s.seq_major ? ((int64_t)b * len + r) * heads + h : ((int64_t)b * heads + h) * len + r) * s.head_dim;
}

// A sequence's keys [0, n) and its first query's position.
struct Sequence {
  int start, n;
};

__device__ __forceinline__ Sequence sequence_of(const AttentionShape& s, int b, int* err) {
  Sequence q{s.k_len - s.q_len, s.k_len};
  if (s.lengths != nullptr) {
    const float v = s.lengths[b];
    if (v >= 0.0f && v <= (float)s.k_len && (int64_t)v <= s.k_len) {
      q.n = (int)v;
    } else {
      q.n = 0;
      atomicCAS(err, 0, (int)kErrSequence);
    }
  }
  if (s.starts != nullptr) {
    const float v = s.starts[b];
    if (v > -1073741824.0f && v < 1073741824.0f) {
      q.start = (int)v;
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

__device__ __forceinline__ Seen seen_by(const AttentionShape& s, const Sequence& q, int64_t p) {
  if (p < 0 || p >= q.n) return {0, 0, 0};
  Seen v{0, 0, (int)p + 1};
  if (s.window > 0 && p + 1 > s.window) {
    v.low = (int)(p + 1 - s.window);
    v.first = min(s.sinks, v.low);
  }
  return v;
}

// ---- every shape and every value: one warp per row --------------------------------

// A row's values over a warp's lanes: lane l holds columns l, l + 32, ...
constexpr int kLaneDims = kMaxHeadDim / 32;

__device__ __forceinline__ void lane_load(const float* __restrict__ p, int dim, float (&v)[kLaneDims]) {
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) {
    const int c = (threadIdx.x & 31) + 32 * i;
    v[i] = c < dim ? p[c] : 0.0f;
  }
}

__device__ __forceinline__ void lane_store(float* __restrict__ p, int dim, const float (&v)[kLaneDims], float scale,
                                           int accumulate) {
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) {
    const int c = (threadIdx.x & 31) + 32 * i;
    if (c < dim) p[c] = accumulate ? p[c] + v[i] * scale : v[i] * scale;
  }
}

__device__ __forceinline__ float lane_dot(const float (&a)[kLaneDims], const float (&b)[kLaneDims]) {
  float d = 0.0f;
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) d += a[i] * b[i];
  return warp_sum(d);
}

__device__ void simple_forward_row(const AttentionShape& s, const Sequence& sq, const float* q, const float* k,
                                   const float* v, float* out, float* stats, int b, int h, int r) {
  const int g = h / (s.heads / s.kv_heads);
  const Seen seen = seen_by(s, sq, (int64_t)sq.start + r);
  float qv[kLaneDims], acc[kLaneDims] = {};
  lane_load(q + row_at(s, b, h, r, s.heads, s.q_len), s.head_dim, qv);
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < seen.high; ++j) {
    if (j == seen.first && j < seen.low) j = seen.low;
    float kv[kLaneDims];
    lane_load(k + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
    const float x = lane_dot(qv, kv) * s.scale;
    const float top = x > m || x != x ? x : m;
    const float keep = m == top ? 1.0f : expf(m - top);
    const float p = x == top && x == -INFINITY ? 0.0f : expf(x - top);
    lane_load(v + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) acc[i] = acc[i] * keep + p * kv[i];
    l = l * keep + p;
    m = top;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  lane_store(out + row_at(s, b, h, r, s.heads, s.q_len), s.head_dim, acc, inv, 0);
  if (stats != nullptr && (threadIdx.x & 31) == 0)
    *(float2*)(stats + 2 * (((int64_t)b * s.heads + h) * s.q_len + r)) = make_float2(m, l);
}

__global__ void __launch_bounds__(256) simple_forward_kernel(AttentionShape s, const float* __restrict__ q,
                                                             const float* __restrict__ k,
                                                             const float* __restrict__ v, float* __restrict__ out,
                                                             float* __restrict__ stats, int* err) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= (int64_t)s.batch * s.heads * s.q_len) return;
  const int r = (int)(i % s.q_len), h = (int)(i / s.q_len % s.heads), b = (int)(i / s.q_len / s.heads);
  simple_forward_row(s, sequence_of(s, b, err), q, k, v, out, stats, b, h, r);
}

__device__ void simple_dq_row(const AttentionShape& s, const Sequence& sq, const float* q, const float* k,
                              const float* v, const float* out, const float* stats, const float* dout, float* dq,
                              int accumulate, int b, int h, int r) {
  const int g = h / (s.heads / s.kv_heads);
  const Seen seen = seen_by(s, sq, (int64_t)sq.start + r);
  const int64_t at = row_at(s, b, h, r, s.heads, s.q_len);
  float qv[kLaneDims], gv[kLaneDims], kv[kLaneDims], vv[kLaneDims], acc[kLaneDims] = {};
  lane_load(out + at, s.head_dim, kv);
  lane_load(dout + at, s.head_dim, gv);
  lane_load(q + at, s.head_dim, qv);
  const float delta = lane_dot(kv, gv);
  const float2 st = *(const float2*)(stats + 2 * (((int64_t)b * s.heads + h) * s.q_len + r));
  for (int j = 0; j < seen.high; ++j) {
    if (j == seen.first && j < seen.low) j = seen.low;
    lane_load(k + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, kv);
    lane_load(v + row_at(s, b, g, j, s.kv_heads, s.k_len), s.head_dim, vv);
    const float p = expf(lane_dot(qv, kv) * s.scale - st.x) / st.y;
    const float ds = p * (lane_dot(gv, vv) - delta);
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) acc[i] += ds * kv[i];
  }
  lane_store(dq + at, s.head_dim, acc, s.scale, accumulate);
}

__global__ void __launch_bounds__(256) simple_dq_kernel(AttentionShape s, const float* __restrict__ q,
                                                        const float* __restrict__ k, const float* __restrict__ v,
                                                        const float* __restrict__ out,
                                                        const float* __restrict__ stats,
                                                        const float* __restrict__ dout, float* __restrict__ dq,
                                                        int accumulate, int* err) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= (int64_t)s.batch * s.heads * s.q_len) return;
  const int r = (int)(i % s.q_len), h = (int)(i / s.q_len % s.heads), b = (int)(i / s.q_len / s.heads);
  simple_dq_row(s, sequence_of(s, b, err), q, k, v, out, stats, dout, dq, accumulate, b, h, r);
}

// The query rows that see key j: those at positions [j, end).
__device__ __forceinline__ void rows_seeing(const AttentionShape& s, const Sequence& sq, int j, int* r0, int* r1) {
  int64_t end = sq.n;
  if (s.window > 0 && j >= s.sinks && end > (int64_t)j + s.window) end = (int64_t)j + s.window;
  const int64_t a = (int64_t)j - sq.start, z = end - sq.start;
  *r0 = (int)(a < 0 ? 0 : a > s.q_len ? s.q_len : a);
  *r1 = j >= sq.n ? *r0 : (int)(z < 0 ? 0 : z > s.q_len ? s.q_len : z);
}

__device__ void simple_dkv_row(const AttentionShape& s, const Sequence& sq, const float* q, const float* k,
                               const float* v, const float* out, const float* stats, const float* dout, float* dk,
                               float* dv, int accumulate_k, int accumulate_v, int b, int g, int j) {
  const int group = s.heads / s.kv_heads;
  const int64_t at = row_at(s, b, g, j, s.kv_heads, s.k_len);
  float kv[kLaneDims], vv[kLaneDims], ak[kLaneDims] = {}, av[kLaneDims] = {};
  int r0, r1;
  rows_seeing(s, sq, j, &r0, &r1);
  if (r0 < r1) {
    lane_load(k + at, s.head_dim, kv);
    lane_load(v + at, s.head_dim, vv);
    for (int h = g * group; h < (g + 1) * group; ++h)
      for (int r = r0; r < r1; ++r) {
        const int64_t row = row_at(s, b, h, r, s.heads, s.q_len);
        float qv[kLaneDims], gv[kLaneDims], ov[kLaneDims];
        lane_load(q + row, s.head_dim, qv);
        lane_load(dout + row, s.head_dim, gv);
        lane_load(out + row, s.head_dim, ov);
        const float2 st = *(const float2*)(stats + 2 * (((int64_t)b * s.heads + h) * s.q_len + r));
        const float p = expf(lane_dot(qv, kv) * s.scale - st.x) / st.y;
        const float ds = p * (lane_dot(gv, vv) - lane_dot(gv, ov));
#pragma unroll
        for (int i = 0; i < kLaneDims; ++i) {
          av[i] += p * gv[i];
          ak[i] += ds * qv[i];
        }
      }
  }
  lane_store(dk + at, s.head_dim, ak, s.scale, accumulate_k);
  lane_store(dv + at, s.head_dim, av, 1.0f, accumulate_v);
}

__global__ void __launch_bounds__(256) simple_dkv_kernel(AttentionShape s, const float* __restrict__ q,
                                                         const float* __restrict__ k, const float* __restrict__ v,
                                                         const float* __restrict__ out,
                                                         const float* __restrict__ stats,
                                                         const float* __restrict__ dout, float* __restrict__ dk,
                                                         float* __restrict__ dv, int accumulate_k, int accumulate_v,
                                                         int* err) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= (int64_t)s.batch * s.kv_heads * s.k_len) return;
  const int j = (int)(i % s.k_len), g = (int)(i / s.k_len % s.kv_heads), b = (int)(i / s.k_len / s.kv_heads);
  simple_dkv_row(s, sequence_of(s, b, err), q, k, v, out, stats, dout, dk, dv, accumulate_k, accumulate_v, b, g, j);
}

}  // namespace

int64_t window_attention_work_elems(const AttentionShape&) { return 1; }
int64_t window_attention_backward_work_elems(const AttentionShape&) { return 1; }

void launch_window_attention(const AttentionShape& s, const float* q, const float* k, const float* v, float* out,
                             float* stats, float*, int* err, cudaStream_t st) {
  const int64_t rows = (int64_t)s.batch * s.heads * s.q_len;
  if (rows <= 0) return;
  simple_forward_kernel<<<(unsigned)ceil_div(rows, 8), 256, 0, st>>>(s, q, k, v, out, stats, err);
  check_launch();
}

void launch_window_attention_backward(const AttentionShape& s, const float* q, const float* k, const float* v,
                                      const float* out, const float* stats, const float* dout, float* dq, float* dk,
                                      float* dv, float*, int accumulate_q, int accumulate_k, int accumulate_v,
                                      int* err, cudaStream_t st) {
  const int64_t rows = (int64_t)s.batch * s.heads * s.q_len, keys = (int64_t)s.batch * s.kv_heads * s.k_len;
  if (rows > 0) {
    simple_dq_kernel<<<(unsigned)ceil_div(rows, 8), 256, 0, st>>>(s, q, k, v, out, stats, dout, dq, accumulate_q, err);
    check_launch();
  }
  if (keys > 0) {
    simple_dkv_kernel<<<(unsigned)ceil_div(keys, 8), 256, 0, st>>>(s, q, k, v, out, stats, dout, dk, dv, accumulate_k,
                                                                    accumulate_v, err);
    check_launch();
  }
}

}  // namespace tysor
