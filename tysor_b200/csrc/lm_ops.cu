// Layer norm, rotary positions over several axes and distillation from a
// teacher's top logits (lm_ops.cuh), forward and backward.  All of them move
// memory far more than they compute: every kernel reads and writes each value
// once, and what limits it is HBM (or, for a few rows, one launch's latency).
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "lm_ops.cuh"

namespace tysor {
namespace {

void check_launch() {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  TYSOR_CUDA(cudaGetLastError());
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of (a, b) over the threads of a group of TPR threads (TPR a multiple
// of the warp).  `red` is the group's own shared array of 2 * TPR / 32 floats;
// groups of one block wait on barriers of their own.  `phase` alternates
// between calls so that one barrier per call is enough.
template <int TPR>
__device__ __forceinline__ void group_sum2(float& a, float& b, float2* red, int group, int phase) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (TPR > 32) {
    constexpr int W = TPR / 32;
    const int t = threadIdx.x % TPR;
    float2* r = red + phase * W;
    if ((t & 31) == 0) r[t >> 5] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
    a = 0.0f;
    b = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a += r[i].x;
      b += r[i].y;
    }
  }
}

// The sum of one value, likewise.
template <int TPR>
__device__ __forceinline__ float group_sum(float a, float* red, int group, int phase) {
  a = warp_sum(a);
  if (TPR > 32) {
    constexpr int W = TPR / 32;
    const int t = threadIdx.x % TPR;
    float* r = red + phase * W;
    if ((t & 31) == 0) r[t >> 5] = a;
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
    a = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) a += r[i];
  }
  return a;
}

// A thread's share of a row: NV float4 at columns 4 (t + i TPR), or, where a
// row may start off a 16-byte boundary, 4 NV floats at columns t + i TPR.
template <int TPR, int NV, bool VEC>
struct RowPart {
  static constexpr int E = 4 * NV;
  __device__ static __forceinline__ int col(int t, int e) {
    return VEC ? 4 * (t + (e / 4) * TPR) + e % 4 : t + e * TPR;
  }
  __device__ static __forceinline__ void load(const float* __restrict__ p, int width, int t, float (&v)[E],
                                              float fill) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 4 * (t + i * TPR);
        const float4 f = c < width ? *(const float4*)(p + c) : make_float4(fill, fill, fill, fill);
        v[4 * i] = f.x;
        v[4 * i + 1] = f.y;
        v[4 * i + 2] = f.z;
        v[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = t + i * TPR;
        v[i] = c < width ? p[c] : fill;
      }
    }
  }
  __device__ static __forceinline__ void store(float* __restrict__ p, int width, int t, const float (&v)[E]) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 4 * (t + i * TPR);
        if (c < width) *(float4*)(p + c) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = t + i * TPR;
        if (c < width) p[c] = v[i];
      }
    }
  }
};

// ---- layer norm -------------------------------------------------------------

// One group of TPR threads per row, the row in registers: the mean first,
// then the squared distances from it (no difference of large sums).  HBM bounds
// it: 16384 rows of 2048, 268 MB, 45 us = 5.9 TB/s; 16 rows 4.7 us a call, a launch.
template <int TPR, int NV, bool VEC, int kThreads>
__global__ void __launch_bounds__(kThreads) layer_norm_kernel(const float* __restrict__ x,
                                                              const float* __restrict__ gain,
                                                              const float* __restrict__ bias, float* __restrict__ y,
                                                              float* __restrict__ stats, int64_t rows, int width,
                                                              float eps) {
  using Part = RowPart<TPR, NV, VEC>;
  constexpr int G = kThreads / TPR;
  __shared__ float red[G][2 * (TPR > 32 ? TPR / 32 : 1)];
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const float inv = 1.0f / (float)width;
  for (int64_t r = (int64_t)blockIdx.x * G + group; r < rows; r += (int64_t)gridDim.x * G) {
    float v[Part::E];
    Part::load(x + r * width, width, t, v, 0.0f);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < Part::E; ++e) s += v[e];
    const float mean = group_sum<TPR>(s, red[group], group, 0) * inv;
    float q = 0.0f;
#pragma unroll
    for (int e = 0; e < Part::E; ++e) {
      const float d = v[e] - mean;
      q += Part::col(t, e) < width ? d * d : 0.0f;
    }
    const float rstd = rsqrtf(group_sum<TPR>(q, red[group], group, 1) * inv + eps);
    float w[Part::E];
    if (gain != nullptr) {
      Part::load(gain, width, t, w, 0.0f);
#pragma unroll
      for (int e = 0; e < Part::E; ++e) v[e] = (v[e] - mean) * rstd * w[e];
    } else {
#pragma unroll
      for (int e = 0; e < Part::E; ++e) v[e] = (v[e] - mean) * rstd;
    }
    if (bias != nullptr) {
      Part::load(bias, width, t, w, 0.0f);
#pragma unroll
      for (int e = 0; e < Part::E; ++e) v[e] += w[e];
    }
    Part::store(y + r * width, width, t, v);
    if (stats != nullptr && t == 0) *(float2*)(stats + 2 * r) = make_float2(mean, rstd);
  }
}

// Rows wider than a block's registers hold: three passes over the row, the
// later ones from L2.
__global__ void __launch_bounds__(1024) layer_norm_wide_kernel(const float* __restrict__ x,
                                                               const float* __restrict__ gain,
                                                               const float* __restrict__ bias, float* __restrict__ y,
                                                               float* __restrict__ stats, int64_t rows,
                                                               int64_t width, float eps) {
  __shared__ float red[64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* xr = x + r * width;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += 1024) s += xr[c];
    const float mean = group_sum<1024>(s, red, 0, 0) / (float)width;
    float q = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
      const float d = xr[c] - mean;
      q += d * d;
    }
    const float rstd = rsqrtf(group_sum<1024>(q, red, 0, 1) / (float)width + eps);
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
      const float n = (xr[c] - mean) * rstd * (gain ? gain[c] : 1.0f);
      y[r * width + c] = bias ? n + bias[c] : n;
    }
    if (stats != nullptr && threadIdx.x == 0) *(float2*)(stats + 2 * r) = make_float2(mean, rstd);
  }
}

__device__ __forceinline__ void copy16(const float4* to, const float4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}

// Rows of more than kLayerNormWide values, held in shared memory (each thread's
// columns by the thread that reads them, so that only the sums wait): two and
// more rows per SM are under way where registers would hold one.  8192 rows of
// 16384, 1.07 GB, 171 us = 6.3 TB/s (in registers 262), 4096 of 20000 121 us (from
// L2 in three passes 222).
constexpr int kSharedRowThreads = 512;
__global__ void __launch_bounds__(kSharedRowThreads) layer_norm_shared_kernel(
    const float* __restrict__ x, const float* __restrict__ gain, const float* __restrict__ bias, float* __restrict__ y,
    float* __restrict__ stats, int64_t rows, int width, float eps) {
  extern __shared__ __align__(16) float4 held[];  // [width / 4]
  __shared__ float red[2 * kSharedRowThreads / 32];
  const int quads = width / 4;
  const float inv = 1.0f / (float)width;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float4* src = (const float4*)(x + r * width);
    for (int i = threadIdx.x; i < quads; i += kSharedRowThreads) copy16(held + i, src + i);
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    float s = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x; i < quads; i += kSharedRowThreads) {
      const float4 f = held[i];
      s += (f.x + f.y) + (f.z + f.w);
    }
    const float mean = group_sum<kSharedRowThreads>(s, red, 0, 0) * inv;
    float q = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x; i < quads; i += kSharedRowThreads) {
      const float4 f = held[i];
      const float a = f.x - mean, b = f.y - mean, c = f.z - mean, d = f.w - mean;
      q += (a * a + b * b) + (c * c + d * d);
    }
    const float rstd = rsqrtf(group_sum<kSharedRowThreads>(q, red, 0, 1) * inv + eps);
    float4* dst = (float4*)(y + r * width);
#pragma unroll 4
    for (int i = threadIdx.x; i < quads; i += kSharedRowThreads) {
      float4 f = held[i];
      f.x = (f.x - mean) * rstd, f.y = (f.y - mean) * rstd, f.z = (f.z - mean) * rstd, f.w = (f.w - mean) * rstd;
      if (gain != nullptr) {
        const float4 w = ((const float4*)gain)[i];
        f.x *= w.x, f.y *= w.y, f.z *= w.z, f.w *= w.w;
      }
      if (bias != nullptr) {
        const float4 w = ((const float4*)bias)[i];
        f.x += w.x, f.y += w.y, f.z += w.z, f.w += w.w;
      }
      dst[i] = f;
    }
    if (stats != nullptr && threadIdx.x == 0) *(float2*)(stats + 2 * r) = make_float2(mean, rstd);
  }
}

// Their gradients: x and dy of a row in shared memory, the next row's on their
// way where `stages` is 2; dgain and dbias as below, a thread owning its columns.
// 8192 rows of 16384, 1.6 GB, 305 us = 5.3 TB/s, of 8196 185 us (two passes over the
// row and a third for the columns 817 and 449).
constexpr int kSharedQuads = 8;  // of a thread: rows up to 16384 values
__global__ void __launch_bounds__(kSharedRowThreads) layer_norm_backward_shared_kernel(
    const float* __restrict__ x, const float* __restrict__ gain, const float* __restrict__ stats,
    const float* __restrict__ dy, float* __restrict__ dx, float* __restrict__ partial, int64_t rows, int width,
    int stages, int accumulate) {
  extern __shared__ __align__(16) float4 held[];  // [stages][x, dy][width / 4]
  __shared__ float2 red[2 * kSharedRowThreads / 32];
  const int quads = width / 4;
  const float inv = 1.0f / (float)width;
  float4 dg[kSharedQuads], db[kSharedQuads];
#pragma unroll
  for (int k = 0; k < kSharedQuads; ++k) dg[k] = db[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto fetch = [&](int64_t r, int stage) {
    if (r < rows) {
      const float4* xs = (const float4*)(x + r * width);
      const float4* ys = (const float4*)(dy + r * width);
      float4* to = held + (int64_t)stage * 2 * quads;
      for (int i = threadIdx.x; i < quads; i += kSharedRowThreads) copy16(to + i, xs + i), copy16(to + quads + i, ys + i);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (stages == 2) fetch(blockIdx.x, 0);
  int phase = 0, stage = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    if (stages == 2) {
      fetch(r + gridDim.x, stage ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      fetch(r, 0);
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    const float4 *xs = held + (int64_t)stage * 2 * quads, *ys = xs + quads;
    const float2 st = *(const float2*)(stats + 2 * r);
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int k = 0; k < kSharedQuads; ++k) {
      const int i = threadIdx.x + k * kSharedRowThreads;
      if (i >= quads) break;
      const float4 f = xs[i], g = ys[i];
      const float4 w = gain ? ((const float4*)gain)[i] : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      const float4 n = make_float4((f.x - st.x) * st.y, (f.y - st.x) * st.y, (f.z - st.x) * st.y, (f.w - st.x) * st.y);
      dg[k].x += g.x * n.x, dg[k].y += g.y * n.y, dg[k].z += g.z * n.z, dg[k].w += g.w * n.w;
      db[k].x += g.x, db[k].y += g.y, db[k].z += g.z, db[k].w += g.w;
      a += (g.x * w.x + g.y * w.y) + (g.z * w.z + g.w * w.w);
      b += (g.x * w.x * n.x + g.y * w.y * n.y) + (g.z * w.z * n.z + g.w * w.w * n.w);
    }
    group_sum2<kSharedRowThreads>(a, b, red, 0, phase);
    phase ^= 1;
    a *= inv;
    b *= inv;
    float4* dst = (float4*)(dx + r * width);
#pragma unroll
    for (int k = 0; k < kSharedQuads; ++k) {
      const int i = threadIdx.x + k * kSharedRowThreads;
      if (i >= quads) break;
      const float4 f = xs[i], g = ys[i];
      const float4 w = gain ? ((const float4*)gain)[i] : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      float4 o = make_float4((g.x * w.x - a - (f.x - st.x) * st.y * b) * st.y, (g.y * w.y - a - (f.y - st.x) * st.y * b) * st.y,
                             (g.z * w.z - a - (f.z - st.x) * st.y * b) * st.y, (g.w * w.w - a - (f.w - st.x) * st.y * b) * st.y);
      if (accumulate) {
        const float4 p = dst[i];
        o.x += p.x, o.y += p.y, o.z += p.z, o.w += p.w;
      }
      dst[i] = o;
    }
    if (stages == 2) stage ^= 1;
  }
  if (partial == nullptr) return;
  float4* line = (float4*)(partial + (int64_t)blockIdx.x * 2 * width);
#pragma unroll
  for (int k = 0; k < kSharedQuads; ++k) {
    const int i = threadIdx.x + k * kSharedRowThreads;
    if (i < quads) line[i] = dg[k], line[quads + i] = db[k];
  }
}

// dx of one row per group and step; each thread owns its columns' share of
// dgain and dbias in registers over all rows of the block.  The block's groups
// add theirs in order in shared memory, and `partial` gets one line per block
// (summed in a fixed order by column_sum_kernel).  HBM bounds it: 16384 rows of
// 2048, 403 MB, 68 us = 5.9 TB/s, and 8 us for the 296 lines of partial sums.
template <int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(512, NV <= 2 ? 2 : 1) layer_norm_backward_kernel(
    const float* __restrict__ x, const float* __restrict__ gain, const float* __restrict__ stats,
    const float* __restrict__ dy, float* __restrict__ dx, float* __restrict__ partial, int64_t rows, int width,
    int accumulate) {
  using Part = RowPart<TPR, NV, VEC>;
  constexpr int G = 512 / TPR;
  __shared__ float2 red[G][2 * (TPR > 32 ? TPR / 32 : 1)];
  extern __shared__ float sums[];  // [2][width]
  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  float w[Part::E], dg[Part::E], db[Part::E];
  if (gain != nullptr) Part::load(gain, width, t, w, 0.0f);
#pragma unroll
  for (int e = 0; e < Part::E; ++e) {
    if (gain == nullptr) w[e] = 1.0f;
    dg[e] = 0.0f;
    db[e] = 0.0f;
  }
  const float inv = 1.0f / (float)width;
  int phase = 0;
  for (int64_t r = (int64_t)blockIdx.x * G + group; r < rows; r += (int64_t)gridDim.x * G) {
    float n[Part::E], g[Part::E];
    Part::load(x + r * width, width, t, n, 0.0f);
    Part::load(dy + r * width, width, t, g, 0.0f);
    const float2 st = *(const float2*)(stats + 2 * r);
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int e = 0; e < Part::E; ++e) {
      n[e] = (n[e] - st.x) * st.y;
      // Columns past the row hold g = 0 and add nothing anywhere.
      dg[e] += g[e] * n[e];
      db[e] += g[e];
      g[e] *= w[e];
      a += g[e];
      b += g[e] * n[e];
    }
    group_sum2<TPR>(a, b, red[group], group, phase);
    phase ^= 1;
    a *= inv;
    b *= inv;
#pragma unroll
    for (int e = 0; e < Part::E; ++e) g[e] = (g[e] - a - n[e] * b) * st.y;
    if (accumulate) {
      Part::load(dx + r * width, width, t, n, 0.0f);
#pragma unroll
      for (int e = 0; e < Part::E; ++e) g[e] = n[e] + g[e];
    }
    Part::store(dx + r * width, width, t, g);
  }
  if (partial == nullptr) return;
  for (int k = 0; k < G; ++k) {
    if (k == group)
#pragma unroll
      for (int e = 0; e < Part::E; ++e) {
        const int c = Part::col(t, e);
        if (c < width) {
          sums[c] = k == 0 ? dg[e] : sums[c] + dg[e];
          sums[width + c] = k == 0 ? db[e] : sums[width + c] + db[e];
        }
      }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * width; c += 512) partial[(int64_t)blockIdx.x * 2 * width + c] = sums[c];
}

// Wide rows: dx alone, two passes over the row.
__global__ void __launch_bounds__(1024) layer_norm_backward_wide_kernel(
    const float* __restrict__ x, const float* __restrict__ gain, const float* __restrict__ stats,
    const float* __restrict__ dy, float* __restrict__ dx, int64_t rows, int64_t width, int accumulate) {
  __shared__ float2 red[64];
  int phase = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* xr = x + r * width;
    const float* yr = dy + r * width;
    const float2 st = *(const float2*)(stats + 2 * r);
    float a = 0.0f, b = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
      const float g = yr[c] * (gain ? gain[c] : 1.0f);
      a += g;
      b += g * ((xr[c] - st.x) * st.y);
    }
    group_sum2<1024>(a, b, red, 0, phase);
    phase ^= 1;
    a /= (float)width;
    b /= (float)width;
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
      const float g = yr[c] * (gain ? gain[c] : 1.0f);
      const float d = (g - a - (xr[c] - st.x) * st.y * b) * st.y;
      float* o = dx + r * width + c;
      *o = accumulate ? *o + d : d;
    }
  }
}

// Wide rows: the partial column sums of dy * n and dy over one block's rows.
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const float* __restrict__ x,
                                                                 const float* __restrict__ stats,
                                                                 const float* __restrict__ dy,
                                                                 float* __restrict__ partial, int64_t rows,
                                                                 int64_t width) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  float dg = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = dy[r * width + c];
    dg += g * ((x[r * width + c] - stats[2 * r]) * stats[2 * r + 1]);
    db += g;
  }
  partial[(int64_t)blockIdx.y * 2 * width + c] = dg;
  partial[(int64_t)blockIdx.y * 2 * width + width + c] = db;
}

// dgain / dbias (+)= the sum of `lines` partial lines of 2 * width floats: 32
// columns per block, 16 threads a column, their parts added in order.
__global__ void __launch_bounds__(512) column_sum_kernel(const float* __restrict__ partial, float* __restrict__ dgain,
                                                         float* __restrict__ dbias, int lines, int64_t width,
                                                         int accumulate) {
  __shared__ float part[16][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < 2 * width)
#pragma unroll 4
    for (int l = slice; l < lines; l += 16) s += partial[(int64_t)l * 2 * width + c];
  part[slice][lane] = s;
  __syncthreads();
  if (slice != 0 || c >= 2 * width) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += part[i][lane];
  float* out = c < width ? dgain : dbias;
  if (out == nullptr) return;
  out += c < width ? c : c - width;
  *out = accumulate ? *out + s : s;
}

// ---- rotary positions ---------------------------------------------------------

struct RopeArgs {
  RopeAxes s;
  int head_chunk;  // heads a thread turns
  int back, accumulate;
};

// Each thread turns V neighbouring pairs of one token in `head_chunk` heads
// with one evaluation of their angles: positions times rates in 64 bits,
// reduced to a fraction of a revolution, so that far positions lose nothing.  HBM
// bounds it: 16 heads of 128 values, 16384 tokens, 268 MB in 42 us = 6.4 TB/s.
template <int V>
__global__ void __launch_bounds__(256) rope_axes_kernel(const float* __restrict__ x,
                                                        const float* __restrict__ positions,
                                                        const double* __restrict__ rates, float* __restrict__ out,
                                                        RopeArgs a) {
  const RopeAxes& s = a.s;
  const int per = s.half / V;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t tokens = (int64_t)s.batch * s.seq;
  if (item >= tokens * per) return;
  const int64_t token = item / per;
  const int i0 = (int)(item - token * per) * V;
  const int64_t b = token / s.seq, at = token - b * s.seq;
  float cs[V], sn[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    int axis = 0;
#pragma unroll
    for (int e = 0; e < kMaxRopeAxes - 1; ++e) axis += i0 + v >= s.ends[e];
    const double turns = (double)positions[(b * s.axes + axis) * s.seq + at] * rates[i0 + v];
    sincospif(2.0f * (float)(turns - rint(turns)), &sn[v], &cs[v]);
    if (a.back) sn[v] = -sn[v];
  }
  const int64_t step = s.seq_major ? 2 * (int64_t)s.half : 2 * (int64_t)s.half * s.seq;
  const int64_t base =
      (s.seq_major ? (b * s.seq + at) * s.heads : b * s.heads * s.seq + at) * 2 * (int64_t)s.half + i0;
  const int h0 = blockIdx.y * a.head_chunk;
  const int h1 = min(s.heads, h0 + a.head_chunk);
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const int64_t o = base + h * step;
    float lo[V], hi[V];
    if (V == 4) {
      const float4 l = *(const float4*)(x + o), u = *(const float4*)(x + o + s.half);
      lo[0] = l.x, lo[1 % V] = l.y, lo[2 % V] = l.z, lo[3 % V] = l.w;
      hi[0] = u.x, hi[1 % V] = u.y, hi[2 % V] = u.z, hi[3 % V] = u.w;
    } else {
      lo[0] = x[o];
      hi[0] = x[o + s.half];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float p = lo[v] * cs[v] - hi[v] * sn[v];
      hi[v] = lo[v] * sn[v] + hi[v] * cs[v];
      lo[v] = p;
    }
    if (a.accumulate) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        lo[v] = out[o + v] + lo[v];
        hi[v] = out[o + s.half + v] + hi[v];
      }
    }
    if (V == 4) {
      *(float4*)(out + o) = make_float4(lo[0], lo[1 % V], lo[2 % V], lo[3 % V]);
      *(float4*)(out + o + s.half) = make_float4(hi[0], hi[1 % V], hi[2 % V], hi[3 % V]);
    } else {
      out[o] = lo[0];
      out[o + s.half] = hi[0];
    }
  }
}

// ---- distillation -------------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;

// 2^x to about 2^-22, subnormal results as 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The index an id stands for: -1 for an absent entry.
__device__ __forceinline__ int entry_id(float id, int64_t width, int* err) {
  if (id < 0.0f) return -1;
  if (!(id < (float)width) || (int64_t)id >= width) {  // NaN too
    atomicCAS(err, 0, (int)kErrIndexRange);
    return -1;
  }
  return (int)id;
}

// The teacher's probabilities of one row into p[0..top), its ids into ids[],
// by one warp; returns whether the row has an entry of any weight.  Entries
// that are absent get p = 0.  `log_mass` is ln(sum of exp((t - best) / T)).
__device__ __forceinline__ bool teacher_row(const float* __restrict__ idr, const float* __restrict__ tr, int top,
                                            int64_t width, float inv_t, int* ids, float* p, float* best_out,
                                            double* log_mass, int* err) {
  const int lane = threadIdx.x & 31;
  float best = -INFINITY;
  bool bad = false;
#pragma unroll 4
  for (int e = lane; e < top; e += 32) {
    const int id = entry_id(idr[e], width, err);
    ids[e] = id;
    const float w = id < 0 ? -INFINITY : tr[e];
    p[e] = w;
    bad |= w != w;
    best = fmaxf(best, w);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (__any_sync(0xffffffffu, bad)) best = NAN;
  float mass = 0.0f;
  for (int e = lane; e < top; e += 32) {
    const float w = best == -INFINITY || p[e] == -INFINITY ? 0.0f : exp2f((p[e] - best) * inv_t * kLog2e);
    p[e] = w;
    mass += w;
  }
  mass = warp_sum(mass);
  const float scale = mass > 0.0f ? 1.0f / mass : 0.0f;
  // Where a weight is NaN so are all; an absent entry stays 0 (nothing reads its id).
  for (int e = lane; e < top; e += 32) p[e] = ids[e] < 0 ? 0.0f : mass == mass ? p[e] * scale : NAN;
  __syncwarp();
  *best_out = best;
  *log_mass = log((double)mass);
  return best != -INFINITY;
}

struct Online {
  float m, s;  // greatest value, sum of exp2((v - m) * c)
};

__device__ __forceinline__ Online join(Online a, Online b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s};
  return {m, a.s * exp2_fast((a.m - m) * c) + b.s * exp2_fast((b.m - m) * c)};
}

__device__ __forceinline__ void take(Online& o, float v, float c) {
  if (v > o.m) {
    o.s = o.s * exp2_fast((o.m - v) * c) + 1.0f;
    o.m = v;
  } else {
    o.s += v == o.m && v == -INFINITY ? 0.0f : exp2_fast((v - o.m) * c);
  }
}

// Greatest logit and sum of one row in one pass, the row split over a cluster
// of gridDim.y blocks (one for many rows) whose parts the first block joins in
// order through distributed shared memory; then the loss of the row's entries.
// Eight small blocks per SM rather than four: while one ends its row (its few
// entries, the logarithms), the others keep loads in flight.  HBM bounds it: 8192
// rows of 32000, 1.05 GB in 181 us = 5.8 TB/s.
constexpr int kDistillThreads = 256;
__global__ void __launch_bounds__(kDistillThreads) distill_loss_kernel(
    const float* __restrict__ logits, const float* __restrict__ ids, const float* __restrict__ teacher,
    float* __restrict__ loss, float* __restrict__ stats, int64_t rows, int64_t width, int top, float temperature,
    int* err) {
  __shared__ Online warp_part[kDistillThreads / 32];
  __shared__ Online part[8];  // block 0's: one entry per block of the cluster
  __shared__ struct {
    float best;
    double log_mass;
    bool any;
  } teach;
  extern __shared__ __align__(8) uint8_t entries[];  // [top] each: gaps (double), ids, probabilities
  const int64_t r = blockIdx.x;
  const int parts = gridDim.y, rank = blockIdx.y, tid = threadIdx.x;
  // Arrives for "this block runs": the first block's shared memory is written
  // only once every block of the cluster has got here.
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const float inv_t = 1.0f / temperature, c = inv_t * kLog2e;
  const float* row = logits + r * width;
  // Chunks of whole float4 from the row's first 16-byte boundary; the values
  // before it and after the last whole float4 go to the first block.
  const int64_t head = min(width, (int64_t)((4 - (((uintptr_t)row >> 2) & 3)) & 3));
  const int64_t quads = (width - head) / 4;
  const int64_t per = (quads + parts - 1) / parts;
  const int64_t q0 = min(quads, rank * per), q1 = min(quads, q0 + per);
  const float4* body = (const float4*)(row + head);
  // The last warp of the first block prepares the teacher's entries meanwhile.
  double* gap = (double*)entries;
  int* eid = (int*)(gap + top);
  float* p = (float*)(eid + top);
  if (rank == 0 && tid >= kDistillThreads - 32) {
    float best;
    double log_mass;
    const bool any = teacher_row(ids + r * top, teacher + r * top, top, width, inv_t, eid, p, &best, &log_mass, err);
    if ((tid & 31) == 0) teach = {best, log_mass, any};
    // What the end needs of each entry: the teacher's logarithm less the
    // student's logit, in 64 bits (the two logarithms nearly cancel where the
    // student follows the teacher).
#pragma unroll 4
    for (int e = tid & 31; e < top; e += 32)
      if (p[e] != 0.0f)
        gap[e] = ((double)teacher[r * top + e] - (double)best - (double)row[eid[e]]) / temperature - log_mass;
  }
  Online o{-INFINITY, 0.0f};
  bool bad = false;
  for (int64_t i = q0 + tid; i < q1; i += 4 * kDistillThreads) {
    float4 f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      f[u] = i + u * kDistillThreads < q1 ? body[i + u * kDistillThreads]
                                          : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    float m = o.m;
#pragma unroll
    for (int u = 0; u < 4; ++u) m = fmaxf(m, fmaxf(fmaxf(f[u].x, f[u].y), fmaxf(f[u].z, f[u].w)));
    if (m == -INFINITY) {  // nothing but -inf so far, or NaN, which fmaxf drops
#pragma unroll
      for (int u = 0; u < 4; ++u) bad |= f[u].x != f[u].x || f[u].y != f[u].y || f[u].z != f[u].z || f[u].w != f[u].w;
      continue;
    }
    float s = o.s * exp2_fast((o.m - m) * c);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      s += (exp2_fast((f[u].x - m) * c) + exp2_fast((f[u].y - m) * c)) +
           (exp2_fast((f[u].z - m) * c) + exp2_fast((f[u].w - m) * c));
    o.m = m;
    o.s = s;
  }
  if (rank == 0) {
    const int64_t tail = head + 4 * quads;
    if (tid < head) take(o, row[tid], c), bad |= row[tid] != row[tid];
    if (tid < width - tail) take(o, row[tail + tid], c), bad |= row[tail + tid] != row[tail + tid];
  }
  if (bad) o.s = NAN;
  float top_of_warp = o.m;
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top_of_warp = fmaxf(top_of_warp, __shfl_xor_sync(0xffffffffu, top_of_warp, k));
  // A lane without a finite value holds a sum of 0, or NaN.
  o.s = warp_sum(o.m == -INFINITY ? o.s : o.s * exp2_fast((o.m - top_of_warp) * c));
  o.m = top_of_warp;
  if ((tid & 31) == 0) warp_part[tid >> 5] = o;
  __syncthreads();
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid == 0) {
    for (int w = 1; w < kDistillThreads / 32; ++w) o = join(o, warp_part[w], c);
    uint32_t dst;
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&part[rank]);
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"(mine));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(o.m), "f"(o.s) : "memory");
  }
  if (parts > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  if (tid >= 32) return;
  Online all = part[0];
  for (int w = 1; w < parts; ++w) all = join(all, part[w], c);
  if (stats != nullptr && tid == 0) *(float2*)(stats + 2 * r) = make_float2(all.m, all.s);
  // Sum of p (ln p - ln q), ln q = (z - max) / T - ln sum.
  const double log_sum = log((double)all.s) + (double)all.m / temperature;
  float sum = 0.0f;
  if (teach.any)
    for (int e = tid; e < top; e += 32)
      if (p[e] != 0.0f) sum += (float)((double)p[e] * (gap[e] + log_sum));
  sum = warp_sum(sum);
  if (tid == 0) loss[r] = temperature * temperature * sum;
}

// One block per row and chunk of columns: T * dloss * q in one pass from the
// row's statistics, then the few entries' own terms.  Entries of one id go
// together: a table of `slots` (a power of two, at least twice `top`) finds each
// id's first entry, which takes the others' in order where there are any.  HBM
// bounds it: 8192 rows of 32000, 2.1 GB in 330 us = 6.4 TB/s.  Comparing each pair of
// entries instead, loss and gradient took 533 us with 64 entries a row where this
// takes 521, and 2858 where this takes 1085 with 1024.
template <bool VEC>
__global__ void __launch_bounds__(kDistillThreads) distill_backward_kernel(
    const float* __restrict__ logits, const float* __restrict__ ids, const float* __restrict__ teacher,
    const float* __restrict__ stats, const float* __restrict__ dloss, float* __restrict__ grad, int64_t rows,
    int64_t width, int64_t chunk, int top, int slots, float temperature, int accumulate, int* err) {
  extern __shared__ float entry[];  // [2][top], then [slots] each: id, its first entry, its entries
  __shared__ int any_entry;
  const int64_t r = blockIdx.x;
  const int64_t c0 = blockIdx.y * chunk, c1 = min(width, c0 + chunk);
  const int tid = threadIdx.x;
  int* eid = (int*)entry;
  float* p = entry + top;
  int *key = (int*)(p + top), *first = key + slots, *count = first + slots;
  for (int i = tid; i < slots; i += kDistillThreads) key[i] = -1, first[i] = INT_MAX, count[i] = 0;
  if (tid >= kDistillThreads - 32) {
    float best;
    double log_mass;
    const bool any = teacher_row(ids + r * top, teacher + r * top, top, width, 1.0f / temperature, eid, p, &best,
                                 &log_mass, err);
    if ((tid & 31) == 0) any_entry = any;
  }
  const float* row = logits + r * width;
  float* out = grad + r * width;
  const float2 st = *(const float2*)(stats + 2 * r);
  const float c = kLog2e / temperature;
  const float up = temperature * (dloss ? dloss[r] : 1.0f);
  const float coef = up / st.y;
  if (accumulate) {  // a row without entries stays as it is
    __syncthreads();
    if (!any_entry) return;
  }
  const int64_t head = VEC ? min(c1 - c0, (int64_t)((4 - (((uintptr_t)(row + c0) >> 2) & 3)) & 3)) : 0;
  const int64_t quads = VEC ? (c1 - c0 - head) / 4 : 0;
  const float4* src = (const float4*)(row + c0 + head);
  float4* dst = (float4*)(out + c0 + head);
  for (int64_t i = tid; i < quads; i += 4 * kDistillThreads) {
    float4 f[4], old[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * kDistillThreads < quads) f[u] = src[i + u * kDistillThreads];
    if (accumulate)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * kDistillThreads < quads) old[u] = dst[i + u * kDistillThreads];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u * kDistillThreads >= quads) break;
      float4 g = make_float4(coef * exp2_fast((f[u].x - st.x) * c), coef * exp2_fast((f[u].y - st.x) * c),
                             coef * exp2_fast((f[u].z - st.x) * c), coef * exp2_fast((f[u].w - st.x) * c));
      if (accumulate) g.x += old[u].x, g.y += old[u].y, g.z += old[u].z, g.w += old[u].w;
      dst[i + u * kDistillThreads] = g;
    }
  }
  auto one = [&](int64_t at) {
    const float g = coef * exp2_fast((row[at] - st.x) * c);
    out[at] = accumulate ? out[at] + g : g;
  };
  if (VEC && tid < head) one(c0 + tid);
  for (int64_t at = c0 + head + 4 * quads + tid; at < c1; at += kDistillThreads) one(at);
  __syncthreads();
  if (!any_entry) {  // 0, whatever the row holds
    for (int64_t at = c0 + tid; at < c1; at += kDistillThreads) out[at] = 0.0f;
    return;
  }
  auto start_of = [&](int id) { return (int)((uint32_t)id * 2654435769u >> 16) & (slots - 1); };
  for (int e = tid; e < top; e += kDistillThreads) {
    const int id = eid[e];
    if (id < c0 || id >= c1) continue;
    int at = start_of(id);
    for (;; at = (at + 1) & (slots - 1)) {  // ends: at most half of the slots are taken
      const int held = atomicCAS(&key[at], -1, id);
      if (held == -1 || held == id) break;
    }
    atomicMin(&first[at], e);
    atomicAdd(&count[at], 1);
  }
  __syncthreads();
  for (int e = tid; e < top; e += kDistillThreads) {
    const int id = eid[e];
    if (id < c0 || id >= c1) continue;
    int at = start_of(id);
    while (key[at] != id) at = (at + 1) & (slots - 1);  // every id in [c0, c1) has its slot
    if (first[at] != e) continue;
    float mass = p[e];
    for (int f = e + 1, more = count[at] - 1; more > 0 && f < top; ++f)
      if (eid[f] == id) mass += p[f], --more;
    out[id] -= up * mass;
  }
}

}  // namespace

// ---- launchers ------------------------------------------------------------------

namespace {

template <int TPR, int NV, bool VEC>
void layer_norm_run(const float* x, const float* gain, const float* bias, float* y, float* stats, int64_t rows,
                    int width, float eps, cudaStream_t st) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  const int64_t want = ceil_div(rows, kThreads / TPR);
  const int blocks = (int)(want < 148 * 64 ? want : 148 * 64);
  layer_norm_kernel<TPR, NV, VEC, kThreads><<<blocks, kThreads, 0, st>>>(x, gain, bias, y, stats, rows, width, eps);
  check_launch();
}

// A row takes the fewest threads that hold it 16 values each: below that a
// block has too few loads in flight, above it the sums' barriers cost more.
template <bool VEC>
void layer_norm_pick(const float* x, const float* gain, const float* bias, float* y, float* stats, int64_t rows,
                     int64_t width, float eps, cudaStream_t st) {
  const int w = (int)width;
  if (width <= 128) layer_norm_run<32, 1, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
  else if (width <= 512) layer_norm_run<32, 4, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
  else if (width <= 1024) layer_norm_run<64, 4, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
  else if (width <= 2048) layer_norm_run<128, 4, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
  else if (width <= 4096) layer_norm_run<256, 4, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
  else if (width <= 8192) layer_norm_run<512, 4, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
  else layer_norm_run<1024, 4, VEC>(x, gain, bias, y, stats, rows, w, eps, st);
}

constexpr int64_t kLayerNormMost = 16384;         // widest row in registers, forward
constexpr int64_t kLayerNormBackwardMost = 8192;  // backward
// Rows above 8192 values that may be loaded 16 bytes at a time are held in shared
// memory as far as it goes, others in registers or read again from L2.
constexpr int64_t kLayerNormWide = 8192;
constexpr int64_t kSharedBytes = 224 * 1024;
constexpr int64_t kSharedBackwardMost = 4 * kSharedQuads * kSharedRowThreads;

int layer_norm_lines(int64_t rows, int64_t width) {
  if (width > kLayerNormBackwardMost) return (int)(rows < 148 ? rows : 148);
  int tpr = 32;
  while (tpr * 8 < width && tpr < 512) tpr *= 2;
  const int64_t want = ceil_div(rows, 512 / tpr);
  return (int)(want < 148 * 2 ? want : 148 * 2);
}

template <int TPR, int NV, bool VEC>
void layer_norm_backward_run(const float* x, const float* gain, const float* stats, const float* dy, float* dx,
                             float* partial, int64_t rows, int width, int accumulate, cudaStream_t st) {
  const size_t smem = partial ? sizeof(float) * 2 * (size_t)width : 0;
  // 48 KB without the attribute, the kernel's own `red` among them.
  constexpr size_t kRed = sizeof(float2) * 2 * (512 / TPR) * (TPR / 32);
  if (smem + kRed > 48 * 1024)
    TYSOR_CUDA(cudaFuncSetAttribute(layer_norm_backward_kernel<TPR, NV, VEC>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
  layer_norm_backward_kernel<TPR, NV, VEC><<<layer_norm_lines(rows, width), 512, smem, st>>>(
      x, gain, stats, dy, dx, partial, rows, width, accumulate);
  check_launch();
}

// Eight values of a row per thread up to 4096: two blocks of 512 threads then
// fit an SM.
template <bool VEC>
void layer_norm_backward_pick(const float* x, const float* gain, const float* stats, const float* dy, float* dx,
                              float* partial, int64_t rows, int64_t width, int accumulate, cudaStream_t st) {
  const int w = (int)width;
  if (width <= 256) layer_norm_backward_run<32, 2, VEC>(x, gain, stats, dy, dx, partial, rows, w, accumulate, st);
  else if (width <= 512) layer_norm_backward_run<64, 2, VEC>(x, gain, stats, dy, dx, partial, rows, w, accumulate, st);
  else if (width <= 1024) layer_norm_backward_run<128, 2, VEC>(x, gain, stats, dy, dx, partial, rows, w, accumulate, st);
  else if (width <= 2048) layer_norm_backward_run<256, 2, VEC>(x, gain, stats, dy, dx, partial, rows, w, accumulate, st);
  else if (width <= 4096) layer_norm_backward_run<512, 2, VEC>(x, gain, stats, dy, dx, partial, rows, w, accumulate, st);
  else layer_norm_backward_run<512, 4, VEC>(x, gain, stats, dy, dx, partial, rows, w, accumulate, st);
}

}  // namespace

void launch_layer_norm(const float* x, const float* gain, const float* bias, float* y, float* stats, int64_t rows,
                       int64_t width, float eps, cudaStream_t st) {
  if (rows <= 0 || width <= 0) return;
  const bool vec = width % 4 == 0 && aligned16(x) && aligned16(y) && aligned16(gain) && aligned16(bias);
  if (vec && width > kLayerNormWide && width * 4 <= kSharedBytes) {
    const int bytes = (int)width * 4, blocks = 148 * (int)std::min<int64_t>(4, kSharedBytes / (bytes + 1024));
    TYSOR_CUDA(cudaFuncSetAttribute(layer_norm_shared_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedBytes));
    layer_norm_shared_kernel<<<(int)std::min<int64_t>(rows, std::max(blocks, 148)), kSharedRowThreads, bytes, st>>>(
        x, gain, bias, y, stats, rows, (int)width, eps);
    check_launch();
    return;
  }
  if (width > kLayerNormMost) {
    layer_norm_wide_kernel<<<(int)(rows < 148 * 2 ? rows : 148 * 2), 1024, 0, st>>>(x, gain, bias, y, stats, rows,
                                                                                    width, eps);
    check_launch();
    return;
  }
  if (vec) layer_norm_pick<true>(x, gain, bias, y, stats, rows, width, eps, st);
  else layer_norm_pick<false>(x, gain, bias, y, stats, rows, width, eps, st);
}

int64_t layer_norm_partial_elems(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0) return 1;
  return (int64_t)layer_norm_lines(rows, width) * 2 * width;
}

void launch_layer_norm_backward(const float* x, const float* gain, const float* stats, const float* dy, float* dx,
                                float* dgain, float* dbias, float* partial, int64_t rows, int64_t width,
                                int accumulate_dx, int accumulate_params, cudaStream_t st) {
  if (width <= 0) return;
  const bool columns = dgain != nullptr || dbias != nullptr;
  int lines = 0;
  if (rows > 0) {
    lines = layer_norm_lines(rows, width);
    float* part = columns ? partial : nullptr;
    const bool vec = width % 4 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(gain);
    if (vec && width > kLayerNormBackwardMost && width <= kSharedBackwardMost && aligned16(partial)) {
      const int stages = 16 * width <= kSharedBytes ? 2 : 1;
      TYSOR_CUDA(cudaFuncSetAttribute(layer_norm_backward_shared_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)kSharedBytes));
      layer_norm_backward_shared_kernel<<<lines, kSharedRowThreads, (size_t)(8 * width * stages), st>>>(
          x, gain, stats, dy, dx, part, rows, (int)width, stages, accumulate_dx);
      check_launch();
    } else if (width > kLayerNormBackwardMost) {
      layer_norm_backward_wide_kernel<<<(int)(rows < 148 * 2 ? rows : 148 * 2), 1024, 0, st>>>(
          x, gain, stats, dy, dx, rows, width, accumulate_dx);
      check_launch();
      if (columns) {
        const dim3 grid((unsigned)ceil_div(width, 256), (unsigned)lines);
        layer_norm_columns_kernel<<<grid, 256, 0, st>>>(x, stats, dy, part, rows, width);
        check_launch();
      }
    } else {
      if (vec) layer_norm_backward_pick<true>(x, gain, stats, dy, dx, part, rows, width, accumulate_dx, st);
      else layer_norm_backward_pick<false>(x, gain, stats, dy, dx, part, rows, width, accumulate_dx, st);
    }
  }
  if (!columns) return;
  column_sum_kernel<<<(unsigned)ceil_div(2 * width, 32), 512, 0, st>>>(partial, dgain, dbias, lines, width,
                                                                       accumulate_params);
  check_launch();
}

void launch_rope_axes(const float* x, const float* positions, const double* rates, float* out, const RopeAxes& shape,
                      int back, int accumulate, cudaStream_t st) {
  const int64_t tokens = (int64_t)shape.batch * shape.seq;
  if (tokens <= 0 || shape.heads <= 0 || shape.half <= 0) return;
  const bool vec = shape.half % 4 == 0 && aligned16(x) && aligned16(out);
  const int64_t items = tokens * (shape.half / (vec ? 4 : 1));
  // All heads of a token in one thread share its angles; where that leaves
  // fewer than two blocks per SM, the heads are spread over more threads.
  int64_t chunk = shape.heads * items / (148 * 2 * 256);
  const int64_t least = ceil_div(shape.heads, 65535);  // blocks of the grid's second axis
  chunk = chunk < least ? least : chunk > shape.heads ? shape.heads : chunk;
  RopeArgs a{shape, (int)chunk, back, accumulate};
  for (int e = shape.axes - 1; e < kMaxRopeAxes; ++e) a.s.ends[e] = INT_MAX;  // the last axis takes the rest
  const dim3 grid((unsigned)ceil_div(items, 256), (unsigned)ceil_div(shape.heads, chunk));
  if (vec) rope_axes_kernel<4><<<grid, 256, 0, st>>>(x, positions, rates, out, a);
  else rope_axes_kernel<1><<<grid, 256, 0, st>>>(x, positions, rates, out, a);
  check_launch();
}

void launch_distill_loss(const float* logits, const float* ids, const float* teacher, float* loss, float* stats,
                         int64_t rows, int64_t width, int top, float temperature, int* err, cudaStream_t st) {
  if (rows <= 0) return;
  if (rows > INT_MAX) throw CudaError("distill_loss takes up to 2^31 - 1 rows");
  // A row is split over up to eight blocks where whole rows leave SMs idle
  // and a part still gives each thread a few loads.
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= 148 * 4 && width / (parts * 2) >= 4 * kDistillThreads) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows, (unsigned)parts);
  cfg.blockDim = dim3(kDistillThreads);
  cfg.dynamicSmemBytes = (sizeof(double) + sizeof(int) + sizeof(float)) * (size_t)top;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {1, (unsigned)parts, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TYSOR_CUDA(cudaLaunchKernelEx(&cfg, distill_loss_kernel, logits, ids, teacher, loss, stats, rows, width, top,
                                temperature, err));
  check_launch();
}

void launch_distill_loss_backward(const float* logits, const float* ids, const float* teacher, const float* stats,
                                  const float* dloss, float* grad, int64_t rows, int64_t width, int top,
                                  float temperature, int accumulate, int* err, cudaStream_t st) {
  if (rows <= 0) return;
  if (rows > INT_MAX) throw CudaError("distill_loss takes up to 2^31 - 1 rows");
  int64_t parts = 1;
  while (rows * parts < 148 * 4 && width / (parts * 2) >= 4 * kDistillThreads && parts < 1024) parts *= 2;
  const int64_t chunk = ceil_div(ceil_div(width, parts), 4) * 4;
  const dim3 grid((unsigned)rows, (unsigned)ceil_div(width, chunk));
  int slots = 16;
  while (slots < 2 * top) slots *= 2;
  const size_t smem = sizeof(float) * (2 * (size_t)top + 3 * (size_t)slots);  // 32 KB at most
  // Rows of both tensors then start at the same offset from a 16-byte boundary.
  const bool vec = (((uintptr_t)logits ^ (uintptr_t)grad) & 15) == 0;
  if (vec)
    distill_backward_kernel<true><<<grid, kDistillThreads, smem, st>>>(logits, ids, teacher, stats, dloss, grad, rows,
                                                                       width, chunk, top, slots, temperature, accumulate, err);
  else
    distill_backward_kernel<false><<<grid, kDistillThreads, smem, st>>>(
        logits, ids, teacher, stats, dloss, grad, rows, width, chunk, top, slots, temperature, accumulate, err);
  check_launch();
}

}  // namespace tysor
