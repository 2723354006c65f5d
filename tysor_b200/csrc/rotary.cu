// Rotary positions on part of a head, in either layout, scaled for long contexts
// (lm_ops.cuh), forward and backward.
#include <limits.h>
#include <math.h>

#include "lm_ops.cuh"

namespace tysor {
namespace {

constexpr int kRotaryThreads = 256;

// N neighbouring values, at an address that is a multiple of theirs.
template <int N>
__device__ __forceinline__ void load_values(float* f, const float* p) {
  if constexpr (N == 4) {
    const float4 w = *(const float4*)p;
    f[0] = w.x, f[1] = w.y, f[2] = w.z, f[3] = w.w;
  } else if constexpr (N == 2) {
    const float2 w = *(const float2*)p;
    f[0] = w.x, f[1] = w.y;
  } else {
    f[0] = *p;
  }
}
template <int N>
__device__ __forceinline__ void store_values(float* p, const float* f) {
  if constexpr (N == 4) *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
  else if constexpr (N == 2) *(float2*)p = make_float2(f[0], f[1]);
  else *p = f[0];
}

// A thread takes V pairs of a token (or 2 V values behind the turned part, which
// it copies), forms their angles once, in 64 bits, and goes over a range of heads.
// Each value is read and written once: HBM bounds it (8 x 2048 tokens of 16 heads of 128,
// half of them turned, 268 MB in 51 us = 5.3 TB/s), or one launch's latency (6 us for one
// token of 32 sequences).  An odd number of pairs
// moves 4 bytes at a time: 16385 x 5 heads of 90, 59 MB in 19 us = 3.1 TB/s (8 bytes for
// neighbours that turn together are no faster); pairs by two, 8 x 2048 tokens of 16 heads of
// 128 with 44 turned, take 63 us, one at a time 86.
// `Index` counts the units: 64-bit divisions would take as long as the rest.
template <int V, bool INTERLEAVED, typename Index>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const float* __restrict__ x,
                                                                const float* __restrict__ positions,
                                                                float* __restrict__ out,
                                                                const __grid_constant__ RotaryShape s, int head_chunk,
                                                                int back, int accumulate) {
  constexpr int W = INTERLEAVED && V == 2 ? 4 : V;  // the turned values of one load
  const int turned = s.half / V;                                            // units that turn
  const int per = turned + (s.head_dim - 2 * s.half + 2 * V - 1) / (2 * V);  // and those that do not
  const Index item = (Index)blockIdx.x * kRotaryThreads + threadIdx.x;
  if (item >= (Index)s.batch * (Index)s.seq * (Index)per) return;
  const Index token32 = item / (Index)per;
  const int unit = (int)(item - token32 * (Index)per);
  const int64_t token = (int64_t)token32, b = (int64_t)(token32 / (Index)s.seq), at = token - b * s.seq;
  const int64_t step = s.seq_major ? s.head_dim : (int64_t)s.head_dim * s.seq;
  const int64_t base = (s.seq_major ? (b * s.seq + at) * s.heads : b * s.heads * s.seq + at) * s.head_dim;
  const int h0 = blockIdx.y * head_chunk, h1 = min(s.heads, h0 + head_chunk);
  if (unit >= turned) {
    const int c = 2 * s.half + (unit - turned) * 2 * V;
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      const int64_t o = base + h * step + c;
      if (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          float4 f = *(const float4*)(x + o + 4 * i);
          if (accumulate) {
            const float4 g = *(const float4*)(out + o + 4 * i);
            f.x += g.x, f.y += g.y, f.z += g.z, f.w += g.w;
          }
          *(float4*)(out + o + 4 * i) = f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i)
          if (c + i < s.head_dim) out[o + i] = accumulate ? out[o + i] + x[o + i] : x[o + i];
      }
    }
    return;
  }
  const int i0 = unit * V;
  const double place = positions != nullptr ? (double)positions[token] : (double)at;
  float cs[V], sn[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const double turns = place * s.rates[i0 + v];
    sincospif(2.0f * (float)(turns - rint(turns)), &sn[v], &cs[v]);
    cs[v] *= s.amplitude;
    sn[v] *= back ? -s.amplitude : s.amplitude;
  }
  // The unit's values: V and V of them `half` apart, or 2 V in a row.
  const int first = INTERLEAVED ? 2 * i0 : i0, second = INTERLEAVED ? first + V : first + s.half;
  auto spot = [&](int e) { return e < V ? first + e : second + e - V; };
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const int64_t o = base + h * step;
    float f[2 * V];
#pragma unroll
    for (int e = 0; e < 2 * V; e += W) load_values<W>(f + e, x + o + spot(e));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float &lo = f[INTERLEAVED ? 2 * v : v], &hi = f[INTERLEAVED ? 2 * v + 1 : V + v];
      const float t = lo * cs[v] - hi * sn[v];
      hi = lo * sn[v] + hi * cs[v];
      lo = t;
    }
#pragma unroll
    for (int e = 0; e < 2 * V; e += W) {
      if (accumulate) {
        float old[W];
        load_values<W>(old, out + o + spot(e));
#pragma unroll
        for (int i = 0; i < W; ++i) f[e + i] += old[i];
      }
      store_values<W>(out + o + spot(e), f + e);
    }
  }
}

}  // namespace

const char* rotary_rates_problem(const RotaryRates& r, double amplitude) {
  if (r.half < 1 || r.half > kMaxRotaryPairs) return "rotary turns 2 to 512 values of a head, an even number";
  if (!(r.theta > 0.0) || std::isinf(r.theta)) return "rotary requires a finite theta > 0";
  if (!(fabs(amplitude) <= 3.4e38)) return "rotary requires a finite amplitude";
  if (r.scaling < kRotaryPlain || r.scaling > kRotaryLogTurns) return "rotary takes scalings 0 to 3";
  if (r.scaling != kRotaryPlain && (!(r.factor > 0.0) || std::isinf(r.factor)))
    return "rotary requires a finite factor > 0";
  if (r.scaling >= kRotaryTurns) {
    if (!(r.context > 0.0) || std::isinf(r.context)) return "rotary requires a finite original length > 0";
    if (!(r.low >= 0.0) || !(r.high > r.low) || std::isinf(r.high) || (r.scaling == kRotaryLogTurns && r.low == 0.0))
      return "rotary requires turns 0 <= low < high (0 < low by logarithms)";
  }
  return nullptr;
}

void rotary_fill_rates(const RotaryRates& r, double* rates) {
  const double circle = 2.0 * 3.14159265358979323846;
  for (int i = 0; i < r.half; ++i) {
    const double rate = pow(r.theta, -(double)i / r.half) / circle;  // revolutions a position
    double keep = r.scaling == kRotaryPlain ? 1.0 : 0.0;
    if (r.scaling >= kRotaryTurns) {
      const double turns = r.context * rate;
      keep = r.scaling == kRotaryTurns ? (turns - r.low) / (r.high - r.low) : log(turns / r.low) / log(r.high / r.low);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
    }
    rates[i] = r.scaling == kRotaryPlain ? rate : rate * (keep + (1.0 - keep) / r.factor);
  }
}

void launch_rotary(const float* x, const float* positions, float* out, const RotaryShape& shape, int back,
                   int accumulate, cudaStream_t st) {
  const int64_t tokens = (int64_t)shape.batch * shape.seq;
  if (tokens <= 0 || shape.heads <= 0) return;
  // As wide as a head's halves and width and the tensors' starts allow.
  const uintptr_t starts = (uintptr_t)x | (uintptr_t)out;
  const int V = shape.half % 4 == 0 && shape.head_dim % 8 == 0 && starts % 16 == 0   ? 4
                : shape.half % 2 == 0 && shape.head_dim % 4 == 0 && starts % 16 == 0 ? 2
                                                                                     : 1;
  const int64_t items = tokens * (shape.half / V + ceil_div(shape.head_dim - 2 * shape.half, 2 * V));
  // The heads of a token in one thread share its angles; where that leaves fewer than
  // eight blocks per SM, they are spread over more threads (8 x 2048 tokens of 16 heads
  // forward and back 107 us with two, 103 with eight, 117 with 32).
  int64_t chunk = shape.heads * items / (148 * 8 * kRotaryThreads);
  const int64_t least = ceil_div(shape.heads, 65535);  // blocks of the grid's second axis
  chunk = chunk < least ? least : chunk > shape.heads ? shape.heads : chunk;
  const dim3 grid((unsigned)ceil_div(items, kRotaryThreads), (unsigned)ceil_div(shape.heads, chunk));
  auto go = [&](auto kernel) {
    kernel<<<grid, kRotaryThreads, 0, st>>>(x, positions, out, shape, (int)chunk, back, accumulate);
  };
  auto pick = [&]<typename Index>(Index) {
    if (V == 4) shape.interleaved ? go(rotary_kernel<4, true, Index>) : go(rotary_kernel<4, false, Index>);
    else if (V == 2) shape.interleaved ? go(rotary_kernel<2, true, Index>) : go(rotary_kernel<2, false, Index>);
    else shape.interleaved ? go(rotary_kernel<1, true, Index>) : go(rotary_kernel<1, false, Index>);
  };
  if (items < INT64_C(4000000000)) pick(uint32_t{});
  else pick(int64_t{});
  g_launches.fetch_add(1, std::memory_order_relaxed);
  TYSOR_CUDA(cudaGetLastError());
}

}  // namespace tysor
