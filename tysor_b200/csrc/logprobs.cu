// Log probabilities of given tokens with entropy and best alternatives
// (lm_ops.cuh), forward and backward.  Both read the logits once (the gradient
// writes as much): HBM bounds them, or for a few rows a launch.
#include <limits.h>
#include <math.h>
#include <stddef.h>

#include <algorithm>

#include "lm_ops.cuh"

namespace tysor {
namespace {

constexpr int kThreads = 256;
constexpr int kLoads = 4;                       // float4 that a thread has on their way
constexpr int kSlab = 4 * kLoads * kThreads;    // values that a block takes at a time
constexpr int kMostParts = 8;                   // blocks of a cluster
constexpr float kLog2e = 1.4426950408889634f;

void check_launch() {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  TYSOR_CUDA(cudaGetLastError());
}

// 2^x to about 2^-22, subnormal results as 0.  (Its error and the rounding of x log2 e make log
// probabilities 1.0e-7 to 1.2e-7 of their norm off, where elementary fp32 operations are 4e-8 to 6e-8.)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The greatest of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ int token_of(float id, int width, int* err) {
  if (id < 0.0f) return -1;
  if (!(id < (float)width)) {  // NaN too; width is at most 2^24, which fp32 holds
    atomicCAS(err, 0, (int)kErrIndexRange);
    return -1;
  }
  return (int)id;
}

// Of some logits: the greatest m, the sum s of 2^y and the sum t of 2^y y, with
// y = (logit - m) log2(e) / T.  (-inf, 0, 0) of none; NaN or +inf as m: not finite.
struct Sums {
  float m, s, t;
};
// y is kept from -inf, whose 2^y = 0 must stay 0 when multiplied by it.
__device__ __forceinline__ float exponent(float z, float m, float c) { return fmaxf((z - m) * c, -200.0f); }
__device__ __forceinline__ bool finite_top(float m) { return m > -INFINITY && m < INFINITY; }
// The sums over a greater greatest value.
__device__ __forceinline__ void raise(Sums& a, float m, float c) {
  const float d = exponent(a.m, m, c), f = exp2_fast(d);
  a.t = f * fmaf(a.s, d, a.t);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  const float m = max3(a.m, b.m, -INFINITY);
  if (!finite_top(m)) return {m, 0.0f, 0.0f};
  if (a.m == -INFINITY) return b;
  if (b.m == -INFINITY) return a;
  raise(a, m, c);
  raise(b, m, c);
  return {m, a.s + b.s, a.t + b.t};
}

// A token and its logit as one number: the greater logit, then the lower id, is the
// greater number.  (-0 counts as 0.)
__device__ __forceinline__ uint64_t key_of(float z, int id) {
  const uint32_t u = __float_as_uint(z == 0.0f ? 0.0f : z);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int id_of(uint64_t key) { return (int)~(uint32_t)key; }

// The candidates for a row's best tokens: keys above `low` so far.  When more than
// `limit` have come, the best `top` stay and `low` rises to the last of them.
constexpr int kListSize = 1024, kCounted = 256;
struct TopList {
  uint64_t key[kListSize];
  uint64_t best[kMaxTopTokens];
  uint64_t low;
  int count, found, digit, need, same;
  int hist[256];
  float warp_floor[kThreads / 32];
  uint64_t incoming[kMostParts * kMaxTopTokens];  // a cluster's, in its first block; not there without one
};

// Leaves the greatest `top` of the list's keys at its start and the last of them as
// `low`: of a few by counting the greater ones, of more by their digits of 8 bits from the
// highest on.  All of the block's threads.
__device__ void keep_best(TopList& l, int top) {
  const int tid = threadIdx.x, n = min(l.count, kListSize);
  __syncthreads();
  if (n <= top) return;
  constexpr int kPer = (kCounted + kThreads - 1) / kThreads;
  if (n <= kCounted) {
    uint64_t mine[kPer];
    int place[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      mine[k] = tid + k * kThreads < n ? l.key[tid + k * kThreads] : 0;
      place[k] = 0;
      if ((tid & ~31) + k * kThreads < n)
#pragma unroll 4
        for (int i = 0; i < n; ++i) place[k] += l.key[i] > mine[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (tid + k * kThreads < n && place[k] < top) {
        l.key[place[k]] = mine[k];
        if (place[k] == top - 1) l.low = mine[k];
      }
    if (tid == 0) l.count = top;
    __syncthreads();
    return;
  }
  uint64_t prefix = 0, mask = 0;
  int need = top;
  for (int shift = 56;; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) l.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads)
      if ((l.key[i] & mask) == prefix) atomicAdd(&l.hist[(int)(l.key[i] >> shift) & 255], 1);
    __syncthreads();
    if (tid < 32) {
      // Lane l counts the digits 8 (31 - l) ... of the greatest first.
      const int first = 8 * (31 - tid);
      int sum = 0;
      for (int i = 0; i < 8; ++i) sum += l.hist[first + i];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (tid >= o) before += x;
      }
      before -= sum;
      if (before < need && before + sum >= need) {
        int d = first + 7;
        while (before + l.hist[d] < need) before += l.hist[d--];
        l.digit = d;
        l.need = need - before;
        l.same = l.hist[d];
      }
    }
    __syncthreads();
    prefix |= (uint64_t)l.digit << shift;
    mask |= (uint64_t)255 << shift;
    need = l.need;
    if (l.same == need || shift == 0) break;  // keys differ: at the last digit they are alone
  }
  if (tid == 0) l.found = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kThreads)
    if ((l.key[i] & mask) >= prefix) l.best[atomicAdd(&l.found, 1)] = l.key[i];
  __syncthreads();
  if (tid < top) l.key[tid] = l.best[tid];
  if (tid < 32) {
    uint64_t least = ~0ull;
    for (int k = tid; k < top; k += 32) least = min(least, l.best[k]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) least = min(least, (uint64_t)__shfl_xor_sync(0xffffffffu, least, k));
    if (tid == 0) l.low = least, l.count = top;
  }
  __syncthreads();
}

// A first floor from a slab's greatest values, one a thread: of each warp's 32 the
// one that enough are not below, so that all warps together hold `top` of at least that.
__device__ __forceinline__ float first_floor(TopList& l, float most, int top) {
  const int lane = threadIdx.x & 31, each = (top + kThreads / 32 - 1) / (kThreads / 32);
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {  // sorted to fall from lane 0 on
      const float other = __shfl_xor_sync(0xffffffffu, most, j);
      const bool first = (lane & j) == 0, falling = (lane & k) == 0;
      most = first == falling ? fmaxf(most, other) : fminf(most, other);
    }
  most = __shfl_sync(0xffffffffu, most, each - 1);
  if (lane == 0) l.warp_floor[threadIdx.x >> 5] = most;
  __syncthreads();
  float floor = l.warp_floor[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) floor = fminf(floor, l.warp_floor[w]);
  return floor;
}

// Adds a key; whether it found no room.
__device__ __forceinline__ bool add_candidate(TopList& l, uint64_t key) {
  const int at = atomicAdd(&l.count, 1);
  if (at < kListSize) l.key[at] = key;
  return at >= kListSize;
}

// Candidates among a slab's values; the bits of those that found no room.
__device__ __forceinline__ uint32_t add_candidates(TopList& l, const float4 (&f)[kLoads], int id, float floor,
                                                   uint64_t low, uint32_t among) {
  uint32_t left = 0;
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const float z[4] = {f[u].x, f[u].y, f[u].z, f[u].w};
    if (!(max3(fmaxf(z[0], z[1]), z[2], z[3]) >= floor)) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (z[e] >= floor && (among >> (4 * u + e) & 1)) {
        const uint64_t key = key_of(z[e], id + 4 * u * kThreads + e);
        if (key > low && add_candidate(l, key)) left |= 1u << (4 * u + e);
      }
  }
  return left;
}

__device__ __forceinline__ void load_slab(float4 (&f)[kLoads], const float4* body, int base, int end) {
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const int i = base + threadIdx.x + u * kThreads;
    f[u] = i < end ? body[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  }
}

// The candidates of [begin, end) once more, where they were more than the list holds
// (rows that rise, or repeat one value): after each slab the best stay, until all have
// found room or are behind.
__device__ __noinline__ void add_slowly(TopList& l, const float4* body, int begin, int end, int head, int top) {
  for (int base = begin; base < end; base += kLoads * kThreads) {
    float4 f[kLoads];
    load_slab(f, body, base, end);
    uint32_t left = 0xffffu;
    for (;;) {
      const uint64_t low = l.low;
      left = add_candidates(l, f, head + 4 * (base + (int)threadIdx.x), logit_of(low), low, left);
      __syncthreads();
      const bool more = l.count > kListSize;
      keep_best(l, top);
      __syncthreads();
      if (!more) break;
    }
  }
}

// One pass over a row, which a cluster of gridDim.y blocks shares where rows are few
// (its first block joins their sums, and their best tokens through distributed shared
// memory).  Without best tokens HBM bounds it: 8192 rows of 32000, 1.05 GB, 164 us = 6.4
// TB/s.  With them the block's waits and choices add up: 2048 rows of 32000 52 us without,
// 65 with the best, 76 with 20, 125 with 128; they want many blocks on an SM (four instead
// of seven, 104 us with 20) more than registers.  32 rows of 32000 take 8 us, with the 20
// best 15: a launch, two exchanges of a cluster, and the choice among its blocks' best.
template <bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? 7 : 6) logprobs_kernel(LogprobShape s, const float* __restrict__ logits,
                                                            const float* __restrict__ ids, float* __restrict__ out,
                                                            float* __restrict__ entropy, float* __restrict__ top_ids,
                                                            float* __restrict__ top_logprobs,
                                                            float* __restrict__ stats, int* err) {
  __shared__ Sums warp_part[kThreads / 32];
  __shared__ Sums part[kMostParts];
  __shared__ int part_count[kMostParts];
  extern __shared__ __align__(16) uint8_t dynamic[];
  TopList& list = *(TopList*)dynamic;  // with TOP alone
  static_assert(kMostParts * kMaxTopTokens <= kListSize, "the cluster's tokens fit the list");
  const int64_t r = blockIdx.x;
  const int parts = gridDim.y, rank = blockIdx.y, tid = threadIdx.x;
  // Arrives for "this block runs": the first block's shared memory is written
  // only once every block of the cluster has got here.
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const float c = kLog2e / s.temperature;
  const float* row = logits + r * s.width;
  // Chunks of whole float4 from the row's first 16-byte boundary; the values before it
  // and after the last whole float4 go to the first block.
  const int head = min(s.width, (int)((4 - (((uintptr_t)row >> 2) & 3)) & 3));
  const int quads = (s.width - head) / 4, per = (quads + parts - 1) / parts;
  const int q0 = min(quads, rank * per), q1 = min(quads, q0 + per);
  const int tail = head + 4 * quads;
  const float4* body = (const float4*)(row + head);
  // Candidates that stay without a choice: choosing early raises the floor, and of more
  // than kCounted takes longer (2048 rows of 32000, 20 best: 76 us, with 84 staying 82; 128
  // best: 125 us, with 160 staying 164).
  const int limit = s.top <= 64 ? s.top + max(8, s.top / 4) : 2 * s.top + 8;
  Sums o{-INFINITY, 0.0f, 0.0f};
  bool bad = false;
  float floor = -INFINITY;
  auto one = [&](float z) {
    if (!finite_top(z)) {
      bad |= !(z == -INFINITY);
      return;
    }
    if (z > o.m) {
      if (o.m > -INFINITY) raise(o, z, c);
      o.m = z;
    }
    const float y = exponent(z, o.m, c), e = exp2_fast(y);
    o.s += e;
    o.t = fmaf(e, y, o.t);
  };
  if (TOP) {
    if (tid == 0) list.count = 0, list.low = key_of(-INFINITY, 0);  // tokens of -inf are not above
    __syncthreads();
  }
  if (rank == 0) {
    const bool here = tid < head;
    const float z = here ? row[tid] : -INFINITY;
    if (here) one(z);
    if (TOP && here && z > -INFINITY) add_candidate(list, key_of(z, tid));
  }
  // The list is looked after when twice as much of the row has been seen, not once a slab:
  // the block's warps then seldom wait for one another.
  int settled = q0, next = q0 + kLoads * kThreads, held = 0;
  if (TOP) {
    __syncthreads();
    held = list.count;
  }
  for (int base = q0; base < q1; base += kLoads * kThreads) {
    float4 f[kLoads];
    load_slab(f, body, base, q1);
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) most = max3(max3(most, f[u].x, f[u].y), f[u].z, f[u].w);
    if (finite_top(most)) {
      if (most > o.m) {
        if (o.m > -INFINITY) raise(o, most, c);
        o.m = most;
      }
      float sum = 0.0f, dot = 0.0f;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const float y0 = exponent(f[u].x, o.m, c), y1 = exponent(f[u].y, o.m, c);
        const float y2 = exponent(f[u].z, o.m, c), y3 = exponent(f[u].w, o.m, c);
        const float e0 = exp2_fast(y0), e1 = exp2_fast(y1), e2 = exp2_fast(y2), e3 = exp2_fast(y3);
        sum += (e0 + e1) + (e2 + e3);
        dot = fmaf(e0, y0, fmaf(e1, y1, fmaf(e2, y2, fmaf(e3, y3, dot))));
      }
      o.s += sum;
      o.t += dot;
    } else {
      bad |= !(most == -INFINITY);
    }
    if (TOP) {
      if (base == q0) floor = first_floor(list, most == most ? most : -INFINITY, s.top);
      if (most >= floor) add_candidates(list, f, head + 4 * (base + tid), floor, list.low, 0xffffu);
      const int end = base + kLoads * kThreads;
      if (end >= next || end >= q1) {
        next = q0 + 2 * (end - q0);
        __syncthreads();
        const int count = list.count;
        __syncthreads();
        if (count > kListSize) {
          if (tid == 0) list.count = held;
          __syncthreads();
          add_slowly(list, body, settled, min(end, q1), head, s.top);
        } else if (count > limit) {
          keep_best(list, s.top);
        }
        held = list.count;
        if (list.low > key_of(-INFINITY, 0)) floor = logit_of(list.low);
        settled = end;
        __syncthreads();
      }
    }
  }
  if (rank == 0) {
    const bool here = tid < s.width - tail;
    const float z = here ? row[tail + tid] : -INFINITY;
    if (here) one(z);
    if (TOP && here && key_of(z, tail + tid) > list.low) add_candidate(list, key_of(z, tail + tid));
  }
  if (bad) o = {NAN, 0.0f, 0.0f};
#pragma unroll
  for (int k = 16; k > 0; k >>= 1)
    o = join(o, {__shfl_xor_sync(0xffffffffu, o.m, k), __shfl_xor_sync(0xffffffffu, o.s, k), __shfl_xor_sync(0xffffffffu, o.t, k)}, c);
  if ((tid & 31) == 0) warp_part[tid >> 5] = o;
  __syncthreads();
  if (TOP) keep_best(list, s.top);
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) o = join(o, warp_part[w], c);
    uint32_t dst;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"((uint32_t)__cvta_generic_to_shared(&part[rank])));
    asm volatile("st.shared::cluster.f32 [%0], %1;\n\tst.shared::cluster.f32 [%0 + 4], %2;\n\tst.shared::cluster.f32 [%0 + 8], %3;" ::"r"(
                     dst), "f"(o.m), "f"(o.s), "f"(o.t)
                 : "memory");
    if (TOP) {
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"((uint32_t)__cvta_generic_to_shared(&part_count[rank])));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(list.count) : "memory");
    }
  }
  if (parts > 1) {
    if (TOP && tid < list.count) {  // at most `top`
      uint32_t dst;
      const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&list.incoming[rank * kMaxTopTokens + tid]);
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"(mine));
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(dst), "l"(list.key[tid]) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
    if (TOP) {
      int n = 0;
      for (int p = 0; p < parts; ++p) {
        if (tid < part_count[p]) list.key[n + tid] = list.incoming[p * kMaxTopTokens + tid];
        n += part_count[p];
      }
      if (tid == 0) list.count = n;
      __syncthreads();
      keep_best(list, s.top);
    }
  }
  __syncthreads();
  Sums all = part[0];
  for (int w = 1; w < parts; ++w) all = join(all, part[w], c);
  const bool none = all.m == -INFINITY, fine = finite_top(all.m);
  const double log_sum = log((double)all.s);
  if (tid == 0) {
    if (stats != nullptr) *(float2*)(stats + 2 * r) = none || fine ? make_float2(all.m, all.s) : make_float2(NAN, NAN);
    if (entropy != nullptr)
      entropy[r] = none ? 0.0f : fine ? (float)(log_sum - 0.6931471805599453 * (double)all.t / (double)all.s) : NAN;
  }
  auto value = [&](float z) {
    return none ? -INFINITY : fine ? (float)(((double)z - (double)all.m) / (double)s.temperature - log_sum) : NAN;
  };
  for (int e = tid; e < s.given; e += kThreads) {
    const int id = token_of(ids[r * s.given + e], s.width, err);
    out[r * s.given + e] = id < 0 ? 0.0f : value(row[id]);
  }
  if (TOP && tid < s.top) {
    const int n = fine ? list.count : 0;
    if (tid < n) {
      const uint64_t key = list.key[tid];
      int place = 0;
      for (int k = 0; k < n; ++k) place += list.key[k] > key;
      top_ids[r * s.top + place] = (float)id_of(key);
      top_logprobs[r * s.top + place] = value(logit_of(key));
    } else {
      top_ids[r * s.top + tid] = -1.0f;
      top_logprobs[r * s.top + tid] = none || fine ? -INFINITY : NAN;
    }
  }
}

// With y as above, p = 2^y / s and ln p = y ln 2 - ln s, a value's gradient is 2^y (a + b y)
// with a and b of the row; the given tokens' own terms are added after.  One block per row
// and chunk of columns.  HBM bounds it: 8192 rows of 32000, 2.1 GB, 333 us = 6.3 TB/s.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(
    LogprobShape s, int chunk, const float* __restrict__ logits, const float* __restrict__ ids,
    const float* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ dout,
    const float* __restrict__ dentropy, float* __restrict__ grad, int accumulate, int* err) {
  __shared__ int token[kMaxGivenTokens];
  __shared__ float up[kMaxGivenTokens];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, c0 = blockIdx.y * chunk, c1 = min(s.width, c0 + chunk);
  const float* row = logits + r * s.width;
  float* g = grad + r * s.width;
  const float2 st = *(const float2*)(stats + 2 * r);
  const float dh = dentropy != nullptr ? dentropy[r] : 0.0f, h = dentropy != nullptr ? entropy[r] : 0.0f;
  for (int e = tid; e < s.given; e += kThreads) {
    token[e] = dout != nullptr ? token_of(ids[r * s.given + e], s.width, err) : -1;
    up[e] = token[e] < 0 ? 0.0f : dout[r * s.given + e];
  }
  __syncthreads();
  if (st.x == -INFINITY) {  // nothing but -inf
    if (!accumulate)
      for (int i = c0 + tid; i < c1; i += kThreads) g[i] = 0.0f;
    return;
  }
  float sum = 0.0f;
  for (int e = 0; e < s.given; ++e) sum += up[e];
  const float inv_t = 1.0f / s.temperature, c = kLog2e / s.temperature;
  const float over = -inv_t / st.y;
  const float a = over * (sum + dh * (h - logf(st.y))), b = over * dh * 0.6931471805599453f;
  auto of = [&](float z) {
    const float y = exponent(z, st.x, c);
    return exp2_fast(y) * fmaf(b, y, a);
  };
  const int head = VEC ? min(c1 - c0, (int)((4 - (((uintptr_t)(row + c0) >> 2) & 3)) & 3)) : 0;
  const int quads = VEC ? (c1 - c0 - head) / 4 : 0;
  const float4* src = (const float4*)(row + c0 + head);
  float4* dst = (float4*)(g + c0 + head);
  for (int i = tid; i < quads; i += kLoads * kThreads) {
    float4 f[kLoads], old[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (i + u * kThreads < quads) f[u] = src[i + u * kThreads];
    if (accumulate)
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
        if (i + u * kThreads < quads) old[u] = dst[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      if (i + u * kThreads >= quads) break;
      float4 d = make_float4(of(f[u].x), of(f[u].y), of(f[u].z), of(f[u].w));
      if (accumulate) d.x += old[u].x, d.y += old[u].y, d.z += old[u].z, d.w += old[u].w;
      dst[i + u * kThreads] = d;
    }
  }
  auto one = [&](int at) {
    const float d = of(row[at]);
    g[at] = accumulate ? g[at] + d : d;
  };
  if (VEC && tid < head) one(c0 + tid);
  for (int at = c0 + head + 4 * quads + tid; at < c1; at += kThreads) one(at);
  __syncthreads();
  // A token given twice takes its terms in order.
  for (int e = tid; e < s.given; e += kThreads) {
    const int id = token[e];
    if (id < c0 || id >= c1) continue;
    bool first = true;
    for (int f = 0; f < e; ++f) first = first && token[f] != id;
    if (!first) continue;
    float d = up[e];
    for (int f = e + 1; f < s.given; ++f)
      if (token[f] == id) d += up[f];
    g[id] += d * inv_t;
  }
}

}  // namespace

void launch_token_logprobs(const LogprobShape& s, const float* logits, const float* ids, float* out, float* entropy,
                           float* top_ids, float* top_logprobs, float* stats, int* err, cudaStream_t st) {
  if (s.rows <= 0) return;
  // Rows that would leave SMs without a block are shared by a cluster's.
  int parts = 1;
  while (parts < kMostParts && s.rows * parts * 2 <= 148 * 4 && s.width / parts > kSlab) parts *= 2;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)s.rows, (unsigned)parts);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = s.top == 0 ? 0 : parts > 1 ? sizeof(TopList) : offsetof(TopList, incoming);
  config.stream = st;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim = {1, (unsigned)parts, 1};
  config.attrs = &cluster;
  config.numAttrs = 1;
  auto kernel = s.top > 0 ? logprobs_kernel<true> : logprobs_kernel<false>;
  TYSOR_CUDA(cudaLaunchKernelEx(&config, kernel, s, logits, ids, out, entropy, top_ids, top_logprobs, stats, err));
  check_launch();
}

void launch_token_logprobs_backward(const LogprobShape& s, const float* logits, const float* ids, const float* stats,
                                    const float* entropy, const float* dout, const float* dentropy, float* grad,
                                    int accumulate, int* err, cudaStream_t st) {
  if (s.rows <= 0) return;
  // Chunks of a row that fill the SMs where rows are few, of at least a slab.
  int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(148 * 8, s.rows), ceil_div(s.width, kSlab)));
  const int chunk = (int)(ceil_div(ceil_div(s.width, chunks), 4) * 4);
  const dim3 grid((unsigned)s.rows, (unsigned)ceil_div(s.width, chunk));
  auto kernel = (((uintptr_t)logits ^ (uintptr_t)grad) & 15) == 0 ? logprobs_backward_kernel<true> : logprobs_backward_kernel<false>;
  kernel<<<grid, kThreads, 0, st>>>(s, chunk, logits, ids, stats, entropy, dout, dentropy, grad, accumulate, err);
  check_launch();
}

}  // namespace tysor
