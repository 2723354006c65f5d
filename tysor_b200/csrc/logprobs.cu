// Log probabilities of given tokens with entropy and best alternatives
// (lm_ops.cuh), forward and backward.
#include <limits.h>
#include <math.h>

#include "lm_ops.cuh"

namespace tysor {
namespace {

constexpr int kThreads = 256;

void check_launch() {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  TYSOR_CUDA(cudaGetLastError());
}

__device__ __forceinline__ int token_of(float id, int width, int* err) {
  if (id < 0.0f) return -1;
  if (!(id < (float)width)) {  // NaN too; width is at most 2^24, which fp32 holds
    atomicCAS(err, 0, (int)kErrIndexRange);
    return -1;
  }
  return (int)id;
}

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* red, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kThreads / 32; ++w) v = f(v, red[w]);
  return v;
}

__global__ void __launch_bounds__(kThreads) logprobs_kernel(LogprobShape s, const float* __restrict__ logits,
                                                            const float* __restrict__ ids, float* __restrict__ out,
                                                            float* __restrict__ entropy, float* __restrict__ top_ids,
                                                            float* __restrict__ top_logprobs,
                                                            float* __restrict__ stats, int* err) {
  __shared__ float red[kThreads / 32];
  const int64_t r = blockIdx.x;
  const float* row = logits + r * s.width;
  auto add = [](float a, float b) { return a + b; };
  auto most = [](float a, float b) { return a > b || a != a ? a : b; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < s.width; i += kThreads) m = most(row[i], m);
  m = block_reduce(m, red, most);
  const bool none = m == -INFINITY, bad = !(m < INFINITY);
  float sum = 0.0f, dot = 0.0f;
  if (!none && !bad)
    for (int i = threadIdx.x; i < s.width; i += kThreads) {
      const float y = (row[i] - m) / s.temperature, e = expf(y);
      sum += e;
      if (e > 0.0f) dot += e * y;
    }
  sum = block_reduce(sum, red, add);
  dot = block_reduce(dot, red, add);
  if (bad) m = sum = NAN;
  const float log_sum = logf(sum);
  if (threadIdx.x == 0) {
    if (stats != nullptr) *(float2*)(stats + 2 * r) = make_float2(m, sum);
    if (entropy != nullptr) entropy[r] = none ? 0.0f : log_sum - dot / sum;
  }
  auto value = [&](int id) { return none ? -INFINITY : (row[id] - m) / s.temperature - log_sum; };
  for (int e = threadIdx.x; e < s.given; e += kThreads) {
    const int id = token_of(ids[r * s.given + e], s.width, err);
    out[r * s.given + e] = id < 0 ? 0.0f : value(id);
  }
  // The best token below the one before, one by one.
  float last = INFINITY;
  int last_id = -1;
  for (int k = 0; k < s.top; ++k) {
    float best = -INFINITY;
    int id = INT_MAX;
    for (int i = threadIdx.x; i < s.width; i += kThreads) {
      const float v = row[i];
      if ((v < last || (v == last && i > last_id)) && v > best) best = v, id = i;
    }
    const float all = block_reduce(best, red, most);
    const float at = block_reduce(best == all ? (float)id : 1e30f, red, [](float a, float b) { return fminf(a, b); });
    const bool found = all > -INFINITY && !bad;
    last = all, last_id = found ? (int)at : 0;
    if (threadIdx.x == 0) {
      top_ids[r * s.top + k] = found ? at : -1.0f;
      top_logprobs[r * s.top + k] = bad ? NAN : found ? value(last_id) : -INFINITY;
    }
  }
}

__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(
    LogprobShape s, const float* __restrict__ logits, const float* __restrict__ ids, const float* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ dout, const float* __restrict__ dentropy,
    float* __restrict__ grad, int accumulate, int* err) {
  __shared__ int token[kMaxGivenTokens];
  __shared__ float up[kMaxGivenTokens];
  const int64_t r = blockIdx.x;
  const float* row = logits + r * s.width;
  float* g = grad + r * s.width;
  const float2 st = *(const float2*)(stats + 2 * r);
  for (int e = threadIdx.x; e < s.given; e += kThreads) {
    token[e] = dout != nullptr ? token_of(ids[r * s.given + e], s.width, err) : -1;
    up[e] = token[e] < 0 ? 0.0f : dout[r * s.given + e];
  }
  __syncthreads();
  float sum = 0.0f;
  for (int e = 0; e < s.given; ++e) sum += up[e];
  const float dh = dentropy != nullptr ? dentropy[r] : 0.0f, h = dentropy != nullptr ? entropy[r] : 0.0f;
  const bool none = st.x == -INFINITY;
  const float log_sum = logf(st.y), inv = 1.0f / s.temperature;
  for (int i = threadIdx.x; i < s.width; i += kThreads) {
    float d = 0.0f;
    if (!none) {
      const float lp = (row[i] - st.x) / s.temperature - log_sum, p = expf(lp);
      d = p == 0.0f ? 0.0f : -p * (sum + dh * (lp + h)) * inv;
    }
    g[i] = accumulate ? g[i] + d : d;
  }
  __syncthreads();
  if (none) return;
  for (int e = threadIdx.x; e < s.given; e += kThreads) {
    bool first = token[e] >= 0;
    for (int f = 0; f < e; ++f) first = first && token[f] != token[e];
    if (!first) continue;
    float d = 0.0f;
    for (int f = e; f < s.given; ++f)
      if (token[f] == token[e]) d += up[f];
    g[token[e]] += d * inv;
  }
}

}  // namespace

void launch_token_logprobs(const LogprobShape& s, const float* logits, const float* ids, float* out, float* entropy,
                           float* top_ids, float* top_logprobs, float* stats, int* err, cudaStream_t st) {
  if (s.rows <= 0) return;
  logprobs_kernel<<<(unsigned)s.rows, kThreads, 0, st>>>(s, logits, ids, out, entropy, top_ids, top_logprobs, stats,
                                                         err);
  check_launch();
}

void launch_token_logprobs_backward(const LogprobShape& s, const float* logits, const float* ids, const float* stats,
                                    const float* entropy, const float* dout, const float* dentropy, float* grad,
                                    int accumulate, int* err, cudaStream_t st) {
  if (s.rows <= 0) return;
  logprobs_backward_kernel<<<(unsigned)s.rows, kThreads, 0, st>>>(s, logits, ids, stats, entropy, dout, dentropy, grad,
                                                                  accumulate, err);
  check_launch();
}

}  // namespace tysor
