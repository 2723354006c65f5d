// Linear attention with a decay for each head (lm_ops.cuh), forward and backward.
//
// One recurrence does all of it.  A scan takes tokens with a query, a key and a
// value each, and holds a state X (rows as wide as keys, columns as values):
//   forward in time:   X = a X + k v^T,  out = scale * q X
//   back in time:      X = X + k v^T,    out = scale * q X,  X = a X
// The forward pass is a scan of (q, k, v); its gradients are three more, since
//   dq = a scan of (dout, v, k), whose state is the forward's transposed,
//   dv = a scan back of (k, q, dout) and dk of (v, dout, q) (the same, transposed).
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

// Rows of one operand: those of sequence b, head h start at b * batch + (h / share) * head.
struct Rows {
  const float* p;
  int64_t batch, head, token;
  int share;
  __device__ __forceinline__ const float* at(int b, int h) const { return p + b * batch + (h / share) * head; }
};

// A state's value of key row i and value column j is at unit * rows * cols + i * si + j * sj.
struct StateAt {
  float* p;
  int64_t si, sj;
};

struct Scan {
  int batch, heads, seq, rows, cols;  // rows: the keys' width, cols: the values'
  Rows q, k, v, out;                  // out.p is written
  const float *decay, *lengths;
  StateAt from, to;                   // where the state starts and ends, or null
  float scale, from_factor, to_factor;  // of the outputs, the first and the last state
  int back;
  int accumulate, accumulate_state;
};

// The number of tokens of sequence b.
__device__ __forceinline__ int tokens_of(const Scan& s, int b, int* err) {
  if (s.lengths == nullptr) return s.seq;
  const float v = s.lengths[b];
  if (v >= 0.0f && v <= (float)s.seq) {
    const int n = (int)fminf(v, 2147483520.0f);
    if (n <= s.seq && (float)n == v) return n;
  }
  atomicCAS(err, 0, (int)kErrSequence);
  return 0;
}

// A head's decay per token in powers of e, at least 0.
__device__ __forceinline__ float decay_of(const Scan& s, int h, int* err) {
  const float d = s.decay[h];
  if (d >= 0.0f) return d;
  atomicCAS(err, 0, (int)kErrDecay);
  return 0.0f;
}

// exp(-decay * steps) as a sum of two floats: a state is multiplied by it once per
// step, so the rounding of one float alone would grow with their number.
__device__ __forceinline__ float2 decay_over(float decay, int steps) {
  const double a = steps == 0 ? 1.0 : exp(-(double)decay * steps);
  const float hi = (float)a;
  return make_float2(hi, (float)(a - (double)hi));
}

// ---- token by token --------------------------------------------------------------

// A block holds `kSlice` columns of one head's state, four columns and every 32nd
// row a thread, and takes the tokens one after the other.  For few tokens what
// counts is reading and writing the state.
constexpr int kStepThreads = 256, kSlice = 32, kStage = 16;
constexpr int kMostDim = 128;

template <bool VEC>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const __grid_constant__ Scan s, int* err) {
  __shared__ float qs[kStage][kMostDim], ks[kStage][kMostDim];
  __shared__ __align__(16) float vs[kStage][kSlice];
  __shared__ __align__(16) float red[2][kStepThreads / 32][kSlice];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x, b = unit / s.heads, h = unit - b * s.heads;
  const int c0 = blockIdx.y * kSlice, width = min(kSlice, s.cols - c0);
  const int c = 4 * (lane & 7), r0 = warp * 4 + (lane >> 3);
  const int64_t state = (int64_t)unit * s.rows * s.cols;
  float x[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 32 * i;
    if (VEC) {
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (s.from.p != nullptr && r < s.rows && c < width)
        f = *(const float4*)(s.from.p + state + (int64_t)r * s.cols + c0 + c);
      x[i][0] = f.x, x[i][1] = f.y, x[i][2] = f.z, x[i][3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[i][j] = s.from.p != nullptr && r < s.rows && c + j < width
                      ? s.from.p[state + r * s.from.si + (c0 + c + j) * s.from.sj]
                      : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i][j] *= s.from_factor;
  }
  const int n = tokens_of(s, b, err);
  const float2 a = decay_over(decay_of(s, h, err), 1);
  const float *q = s.q.at(b, h), *k = s.k.at(b, h), *v = s.v.at(b, h) + c0;
  float* out = const_cast<float*>(s.out.at(b, h)) + c0;
  auto fade = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = fmaf(x[i][j], a.x, x[i][j] * a.y);
  };
  for (int t0 = 0; t0 < n; t0 += kStage) {
    const int m = min(kStage, n - t0);
    auto token = [&](int t) { return (int64_t)(s.back ? n - 1 - t0 - t : t0 + t); };
    __syncthreads();
    for (int i = tid; i < m * kMostDim; i += kStepThreads) {
      const int t = i / kMostDim, r = i % kMostDim;
      qs[t][r] = r < s.rows ? q[token(t) * s.q.token + r] : 0.0f;
      ks[t][r] = r < s.rows ? k[token(t) * s.k.token + r] : 0.0f;
    }
    for (int i = tid; i < m * kSlice; i += kStepThreads) {
      const int t = i / kSlice, j = i % kSlice;
      vs[t][j] = j < width ? v[token(t) * s.v.token + j] : 0.0f;
    }
    __syncthreads();
    for (int t = 0; t < m; ++t) {
      const float4 w = *(const float4*)&vs[t][c];
      float o[4] = {};
      if (!s.back) fade();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float key = ks[t][r0 + 32 * i], query = qs[t][r0 + 32 * i];
        x[i][0] = fmaf(key, w.x, x[i][0]), x[i][1] = fmaf(key, w.y, x[i][1]);
        x[i][2] = fmaf(key, w.z, x[i][2]), x[i][3] = fmaf(key, w.w, x[i][3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(query, x[i][j], o[j]);
      }
      if (s.back) fade();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] += __shfl_xor_sync(0xffffffffu, o[j], 8);
        o[j] += __shfl_xor_sync(0xffffffffu, o[j], 16);
      }
      if (lane < 8) *(float4*)&red[t & 1][warp][c] = make_float4(o[0], o[1], o[2], o[3]);
      __syncthreads();
      if (tid < width) {
        float sum = 0.0f;
#pragma unroll
        for (int w2 = 0; w2 < kStepThreads / 32; ++w2) sum += red[t & 1][w2][tid];
        float* to = out + token(t) * s.out.token + tid;
        *to = s.accumulate ? *to + sum * s.scale : sum * s.scale;
      }
    }
  }
  if (!s.accumulate)  // rows behind the sequence's end
    for (int i = tid; i < (s.seq - n) * kSlice; i += kStepThreads)
      if (i % kSlice < width) out[(int64_t)(n + i / kSlice) * s.out.token + i % kSlice] = 0.0f;
  if (s.to.p == nullptr) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 32 * i;
    if (r >= s.rows || c >= width) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i][j] *= s.to_factor;
    if (VEC) {
      float4* to = (float4*)(s.to.p + state + (int64_t)r * s.cols + c0 + c);
      float4 f = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
      if (s.accumulate_state) {
        const float4 g = *to;
        f.x += g.x, f.y += g.y, f.z += g.z, f.w += g.w;
      }
      *to = f;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < width) {
          float* to = s.to.p + state + r * s.to.si + (c0 + c + j) * s.to.sj;
          *to = s.accumulate_state ? *to + x[i][j] : x[i][j];
        }
    }
  }
}

// dst[b][g] (+)= sum over the heads that share key head g of src[b][h], in order.
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* __restrict__ src, Rows dst, int batch,
                                                        int kv_heads, int group, int seq, int dim, int accumulate) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)batch * kv_heads * seq * dim;
  if (i >= n) return;
  const int64_t row = i / dim, c = i - row * dim;
  const int64_t bg = row / seq, t = row - bg * seq;
  const float* from = src + (bg * group * seq + t) * dim + c;
  float sum = 0.0f;
  for (int k = 0; k < group; ++k) sum += from[(int64_t)k * seq * dim];
  float* to = const_cast<float*>(dst.p) + bg / kv_heads * dst.batch + bg % kv_heads * dst.head + t * dst.token + c;
  *to = accumulate ? *to + sum : sum;
}

void run_scan(const Scan& s, int* err, cudaStream_t st) {
  if (s.batch <= 0 || s.heads <= 0) return;
  auto plain = [&](const StateAt& x) {
    return x.p == nullptr || (x.si == s.cols && x.sj == 1 && ((uintptr_t)x.p & 15) == 0);
  };
  const dim3 grid((unsigned)(s.batch * s.heads), (unsigned)ceil_div(s.cols, kSlice));
  if (s.cols % 4 == 0 && plain(s.from) && plain(s.to)) step_kernel<true><<<grid, kStepThreads, 0, st>>>(s, err);
  else step_kernel<false><<<grid, kStepThreads, 0, st>>>(s, err);
  check_launch();
}

Rows rows_of(const DecayShape& s, const float* p, int heads, int dim, int share) {
  if (s.seq_major) return {p, (int64_t)s.seq * heads * dim, dim, (int64_t)heads * dim, share};
  return {p, (int64_t)heads * s.seq * dim, (int64_t)s.seq * dim, dim, share};
}

Scan scan_of(const DecayShape& s, const DecayInputs& in) {
  Scan c{};
  c.batch = s.batch;
  c.heads = s.heads;
  c.seq = s.seq;
  c.decay = in.decay;
  c.lengths = in.lengths;
  c.scale = s.scale;
  c.from_factor = c.to_factor = 1.0f;
  return c;
}

}  // namespace

const char* decay_attention_problem(uint64_t batch, uint64_t heads, uint64_t kv_heads, uint64_t seq, uint64_t key_dim,
                                    uint64_t value_dim, float scale) {
  if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0)
    return "decay_attention: the key heads must divide the query heads";
  if (key_dim == 0 || value_dim == 0 || key_dim > kMostDim || value_dim > kMostDim)
    return "decay_attention takes keys and values of 1 to 128";
  const uint64_t most = 1u << 29;
  if (seq > most || batch > most || heads > most || batch * heads > INT32_MAX)
    return "decay_attention takes lengths, batches and heads up to 2^29, and 2^31 - 1 heads in all";
  if (!(scale >= 0x1p-60f && scale <= 0x1p60f)) return "decay_attention requires a scale from 2^-60 to 2^60";
  return nullptr;
}

int64_t decay_attention_work_elems(const DecayShape&) { return 0; }

int64_t decay_attention_backward_work_elems(const DecayShape& s) {
  if (s.heads == s.kv_heads) return 0;
  return (int64_t)s.batch * s.heads * s.seq * std::max(s.key_dim, s.value_dim);
}

void launch_decay_attention(const DecayShape& s, const DecayInputs& in, float* out, float* new_state, float*,
                            int* err, cudaStream_t st) {
  const int share = s.heads / s.kv_heads;
  Scan c = scan_of(s, in);
  c.rows = s.key_dim;
  c.cols = s.value_dim;
  c.q = rows_of(s, in.q, s.heads, s.key_dim, 1);
  c.k = rows_of(s, in.k, s.kv_heads, s.key_dim, share);
  c.v = rows_of(s, in.v, s.kv_heads, s.value_dim, share);
  c.out = rows_of(s, out, s.heads, s.value_dim, 1);
  c.from = {const_cast<float*>(in.state), s.value_dim, 1};
  c.to = {new_state, s.value_dim, 1};
  run_scan(c, err, st);
}

void launch_decay_attention_backward(const DecayShape& s, const DecayInputs& in, const float* dout,
                                     const float* dnew_state, float* dq, float* dk, float* dv, float* dstate,
                                     float* work, int accumulate_q, int accumulate_k, int accumulate_v,
                                     int accumulate_state, int* err, cudaStream_t st) {
  const int share = s.heads / s.kv_heads;
  const Rows q = rows_of(s, in.q, s.heads, s.key_dim, 1), k = rows_of(s, in.k, s.kv_heads, s.key_dim, share);
  const Rows v = rows_of(s, in.v, s.kv_heads, s.value_dim, share), g = rows_of(s, dout, s.heads, s.value_dim, 1);
  Scan c = scan_of(s, in);
  c.rows = s.value_dim;
  c.cols = s.key_dim;
  c.q = g;
  c.k = v;
  c.v = k;
  c.out = rows_of(s, dq, s.heads, s.key_dim, 1);
  c.from = {const_cast<float*>(in.state), 1, s.value_dim};
  c.accumulate = accumulate_q;
  run_scan(c, err, st);

  // The states of the scans back are the gradients' over `scale`.
  c.back = 1;
  c.from_factor = 1.0f / s.scale;
  c.to_factor = s.scale;
  auto keys = [&](float* grad, int dim, int accumulate) {
    const Rows to = rows_of(s, grad, s.kv_heads, dim, 1);
    if (share == 1) {
      c.out = to;
      c.accumulate = accumulate;
      run_scan(c, err, st);
      return;
    }
    c.out = {work, (int64_t)s.heads * s.seq * dim, (int64_t)s.seq * dim, dim, 1};
    c.accumulate = 0;
    run_scan(c, err, st);
    const int64_t n = (int64_t)s.batch * s.kv_heads * s.seq * dim;
    if (n <= 0) return;
    sum_heads_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, st>>>(work, to, s.batch, s.kv_heads, share, s.seq, dim,
                                                                 accumulate);
    check_launch();
  };
  c.q = v;
  c.k = g;
  c.v = q;
  c.from = {const_cast<float*>(dnew_state), 1, s.value_dim};
  keys(dk, s.key_dim, accumulate_k);
  c.rows = s.key_dim;
  c.cols = s.value_dim;
  c.q = k;
  c.k = q;
  c.v = g;
  c.from = {const_cast<float*>(dnew_state), s.value_dim, 1};
  c.to = {dstate, s.value_dim, 1};
  c.accumulate_state = accumulate_state;
  keys(dv, s.value_dim, accumulate_v);
}

}  // namespace tysor
