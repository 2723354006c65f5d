// Linear attention with a decay for each head (lm_ops.cuh), forward and backward.
//
// One recurrence does all of it.  A scan takes tokens with a query, a key and a
// value each, and holds a state X (rows as wide as keys, columns as values):
//   forward in time:   X = a X + k v^T,  out = scale * q X
//   back in time:      X = X + k v^T,    out = scale * q X,  X = a X
// The forward pass is a scan of (q, k, v); its gradients are three more, since
//   dq = a scan of (dout, v, k), whose state is the forward's transposed,
//   dv = a scan back of (k, q, dout) and dk of (v, dout, q) (the same, transposed).
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

// A bounded wait of a warp whose lanes sleep meanwhile (try_wait with a hint of 2 ms): the
// pipeline's roles wait for most of a step, and asking again and again takes issue slots
// from those that work.
__device__ __forceinline__ bool sleep_wait(uint32_t bar, uint32_t parity, int* err) {
  auto done = [&] {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(2000000u)
        : "memory");
    return ok != 0;
  };
  bool ok = done();
  if (!ok) {
    const long long start = clock64();
    while (!(ok = done()))
      if (clock64() - start > kWaitCycles) {
        atomicCAS(err, 0, (int)kErrBarrierTimeout);
        break;
      }
  }
  return __all_sync(0xffffffffu, ok);
}

// Two fp32 values for the paired instructions.
typedef float2 Pair;
__device__ __forceinline__ Pair pair_of(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { return __ffma2_rn(a, b, c); }

// ---- token by token --------------------------------------------------------------

// A block holds `kSlice` columns of one head's state, four columns and every 16th
// row a thread, and takes the tokens one after the other.  For few tokens what
// counts is reading and writing the state: one token of 32 sequences of 16 heads of 128, 67 MB,
// 18 us out of HBM = 3.8 TB/s, 13 us where the state is still in L2; 16 states take 9 us, a
// launch and the way to memory and back.  The blocks' number counts: 256 threads with 64
// bytes of state each, four blocks an SM, took 22 us, and the first token's loads
// before the state is waited for need registers that the threads do not have (15 us in place
// of 13).  Every further token is 2.3 us, for its sums over the threads.
constexpr int kMostDim = 128;
constexpr int kStepThreads = 128, kSlice = 32, kStage = 8;
constexpr int kStepRows = kStepThreads / 8, kStepMine = kMostDim / kStepRows;  // rows at a time, and of a thread

template <bool VEC>
__global__ void __launch_bounds__(kStepThreads, 8) step_kernel(const __grid_constant__ Scan s, int* err) {
  __shared__ float qs[kStage][kMostDim], ks[kStage][kMostDim];
  __shared__ __align__(16) float vs[kStage][kSlice];
  __shared__ __align__(16) float red[2][kStepThreads / 32][kSlice];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x, b = unit / s.heads, h = unit - b * s.heads;
  const int c0 = blockIdx.y * kSlice, width = min(kSlice, s.cols - c0);
  const int c = 4 * (lane & 7), r0 = warp * 4 + (lane >> 3);
  const int64_t state = (int64_t)unit * s.rows * s.cols;
  Pair x[kStepMine][2];
#pragma unroll
  for (int i = 0; i < kStepMine; ++i) {
    const int r = r0 + kStepRows * i;
    float f[4] = {};
    if (VEC) {
      if (s.from.p != nullptr && r < s.rows && c < width) {
        const float4 w = *(const float4*)(s.from.p + state + (int64_t)r * s.cols + c0 + c);
        f[0] = w.x, f[1] = w.y, f[2] = w.z, f[3] = w.w;
      }
    } else if (s.from.p != nullptr && r < s.rows) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < width) f[j] = s.from.p[state + r * s.from.si + (c0 + c + j) * s.from.sj];
    }
    x[i][0] = pair_of(f[0] * s.from_factor, f[1] * s.from_factor);
    x[i][1] = pair_of(f[2] * s.from_factor, f[3] * s.from_factor);
  }
  const int n = tokens_of(s, b, err);
  const float2 a = decay_over(decay_of(s, h, err), 1);
  const float *q = s.q.at(b, h), *k = s.k.at(b, h), *v = s.v.at(b, h) + c0;
  float* out = const_cast<float*>(s.out.at(b, h)) + c0;
  const Pair fade_hi = pair_of(a.x, a.x), fade_lo = pair_of(a.y, a.y);
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
      const Pair w2[2] = {pair_of(w.x, w.y), pair_of(w.z, w.w)};
      Pair sum[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll
      for (int i = 0; i < kStepMine; ++i) {
        const float key = ks[t][r0 + kStepRows * i], query = qs[t][r0 + kStepRows * i];
        const Pair key2 = pair_of(key, key), query2 = pair_of(query, query);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          Pair& y = x[i][j];
          const Pair add = mul2(key2, w2[j]);
          // Forward in time the state fades first, back in time afterwards.
          y = s.back ? fma2(key2, w2[j], y) : fma2(y, fade_hi, fma2(y, fade_lo, add));
          sum[j] = fma2(query2, y, sum[j]);
          if (s.back) y = fma2(y, fade_hi, mul2(y, fade_lo));
        }
      }
      float o[4] = {sum[0].x, sum[0].y, sum[1].x, sum[1].y};
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
  for (int i = 0; i < kStepMine; ++i) {
    const int r = r0 + kStepRows * i;
    if (r >= s.rows || c >= width) continue;
    const float2 y0 = x[i][0], y1 = x[i][1];
    float4 f = make_float4(y0.x * s.to_factor, y0.y * s.to_factor, y1.x * s.to_factor, y1.y * s.to_factor);
    if (VEC) {
      float4* to = (float4*)(s.to.p + state + (int64_t)r * s.cols + c0 + c);
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
          const float y = j == 0 ? f.x : j == 1 ? f.y : j == 2 ? f.z : f.w;
          *to = s.accumulate_state ? *to + y : y;
        }
    }
  }
}

// ---- 64 tokens at a time ----------------------------------------------------------

// With X the state before 64 tokens, i and j counting them, lead = 1 and tail = 0
// forward in time (0 and 1 back), a scan is four matrix products:
//   out_i = scale * (a^(i + lead) q_i X + sum over j <= i of P_ij v_j),  P_ij = a^(i - j) q_i.k_j
//   X <- a^64 X + sum over j of a^(63 - j + tail) k_j v_j^T
// fp32 accuracy out of fp16 matrix instructions, as in the attention kernels: an
// operand is scaled by a power of two and split into hi = fp16(x) and lo =
// fp16(x - hi), and a product is hi.hi + lo.hi + hi.lo.  hi and lo hold 22 bits of a value down
// to 2^-16 of the greatest that shares its power, and one fewer for each power of two below:
//   q and k: a power for each row (token);
//   v: one for each column, of rows each by its own power where rows differ by more than 2^4;
//   P: one for each row, of the greatest key (with v's row's power) that the token sees, faded as it is
//     for the token; what comes later does not count.  One for all rows where none differ by more than 2^4;
//   w: one for each column, of its greatest product (the greatest key times the column's greatest
//     value lost the columns in which a large key meets a small value);
//   X: one for each column, of a bound of what w's have added to it.
// The matrix unit adds with truncation, so a step's sums leave it and X is kept
// in fp32 registers.  Products are formed transposed (values' columns in the unit's
// 128 rows), so that X^T, v^T and w^T = (a^(63 - j + tail) v_j)^T are operands in tensor
// memory, written there by the threads that hold them.
//
// A block takes one head's tokens (or a segment of them) step by step: a loading warp
// brings the next step's rows into shared memory (by tensor maps; rows that are no whole
// 16-byte pieces by three warps, 4 bytes at a time), two that would be idle look at the sizes of
// v's rows, sixteen warps split the rows, form P and
// keep X, an issuing warp feeds the matrix unit.  Values that fp16's range would spoil
// (2^60 and more, below 2^-80, not finite, rows too far apart) send their step through the registers
// token by token.
//
// What bounds it: the sixteen warps' instructions, one behind the other.  A step takes 5.1 us, some
// 9300 cycles.  Of the 8900 before columns' products and rows' sizes were looked at, 1800 split the
// q and k rows, 900 were for the values and the barrier, 1400
// for v and w, 1200 for P, 500 for X, 800 to lay it into tensor memory, the rest for the
// outputs and waits.  The tensor pipe is busy for a quarter of them and the schedulers issue
// in 57% of cycles (21 K warp instructions a step).  Tensor memory's 512 columns and 226 KB of
// shared memory leave room for one block an SM.  8 x 2048 tokens of 16 heads of 128, 128
// blocks: 162 us with the same inputs again and 171 with others between (154 and 168 with one power
// of two for all of P and of w, which lost digits where tokens differ in size).  Rows unlike by more
// than 2^4 cost 182 us in place of 170, sizes spread over 2^20 270 to 330, all tokens one by one 1970.
// Heads of 64 wide leave half of the unit's 128 rows idle: 133 us.  Rows of 4-byte pieces: 127 wide 303 us.
// Tried, same inputs, each beside what was there then: outputs stored by the sixteen warps (163 us, 158),
// all of X q^T before the sums (170, 158), warps of their own for splitting and for X (182 to
// 238 us, 166 without: more instructions and exchanges), the next step's rows split while the
// matrix unit works (171 to 254, registers), row by row bulk copies (80 cycles each to issue),
// stores of single values (190, 178 with boxes), no work on P's blocks of zeros (171, 169), v's rows looked
// at by the sixteen warps themselves (181 in place of 173, others between).
constexpr int kStep = 64;
constexpr int kWorkers = 512, kScanThreads = kWorkers + 128, kLoaders = 3;  // loading warps
constexpr int kWorkerRegs = 104, kOtherRegs = 64;  // 4 x 104 + 64 = 5 x 96, what a quarter of an SM is launched with
constexpr int kBoxBytes = kStep * 128;             // 64 rows of 64 fp16 values
constexpr uint32_t kLeastBiased = 127 - 80, kFarRange = 140;  // exponents from 2^-80 to 2^60

// Columns of tensor memory.
template <int DK>
struct ScanTmem {
  static constexpr uint32_t kState = 0, kStateLo = DK / 2, kDelta = DK, kFrom = 2 * DK, kScore = kFrom + 64,
                            kV = kScore + 64, kW = kV + 64;  // hi; lo 32 columns behind
};
constexpr uint32_t kTmemColumns = 512;
// How far the factors of a step may lie apart, so that the columns need not be looked at, and so that
// it does not go token by token.
constexpr float kApart = 0x1p10f, kFarApart = 0x1p60f;

template <int DK>
struct ScanSmem {
  static constexpr int kBoxes = DK / 64;
  static constexpr int kQ = 0;                              // [kBoxes][hi, lo] boxes
  static constexpr int kK = kQ + 2 * kBoxes * kBoxBytes;    // [hi, lo][kBoxes]
  static constexpr int kP = kK + 2 * kBoxes * kBoxBytes;    // hi, lo, and what q's lo adds
  static constexpr int kRawQ = kP + 3 * kBoxBytes;          // fp32 rows of the next step
  static constexpr int kRawK = kRawQ + kStep * DK * 4;
  static constexpr int kRawV = kRawK + kStep * DK * 4;
  static constexpr int kOut = kRawV + kStep * kMostDim * 4;  // a step's outputs, as the tensor holds them
  static constexpr int kMisc = kOut + kStep * kMostDim * 4;
  static constexpr int kMiscBytes = 4 * (64 + 5 * 128 + 1024 + 512 + 2 * 64) + 20 * 8;  // factors, sizes, barriers
  static constexpr int kBytes = kMisc + kMiscBytes + 1023;                           // and what the alignment takes
  static_assert(kBytes <= 227 * 1024);
};

// Boxes of 64 rows of a head's q, k and v, where rows are whole 16-byte pieces, and of
// the output, if its rows are (`stores`).
struct ScanMaps {
  CUtensorMap q, k, v, out;
  int stores;
};
__device__ __forceinline__ void load_rows(uint32_t to, const CUtensorMap* map, int row, int head, int batch, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          to),
      "l"((uint64_t)map), "r"(0), "r"(row), "r"(head), "r"(batch), "r"(bar)
      : "memory");
}

// The same box into L2.
__device__ __forceinline__ void prefetch_rows(const CUtensorMap* map, int row, int head, int batch) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"((uint64_t)map), "r"(0),
               "r"(row), "r"(head), "r"(batch)
               : "memory");
}

// A box of shared memory to a head's output, or added to it.
__device__ __forceinline__ void store_rows(const CUtensorMap* map, uint32_t from, int row, int head, int batch,
                                           int accumulate) {
  if (accumulate)
    asm volatile(
        "cp.reduce.async.bulk.tensor.4d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
            (uint64_t)map),
        "r"(0), "r"(row), "r"(head), "r"(batch), "r"(from)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"((uint64_t)map),
        "r"(0), "r"(row), "r"(head), "r"(batch), "r"(from)
        : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

struct ScanParts {
  // [unit][slots][rows * cols], with several segments: the state that the first starts from,
  // then each piece's own state, and in their places the states behind the pieces.  (The call's
  // new state may replace the old one, so no segment but a head's only one reads that.)
  float* states;
  int si, sj;  // between their key rows and value columns, for the segments that start from them
};

// How a head's tokens are shared: `segments` blocks take turns of whole steps, and where
// there is more than one, `pieces` blocks each form the own states of all but the last.
struct Split {
  int segments, pieces;
  int slots;  // a head's states: (segments - 1) * pieces + 1
};
constexpr int kMostSlots = 64;
// Scans of one launch: all of as many sequences and heads, and of one kind.
constexpr int kMostScans = 3;
struct Scans {
  Split split;
  ScanMaps maps[kMostScans];
  Scan scan[kMostScans];
  ScanParts parts[kMostScans];
};

__device__ __forceinline__ void worker_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

// The greatest magnitude; NaN if one is.
__device__ __forceinline__ float most_of(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float warp_most(float v) {
  float r;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ uint32_t biased_of(float magnitude) { return __float_as_uint(magnitude) >> 23; }
__device__ __forceinline__ float power_of(uint32_t biased) { return __uint_as_float(biased << 23); }
// 2^(14 - e) for a greatest magnitude of 2^e to 2^(e+1), and its inverse; for 0, 1.
__device__ __forceinline__ uint32_t scale_biased(float most) { return most == 0.0f ? 141u : max(biased_of(most), 16u); }
// The same, of powers below fp32's normal numbers too.
__device__ __forceinline__ float small_power_of(int biased) {
  return biased > 0 ? power_of(biased) : power_of(max(biased + 64, 0)) * 0x1p-64f;
}
// 1 / x of a power of two, 0 of 0.
__device__ __forceinline__ float inverse_of(float x) { return x > 0.0f ? power_of(254u - biased_of(x)) : 0.0f; }
// Whether a tile of this greatest magnitude (0 apart) goes token by token; NaN does.
__device__ __forceinline__ bool far_biased(uint32_t biased) { return biased - kLeastBiased >= kFarRange; }

__device__ __forceinline__ uint32_t half_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
// Pairs of values as pairs of halves: hi, and what is left.
__device__ __forceinline__ void split_pair(Pair v, uint32_t& hi, uint32_t& lo) {
  const float2 f = v;
  hi = half_pair(f.x, f.y);
  const float2 back = __half22float2(*(const __half2*)&hi);
  const float2 rest = fma2(pair_of(back.x, back.y), pair_of(-1.0f, -1.0f), v);
  lo = half_pair(rest.x, rest.y);
}

__device__ __forceinline__ void copy_async4(uint32_t to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// The tokens of a sequence that segment `part` takes, or its piece `piece` (or all of it, -1):
// [first, last) of the order of the scan.
__device__ __forceinline__ void segment_of(int n, const Split& split, int part, int piece, int* first, int* last) {
  const int steps = (n + kStep - 1) / kStep, per = (steps + split.segments - 1) / split.segments;
  int from = part * per, to = from + per;
  if (piece >= 0) {
    const int each = (per + split.pieces - 1) / split.pieces;
    from += piece * each;
    to = min(to, from + each);
  }
  *first = min(n, from * kStep);
  *last = max(*first, min(n, to * kStep));
}

// STATE_ONLY: the segment's own state (from 0), for the segments behind it.  Its steps have
// but one product, which they take in turns of two sets of operands and sums: a step's sums
// are added while the matrix unit is at the next.  VEC: rows of
// whole 16-byte pieces.
template <int DK, bool STATE_ONLY, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 1) scan_kernel(const __grid_constant__ Scans all, int* err) {
  const Scan& s = all.scan[blockIdx.y];
  const ScanMaps& maps = all.maps[blockIdx.y];
  const ScanParts& parts = all.parts[blockIdx.y];
  const int segments = all.split.segments;
  using Tm = ScanTmem<DK>;
  using Sm = ScanSmem<DK>;
  constexpr int kBoxes = DK / 64, kMine = DK / 4;  // state values of a thread
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (As an offset: the compiler then knows what is derived from it for shared memory.)
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  float* since = (float*)(smem + Sm::kMisc);  // [64] a^(i + lead)
  float* lefts = since + 64;                  // [2][64] 2^20 a^(63 - j + tail), and the same of a last, shorter step
  float* nears = lefts + 128;                 // [128] a^(d - 63), 0 below
  float* q_downs = nears + 128;               // [2][64] what undoes the rows' factors (q's times 2^14 scale), steps in turn
  float* k_downs = q_downs + 128;             // [2][64]
  float* v_mosts = k_downs + 128;             // [4][128] pairs
  float* x_most = v_mosts + 1024;             // [4][128]
  float* p_downs = x_most + 512;              // [64] what undoes the factors of P's rows
  float* v_ups = p_downs + 64;                // [2][64] the powers of two of v's rows
  float* kv_downs = v_ups + 128;              // [64] what undoes k's and v's rows' factors together
  uint64_t* bars = (uint64_t*)(kv_downs + 64);
  int* far_step = (int*)(bars + 14);              // [2]
  int* uneven = far_step + 2;                     // [2] whether k's or v's rows differ in size from `usual`
  uint32_t* usual = (uint32_t*)(uneven + 2);      // [2][2] the exponents of the first key and value of the step before
  uint32_t* tmem_slot = usual + 4;
  const uint32_t base = smem_u32(smem);
  const uint32_t raw_full = smem_u32(bars), raw_empty = raw_full + 8, ready = raw_full + 16, values_ready = raw_full + 24,
                 score_full = raw_full + 32, sums_full = raw_full + 40, p_ready = raw_full + 48,
                 out_full = raw_full + 56, far_seen = raw_full + 64,
                 // Of every second step: with STATE_ONLY the warps may be a step ahead of the issuing one.
                 ready_odd = raw_full + 72, from_full = raw_full + 80, out_ready = raw_full + 88, out_free = raw_full + 96;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int runs = STATE_ONLY ? (segments - 1) * all.split.pieces : segments;
  const int unit = blockIdx.x / runs, run = blockIdx.x - unit * runs;
  const int part = STATE_ONLY ? run / all.split.pieces : run, piece = STATE_ONLY ? run - part * all.split.pieces : -1;
  const int b = unit / s.heads, h = unit - b * s.heads;
  const int n = tokens_of(s, b, err);
  int t0, t1;
  segment_of(n, all.split, part, piece, &t0, &t1);
  const float decay = decay_of(s, h, err);
  const int lead = s.back ? 0 : 1, tail = 1 - lead;
  auto power = [&](int steps) { return steps == 0 ? 1.0f : expf(-decay * steps); };

  if (tid == 0) {
    mbar_init(raw_full, VEC ? 1 : 32 * kLoaders);
    mbar_init(raw_empty, 1);
    mbar_init(ready, 1);
    mbar_init(ready_odd, 1);
    mbar_init(values_ready, kWorkers / 32);
    mbar_init(score_full, 1);
    mbar_init(sums_full, 1);
    mbar_init(p_ready, kWorkers / 32);
    mbar_init(out_full, 1);
    mbar_init(far_seen, 1);
    mbar_init(from_full, 1);
    mbar_init(out_ready, kWorkers / 32);
    mbar_init(out_free, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    far_step[0] = far_step[1] = uneven[0] = uneven[1] = 0;
    usual[0] = usual[1] = 0;
  }
  if (tid < 64) since[tid] = power(tid + lead);
  if (tid >= 64 && tid < 192) {
    const int j = tid & 63, m = tid < 128 ? kStep : (t1 - t0) % kStep;
    lefts[tid - 64] = j < m ? power(m - 1 - j + tail) * 0x1p20f : 0.0f;
  }
  if (tid >= 192 && tid < 320) nears[tid - 192] = tid - 192 < 63 ? 0.0f : power(tid - 192 - 63);
  if (warp == kWorkers / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // Columns that no copy writes are 0.
  if (!VEC && (s.rows != DK || s.cols != kMostDim))
    for (int i = tid; i < (Sm::kOut - Sm::kRawQ) / 16; i += kScanThreads)
      ((uint4*)(smem + Sm::kRawQ))[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const float *q = s.q.at(b, h), *k = s.k.at(b, h), *v = s.v.at(b, h);
  auto token = [&](int t) { return (int64_t)(s.back ? n - 1 - t : t); };
  // Rows of a step as they lie in shared memory: boxes hold them as the tensor does.
  const int key_pitch = VEC ? s.rows : DK, value_pitch = VEC ? s.cols : kMostDim;
  const bool turned = VEC && s.back;
  auto place = [&](int i) { return turned ? kStep - 1 - i : i; };

  // The sizes of v's rows from `row0` on, `rows` (up to 32) of them, and whether they are as usual, as the
  // splitting warps do for k.
  auto look_at_values = [&](int row0, auto rows, int turn, int m) {
    const float* raw = (const float*)(smem + Sm::kRawV) + (!VEC || 4 * lane < s.cols ? 4 * lane : 0);
    float mine = 0.0f;  // of row `lane`
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      if (row0 + r >= m) break;
      const float4 w = *(const float4*)(raw + place(row0 + r) * value_pitch);
      const float most = warp_most(most_of(most_of(w.x, w.y, w.z), w.w, 0.0f));
      if (lane == r) mine = most;
    }
    const uint32_t biased = scale_biased(mine), was = usual[2 * turn + 1];
    if (lane < rows) v_ups[64 * turn + row0 + lane] = mine == 0.0f ? 0.0f : power_of(251u - biased);
    if (row0 + lane == 0) usual[2 * (turn ^ 1) + 1] = biased;
    if (far_biased(biased)) far_step[turn] = 1;
    if (lane < rows && row0 + lane < m && (mine == 0.0f || biased - was + 2 > 4)) uneven[turn] = 1;
  };

  if (warp >= kWorkers / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kWorkers / 32) {
      // The issuing warp.
      constexpr uint32_t kNarrow = umma_idesc(kStep, false), kRows = umma_idesc(DK, true);
      const bool leader = elect_one();
      uint32_t steps = 0;  // those of the matrix unit
      bool ok = true;
      // The outputs of the step before, which its warps have left in shared memory, go from here:
      // issuing a copy takes as long as a tenth of what they do in a step.
      bool storing = false;
      uint32_t stores = 0;
      auto store_outputs = [&](int t) {
        ok = sleep_wait(out_ready, stores++ & 1, err);
        if (ok && leader)
          store_rows(&maps.out, base + Sm::kOut, s.back ? n - kStep - t : t, h / s.out.share, b, s.accumulate);
        __syncwarp();
      };
      for (int t = t0, c = 0; t < t1 && ok; t += kStep, ++c) {
        const bool second = STATE_ONLY && (c & 1);
        if (VEC && !STATE_ONLY && storing) store_outputs(t - kStep);
        if (ok) ok = sleep_wait(c & 1 ? ready_odd : ready, (c >> 1) & 1, err);
        if (!ok) break;
        if (VEC && !STATE_ONLY && storing) {
          if (leader) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            mbar_arrive(out_free);
          }
          __syncwarp();
          storing = false;
        }
        tc_fence_after();
        if (*(volatile int*)&far_step[c & 1]) {
          if (leader) mbar_arrive(far_seen);
          continue;
        }
        if (!STATE_ONLY && leader) {
          // P: [q hi; q lo] times k hi, then k lo.
#pragma unroll
          for (int pass = 0; pass < 2; ++pass)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) {
              const uint32_t a = column_word(base + Sm::kQ + (i / 4) * 2 * kBoxBytes) + (i & 3) * kColumnStep;
              const uint32_t k = column_word(base + Sm::kK + (pass * kBoxes + i / 4) * kBoxBytes) + (i & 3) * kColumnStep;
              umma_ss(tmem + Tm::kScore, a, k, kNarrow, pass + i > 0);
            }
          umma_commit(score_full);
        }
        // X^T q^T: lo.hi, hi.lo, hi.hi; the first half (with narrow keys all) while the values are
        // split, the second behind the sums, which the warps need earlier.
        auto from_state = [&](bool first_half) {
#pragma unroll
          for (int pass = 0; pass < 3; ++pass)
#pragma unroll
            for (int i = 0; i < DK / 16; ++i)
              if ((DK == 64 || 2 * (pass * (DK / 16) + i) < 3 * (DK / 16)) == first_half) {
                const uint32_t x = tmem + (pass == 0 ? Tm::kStateLo : Tm::kState) + i * 8;
                const uint32_t q = column_word(base + Sm::kQ + ((i / 4) * 2 + (pass == 1)) * kBoxBytes) + (i & 3) * kColumnStep;
                umma_ts(tmem + Tm::kFrom, x, q, kNarrow, pass + i > 0);
              }
        };
        if (!STATE_ONLY && leader) from_state(true);
        __syncwarp();
        ok = sleep_wait(values_ready, steps & 1, err);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          // w^T k.
#pragma unroll
          for (int pass = 0; pass < 3; ++pass)
#pragma unroll
            for (int i = 0; i < kStep / 16; ++i) {
              const uint32_t w = tmem + (second ? Tm::kV : Tm::kW) + (pass == 0 ? 32 : 0) + i * 8;
              const uint32_t k =
                  row_word(base + (second ? Sm::kQ : Sm::kK) + (pass == 1) * kBoxes * kBoxBytes, kBoxBytes) + i * kRowStep;
              umma_ts(tmem + (second ? Tm::kFrom : Tm::kDelta), w, k, kRows, pass + i > 0);
            }
          umma_commit(sums_full);
          if (!STATE_ONLY) {
            from_state(false);
            umma_commit(from_full);
          }
        }
        if (!STATE_ONLY) {
          __syncwarp();
          ok = sleep_wait(p_ready, steps & 1, err);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            // v^T P^T: lo.hi, hi.lo, hi.(q's lo), hi.hi.
#pragma unroll
            for (int pass = 0; pass < 4; ++pass)
#pragma unroll
              for (int i = 0; i < kStep / 16; ++i) {
                const uint32_t v = tmem + Tm::kV + (pass == 0 ? 32 : 0) + i * 8;
                const int box = pass == 1 ? 1 : pass == 2 ? 2 : 0;
                const uint32_t p = column_word(base + Sm::kP + box * kBoxBytes) + i * kColumnStep;
                umma_ts(tmem + Tm::kScore, v, p, kNarrow, pass + i > 0);
              }
            umma_commit(out_full);
          }
          storing = VEC && maps.stores && t1 - t >= kStep;
        }
        ++steps;
        __syncwarp();
      }
      if (VEC && !STATE_ONLY) {
        if (ok && storing) store_outputs(t0 + (t1 - t0 - 1) / kStep * kStep);
        if (leader) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
      }
    } else if (VEC) {
      // The loading warp: a box of each operand a step.
      if (warp == kWorkers / 32 + 1) {
        const bool leader = elect_one();
        bool ok = true;
        int c = 0;
        for (int t = t0; t < t1; t += kStep, ++c) {
          if (c > 0) ok = sleep_wait(raw_empty, (c - 1) & 1, err);
          if (!ok) break;
          if (leader) {
            // What lies outside the tensor comes as 0, what lies behind the sequence's end as it is.
            const int row = s.back ? n - kStep - t : t;
            mbar_expect_tx(raw_full, kStep * 4 * ((STATE_ONLY ? 1 : 2) * s.rows + s.cols));
            load_rows(base + Sm::kRawK, &maps.k, row, h / s.k.share, b, raw_full);
            if (!STATE_ONLY) load_rows(base + Sm::kRawQ, &maps.q, row, h / s.q.share, b, raw_full);
            load_rows(base + Sm::kRawV, &maps.v, row, h / s.v.share, b, raw_full);
            // The step after next's on their way to L2 (without, 65536 tokens took 260 us for 247 and
            // training on 8192 467 for 446), where it is whole.
            if (t + 2 * kStep <= t1) {
              const int next = s.back ? row - kStep : row + kStep;
              prefetch_rows(&maps.k, next, h / s.k.share, b);
              if (!STATE_ONLY) prefetch_rows(&maps.q, next, h / s.q.share, b);
              prefetch_rows(&maps.v, next, h / s.v.share, b);
            }
          }
          __syncwarp();
        }
        // The last copies end before the block does.
        if (c > 0) sleep_wait(raw_full, (c - 1) & 1, err);
      } else if (!STATE_ONLY) {
        // The other two look at a step's values while the sixteen split q and k.
        bool ok = true;
        for (int t = t0, c = 0; t < t1; t += kStep, ++c) {
          if (ok) ok = sleep_wait(raw_full, c & 1, err);
          look_at_values((warp & 1) * 32, std::integral_constant<int, 32>{}, c & 1, min(kStep, t1 - t));
          asm volatile("bar.arrive 6, %0;" ::"n"(kWorkers + 64) : "memory");
        }
      }
    } else {
      // The loading warps, a row at a time.
      const int loader = warp - kWorkers / 32 - 1;
      bool ok = true;
      for (int t = t0, c = 0; t < t1 && ok; t += kStep, ++c) {
        if (c > 0) ok = sleep_wait(raw_empty, (c - 1) & 1, err);
        if (!ok) break;
        const int m = min(kStep, t1 - t);
        auto row = [&](const float* from, int dim, uint32_t to) {
#pragma unroll
          for (int i = 0; i < kMostDim / 32; ++i)
            if (lane + 32 * i < dim) copy_async4(to + 4 * (lane + 32 * i), from + lane + 32 * i);
        };
#pragma unroll 4
        for (int r = loader; r < m; r += kLoaders) {
          const int64_t at = token(t + r);
          row(k + at * s.k.token, s.rows, base + Sm::kRawK + r * DK * 4);
          if (!STATE_ONLY) row(q + at * s.q.token, s.rows, base + Sm::kRawQ + r * DK * 4);
          row(v + at * s.v.token, s.cols, base + Sm::kRawV + r * kMostDim * 4);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(raw_full) : "memory");
      }
      // The last copies end before the block does.
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWorkerRegs));
    const int quarter = warp & 3, group = warp >> 2;  // tensor memory lanes, and which 16 tokens or quarter of the rows
    const int col = quarter * 32 + lane;              // the value column of this thread
    const uint32_t at_lane = tmem + ((uint32_t)(quarter * 32) << 16);
    float* out = const_cast<float*>(s.out.at(b, h));
    const int64_t state = (int64_t)unit * s.rows * s.cols;
    Pair x[kMine / 2];  // X^T: this column, rows group * kMine + i
    {
      float first[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) first[i] = 0.0f;
      if (!STATE_ONLY && col < s.cols) {
        if (segments > 1) {
          const float* from = parts.states + ((int64_t)unit * all.split.slots + part * all.split.pieces) * s.rows * s.cols;
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            const int r = group * kMine + i;
            if (r < s.rows) first[i] = from[r * parts.si + col * parts.sj];
          }
        } else if (s.from.p != nullptr) {
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            const int r = group * kMine + i;
            if (r < s.rows) first[i] = s.from.p[state + r * s.from.si + col * s.from.sj] * s.from_factor;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kMine / 2; ++i) x[i] = pair_of(first[2 * i], first[2 * i + 1]);
    }
    // X^T's greatest magnitude in this column, over the four threads that hold it.
    auto most_of_state = [&] {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < kMine / 2; ++i) {
        const float2 f = x[i];
        m = most_of(m, f.x, f.y);
      }
      x_most[group * 128 + col] = m;
      worker_sync();
      return most_of(most_of(x_most[col], x_most[128 + col], x_most[256 + col]), x_most[384 + col], 0.0f);
    };
    float x_down = 1.0f;  // undoes the factor of the state in tensor memory
    auto put_state = [&](float bound) {
      const uint32_t biased = scale_biased(bound);
      x_down = power_of(biased - 14u);
      const float up = power_of(268u - biased);
      const Pair up2 = pair_of(up, up);
      uint32_t hi[kMine / 2], lo[kMine / 2];
#pragma unroll
      for (int i = 0; i < kMine / 2; ++i) split_pair(mul2(x[i], up2), hi[i], lo[i]);
      if constexpr (DK == 128) {
        tmem_st16(at_lane + Tm::kState + group * (kMine / 2), hi);
        tmem_st16(at_lane + Tm::kStateLo + group * (kMine / 2), lo);
      } else {
        tmem_st8(at_lane + Tm::kState + group * (kMine / 2), hi);
        tmem_st8(at_lane + Tm::kStateLo + group * (kMine / 2), lo);
      }
    };
    const int row_i = col & (kStep - 1);  // of P
    const float2 fade = decay_over(decay, kStep);
    bool ok = true;
    uint32_t steps = 0, far_steps = 0, stores = 0;
    float bound = 0.0f;  // at least X^T's greatest magnitude in this column
    bool far_state = false;
    if (t0 < t1) {
      if (!STATE_ONLY) {
        bound = most_of_state();
        far_state = biased_of(bound) >= 254;
        put_state(bound);
      }
    }
    uint32_t sums = 0;
    // Adds a step's sums to X once the matrix unit has them.
    auto add_sums = [&](uint32_t at, int m, float w_down) {
      const float2 a = m == kStep ? fade : decay_over(decay, m);
      if (ok) ok = sleep_wait(sums_full, sums & 1, err);
      ++sums;
      tc_fence_after();
      const Pair a_hi = pair_of(a.x, a.x), a_lo = pair_of(a.y, a.y), w2 = pair_of(w_down, w_down);
#pragma unroll
      for (int part = 0; part < kMine / 16; ++part) {
        float d[16];
        tmem_ld16(at_lane + at + group * kMine + 16 * part, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          Pair& y = x[8 * part + i];
          y = fma2(y, a_hi, fma2(y, a_lo, mul2(pair_of(d[2 * i], d[2 * i + 1]), w2)));
        }
      }
    };
    bool pending = false;  // of STATE_ONLY: the step before has sums to add
    float pending_w = 0.0f;
    int pending_turn = 0, pending_m = kStep;
    auto flush = [&] {
      if (pending) add_sums(pending_turn ? Tm::kFrom : Tm::kDelta, pending_m, pending_w);
      pending = false;
    };
    for (int t = t0, c = 0; t < t1; t += kStep, ++c) {
      const int m = min(kStep, t1 - t);
      const int turn = c & 1;
      float *q_down = q_downs + 64 * turn, *k_down = k_downs + 64 * turn, *v_up = v_ups + 64 * turn;
      const uint32_t usual_k = STATE_ONLY ? 0 : usual[2 * turn];
      if (ok) ok = sleep_wait(raw_full, turn, err);
      if (m < kStep) {  // zeros behind the sequence's end
        const int first = turned ? 0 : m;
        for (int i = tid; i < (kStep - m) * key_pitch; i += kWorkers) {
          ((float*)(smem + Sm::kRawQ))[first * key_pitch + i] = 0.0f;
          ((float*)(smem + Sm::kRawK))[first * key_pitch + i] = 0.0f;
        }
        for (int i = tid; i < (kStep - m) * value_pitch; i += kWorkers)
          ((float*)(smem + Sm::kRawV))[first * value_pitch + i] = 0.0f;
        worker_sync();
      }
      // q and k rows, a warp eight of one of them.
      bool far = far_state, odd = false;
      {
        constexpr int kRowsPer = STATE_ONLY ? 4 : 8;
        const bool is_k = STATE_ONLY || warp >= 8;
        const int row0 = STATE_ONLY ? warp * 4 : (warp & 7) * 8;
        // (Where rows hold fewer than DK values, the lanes behind them read the first once more
        // and take them 0 times.)
        const bool held = !VEC || lane * (DK / 32) < s.rows;
        const float* raw = (const float*)(smem + (is_k ? Sm::kRawK : Sm::kRawQ)) + place(row0) * key_pitch +
                           (held ? lane * (DK / 32) : 0);
        const int next_row = turned ? -key_pitch : key_pitch;
        Pair f[kRowsPer][kBoxes];
        float mine = 0.0f;  // of row `lane`
#pragma unroll
        for (int r = 0; r < kRowsPer; ++r) {
          float most;
          if constexpr (DK == 128) {
            const float4 w = *(const float4*)(raw + r * next_row);
            f[r][0] = pair_of(w.x, w.y), f[r][kBoxes - 1] = pair_of(w.z, w.w);
            most = most_of(most_of(w.x, w.y, w.z), w.w, 0.0f);
          } else {
            const float2 w = *(const float2*)(raw + r * next_row);
            f[r][0] = pair_of(w.x, w.y);
            most = most_of(w.x, w.y, 0.0f);
          }
          most = warp_most(most);
          if (lane == r) mine = most;
        }
        const uint32_t biased = scale_biased(mine);
        far |= far_biased(biased);
        if (!STATE_ONLY && is_k) {
          odd = lane < kRowsPer && row0 + lane < m && (mine == 0.0f || biased - usual_k + 2 > 4);
          if (row0 + lane == 0) usual[2 * (turn ^ 1)] = biased;
        }
        // A row of zeros has no part in the greatest factor.
        if (lane < kRowsPer)
          (is_k ? k_down : q_down)[row0 + lane] = mine == 0.0f ? 0.0f : is_k ? power_of(biased - 14u) : power_of(biased) * s.scale;
        const float up = power_of(268u - biased);
        uint8_t* box = smem + (is_k && !(STATE_ONLY && turn) ? Sm::kK : Sm::kQ);
        const int other = (is_k ? kBoxes : 1) * kBoxBytes;  // from hi to lo
        if (DK == 128) box += (lane >> 4) * (is_k ? 1 : 2) * kBoxBytes;
#pragma unroll
        for (int r = 0; r < kRowsPer; ++r) {
          float u = __shfl_sync(0xffffffffu, up, r);
          if (VEC && !held) u = 0.0f;
          const Pair u2 = pair_of(u, u);
          const int row = row0 + r;
          if constexpr (DK == 128) {
            uint2 hi, lo;
            split_pair(mul2(f[r][0], u2), hi.x, lo.x);
            split_pair(mul2(f[r][kBoxes - 1], u2), hi.y, lo.y);
            uint8_t* to = box + row * 128 + ((((lane & 15) >> 1) ^ (row & 7)) << 4) + ((lane & 1) << 3);
            *(uint2*)to = hi;
            *(uint2*)(to + other) = lo;
          } else {
            uint32_t hi, lo;
            split_pair(mul2(f[r][0], u2), hi, lo);
            uint8_t* to = box + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + ((lane & 3) << 2);
            *(uint32_t*)to = hi;
            *(uint32_t*)(to + other) = lo;
          }
        }
      }
      // This column's values of 16 tokens.
      Pair val[8];
      float val_most = 0.0f;
      {
        // (Threads behind the last column read the first; nothing takes what they hold.)
        const float* raw = (const float*)(smem + Sm::kRawV) + place(group * 16) * value_pitch + (VEC && col >= s.cols ? 0 : col);
        const int next_row = turned ? -value_pitch : value_pitch;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = raw[2 * i * next_row], d = raw[(2 * i + 1) * next_row];
          val[i] = pair_of(a, d);
          val_most = most_of(val_most, a, d);
        }
        if (STATE_ONLY) far |= far_biased(scale_biased(val_most));
      }
      if (!STATE_ONLY && !VEC) look_at_values(warp * 4, std::integral_constant<int, 4>{}, turn, m);
      if (far) far_step[turn] = 1;
      if (odd) uneven[turn] = 1;
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (STATE_ONLY || !VEC) worker_sync();
      else asm volatile("bar.sync 6, %0;" ::"n"(kWorkers + 64) : "memory");
      bool far_now = *(volatile int*)&far_step[turn];
      // Where the rows of k or of v differ by more than 2^4, which they mostly do not, each row of v goes by its
      // own power of two as those of k do, and a row of P takes the greatest factor of the two among the
      // tokens that it sees, as far as they have not faded: what comes later, or has faded, does not take
      // its digits.  Of row `row_i`:
      uint32_t p_biased = 0;
      const bool even = STATE_ONLY || !*(volatile int*)&uneven[turn];
      if (!STATE_ONLY) {
        p_biased = usual_k + 2 - 14;
        if (!even) {
          const float k0 = k_down[lane] * inverse_of(v_up[lane]);  // tokens `lane` and `lane + 32`
          const float k1 = k_down[lane + 32] * inverse_of(v_up[lane + 32]);
          if (warp == 0) kv_downs[lane] = k0, kv_downs[lane + 32] = k1;
          far_now |= __any_sync(0xffffffffu, (k0 > 0.0f && k0 < 0x1p-126f) || (k1 > 0.0f && k1 < 0x1p-126f));
          k_down = kv_downs;
          val_most = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 u = *(const float4*)(v_up + group * 16 + 4 * i);
            val[2 * i] = mul2(val[2 * i], pair_of(u.x, u.y));
            val[2 * i + 1] = mul2(val[2 * i + 1], pair_of(u.z, u.w));
            val_most = most_of(most_of(val_most, val[2 * i].x, val[2 * i].y), val[2 * i + 1].x, val[2 * i + 1].y);
          }
          float seen0 = k0, seen1 = k1;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const float faded = nears[63 + d];
            const float u0 = __shfl_up_sync(0xffffffffu, seen0, d) * faded, u1 = __shfl_up_sync(0xffffffffu, seen1, d) * faded;
            if (lane >= d) seen0 = fmaxf(seen0, u0), seen1 = fmaxf(seen1, u1);
          }
          seen1 = fmaxf(seen1, __shfl_sync(0xffffffffu, seen0, 31) * nears[64 + lane]);
          const float most = warp_most(fmaxf(k0, k1)), least_inv = warp_most(fmaxf(inverse_of(k0), inverse_of(k1)));
          far_now |= most * least_inv > kFarApart;
          // (Rounded up to a power of two; at least 2^-126 of the greatest, so that no later key's factor
          // over it is infinite.)
          p_biased = (__float_as_uint(fmaxf(quarter & 1 ? seen1 : seen0, most * 0x1p-126f)) + 0x7fffffu) >> 23;
          if (warp < 2) p_downs[warp * 32 + lane] = power_of(p_biased);
          worker_sync();  // kv_downs, p_downs
          if (most * least_inv > kApart && !far_now) {
            // Small tokens behind a large one: P holds their scores relative to the large one's, which does
            // where a column's greatest product so far (`seen`, faded) is near what P's row is relative to
            // times the column's greatest value.  Where it is below 2^-15 of that, the step goes token by token.
            float v_all[16], seen = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              v_all[i] = fabsf(i & 1 ? val[i / 2].y : val[i / 2].x) * k_down[group * 16 + i];
              seen = fmaxf(seen * nears[64], v_all[i]);
            }
            ((float2*)v_mosts)[group * 128 + col] = make_float2(val_most, seen);
            worker_sync();
            float column = 0.0f;
            seen = 0.0f;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2 of_group = ((const float2*)v_mosts)[g * 128 + col];
              column = fmaxf(column, of_group.x);
              if (g < group) seen = fmaxf(seen * nears[63 + 16], of_group.y);
            }
            bool lost = false;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              seen = fmaxf(seen * nears[64], v_all[i]);
              lost |= seen > 0.0f && seen < 0x1p-15f * column * p_downs[group * 16 + i];
            }
            if (lost) far_step[turn] = 1;
            worker_sync();
            far_now = *(volatile int*)&far_step[turn];
          }
        }
      }
      if (tid == 0) {
        far_step[turn ^ 1] = uneven[turn ^ 1] = 0;
        if (far_now) far_step[turn] = 1;
        mbar_arrive(turn ? ready_odd : ready);
      }
      if (far_now) {
        // Token by token.
        if (STATE_ONLY) flush();
        const float2 one = decay_over(decay, 1);
        const Pair hi = pair_of(one.x, one.x), lo = pair_of(one.y, one.y);
        for (int i = 0; i < m; ++i) {
          const float* kr = (const float*)(smem + Sm::kRawK) + place(i) * key_pitch;
          const float* qr = (const float*)(smem + Sm::kRawQ) + place(i) * key_pitch;
          const float w = col < s.cols ? ((const float*)(smem + Sm::kRawV))[place(i) * value_pitch + col] : 0.0f;
          auto two = [&](const float* row, int r) {
            return pair_of(r < s.rows ? row[r] : 0.0f, r + 1 < s.rows ? row[r + 1] : 0.0f);
          };
          const Pair w2 = pair_of(w, w);
          Pair sum = pair_of(0.0f, 0.0f);
#pragma unroll
          for (int j = 0; j < kMine / 2; ++j) {
            const int r = group * kMine + 2 * j;
            if (lead) x[j] = fma2(x[j], hi, mul2(x[j], lo));
            x[j] = fma2(two(kr, r), w2, x[j]);
            if (!STATE_ONLY) sum = fma2(two(qr, r), x[j], sum);
            if (!lead) x[j] = fma2(x[j], hi, mul2(x[j], lo));
          }
          if (!STATE_ONLY) {
            float* sums = i & 1 ? v_mosts : x_most;
            sums[group * 128 + col] = sum.x + sum.y;
            worker_sync();
            if (group == 0 && col < s.cols) {
              const float all = ((sums[col] + sums[128 + col]) + (sums[256 + col] + sums[384 + col])) * s.scale;
              float* to = out + token(t + i) * s.out.token + col;
              *to = s.accumulate ? *to + all : all;
            }
          }
        }
        worker_sync();  // the rows are read, and the sums
        if (tid == 0 && t + kStep < t1) mbar_arrive(raw_empty);
        if (!STATE_ONLY) {
          bound = most_of_state();
          far_state = biased_of(bound) >= 254;
          if (t + kStep < t1) put_state(bound);
        }
        // The issuing warp keeps step.
        if (ok) ok = sleep_wait(far_seen, far_steps & 1, err);
        ++far_steps;
        continue;
      }
      if (tid == 0 && t + kStep < t1) mbar_arrive(raw_empty);
      // v, and w = v_j a^(63 - j + tail) times the key's factor, each column with powers of two of its own: what a
      // large key is not multiplied with does not feel it.  (2^20 w is at most 2^126, and below 2^-126 only
      // where the product of key and value is.)
      float p_down, w_down;
      {
        const float* left = lefts + (m < kStep ? kStep : 0);
        Pair w[8];
        float w_most = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float4 l = *(const float4*)(left + group * 16 + 2 * i), f = *(const float4*)(k_down + group * 16 + 2 * i);
          w[i] = mul2(val[i], mul2(pair_of(f.x, f.y), pair_of(l.x, l.y)));
          w[i + 1] = mul2(val[i + 1], mul2(pair_of(f.z, f.w), pair_of(l.z, l.w)));
          w_most = most_of(most_of(w_most, w[i].x, w[i].y), w[i + 1].x, w[i + 1].y);
        }
        // Over the four threads that hold the column.
        float2* mosts = (float2*)v_mosts + col;
        mosts[group * 128] = make_float2(val_most, w_most);
        // (Before this step's values are ready: its own sums would end another phase of the barrier.)
        if (STATE_ONLY) flush();
        asm volatile("bar.sync %0, 128;" ::"r"(2 + quarter) : "memory");
        {
          const float2 m0 = mosts[0], m1 = mosts[128], m2 = mosts[256], m3 = mosts[384];
          val_most = most_of(most_of(m0.x, m1.x, m2.x), m3.x, 0.0f);
          w_most = most_of(most_of(m0.y, m1.y, m2.y), m3.y, 0.0f);
        }
        uint32_t hi[8], lo[8];
        if (!STATE_ONLY) {
          const uint32_t biased = scale_biased(val_most);
          const float up = power_of(268u - biased);
          const Pair up2 = pair_of(up, up);
#pragma unroll
          for (int i = 0; i < 8; ++i) split_pair(mul2(val[i], up2), hi[i], lo[i]);
          tmem_st8(at_lane + Tm::kV + group * 8, hi);
          tmem_st8(at_lane + Tm::kV + 32 + group * 8, lo);
          p_down = power_of(biased - 14u) * 0x1p8f * (even ? power_of(p_biased) : 1.0f);
        }
        const uint32_t biased = scale_biased(w_most);
        const float up = power_of(268u - biased);
        w_down = w_most > 0.0f ? small_power_of((int)biased - (14 + 20)) : 0.0f;
        const Pair up2 = pair_of(up, up);
#pragma unroll
        for (int i = 0; i < 8; ++i) split_pair(mul2(w[i], up2), hi[i], lo[i]);
        const uint32_t at_w = at_lane + (STATE_ONLY && turn ? Tm::kV : Tm::kW) + group * 8;
        tmem_st8(at_w, hi);
        tmem_st8(at_w + 32, lo);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(values_ready);

      if (!STATE_ONLY) {
        if (ok) ok = sleep_wait(score_full, steps & 1, err);
        tc_fence_after();
        // P of 16 keys: rows (tokens) 0..63 in the lanes of quarters 0 and 1, what q's lo adds in 2 and 3.
        const float inv = power_of(254u - p_biased) * 0x1p-22f;
        const Pair inv2 = pair_of(inv, inv);
        const float* near = nears + 63 + row_i - group * 16;
        float p[16];
        tmem_ld16(at_lane + Tm::kScore + group * 16, p);
        Pair f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 d = *(const float4*)(k_down + group * 16 + 4 * i);
          const float* a = near - 4 * i;
          f[2 * i] = mul2(pair_of(p[4 * i], p[4 * i + 1]), mul2(mul2(pair_of(d.x, d.y), inv2), pair_of(a[0], a[-1])));
          f[2 * i + 1] =
              mul2(pair_of(p[4 * i + 2], p[4 * i + 3]), mul2(mul2(pair_of(d.z, d.w), inv2), pair_of(a[-2], a[-3])));
        }
        uint8_t* row = smem + Sm::kP + row_i * 128;
        const int x0 = ((2 * group) ^ (row_i & 7)) << 4, x1 = ((2 * group + 1) ^ (row_i & 7)) << 4;
        uint32_t hi[8], lo[8];
        if (quarter < 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) split_pair(f[j], hi[j], lo[j]);
          *(uint4*)(row + x0) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *(uint4*)(row + x1) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
          *(uint4*)(row + kBoxBytes + x0) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          *(uint4*)(row + kBoxBytes + x1) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) hi[j] = half_pair(f[j].x, f[j].y);
          *(uint4*)(row + 2 * kBoxBytes + x0) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *(uint4*)(row + 2 * kBoxBytes + x1) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
        }
        tc_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
      }
      if (STATE_ONLY) {
        pending = true;
        pending_w = w_down;
        pending_turn = turn;
        pending_m = m;
        continue;
      }
      // X, and a bound of it: 64 products of packed values are at most 2^36.
      const float from_down = x_down;
      const float2 a = m == kStep ? fade : decay_over(decay, m);
      add_sums(Tm::kDelta, m, w_down);
      if (!STATE_ONLY) {
        bound = fmaf(bound, a.x, 0x1p36f * w_down) * 1.000001f;
        // (It grows by what the sums may be, not by what they are.)
        if ((c & 15) == 15) bound = most_of_state();
        far_state = biased_of(bound) >= 254;
        if (ok) ok = sleep_wait(from_full, steps & 1, err);
        tc_fence_after();
        if (t + kStep < t1) put_state(bound);
        if (ok) ok = sleep_wait(out_full, steps & 1, err);
        tc_fence_after();
        float from[16], own[16];
        tmem_ld16(at_lane + Tm::kFrom + group * 16, from);
        tmem_ld16(at_lane + Tm::kScore + group * 16, own);
        if (!even) {
#pragma unroll
          for (int i = 0; i < 16; ++i) own[i] *= p_downs[group * 16 + i] * p_down;
          p_down = 1.0f;
        }
        // (2^14 of a query's factor stands in q_down: before it is taken, sums are then as large as the
        // outputs of a query of 1, and no power of two is needed that fp32 does not have.)
        const Pair p2 = pair_of(p_down, p_down), f2 = pair_of(from_down * 0x1p-14f, from_down * 0x1p-14f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 w = *(const float4*)(since + group * 16 + 4 * i), d = *(const float4*)(q_down + group * 16 + 4 * i);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int e = 4 * i + 2 * j;
            const Pair o = fma2(mul2(pair_of(from[e], from[e + 1]), j ? pair_of(w.z, w.w) : pair_of(w.x, w.y)), f2,
                                mul2(pair_of(own[e], own[e + 1]), p2));
            const Pair y = mul2(o, j ? pair_of(d.z, d.w) : pair_of(d.x, d.y));
            own[e] = y.x, own[e + 1] = y.y;
          }
        }
        if (VEC && maps.stores && m == kStep) {
          // Through shared memory: a thread's stores of single values would take the load and
          // store units longer than the step's loads.
          if (ok && stores > 0) ok = sleep_wait(out_free, (stores - 1) & 1, err);
          ++stores;
          float* to = (float*)(smem + Sm::kOut) + place(group * 16) * value_pitch + col;
          const int next_row = turned ? -value_pitch : value_pitch;
          if (col < s.cols)
#pragma unroll
            for (int i = 0; i < 16; ++i) to[i * next_row] = own[i];
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(out_ready);
        } else {
          const int rows = col < s.cols ? min(m - group * 16, 16) : 0;  // of this thread's
          const int64_t pitch = s.back ? -s.out.token : s.out.token;
          float* to = out + token(t + group * 16) * s.out.token + col;
#pragma unroll
          for (int i = 0; i < 16; ++i, to += pitch)
            if (i < rows) *to = s.accumulate ? *to + own[i] : own[i];
        }
      }
      ++steps;
    }
    if (STATE_ONLY) flush();
    // Rows behind the sequence's end, spread over its blocks.
    if (!STATE_ONLY && !s.accumulate)
      for (int r = n + part * 4 + group; r < s.seq; r += 4 * segments)
        if (col < s.cols) out[(int64_t)r * s.out.token + col] = 0.0f;
    if (STATE_ONLY || (s.to.p != nullptr && part == segments - 1)) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int r = group * kMine + i;
        const float y = i & 1 ? x[i / 2].y : x[i / 2].x;
        if (r >= s.rows || col >= s.cols) continue;
        if (STATE_ONLY) {
          parts.states[((int64_t)unit * all.split.slots + run + 1) * s.rows * s.cols + (int64_t)r * s.cols + col] = y;
        } else {
          float* to = s.to.p + state + r * s.to.si + col * s.to.sj;
          *to = s.accumulate_state ? *to + y * s.to_factor : y * s.to_factor;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWorkers / 32)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
}

// From each piece's own state the state behind it, in place.
__global__ void __launch_bounds__(256) scan_states_kernel(const __grid_constant__ Scans all, int* err) {
  const Scan& s = all.scan[blockIdx.z];
  const int unit = blockIdx.y, b = unit / s.heads, h = unit - b * s.heads;
  const int i = blockIdx.x * 256 + threadIdx.x, elems = s.rows * s.cols;
  const int n = tokens_of(s, b, err), runs = all.split.slots - 1;
  // What a piece leaves of the state before it, as a sum of two.
  __shared__ float2 fade[kMostSlots];
  if (threadIdx.x < runs) {
    const int part = threadIdx.x / all.split.pieces;
    int t0, t1;
    segment_of(n, all.split, part, threadIdx.x - part * all.split.pieces, &t0, &t1);
    fade[threadIdx.x] = decay_over(decay_of(s, h, err), t1 - t0);
  }
  __syncthreads();
  if (i >= elems) return;
  const int r = i / s.cols, c = i - r * s.cols;
  float x = s.from.p != nullptr ? s.from.p[(int64_t)unit * elems + r * s.from.si + c * s.from.sj] * s.from_factor : 0.0f;
  float* at = all.parts[blockIdx.z].states + (int64_t)unit * all.split.slots * elems + i;
  *at = x;
  constexpr int kAhead = 8;
  for (int j0 = 0; j0 < runs; j0 += kAhead) {
    float own[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) own[k] = j0 + k < runs ? at[(int64_t)(k + 1) * elems] : 0.0f;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (j0 + k >= runs) break;
      const float2 a = fade[j0 + k];
      x = fmaf(x, a.x, fmaf(x, a.y, own[k]));
      at += elems;
      *at = x;
    }
  }
}

// dst[b][g] (+)= sum over the heads that share key head g of src[b][h], in order.
struct HeadSum {
  const float* src;
  Rows dst;
  int dim, accumulate;
};
struct HeadSums {
  HeadSum of[2];
};
template <int V, typename Index>
__global__ void __launch_bounds__(256) sum_heads_kernel(const __grid_constant__ HeadSums sums, Index rows, int kv_heads,
                                                        int group, int seq) {
  const HeadSum& s = sums.of[blockIdx.y];
  const Index i = (Index)blockIdx.x * 256 + threadIdx.x, per = s.dim / V;
  if (i >= rows * per) return;
  const Index row = i / per, bg = row / seq, b = bg / kv_heads;
  const int c = (int)(i - row * per) * V;
  const int64_t t = row - bg * seq, pitch = (int64_t)seq * s.dim;
  const float* from = s.src + (int64_t)bg * group * pitch + t * s.dim + c;
  float* to = const_cast<float*>(s.dst.p) + b * s.dst.batch + (bg - b * kv_heads) * s.dst.head + t * s.dst.token + c;
  float sum[V] = {};
  auto add = [&](const float* p) {
    if constexpr (V == 4) {
      const float4 w = *(const float4*)p;
      sum[0] += w.x, sum[1] += w.y, sum[2] += w.z, sum[3] += w.w;
    } else {
      sum[0] += *p;
    }
  };
#pragma unroll 4
  for (int k = 0; k < group; ++k) add(from + k * pitch);
  if (s.accumulate) add(to);
  if constexpr (V == 4) *(float4*)to = make_float4(sum[0], sum[1], sum[2], sum[3]);
  else *to = sum[0];
}

// From how many tokens on 64 at a time are faster than one by one (24 tokens: 32 sequences of
// 16 heads 73 us one by one and 68 by 64, one sequence 19 and 20).
constexpr int kChunkedFrom = 24;

// How the tokens of each of `units` heads are shared, of `scans` in one launch, of `states` of
// which a first launch forms states.  Times in steps of scan_kernel, 5 us: 2 for a block's
// start and end, half a step for one of the first launch, 1.5 for the join's launch (with 3,
// 3 ragged sequences of 777 train in 114 us in place of 101).  With one segment a head,
// training on 8192 tokens of 16 heads took 1220 us where it took 445 with these; with one piece a
// segment 500.
Split split_of(int64_t units, int seq, int scans, int states) {
  const int64_t steps = ceil_div(seq, kStep);
  double best = (double)ceil_div(scans * units, 148) * (steps + 2.0);
  Split split{1, 1, 1};
  if (units > 1024) return split;
  for (int64_t n = 2; n <= std::min<int64_t>(steps, kMostSlots); ++n) {
    const int64_t per = ceil_div(steps, n);
    for (int64_t p = 1; p <= std::min<int64_t>(per, kMostSlots / n); ++p) {
      const double cost = (double)ceil_div(scans * units * n, 148) * (per + 2.0) +
                          (double)ceil_div(states * units * (n - 1) * p, 148) * (0.5 * ceil_div(per, p) + 2.0) + 1.5;
      if (cost < best) best = cost, split = {(int)n, (int)p, (int)((n - 1) * p + 1)};
    }
  }
  return split;
}
Split forward_split(const DecayShape& s) { return split_of((int64_t)s.batch * s.heads, s.seq, 1, 1); }
Split backward_split(const DecayShape& s) { return split_of((int64_t)s.batch * s.heads, s.seq, 3, 2); }

// Floats of a scan's states.  (What lies behind them starts on a 16-byte boundary.)
int64_t states_elems(const DecayShape& s, const Split& split) {
  if (s.seq < kChunkedFrom || split.segments == 1) return 0;
  return ceil_div((int64_t)s.batch * s.heads * split.slots * s.key_dim * s.value_dim, 4) * 4;
}

// Whether an operand's rows are whole 16-byte pieces.
bool whole_pieces(const Rows& r, int dim) {
  return ((uintptr_t)r.p & 15) == 0 && dim % 4 == 0 && r.token % 4 == 0 && r.head % 4 == 0 && r.batch % 4 == 0;
}

template <int DK, bool STATE_ONLY, bool VEC>
void launch_chunks(const Scans& scans, int count, int* err, cudaStream_t st) {
  auto kernel = scan_kernel<DK, STATE_ONLY, VEC>;
  static std::atomic<uint64_t> set{0};  // devices whose limit is set
  int device;
  TYSOR_CUDA(cudaGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (!(set.load(std::memory_order_relaxed) & bit)) {
    // The warps share out what the block is launched with.
    cudaFuncAttributes made;
    TYSOR_CUDA(cudaFuncGetAttributes(&made, kernel));
    if (made.numRegs * kScanThreads < kWorkers * kWorkerRegs + (kScanThreads - kWorkers) * kOtherRegs)
      throw CudaError("decay_attention: the kernel was built with too few registers");
    TYSOR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ScanSmem<DK>::kBytes));
    set.fetch_or(bit, std::memory_order_relaxed);
  }
  const int units = scans.scan[0].batch * scans.scan[0].heads, runs = STATE_ONLY ? scans.split.slots - 1 : scans.split.segments;
  kernel<<<dim3((unsigned)(units * runs), (unsigned)count), kScanThreads, ScanSmem<DK>::kBytes, st>>>(scans, err);
  check_launch();
}

// A scan and where it has the states of its segments.
struct ScanCall {
  Scan s;
  ScanParts parts;
  bool own_states;  // or those that an earlier call of the launch forms

  bool vec() const { return whole_pieces(s.q, s.rows) && whole_pieces(s.k, s.rows) && whole_pieces(s.v, s.cols); }
};

ScanMaps maps_of(const Scan& s) {
  auto map = [&](const Rows& r, int dim, int box_cols, int box_rows) {
    return rows_map(r.p, {(uint64_t)dim, (uint64_t)s.seq, (uint64_t)(s.heads / r.share), (uint64_t)s.batch},
                    {(uint64_t)r.token, (uint64_t)r.head, (uint64_t)r.batch}, box_cols, box_rows);
  };
  ScanMaps maps{map(s.q, s.rows, s.rows, kStep), map(s.k, s.rows, s.rows, kStep), map(s.v, s.cols, s.cols, kStep), {},
                whole_pieces(s.out, s.cols)};
  if (maps.stores) maps.out = map(s.out, s.cols, s.cols, kStep);
  return maps;
}

// Scans of as many sequences and heads that do not need one another's outputs, each kind of
// kernel in one launch: heads that leave SMs without a block do so once, not once a scan.
void run_scans(const ScanCall* calls, int count, const Split& split, int* err, cudaStream_t st) {
  const Scan& any = calls[0].s;
  if (any.batch <= 0 || any.heads <= 0) return;
  if (any.seq < kChunkedFrom) {
    for (int i = 0; i < count; ++i) {
      const Scan& s = calls[i].s;
      auto plain = [&](const StateAt& x) {
        return x.p == nullptr || (x.si == s.cols && x.sj == 1 && ((uintptr_t)x.p & 15) == 0);
      };
      const dim3 grid((unsigned)(s.batch * s.heads), (unsigned)ceil_div(s.cols, kSlice));
      if (s.cols % 4 == 0 && plain(s.from) && plain(s.to)) step_kernel<true><<<grid, kStepThreads, 0, st>>>(s, err);
      else step_kernel<false><<<grid, kStepThreads, 0, st>>>(s, err);
      check_launch();
    }
    return;
  }
  // (Keys and values of different widths: the gradients' scans still go together.)
  bool wide = false;
  for (int i = 0; i < count; ++i) wide |= calls[i].s.rows > 64;
  auto pass = [&](bool vec, bool state_only) {
    Scans scans{};
    scans.split = split;
    int n = 0;
    for (int i = 0; i < count; ++i) {
      const ScanCall& c = calls[i];
      if (c.vec() != vec || (state_only && !c.own_states)) continue;
      if (vec) scans.maps[n] = maps_of(c.s);
      scans.scan[n] = c.s;
      scans.parts[n++] = c.parts;
    }
    if (n == 0) return;
    auto go = [&]<int DK, bool VEC>() {
      state_only ? launch_chunks<DK, true, VEC>(scans, n, err, st) : launch_chunks<DK, false, VEC>(scans, n, err, st);
    };
    if (wide) vec ? go.template operator()<128, true>() : go.template operator()<128, false>();
    else vec ? go.template operator()<64, true>() : go.template operator()<64, false>();
  };
  auto passes = [&](bool state_only) {
    pass(false, state_only);
    pass(true, state_only);
  };
  if (split.segments > 1) {
    passes(true);
    Scans scans{};
    scans.split = split;
    int n = 0;
    for (int i = 0; i < count; ++i)
      if (calls[i].own_states) scans.scan[n] = calls[i].s, scans.parts[n++] = calls[i].parts;
    scan_states_kernel<<<dim3((unsigned)ceil_div(any.rows * any.cols, 256), (unsigned)(any.batch * any.heads), (unsigned)n),
                         256, 0, st>>>(scans, err);
    check_launch();
  }
  passes(false);
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
  // (A row's power of two times that stays a normal number.)
  if (!(scale >= 0x1p-30f && scale <= 0x1p30f)) return "decay_attention requires a scale from 2^-30 to 2^30";
  return nullptr;
}

int64_t decay_attention_work_elems(const DecayShape& s) { return states_elems(s, forward_split(s)); }

// Floats of a gradient of each query head's own, where they share key heads.
static int64_t by_head_elems(const DecayShape& s, int dim) {
  return s.heads == s.kv_heads ? 0 : ceil_div((int64_t)s.batch * s.heads * s.seq * dim, 4) * 4;
}
int64_t decay_attention_backward_work_elems(const DecayShape& s) {
  return 2 * states_elems(s, backward_split(s)) + by_head_elems(s, s.key_dim) + by_head_elems(s, s.value_dim);
}

void launch_decay_attention(const DecayShape& s, const DecayInputs& in, float* out, float* new_state, float* work,
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
  const ScanCall call{c, {work, s.value_dim, 1}, true};
  run_scans(&call, 1, forward_split(s), err, st);
}

void launch_decay_attention_backward(const DecayShape& s, const DecayInputs& in, const float* dout,
                                     const float* dnew_state, float* dq, float* dk, float* dv, float* dstate,
                                     float* work, int accumulate_q, int accumulate_k, int accumulate_v,
                                     int accumulate_state, int* err, cudaStream_t st) {
  const int share = s.heads / s.kv_heads;
  const Rows q = rows_of(s, in.q, s.heads, s.key_dim, 1), k = rows_of(s, in.k, s.kv_heads, s.key_dim, share);
  const Rows v = rows_of(s, in.v, s.kv_heads, s.value_dim, share), g = rows_of(s, dout, s.heads, s.value_dim, 1);
  const Split split = backward_split(s);
  const int64_t states = states_elems(s, split);
  float* by_head = work + 2 * states;
  Scan c = scan_of(s, in);
  c.rows = s.value_dim;
  c.cols = s.key_dim;
  c.q = g;
  c.k = v;
  c.v = k;
  c.out = rows_of(s, dq, s.heads, s.key_dim, 1);
  c.from = {const_cast<float*>(in.state), 1, s.value_dim};
  c.accumulate = accumulate_q;
  ScanCall calls[3];
  calls[0] = {c, {work, s.key_dim, 1}, true};

  // The states of the scans back are the gradients' over `scale`.  The second one's is the
  // first's transposed: its segments start from the first's states.
  c.back = 1;
  c.from_factor = 1.0f / s.scale;
  c.to_factor = s.scale;
  HeadSums sums;
  auto keys_out = [&](int i, float* grad, int dim, int accumulate) {
    const Rows to = rows_of(s, grad, s.kv_heads, dim, 1);
    if (share == 1) {
      c.out = to;
      c.accumulate = accumulate;
      return;
    }
    float* part = by_head + (i ? by_head_elems(s, s.value_dim) : 0);
    c.out = {part, (int64_t)s.heads * s.seq * dim, (int64_t)s.seq * dim, dim, 1};
    c.accumulate = 0;
    sums.of[i] = {part, to, dim, accumulate};
  };
  c.rows = s.key_dim;
  c.cols = s.value_dim;
  c.q = k;
  c.k = q;
  c.v = g;
  c.from = {const_cast<float*>(dnew_state), s.value_dim, 1};
  c.to = {dstate, s.value_dim, 1};
  c.accumulate_state = accumulate_state;
  keys_out(0, dv, s.value_dim, accumulate_v);
  calls[1] = {c, {work + states, s.value_dim, 1}, true};
  c.rows = s.value_dim;
  c.cols = s.key_dim;
  c.q = v;
  c.k = g;
  c.v = q;
  c.from = {const_cast<float*>(dnew_state), 1, s.value_dim};
  c.to = {};
  keys_out(1, dk, s.key_dim, accumulate_k);
  calls[2] = {c, {work + states, 1, s.value_dim}, false};
  run_scans(calls, 3, split, err, st);

  const int64_t rows = (int64_t)s.batch * s.kv_heads * s.seq;
  if (share == 1 || rows <= 0) return;
  const bool vec = whole_pieces(sums.of[0].dst, s.value_dim) && whole_pieces(sums.of[1].dst, s.key_dim) &&
                   whole_pieces({by_head, 0, 0, 0, 1}, 4);
  const int64_t n = rows * std::max(s.key_dim, s.value_dim) / (vec ? 4 : 1);
  auto go = [&](auto kernel, auto count) {
    kernel<<<dim3((unsigned)ceil_div(n, 256), 2), 256, 0, st>>>(sums, count, s.kv_heads, share, s.seq);
  };
  if (n < INT64_C(4000000000)) vec ? go(sum_heads_kernel<4, uint32_t>, (uint32_t)rows) : go(sum_heads_kernel<1, uint32_t>, (uint32_t)rows);
  else vec ? go(sum_heads_kernel<4, int64_t>, rows) : go(sum_heads_kernel<1, int64_t>, rows);
  check_launch();
}

}  // namespace tysor
