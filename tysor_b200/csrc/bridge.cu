// The C ABI of libtysor_cuda.so: context, buffers, per-op dispatch
// (include/tysor_cuda.h).  Every entry point catches C++ exceptions and
// reports them through tysor_cuda_last_error(), the convention of the
// reference's Metal bridge (native/metal_bridge.mm:14-16, 72-97).
#include <math.h>
#include <string.h>

#include <algorithm>
#include <cstring>
#include <initializer_list>
#include <mutex>
#include <vector>

#include "../../include/tysor_cuda.h"
#include "context.cuh"
#include "lm_ops.cuh"
#include "ops.cuh"

namespace tysor {

std::atomic<int64_t> g_launches{0};

static thread_local std::string t_last_error;

void set_last_error(const std::string& msg) { t_last_error = msg; }
const char* last_error_cstr() { return t_last_error.c_str(); }

const char* device_error_message(int code) {
  switch (code) {
    case kErrIndexRange: return "Embedding index out of range";
    case kErrBarrierTimeout: return "a tensor-core pipeline wait timed out";
    case kErrTmemAlloc: return "tensor memory allocation failed";
    case kErrSequence: return "Attention start or length out of range";
    case kErrDecay: return "Decay below 0 or NaN";
    default: return "unknown device error";
  }
}

void* Context::ensure_scratch(size_t bytes) {
  const bool in_capture = capturing();
  if (bytes <= scratch_bytes) {
    scratch_captured |= in_capture;
    return scratch;
  }
  if (in_capture)
    throw CudaError("the workspace cannot grow while the context's stream is captured: make the call once before");
  TYSOR_CUDA(cudaStreamSynchronize(stream));
  if (scratch_captured) former_scratch.push_back(scratch);
  else if (scratch) TYSOR_CUDA(cudaFree(scratch));
  scratch = nullptr;
  scratch_bytes = 0;
  scratch_captured = false;
  size_t want = bytes + bytes / 4 + 4096;
  TYSOR_CUDA(cudaMalloc(&scratch, want));
  scratch_bytes = want;
  return scratch;
}

bool Context::capturing() const {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  TYSOR_CUDA(cudaStreamIsCapturing(stream, &status));
  return status != cudaStreamCaptureStatusNone;
}

void* Context::new_table(const void* host, size_t bytes) {
  if (capturing())
    throw CudaError("rope's table of these sizes cannot be made while the context's stream is captured: "
                    "make the call once before");
  void* d = nullptr;
  TYSOR_CUDA(cudaMalloc(&d, bytes));
  // On the stream whose kernels read it, which waits for no other stream's copies.
  cudaError_t e = cudaMemcpyAsync(d, host, bytes, cudaMemcpyHostToDevice, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) cudaFree(d);
  TYSOR_CUDA(e);
  return d;
}

const float2* Context::rope_table(int64_t seq, int64_t half, double theta) {
  uint64_t bits;
  std::memcpy(&bits, &theta, sizeof bits);
  auto key = std::make_tuple(seq, half, bits);
  auto it = rope_tables.find(key);
  if (it != rope_tables.end()) return it->second;
  // Angles and their cos/sin are computed on the host with the C library in
  // f32, as layers.rs:254-262 computes them; the kernels then apply the
  // rotation with separately rounded products.
  std::vector<float> inv((size_t)(half > 0 ? half : 1));
  for (int64_t i = 0; i < half; ++i) inv[i] = powf((float)theta, -(float)i / (float)half);
  std::vector<float2> tab((size_t)(seq * half > 0 ? seq * half : 1));
  for (int64_t p = 0; p < seq; ++p)
    for (int64_t i = 0; i < half; ++i) {
      volatile float ang = (float)p * inv[i];
      tab[p * half + i] = make_float2(cosf(ang), sinf(ang));
    }
  auto* d = (const float2*)new_table(tab.data(), sizeof(float2) * tab.size());
  rope_tables[key] = d;
  return d;
}

const double* Context::rope_rate_table(int64_t half, double theta) {
  uint64_t bits;
  std::memcpy(&bits, &theta, sizeof bits);
  auto key = std::make_tuple(half, bits);
  auto it = rope_rates.find(key);
  if (it != rope_rates.end()) return it->second;
  std::vector<double> rate((size_t)half);
  for (int64_t i = 0; i < half; ++i) rate[i] = pow(theta, -(double)i / (double)half) / (2.0 * 3.14159265358979323846);
  auto* d = (const double*)new_table(rate.data(), sizeof(double) * rate.size());
  rope_rates[key] = d;
  return d;
}

const std::vector<double>& Context::rotary_rates(const RotaryRates& r) {
  for (auto& [key, rates] : rotary_rate_lists)
    if (key == r) return rates;
  // Few models in a process; one that changes them from call to call pays for it.
  if (rotary_rate_lists.size() >= 16) rotary_rate_lists.clear();
  std::vector<double> rates((size_t)r.half);
  rotary_fill_rates(r, rates.data());
  return rotary_rate_lists.emplace_back(r, std::move(rates)).second;
}

void Context::sync_and_check() {
  TYSOR_CUDA(cudaStreamSynchronize(stream));
  int code = 0;
  TYSOR_CUDA(cudaMemcpy(&code, d_err, sizeof(int), cudaMemcpyDeviceToHost));
  if (code != 0) {
    int zero = 0;
    TYSOR_CUDA(cudaMemcpy(d_err, &zero, sizeof(int), cudaMemcpyHostToDevice));
    throw CudaError(device_error_message(code));
  }
}

}  // namespace tysor

using namespace tysor;

namespace {

template <typename F>
bool guarded(F&& f) {
  try {
    f();
    return true;
  } catch (const std::exception& e) {
    set_last_error(e.what());
    return false;
  } catch (...) {
    set_last_error("unknown error");
    return false;
  }
}

Context* ctx_of(void* p) {
  if (!p) throw CudaError("null context");
  Context* c = static_cast<Context*>(p);
  TYSOR_CUDA(cudaSetDevice(c->device));
  return c;
}

Buffer* buf_of(void* p) {
  if (!p) throw CudaError("null buffer");
  return static_cast<Buffer*>(p);
}

float* ptr_of(void* p, size_t need, const char* what) {
  Buffer* b = buf_of(p);
  if (b->count < need)
    throw CudaError(std::string(what) + " buffer holds " + std::to_string(b->count) +
                    " elements, " + std::to_string(need) + " needed");
  return b->ptr;
}

GemmScratch gemm_scratch(Context* c, int batch, int64_t M, int64_t N, int64_t K,
                         const GemmOperand& A, const GemmOperand& Bm, int mode) {
  int64_t na = 0, nb = 0;
  gemm_scratch_need(batch, M, N, K, A, Bm, mode, &na, &nb);
  GemmScratch s{nullptr, nullptr, 0, 0};
  if (na + nb == 0) return s;
  const int64_t na_pad = (na + 63) & ~(int64_t)63;
  float* base = (float*)c->ensure_scratch(sizeof(float) * (size_t)(na_pad + nb + 64));
  s.a_lo = base;
  s.b_lo = base + na_pad;
  s.a_elems = na;
  s.b_elems = nb;
  return s;
}

void run_gemm(Context* c, int batch, int64_t M, int64_t N, int64_t K, const GemmOperand& A,
              const GemmOperand& Bm, const GemmOutput& out, const GemmEpilogue& ep_in) {
  GemmEpilogue ep = ep_in;
  ep.chunk_kb = c->accum_chunk_kb;
  const int mode =
      gemm_effective_mode(c->matmul_mode, batch, M, N, K, ep.tri, ep.smx_p != nullptr, out.ld, out.batch_stride);
  GemmScratch s = gemm_scratch(c, batch, M, N, K, A, Bm, mode);
  gemm_launch(batch, M, N, K, A, Bm, out, ep, mode, s, c->d_err, c->stream);
}

float* scratch_floats(Context* c, int64_t n) {
  return (float*)c->ensure_scratch(sizeof(float) * (size_t)(n > 0 ? n : 1));
}

// A dispatch's operands: each holds what the call needs and lies on the
// context's device, pairs of values (statistics) are 8-byte aligned, and no
// output overlaps an input or another output.
struct Operands {
  Context* ctx;
  struct Range {
    uintptr_t begin, end;
    const char* what;
    bool written;
  };
  std::vector<Range> ranges;

  explicit Operands(Context* c) : ctx(c) {}

  float* take(void* p, size_t need, const char* what, bool written) {
    float* f = ptr_of(p, need, what);
    if (buf_of(p)->ctx->device != ctx->device)
      throw CudaError(std::string(what) + " buffer is on another device");
    if (std::strcmp(what, "stats") == 0 && ((uintptr_t)f & 7) != 0)
      throw CudaError("stats buffer must start on an 8-byte boundary");
    ranges.push_back({(uintptr_t)f, (uintptr_t)(f + need), what, written});
    return f;
  }
  const float* in(void* p, size_t need, const char* what) { return take(p, need, what, false); }
  const float* in_or_null(void* p, size_t need, const char* what) { return p ? in(p, need, what) : nullptr; }
  float* out(void* p, size_t need, const char* what) { return take(p, need, what, true); }
  float* out_or_null(void* p, size_t need, const char* what) { return p ? out(p, need, what) : nullptr; }

  // `a_may_be` and `b_may_be`: two operands that may be the very same memory.
  void check_overlap(const char* a_may_be = "", const char* b_may_be = "") const {
    for (const Range& a : ranges)
      for (const Range& b : ranges)
        if (&a != &b && a.begin == b.begin && std::strcmp(a.what, a_may_be) == 0 && std::strcmp(b.what, b_may_be) == 0)
          continue;
        else if (&a != &b && a.written && a.begin < a.end && b.begin < b.end && a.begin < b.end && b.begin < a.end)
          throw CudaError(std::string(a.what) + " overlaps " + b.what);
  }
};

// The product of sizes, refused where no buffer could hold it.
size_t elems(std::initializer_list<uint64_t> sizes) {
  uint64_t n = 1;
  for (uint64_t d : sizes)
    if (d == 0) return 0;
  for (uint64_t d : sizes) {
    if (n > ((uint64_t)1 << 60) / d) throw CudaError("sizes overflow");
    n *= d;
  }
  return (size_t)n;
}

void check_norm(uint32_t width, float eps) {
  if (width == 0) throw CudaError("layer_norm requires a width of at least 1");
  if (!(eps >= 0.0f) || isinf(eps)) throw CudaError("layer_norm requires a finite eps >= 0");
}

void check_distill(uint32_t width, uint32_t top, float temperature) {
  if (width == 0 || width > 0x7fffffffu) throw CudaError("distill_loss requires a width of 1 to 2^31 - 1");
  if (top == 0 || top > (uint32_t)kMaxDistillTop)
    throw CudaError("distill_loss takes 1 to " + std::to_string(kMaxDistillTop) + " entries per row");
  if (!distill_temperature(temperature))
    throw CudaError("distill_loss requires a finite temperature > 0, from 2^-60 to 2^60");
}

AttentionShape attention_shape(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t q_len, uint32_t k_len,
                               uint32_t head_dim, uint32_t window, uint32_t sinks, float scale, bool seq_major) {
  if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0)
    throw CudaError("window_attention: the key heads must divide the query heads");
  if (head_dim == 0 || head_dim > (uint32_t)kMaxHeadDim)
    throw CudaError("window_attention takes heads of 1 to " + std::to_string(kMaxHeadDim) + " values");
  const uint32_t most = 1u << 29;  // positions stay below 2^30
  if (q_len > most || k_len > most || batch > most || heads > most)
    throw CudaError("window_attention takes lengths, batches and heads up to 2^29");
  // A subnormal scale would hold fewer bits than the scores it multiplies, and one
  // above 2^127 leaves fp32 times log2 e.
  if (!(scale >= 0x1p-126f) || scale > 0x1p127f)
    throw CudaError("window_attention requires a finite scale of at least 2^-126 and at most 2^127");
  AttentionShape s{};
  s.batch = (int)batch;
  s.heads = (int)heads;
  s.kv_heads = (int)kv_heads;
  s.q_len = (int)q_len;
  s.k_len = (int)k_len;
  s.head_dim = (int)head_dim;
  s.window = (int)(window < most ? window : most);  // no position lies further back
  s.sinks = (int)(sinks < most ? sinks : most);
  s.scale = scale;
  s.seq_major = seq_major;
  return s;
}

void rope_axes(void* context, void* x, void* positions, void* out, uint32_t batch, uint32_t heads, uint32_t seq_len,
               const int64_t* sections, int axes, double theta, bool seq_major, bool back, bool accumulate) {
  Operands o(ctx_of(context));
  if (sections == nullptr || axes < 1 || axes > kMaxRopeAxes)
    throw CudaError("rope_axes takes 1 to " + std::to_string(kMaxRopeAxes) + " axes");
  if (!(theta > 0.0) || isinf(theta)) throw CudaError("rope_axes requires a finite theta > 0");
  const uint32_t most = 1u << 30;
  if (batch > most || heads > most || seq_len > most) throw CudaError("rope_axes takes sizes up to 2^30");
  RopeAxes s{};
  s.batch = (int)batch;
  s.heads = (int)heads;
  s.seq = (int)seq_len;
  s.axes = axes;
  s.seq_major = seq_major;
  int64_t half = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 1 || sections[a] > 65536) throw CudaError("rope_axes sections hold 1 to 65536 pairs");
    half += sections[a];
    s.ends[a] = (int)half;
  }
  s.half = (int)half;
  const size_t n = elems({batch, heads, seq_len, 2 * (uint64_t)half});
  const float* in = o.in(x, n, back ? "grad" : "input");
  const float* pos = o.in(positions, elems({batch, (uint64_t)axes, seq_len}), "positions");
  float* y = o.out(out, n, back ? "dx" : "out");
  o.check_overlap();
  launch_rope_axes(in, pos, o.ctx->rope_rate_table(half, theta), y, s, back, accumulate, o.ctx->stream);
}

void rotary(void* context, void* x, void* positions, void* out, uint32_t batch, uint32_t heads, uint32_t seq_len,
            uint32_t head_dim, uint32_t rotary_dim, bool interleaved, const RotaryRates& rates, double amplitude,
            bool seq_major, bool back, bool accumulate) {
  Operands o(ctx_of(context));
  if (rotary_dim % 2 != 0 || rotary_dim > head_dim)
    throw CudaError("rotary requires an even number of turned values, at most the head's");
  if (const char* problem = rotary_rates_problem(rates, amplitude)) throw CudaError(problem);
  const uint32_t most = 1u << 30;
  if (batch > most || heads > most || seq_len > most || head_dim > most)
    throw CudaError("rotary takes sizes up to 2^30");
  RotaryShape s{};
  s.batch = (int)batch;
  s.heads = (int)heads;
  s.seq = (int)seq_len;
  s.head_dim = (int)head_dim;
  s.half = rates.half;
  s.interleaved = interleaved;
  s.seq_major = seq_major;
  s.amplitude = (float)amplitude;
  const size_t n = elems({batch, heads, seq_len, head_dim});
  const float* in = o.in(x, n, back ? "grad" : "input");
  const float* pos = o.in_or_null(positions, elems({batch, seq_len}), "positions");
  float* y = o.out(out, n, back ? "dx" : "out");
  o.check_overlap();
  std::copy_n(o.ctx->rotary_rates(rates).begin(), rates.half, s.rates);
  launch_rotary(in, pos, y, s, back, accumulate, o.ctx->stream);
}

DecayShape decay_shape(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t seq_len, uint32_t key_dim,
                       uint32_t value_dim, float scale, bool seq_major) {
  if (const char* problem = decay_attention_problem(batch, heads, kv_heads, seq_len, key_dim, value_dim, scale))
    throw CudaError(problem);
  return {(int)batch, (int)heads, (int)kv_heads, (int)seq_len, (int)key_dim, (int)value_dim, scale, seq_major};
}

// The operands of decay_attention and its gradients; `state` is read alone.
DecayInputs decay_inputs(Operands& o, const DecayShape& s, void* q, void* k, void* v, void* decay, void* state,
                         void* lengths) {
  const uint64_t batch = s.batch, heads = s.heads, kv_heads = s.kv_heads, seq = s.seq;
  const uint64_t key_dim = s.key_dim, value_dim = s.value_dim;
  DecayInputs in{};
  in.q = o.in(q, elems({batch, heads, seq, key_dim}), "q");
  in.k = o.in(k, elems({batch, kv_heads, seq, key_dim}), "k");
  in.v = o.in(v, elems({batch, kv_heads, seq, value_dim}), "v");
  in.decay = o.in(decay, heads, "decay");
  in.state = o.in_or_null(state, elems({batch, heads, key_dim, value_dim}), "state");
  in.lengths = o.in_or_null(lengths, batch, "lengths");
  if (((uintptr_t)in.state & 15) != 0) throw CudaError("state buffer must start on a 16-byte boundary");
  return in;
}

LogprobShape logprob_shape(uint32_t rows, uint32_t width, uint32_t given, uint32_t top, float temperature) {
  if (width == 0 || width > (uint32_t)kMaxLogprobWidth)
    throw CudaError("token_logprobs requires a width of 1 to 2^24");
  if (rows > (uint32_t)INT32_MAX) throw CudaError("token_logprobs takes up to 2^31 - 1 rows");
  if (given > (uint32_t)kMaxGivenTokens)
    throw CudaError("token_logprobs takes up to " + std::to_string(kMaxGivenTokens) + " given ids a row");
  if (top > (uint32_t)kMaxTopTokens)
    throw CudaError("token_logprobs gives up to " + std::to_string(kMaxTopTokens) + " best tokens a row");
  if (!distill_temperature(temperature))
    throw CudaError("token_logprobs requires a finite temperature > 0, from 2^-60 to 2^60");
  return {rows, (int)width, (int)given, (int)top, temperature};
}

}  // namespace

extern "C" {

const char* tysor_cuda_last_error(void) { return last_error_cstr(); }

void* tysor_cuda_context_new(int device) {
  Context* out = nullptr;
  guarded([&] {
    int n = 0;
    TYSOR_CUDA(cudaGetDeviceCount(&n));
    if (device < 0 || device >= n)
      throw CudaError("CUDA device " + std::to_string(device) + " not present (" +
                      std::to_string(n) + " visible)");
    cudaDeviceProp prop;
    TYSOR_CUDA(cudaGetDeviceProperties(&prop, device));
    if (prop.major != 10)
      throw CudaError(std::string("tysor_cuda is built for sm_100a; device is ") + prop.name);
    TYSOR_CUDA(cudaSetDevice(device));
    auto* c = new Context();
    c->device = device;
    TYSOR_CUDA(cudaStreamCreateWithFlags(&c->stream, cudaStreamNonBlocking));
    TYSOR_CUDA(cudaMalloc(&c->d_err, 16));
    TYSOR_CUDA(cudaMemset(c->d_err, 0, 16));
    out = c;
  });
  return out;
}

void tysor_cuda_context_free(void* context) {
  if (!context) return;
  guarded([&] {
    Context* c = static_cast<Context*>(context);
    cudaSetDevice(c->device);
    cudaStreamSynchronize(c->stream);
    for (auto& kv : c->rope_tables) cudaFree((void*)kv.second);
    for (auto& kv : c->rope_rates) cudaFree((void*)kv.second);
    if (c->scratch) cudaFree(c->scratch);
    for (void* p : c->former_scratch) cudaFree(p);
    if (c->d_err) cudaFree(c->d_err);
    if (c->comm) tysor_cuda_comm_free(c);
    cudaStreamDestroy(c->stream);
    delete c;
  });
}

bool tysor_cuda_synchronize(void* context) {
  return guarded([&] { ctx_of(context)->sync_and_check(); });
}

bool tysor_cuda_set_matmul_accumulation(void* context, int kblocks) {
  return guarded([&] {
    if (kblocks < 0 || kblocks > 64) throw CudaError("accumulation chunk must be 0 (default) or 1..64 k-blocks");
    ctx_of(context)->accum_chunk_kb = kblocks;
  });
}

bool tysor_cuda_probe_wait_timeout(void* context, int64_t limit_cycles) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_wait_timeout_probe(c->d_err, (long long)limit_cycles, c->stream);
    c->sync_and_check();
  });
}

void* tysor_cuda_context_stream(void* context) {
  void* out = nullptr;
  guarded([&] { out = (void*)ctx_of(context)->stream; });
  return out;
}

bool tysor_cuda_set_matmul_mode(void* context, int mode) {
  return guarded([&] {
    if (mode < 0 || mode > 3)
      throw CudaError("matmul mode must be 0 (strict), 1 (fast), 2 (exact) or 3 (strict16)");
    ctx_of(context)->matmul_mode = mode;
  });
}

void* tysor_cuda_buffer_new_zeroed(void* context, size_t count) {
  Buffer* out = nullptr;
  guarded([&] {
    Context* c = ctx_of(context);
    auto* b = new Buffer();
    b->ctx = c;
    b->count = count;
    b->owned = true;
    TYSOR_CUDA(cudaMalloc(&b->ptr, sizeof(float) * (count ? count : 1)));
    TYSOR_CUDA(cudaMemsetAsync(b->ptr, 0, sizeof(float) * (count ? count : 1), c->stream));
    out = b;
  });
  return out;
}

void* tysor_cuda_buffer_new_with_data(void* context, const float* data, size_t count) {
  void* b = tysor_cuda_buffer_new_zeroed(context, count);
  if (!b) return nullptr;
  if (!tysor_cuda_buffer_write(b, data, count)) {
    tysor_cuda_buffer_free(b);
    return nullptr;
  }
  return b;
}

void tysor_cuda_buffer_free(void* buffer) {
  if (!buffer) return;
  Buffer* b = static_cast<Buffer*>(buffer);
  if ((b->owned || b->wrapped) && b->ptr) {
    cudaSetDevice(b->ctx->device);
    // What is under way may use the memory, which goes back to its allocator here:
    // the library's, or the caller's.  (A capture is not under way, and no wait for it.)
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaStreamIsCapturing(b->ctx->stream, &capture);
    if (b->owned || capture == cudaStreamCaptureStatusNone) cudaStreamSynchronize(b->ctx->stream);
    if (b->owned) cudaFree(b->ptr);
  }
  delete b;
}

bool tysor_cuda_buffer_read(void* buffer, float* out_data, size_t count) {
  return guarded([&] {
    Buffer* b = buf_of(buffer);
    if (count > b->count) throw CudaError("buffer read past the end");
    ctx_of(b->ctx)->sync_and_check();
    TYSOR_CUDA(cudaMemcpy(out_data, b->ptr, sizeof(float) * count, cudaMemcpyDeviceToHost));
  });
}

bool tysor_cuda_buffer_write(void* buffer, const float* data, size_t count) {
  return guarded([&] {
    Buffer* b = buf_of(buffer);
    if (count > b->count) throw CudaError("buffer write past the end");
    Context* c = ctx_of(b->ctx);
    TYSOR_CUDA(cudaMemcpyAsync(b->ptr, data, sizeof(float) * count, cudaMemcpyHostToDevice, c->stream));
    TYSOR_CUDA(cudaStreamSynchronize(c->stream));
  });
}

void* tysor_cuda_buffer_view(void* base, size_t offset, size_t count) {
  Buffer* out = nullptr;
  guarded([&] {
    Buffer* b = buf_of(base);
    if (offset + count > b->count) throw CudaError("view outside its base buffer");
    auto* v = new Buffer();
    v->ctx = b->ctx;
    v->ptr = b->ptr + offset;
    v->count = count;
    v->owned = false;
    out = v;
  });
  return out;
}

void* tysor_cuda_buffer_wrap(void* context, float* data, size_t count) {
  Buffer* out = nullptr;
  guarded([&] {
    Context* c = ctx_of(context);
    if (data == nullptr) throw CudaError("wrap: null device pointer");
    if (((uintptr_t)data & 3) != 0) throw CudaError("wrap: the memory is not aligned to its fp32 values");
    cudaPointerAttributes attr;
    TYSOR_CUDA(cudaPointerGetAttributes(&attr, data));
    if (attr.type != cudaMemoryTypeDevice || attr.device != c->device)
      throw CudaError("wrap: the memory is not on the context's device");
    auto* b = new Buffer();
    b->ctx = c;
    b->ptr = data;
    b->count = count;
    b->wrapped = true;
    out = b;
  });
  return out;
}

size_t tysor_cuda_buffer_count(void* buffer) { return buffer ? buf_of(buffer)->count : 0; }

// ---- forward dispatch --------------------------------------------------------

bool tysor_cuda_dispatch_matmul(void* context, void* lhs, void* rhs, void* out, uint32_t m,
                                uint32_t n, uint32_t k) {
  return tysor_cuda_dispatch_linear(context, lhs, rhs, nullptr, out, m, n, k, false);
}

bool tysor_cuda_dispatch_linear(void* context, void* input, void* weight, void* bias, void* out,
                                uint32_t m, uint32_t n, uint32_t k, bool with_bias) {
  return guarded([&] {
    Context* c = ctx_of(context);
    GemmOperand A{ptr_of(input, (size_t)m * k, "lhs"), false, (int64_t)k, 0};
    GemmOperand Bm{ptr_of(weight, (size_t)k * n, "rhs"), false, (int64_t)n, 0};
    GemmOutput O{ptr_of(out, (size_t)m * n, "out"), (int64_t)n, 0};
    GemmEpilogue ep{with_bias ? ptr_of(bias, n, "bias") : nullptr, 1.0f, 0, 0};
    run_gemm(c, 1, m, n, k, A, Bm, O, ep);
  });
}

bool tysor_cuda_dispatch_matmul_ex(void* context, uint32_t batch, uint32_t m, uint32_t n,
                                   uint32_t k, void* a, bool trans_a, uint64_t lda,
                                   uint64_t stride_a, void* b, bool trans_b, uint64_t ldb,
                                   uint64_t stride_b, void* cbuf, uint64_t ldc, uint64_t stride_c,
                                   void* bias, float alpha, bool accumulate, bool relu) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (batch == 0) return;
    const uint64_t a_rows = trans_a ? k : m, a_cols = trans_a ? m : k;
    const uint64_t b_rows = trans_b ? n : k, b_cols = trans_b ? k : n;
    if (lda < a_cols || ldb < b_cols || ldc < n) throw CudaError("matmul_ex: leading dimension too small");
    const size_t a_need = (batch - 1) * stride_a + (a_rows ? (a_rows - 1) * lda + a_cols : 0);
    const size_t b_need = (batch - 1) * stride_b + (b_rows ? (b_rows - 1) * ldb + b_cols : 0);
    const size_t c_need = (batch - 1) * stride_c + (m ? (m - 1) * ldc + n : 0);
    GemmOperand A{ptr_of(a, a_need, "a"), trans_a, (int64_t)lda, (int64_t)stride_a};
    GemmOperand Bm{ptr_of(b, b_need, "b"), trans_b, (int64_t)ldb, (int64_t)stride_b};
    GemmOutput O{ptr_of(cbuf, c_need, "c"), (int64_t)ldc, (int64_t)stride_c};
    GemmEpilogue ep{bias ? ptr_of(bias, n, "bias") : nullptr, alpha, accumulate ? 1 : 0, relu ? 1 : 0};
    run_gemm(c, (int)batch, m, n, k, A, Bm, O, ep);
  });
}

bool tysor_cuda_dispatch_unary(void* context, int op, void* input, void* out, uint32_t count,
                               float param) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (op < 0 || op > 3) throw CudaError("unknown unary op");
    launch_unary(op, ptr_of(input, count, "input"), ptr_of(out, count, "out"), count, param, c->stream);
  });
}

bool tysor_cuda_dispatch_binary_tt(void* context, int op, void* lhs, void* rhs, void* out,
                                   uint32_t count) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (op < 0 || op > 3) throw CudaError("unsupported tensor binary op");
    launch_binary_tt(op, ptr_of(lhs, count, "lhs"), ptr_of(rhs, count, "rhs"), ptr_of(out, count, "out"),
                     count, c->stream);
  });
}

bool tysor_cuda_dispatch_binary_ts(void* context, int op, void* input, void* out, uint32_t count,
                                   double scalar) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (op < 0 || op > 3) throw CudaError("unsupported tensor binary op");
    launch_binary_ts(op, ptr_of(input, count, "input"), (float)scalar, ptr_of(out, count, "out"), count,
                     c->stream);
  });
}

bool tysor_cuda_dispatch_binary_st(void* context, int op, void* input, void* out, uint32_t count,
                                   double scalar) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (op < 0 || op > 3) throw CudaError("unsupported tensor binary op");
    launch_binary_st(op, (float)scalar, ptr_of(input, count, "input"), ptr_of(out, count, "out"), count,
                     c->stream);
  });
}

bool tysor_cuda_dispatch_rms_norm(void* context, void* input, void* out, uint32_t rows,
                                  uint32_t width) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    launch_rms_norm(ptr_of(input, n, "input"), ptr_of(out, n, "out"), rows, width, c->stream);
  });
}

bool tysor_cuda_dispatch_softmax(void* context, void* input, void* out, uint32_t rows,
                                 uint32_t width) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    launch_softmax(ptr_of(input, n, "input"), ptr_of(out, n, "out"), rows, width, c->stream);
  });
}

bool tysor_cuda_dispatch_cross_entropy(void* context, void* logits, void* target, void* out,
                                       uint32_t rows, uint32_t width) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    launch_cross_entropy(ptr_of(logits, n, "logits"), ptr_of(target, n, "target"), ptr_of(out, rows, "out"),
                         rows, width, c->stream);
  });
}

bool tysor_cuda_dispatch_embedding(void* context, void* indices, void* weight, void* out,
                                   uint32_t index_count, uint32_t embedding_dim,
                                   uint32_t num_embeddings) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_embedding(ptr_of(indices, index_count, "indices"),
                     ptr_of(weight, (size_t)num_embeddings * embedding_dim, "weight"),
                     ptr_of(out, (size_t)index_count * embedding_dim, "out"), index_count,
                     num_embeddings, embedding_dim, c->d_err, c->stream);
  });
}

bool tysor_cuda_dispatch_repeat_kv(void* context, void* input, void* out, uint32_t outer,
                                   uint32_t out_heads, uint32_t inner, uint32_t repeats) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (repeats == 0 || out_heads % repeats != 0) throw CudaError("repeat_kv repeats must divide the output heads");
    const uint32_t heads = out_heads / repeats;
    launch_repeat_kv(ptr_of(input, (size_t)outer * heads * inner, "input"),
                     ptr_of(out, (size_t)outer * out_heads * inner, "out"), outer, heads, inner, repeats,
                     c->stream);
  });
}

bool tysor_cuda_dispatch_causal_mask(void* context, void* input, void* out, uint32_t outer,
                                     uint32_t q, uint32_t k) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)outer * q * k;
    launch_causal_mask(ptr_of(input, n, "input"), ptr_of(out, n, "out"), outer, q, k, c->stream);
  });
}

bool tysor_cuda_dispatch_rope(void* context, void* input, void* out, uint32_t outer,
                              uint32_t seq_len, uint32_t half_dim, double theta) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)outer * seq_len * half_dim * 2;
    const float2* tab = c->rope_table(seq_len, half_dim, theta);
    launch_rope(ptr_of(input, n, "input"), ptr_of(out, n, "out"), tab, outer, seq_len, half_dim, c->stream);
  });
}

// ---- backward and update -------------------------------------------------------------

bool tysor_cuda_dispatch_relu_backward(void* context, void* out_act, void* grad, void* dx,
                                       uint64_t count, bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_relu_backward(ptr_of(out_act, count, "out"), ptr_of(grad, count, "grad"), ptr_of(dx, count, "dx"),
                         count, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_silu_backward(void* context, void* input, void* grad, void* dx,
                                       uint64_t count, bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_silu_backward(ptr_of(input, count, "input"), ptr_of(grad, count, "grad"), ptr_of(dx, count, "dx"),
                         count, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_softmax_backward(void* context, void* output, void* grad, void* dx,
                                          uint64_t count, bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_softmax_backward(ptr_of(output, count, "output"), ptr_of(grad, count, "grad"),
                            ptr_of(dx, count, "dx"), count, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_cross_entropy_backward(void* context, void* logits, void* target,
                                                void* grad, uint32_t rows, uint32_t width,
                                                bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    launch_cross_entropy_backward(ptr_of(logits, n, "logits"), ptr_of(target, n, "target"),
                                  ptr_of(grad, n, "grad"), rows, width, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_rope_backward(void* context, void* grad, void* dx, uint32_t outer,
                                       uint32_t seq_len, uint32_t half_dim, double theta,
                                       bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)outer * seq_len * half_dim * 2;
    const float2* tab = c->rope_table(seq_len, half_dim, theta);
    launch_rope_backward(ptr_of(grad, n, "grad"), ptr_of(dx, n, "dx"), tab, outer, seq_len, half_dim,
                         accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_repeat_kv_backward(void* context, void* grad, void* dx, uint32_t outer,
                                            uint32_t heads, uint32_t inner, uint32_t repeats,
                                            bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (repeats == 0) throw CudaError("repeat_kv backward requires repeats > 0");
    launch_repeat_kv_backward(ptr_of(grad, (size_t)outer * heads * repeats * inner, "grad"),
                              ptr_of(dx, (size_t)outer * heads * inner, "dx"), outer, heads, inner,
                              repeats, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_causal_mask_backward(void* context, void* grad, void* dx, uint32_t outer,
                                              uint32_t q, uint32_t k, bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)outer * q * k;
    launch_causal_mask_backward(ptr_of(grad, n, "grad"), ptr_of(dx, n, "dx"), outer, q, k, accumulate,
                                c->stream);
  });
}

bool tysor_cuda_dispatch_embedding_backward(void* context, void* grad, void* indices,
                                            void* weight_grad, uint32_t index_count,
                                            uint32_t embedding_dim, uint32_t num_embeddings,
                                            bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    void* work = c->ensure_scratch(embedding_backward_work_bytes(index_count, num_embeddings));
    launch_embedding_backward(ptr_of(grad, (size_t)index_count * embedding_dim, "grad"),
                              ptr_of(indices, index_count, "indices"),
                              ptr_of(weight_grad, (size_t)num_embeddings * embedding_dim, "weight_grad"),
                              index_count, num_embeddings, embedding_dim, work, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_bias_grad(void* context, void* grad, void* bias_grad, uint32_t rows,
                                   uint32_t width, bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    float* partial = scratch_floats(c, colsum_partial_elems(rows, width));
    launch_colsum(ptr_of(grad, (size_t)rows * width, "grad"), ptr_of(bias_grad, width, "bias_grad"), partial,
                  rows, width, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_add_inplace(void* context, void* dst, void* src, uint64_t count) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_add_inplace(ptr_of(dst, count, "dst"), ptr_of(src, count, "src"), count, c->stream);
  });
}

bool tysor_cuda_dispatch_sgd_update(void* context, void* param, void* grad, uint64_t count,
                                    double lr) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_sgd(ptr_of(param, count, "param"), ptr_of(grad, count, "grad"), (float)lr, count, c->stream);
  });
}

bool tysor_cuda_dispatch_reduce_sum(void* context, void* input, void* out, uint64_t count) {
  return guarded([&] {
    Context* c = ctx_of(context);
    float* partial = scratch_floats(c, 1024);
    launch_reduce_sum(ptr_of(input, count, "input"), ptr_of(out, 1, "out"), partial, count, c->stream);
  });
}

bool tysor_cuda_dispatch_rms_norm_gain(void* context, void* input, void* gain, void* out,
                                       uint32_t rows, uint32_t width, float eps) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    launch_rms_norm_gain(ptr_of(input, n, "input"), ptr_of(gain, width, "gain"), ptr_of(out, n, "out"), rows,
                         width, eps, c->stream);
  });
}

bool tysor_cuda_dispatch_rms_norm_gain_backward(void* context, void* input, void* gain, void* dy,
                                                void* dx, void* dgain, uint32_t rows,
                                                uint32_t width, float eps, bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    float* partial = scratch_floats(c, rms_gain_partial_elems(rows, width));
    launch_rms_norm_gain_backward(ptr_of(input, n, "input"), ptr_of(gain, width, "gain"), ptr_of(dy, n, "dy"),
                                  ptr_of(dx, n, "dx"), ptr_of(dgain, width, "dgain"), partial, rows, width,
                                  eps, accumulate, accumulate, c->stream);
  });
}

bool tysor_cuda_dispatch_cross_entropy_labels(void* context, void* logits, void* labels,
                                              void* out, uint32_t rows, uint32_t width) {
  return guarded([&] {
    Context* c = ctx_of(context);
    launch_cross_entropy_labels(ptr_of(logits, (size_t)rows * width, "logits"), ptr_of(labels, rows, "labels"),
                                ptr_of(out, rows, "out"), rows, width, c->d_err, c->stream);
  });
}

bool tysor_cuda_dispatch_cross_entropy_labels_backward(void* context, void* logits, void* labels,
                                                       void* grad, uint32_t rows, uint32_t width,
                                                       bool accumulate) {
  return guarded([&] {
    Context* c = ctx_of(context);
    const size_t n = (size_t)rows * width;
    launch_cross_entropy_labels_backward(ptr_of(logits, n, "logits"), ptr_of(labels, rows, "labels"),
                                         ptr_of(grad, n, "grad"), rows, width, accumulate, c->d_err,
                                         c->stream);
  });
}

bool tysor_cuda_dispatch_layer_norm(void* context, void* input, void* gain, void* bias, void* out,
                                    void* stats, uint32_t rows, uint32_t width, float eps) {
  return guarded([&] {
    Operands o(ctx_of(context));
    check_norm(width, eps);
    const size_t n = (size_t)rows * width;
    const float* x = o.in(input, n, "input");
    const float* g = o.in_or_null(gain, width, "gain");
    const float* b = o.in_or_null(bias, width, "bias");
    float* y = o.out(out, n, "out");
    float* s = o.out_or_null(stats, (size_t)rows * 2, "stats");
    o.check_overlap();
    launch_layer_norm(x, g, b, y, s, rows, width, eps, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_layer_norm_backward(void* context, void* input, void* gain, void* stats, void* dy,
                                             void* dx, void* dgain, void* dbias, uint32_t rows,
                                             uint32_t width, bool accumulate) {
  return guarded([&] {
    Operands o(ctx_of(context));
    check_norm(width, 0.0f);
    const size_t n = (size_t)rows * width;
    const float* x = o.in(input, n, "input");
    const float* g = o.in_or_null(gain, width, "gain");
    const float* s = o.in(stats, (size_t)rows * 2, "stats");
    const float* gy = o.in(dy, n, "dy");
    float* gx = o.out(dx, n, "dx");
    float* gg = o.out_or_null(dgain, width, "dgain");
    float* gb = o.out_or_null(dbias, width, "dbias");
    o.check_overlap();
    float* partial = scratch_floats(o.ctx, layer_norm_partial_elems(rows, width));
    launch_layer_norm_backward(x, g, s, gy, gx, gg, gb, partial, rows, width, accumulate, accumulate,
                               o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_rope_axes(void* context, void* input, void* positions, void* out, uint32_t batch,
                                   uint32_t heads, uint32_t seq_len, const int64_t* sections, int axes,
                                   double theta, bool seq_major) {
  return guarded([&] {
    rope_axes(context, input, positions, out, batch, heads, seq_len, sections, axes, theta, seq_major, false,
              false);
  });
}

bool tysor_cuda_dispatch_rope_axes_backward(void* context, void* grad, void* positions, void* dx,
                                            uint32_t batch, uint32_t heads, uint32_t seq_len,
                                            const int64_t* sections, int axes, double theta, bool seq_major,
                                            bool accumulate) {
  return guarded([&] {
    rope_axes(context, grad, positions, dx, batch, heads, seq_len, sections, axes, theta, seq_major, true,
              accumulate);
  });
}

bool tysor_cuda_dispatch_window_attention(void* context, void* q, void* k, void* v, void* starts,
                                          void* lengths, void* out, void* stats, uint32_t batch,
                                          uint32_t heads, uint32_t kv_heads, uint32_t q_len, uint32_t k_len,
                                          uint32_t head_dim, uint32_t window, uint32_t sinks, float scale,
                                          bool seq_major) {
  return guarded([&] {
    Operands o(ctx_of(context));
    AttentionShape s = attention_shape(batch, heads, kv_heads, q_len, k_len, head_dim, window, sinks, scale, seq_major);
    const size_t nq = elems({batch, heads, q_len, head_dim}), nk = elems({batch, kv_heads, k_len, head_dim});
    const float* qp = o.in(q, nq, "q");
    const float* kp = o.in(k, nk, "k");
    const float* vp = o.in(v, nk, "v");
    s.starts = o.in_or_null(starts, batch, "starts");
    s.lengths = o.in_or_null(lengths, batch, "lengths");
    float* op = o.out(out, nq, "out");
    float* sp = o.out_or_null(stats, elems({batch, heads, q_len, 2}), "stats");
    o.check_overlap();
    float* work = scratch_floats(o.ctx, window_attention_work_elems(s));
    launch_window_attention(s, qp, kp, vp, op, sp, work, o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_window_attention_backward(void* context, void* q, void* k, void* v, void* starts,
                                                   void* lengths, void* out, void* stats, void* dout,
                                                   void* dq, void* dk, void* dv, uint32_t batch,
                                                   uint32_t heads, uint32_t kv_heads, uint32_t q_len,
                                                   uint32_t k_len, uint32_t head_dim, uint32_t window,
                                                   uint32_t sinks, float scale, bool seq_major,
                                                   bool accumulate) {
  return guarded([&] {
    Operands o(ctx_of(context));
    AttentionShape s = attention_shape(batch, heads, kv_heads, q_len, k_len, head_dim, window, sinks, scale, seq_major);
    const size_t nq = elems({batch, heads, q_len, head_dim}), nk = elems({batch, kv_heads, k_len, head_dim});
    const float* qp = o.in(q, nq, "q");
    const float* kp = o.in(k, nk, "k");
    const float* vp = o.in(v, nk, "v");
    s.starts = o.in_or_null(starts, batch, "starts");
    s.lengths = o.in_or_null(lengths, batch, "lengths");
    const float* op = o.in(out, nq, "out");
    const float* sp = o.in(stats, elems({batch, heads, q_len, 2}), "stats");
    const float* gp = o.in(dout, nq, "dout");
    float* gq = o.out(dq, nq, "dq");
    float* gk = o.out(dk, nk, "dk");
    float* gv = o.out(dv, nk, "dv");
    o.check_overlap();
    float* work = scratch_floats(o.ctx, window_attention_backward_work_elems(s));
    launch_window_attention_backward(s, qp, kp, vp, op, sp, gp, gq, gk, gv, work, accumulate, accumulate, accumulate,
                                     o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_distill_loss(void* context, void* logits, void* ids, void* teacher, void* out,
                                      void* stats, uint32_t rows, uint32_t width, uint32_t top,
                                      float temperature) {
  return guarded([&] {
    Operands o(ctx_of(context));
    check_distill(width, top, temperature);
    const float* z = o.in(logits, (size_t)rows * width, "logits");
    const float* id = o.in(ids, (size_t)rows * top, "ids");
    const float* t = o.in(teacher, (size_t)rows * top, "teacher");
    float* l = o.out(out, rows, "out");
    float* s = o.out_or_null(stats, (size_t)rows * 2, "stats");
    o.check_overlap();
    launch_distill_loss(z, id, t, l, s, rows, width, (int)top, temperature, o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_distill_loss_backward(void* context, void* logits, void* ids, void* teacher,
                                               void* stats, void* dloss, void* grad, uint32_t rows,
                                               uint32_t width, uint32_t top, float temperature,
                                               bool accumulate) {
  return guarded([&] {
    Operands o(ctx_of(context));
    check_distill(width, top, temperature);
    const float* z = o.in(logits, (size_t)rows * width, "logits");
    const float* id = o.in(ids, (size_t)rows * top, "ids");
    const float* t = o.in(teacher, (size_t)rows * top, "teacher");
    const float* s = o.in(stats, (size_t)rows * 2, "stats");
    const float* d = o.in_or_null(dloss, rows, "dloss");
    float* g = o.out(grad, (size_t)rows * width, "grad");
    o.check_overlap();
    launch_distill_loss_backward(z, id, t, s, d, g, rows, width, (int)top, temperature, accumulate, o.ctx->d_err,
                                 o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_rotary(void* context, void* input, void* positions, void* out, uint32_t batch,
                                uint32_t heads, uint32_t seq_len, uint32_t head_dim, uint32_t rotary_dim,
                                bool interleaved, double theta, int scaling, double factor,
                                double original_len, double low, double high, double amplitude,
                                bool seq_major) {
  return guarded([&] {
    rotary(context, input, positions, out, batch, heads, seq_len, head_dim, rotary_dim, interleaved,
           {(int)(rotary_dim / 2), theta, scaling, factor, original_len, low, high}, amplitude, seq_major, false, false);
  });
}

bool tysor_cuda_dispatch_rotary_backward(void* context, void* grad, void* positions, void* dx, uint32_t batch,
                                         uint32_t heads, uint32_t seq_len, uint32_t head_dim,
                                         uint32_t rotary_dim, bool interleaved, double theta, int scaling,
                                         double factor, double original_len, double low, double high,
                                         double amplitude, bool seq_major, bool accumulate) {
  return guarded([&] {
    rotary(context, grad, positions, dx, batch, heads, seq_len, head_dim, rotary_dim, interleaved,
           {(int)(rotary_dim / 2), theta, scaling, factor, original_len, low, high}, amplitude, seq_major, true,
           accumulate);
  });
}

bool tysor_cuda_dispatch_decay_attention(void* context, void* q, void* k, void* v, void* decay, void* state,
                                         void* lengths, void* out, void* new_state, uint32_t batch,
                                         uint32_t heads, uint32_t kv_heads, uint32_t seq_len,
                                         uint32_t key_dim, uint32_t value_dim, float scale,
                                         bool seq_major) {
  return guarded([&] {
    Operands o(ctx_of(context));
    const DecayShape s = decay_shape(batch, heads, kv_heads, seq_len, key_dim, value_dim, scale, seq_major);
    const DecayInputs in = decay_inputs(o, s, q, k, v, decay, state, lengths);
    float* op = o.out(out, elems({batch, heads, seq_len, value_dim}), "out");
    float* np = o.out_or_null(new_state, elems({batch, heads, key_dim, value_dim}), "new_state");
    if (((uintptr_t)np & 15) != 0) throw CudaError("new_state buffer must start on a 16-byte boundary");
    o.check_overlap("new_state", "state");
    float* work = scratch_floats(o.ctx, decay_attention_work_elems(s));
    launch_decay_attention(s, in, op, np, work, o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_decay_attention_backward(void* context, void* q, void* k, void* v, void* decay,
                                                  void* state, void* lengths, void* dout, void* dnew_state,
                                                  void* dq, void* dk, void* dv, void* dstate, uint32_t batch,
                                                  uint32_t heads, uint32_t kv_heads, uint32_t seq_len,
                                                  uint32_t key_dim, uint32_t value_dim, float scale,
                                                  bool seq_major, bool accumulate) {
  return guarded([&] {
    Operands o(ctx_of(context));
    const DecayShape s = decay_shape(batch, heads, kv_heads, seq_len, key_dim, value_dim, scale, seq_major);
    const DecayInputs in = decay_inputs(o, s, q, k, v, decay, state, lengths);
    const size_t states = elems({batch, heads, key_dim, value_dim});
    const float* gp = o.in(dout, elems({batch, heads, seq_len, value_dim}), "dout");
    const float* gn = o.in_or_null(dnew_state, states, "dnew_state");
    float* gq = o.out(dq, elems({batch, heads, seq_len, key_dim}), "dq");
    float* gk = o.out(dk, elems({batch, kv_heads, seq_len, key_dim}), "dk");
    float* gv = o.out(dv, elems({batch, kv_heads, seq_len, value_dim}), "dv");
    float* gs = o.out_or_null(dstate, states, "dstate");
    if ((((uintptr_t)gn | (uintptr_t)gs) & 15) != 0)
      throw CudaError("dnew_state and dstate buffers must start on a 16-byte boundary");
    o.check_overlap();
    float* work = scratch_floats(o.ctx, decay_attention_backward_work_elems(s));
    launch_decay_attention_backward(s, in, gp, gn, gq, gk, gv, gs, work, accumulate, accumulate, accumulate, accumulate,
                                    o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_token_logprobs(void* context, void* logits, void* ids, void* out, void* entropy,
                                        void* top_ids, void* top_logprobs, void* stats, uint32_t rows,
                                        uint32_t width, uint32_t given, uint32_t top, float temperature) {
  return guarded([&] {
    Operands o(ctx_of(context));
    const LogprobShape s = logprob_shape(rows, width, given, top, temperature);
    const float* z = o.in(logits, elems({rows, width}), "logits");
    const float* id = given ? o.in(ids, elems({rows, given}), "ids") : nullptr;
    float* op = given ? o.out(out, elems({rows, given}), "out") : nullptr;
    float* ep = o.out_or_null(entropy, rows, "entropy");
    float* ti = top ? o.out(top_ids, elems({rows, top}), "top_ids") : nullptr;
    float* tl = top ? o.out(top_logprobs, elems({rows, top}), "top_logprobs") : nullptr;
    float* sp = o.out_or_null(stats, elems({rows, 2}), "stats");
    o.check_overlap();
    launch_token_logprobs(s, z, id, op, ep, ti, tl, sp, o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_token_logprobs_backward(void* context, void* logits, void* ids, void* stats,
                                                 void* entropy, void* dout, void* dentropy, void* grad,
                                                 uint32_t rows, uint32_t width, uint32_t given,
                                                 float temperature, bool accumulate) {
  return guarded([&] {
    Operands o(ctx_of(context));
    const LogprobShape s = logprob_shape(rows, width, given, 0, temperature);
    const float* z = o.in(logits, elems({rows, width}), "logits");
    const float* id = given && dout ? o.in(ids, elems({rows, given}), "ids") : nullptr;
    const float* sp = o.in(stats, elems({rows, 2}), "stats");
    const float* gp = given ? o.in_or_null(dout, elems({rows, given}), "dout") : nullptr;
    const float* gh = o.in_or_null(dentropy, rows, "dentropy");
    const float* ep = gh ? o.in(entropy, rows, "entropy") : nullptr;
    float* g = o.out(grad, elems({rows, width}), "grad");
    o.check_overlap();
    launch_token_logprobs_backward(s, z, id, sp, ep, gp, gh, g, accumulate, o.ctx->d_err, o.ctx->stream);
  });
}

bool tysor_cuda_dispatch_transpose(void* context, void* input, void* out, const int64_t* dims,
                                   int rank, int a, int b) {
  return guarded([&] {
    Context* c = ctx_of(context);
    if (rank < 1 || rank > 8 || a < 0 || b < 0 || a >= rank || b >= rank)
      throw CudaError("transpose axis out of range");
    size_t n = 1;
    for (int i = 0; i < rank; ++i) n *= (size_t)dims[i];
    launch_transpose(ptr_of(input, n, "input"), ptr_of(out, n, "out"), dims, rank, a < b ? a : b,
                     a < b ? b : a, 0, c->stream);
  });
}

}  // extern "C"
