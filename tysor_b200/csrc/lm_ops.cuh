// Language-model operators without a counterpart in the reference: layer
// norm, rotary positions over several axes, distillation from a teacher's top
// logits (lm_ops.cu), sliding-window attention with sinks (attention.cu), rotary
// positions on part of a head (rotary.cu), linear attention with decay (decay.cu)
// and log probabilities of given tokens (logprobs.cu).
// All fp32.  Gradients are the formulas' own (not the reference's shortened
// backward rules).  Each launcher enqueues on `st` and returns immediately.
#pragma once

#include "common.cuh"

namespace tysor {

// y = (x - mean) * rstd * gain + bias per row, rstd = 1 / sqrt(var + eps) with
// the population variance.  gain and bias may be null (1 and 0); stats, if not
// null, receives [rows][2] = (mean, rstd).
void launch_layer_norm(const float* x, const float* gain, const float* bias, float* y, float* stats, int64_t rows,
                       int64_t width, float eps, cudaStream_t st);
// With n = (x - mean) * rstd and g = dy * gain:
//   dx    (+)= rstd * (g - mean(g) - n * mean(g * n))
//   dgain (+)= column sums of dy * n,   dbias (+)= column sums of dy.
// dgain and dbias may be null.  `partial` needs
// layer_norm_partial_elems(rows, width) floats.
int64_t layer_norm_partial_elems(int64_t rows, int64_t width);
void launch_layer_norm_backward(const float* x, const float* gain, const float* stats, const float* dy, float* dx,
                                float* dgain, float* dbias, float* partial, int64_t rows, int64_t width,
                                int accumulate_dx, int accumulate_params, cudaStream_t st);

// Rotary positions over up to kMaxRopeAxes axes.  Pair i of `half` (elements
// i and half + i of a head) turns by positions[b][axis(i)][s] * rates[i]
// revolutions, axis(i) the axis whose section holds i; `ends[a]` is the end of
// axis a's section.  x is [batch][heads][seq][2 half], or [batch][seq][heads]
// [2 half] with seq_major.  `back` turns the other way (the gradient).
constexpr int kMaxRopeAxes = 8;
struct RopeAxes {
  int batch, heads, seq, half;
  int axes;
  int ends[kMaxRopeAxes];
  int seq_major;
};
void launch_rope_axes(const float* x, const float* positions, const double* rates, float* out, const RopeAxes& shape,
                      int back, int accumulate, cudaStream_t st);

// Distillation from a teacher's best `top` logits per row.  With p the
// softmax of the teacher's entries / T and q the softmax of the row's logits /
// T over the whole width:
//   loss = T^2 * sum_e p_e * (ln p_e - ln q[id_e])
//   grad (+)= dloss * T * (q - sum_e p_e [id_e])       (0 for an empty row)
// An id below 0 is an absent entry; a row without an entry has loss 0.  An id
// not below `width` or NaN sets *err (kErrIndexRange) and counts as absent.
// stats receives [rows][2] = (max logit, sum of exp((logit - max) / T)); the
// gradient reads it.  dloss null: 1 for every row.
constexpr int kMaxDistillTop = 1024;
// Temperatures for which 1 / T and T^2 are far from the ends of fp32.
inline bool distill_temperature(float t) { return t >= 0x1p-60f && t <= 0x1p60f; }
void launch_distill_loss(const float* logits, const float* ids, const float* teacher, float* loss, float* stats,
                         int64_t rows, int64_t width, int top, float temperature, int* err, cudaStream_t st);
void launch_distill_loss_backward(const float* logits, const float* ids, const float* teacher, const float* stats,
                                  const float* dloss, float* grad, int64_t rows, int64_t width, int top,
                                  float temperature, int accumulate, int* err, cudaStream_t st);

// Causal attention over a sliding window and the first keys.  Query row r of
// sequence b stands at p = starts[b] + r; with n = lengths[b] it sees key j if
//   0 <= p < n,  j <= p  and  (window == 0 or p - j < window or j < sinks).
// out = softmax(scale * q.k) . v over the keys it sees (0 for a row that sees
// none).  q and out are [batch][heads][q_len][head_dim], k and v
// [batch][kv_heads][k_len][head_dim] (heads / kv_heads query heads share a key
// head), or with seq_major [batch][len][heads][head_dim].  starts null:
// k_len - q_len; lengths null: k_len.  A length outside [0, k_len] or a start
// that is no number sets *err (kErrSequence); its sequence counts as empty.
constexpr int kMaxHeadDim = 128;
struct AttentionShape {
  int batch, heads, kv_heads, q_len, k_len, head_dim;
  int window, sinks;
  float scale;
  int seq_major;
  const float* starts;
  const float* lengths;
};
// stats (may be null) receives [batch][heads][q_len][2]: the row's greatest
// visible scale * q.k and the sum of exp(score - greatest); (-inf, 0) for a
// row that sees nothing.
void launch_window_attention(const AttentionShape& s, const float* q, const float* k, const float* v, float* out,
                             float* stats, float* work, int* err, cudaStream_t st);
int64_t window_attention_work_elems(const AttentionShape& s);
// Exact gradients: with P the probabilities and dP = dout.v^T,
//   dv (+)= P^T.dout,  dS = P * (dP - rowsum(dout * out)),
//   dq (+)= scale * dS.k,  dk (+)= scale * dS^T.q,
// dk and dv summed over the query heads that share a key head.
void launch_window_attention_backward(const AttentionShape& s, const float* q, const float* k, const float* v,
                                      const float* out, const float* stats, const float* dout, float* dq, float* dk,
                                      float* dv, float* work, int accumulate_q, int accumulate_k, int accumulate_v,
                                      int* err, cudaStream_t st);
int64_t window_attention_backward_work_elems(const AttentionShape& s);

// Rotary positions on the first 2 * half values of each head of `head_dim`: pair
// i turns by positions[b][s] * rates[i] revolutions and grows by `amplitude`;
// the rest is copied.  Pair i is (i, half + i), or (2 i, 2 i + 1) if
// interleaved.  positions null: 0, 1, 2, ...  x is [batch][heads][seq][head_dim],
// or [batch][seq][heads][head_dim] with seq_major.  `back` turns the other way.
constexpr int kMaxRotaryPairs = 256;
struct RotaryShape {
  int batch, heads, seq, head_dim, half;
  int interleaved, seq_major;
  float amplitude;
  double rates[kMaxRotaryPairs];
};
// How the rates of long contexts are scaled: none, all, or by how often a pair
// turns over the context trained on (include/tysor_cuda.h).
enum RotaryScaling : int { kRotaryPlain = 0, kRotaryLinear = 1, kRotaryTurns = 2, kRotaryLogTurns = 3 };
struct RotaryRates {
  int half;
  double theta;
  int scaling;
  double factor, context, low, high;
  bool operator==(const RotaryRates&) const = default;
};
// Null, or what is wrong with them.
const char* rotary_rates_problem(const RotaryRates& r, double amplitude);
void rotary_fill_rates(const RotaryRates& r, double* rates);
void launch_rotary(const float* x, const float* positions, float* out, const RotaryShape& shape, int back,
                   int accumulate, cudaStream_t st);

// Linear attention with a decay for each head.  With a = exp(-decay[h]) and S_0
// the given state, or 0:
//   S_t = a S_(t-1) + k_t v_t^T,   out_t = scale * q_t S_t     (t = 1 .. n)
// and S_n the new state.  q and k are [batch][heads or kv_heads][seq][key_dim],
// v and out [..][seq][value_dim] (with seq_major [batch][seq][heads][dim]), states
// [batch][heads][key_dim][value_dim].  lengths null: n = seq.  A length outside
// [0, seq] sets *err (kErrSequence, the sequence then counts as empty), a decay
// below 0 or NaN kErrDecay (and counts as 0).
struct DecayShape {
  int batch, heads, kv_heads, seq, key_dim, value_dim;
  float scale;
  int seq_major;
};
// Null, or what is wrong with a shape.
const char* decay_attention_problem(uint64_t batch, uint64_t heads, uint64_t kv_heads, uint64_t seq, uint64_t key_dim,
                                    uint64_t value_dim, float scale);
struct DecayInputs {
  const float *q, *k, *v, *decay, *state, *lengths;
};
// new_state may be `state`.
void launch_decay_attention(const DecayShape& s, const DecayInputs& in, float* out, float* new_state, float* work,
                            int* err, cudaStream_t st);
int64_t decay_attention_work_elems(const DecayShape& s);
// With E_n = dnew_state + scale q_n dout_n^T, E_t = a E_(t+1) + scale q_t dout_t^T:
//   dq_t (+)= scale * dout_t S_t^T,  dk_t (+)= v_t E_t^T,  dv_t (+)= k_t E_t,  dstate (+)= a E_1.
void launch_decay_attention_backward(const DecayShape& s, const DecayInputs& in, const float* dout,
                                     const float* dnew_state, float* dq, float* dk, float* dv, float* dstate,
                                     float* work, int accumulate_q, int accumulate_k, int accumulate_v,
                                     int accumulate_state, int* err, cudaStream_t st);
int64_t decay_attention_backward_work_elems(const DecayShape& s);

// Log probabilities under the softmax of a row's logits / T: of the row's `given`
// ids (an id below 0 is absent: 0), the distribution's entropy, and the `top` most
// probable tokens in order (equal ones by id) with theirs; id -1 and -inf where no
// token of probability above 0 is left.  A row that holds nothing but -inf has log
// probabilities -inf and entropy 0; one with NaN or +inf NaN (and no best tokens).
// An id not below `width` or NaN sets *err (kErrIndexRange) and counts as absent.
// stats receives [rows][2] = (greatest logit, sum of exp((logit - greatest) / T)).
constexpr int kMaxGivenTokens = 128, kMaxTopTokens = 128, kMaxLogprobWidth = 1 << 24;
struct LogprobShape {
  int64_t rows;
  int width, given, top;
  float temperature;
};
void launch_token_logprobs(const LogprobShape& s, const float* logits, const float* ids, float* out, float* entropy,
                           float* top_ids, float* top_logprobs, float* stats, int* err, cudaStream_t st);
// With p the probabilities and H the entropy:
//   grad (+)= (1 / T) (sum over given of dout ([id] - p) - dentropy * p (ln p + H)).
// dout null: 0 for all; dentropy null: 0.  Rows of nothing but -inf have gradient 0.
void launch_token_logprobs_backward(const LogprobShape& s, const float* logits, const float* ids, const float* stats,
                                    const float* entropy, const float* dout, const float* dentropy, float* grad,
                                    int accumulate, int* err, cudaStream_t st);

}  // namespace tysor
