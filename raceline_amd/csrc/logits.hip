// Adjustments of a row of logits before a token is chosen from it: penalties for tokens that
// were said already, biases, and a mask of the tokens that may follow. Stands between rl_head
// and rl_top_k_device.
#include "rlq_common.h"
#include "../../include/rlq.h"

namespace rlq {
namespace {

constexpr int kLogitThreads = 256, kLogitSpan = 4096, kMaxBiases = 1024;

struct LogitArgs {
  const float *x;
  float *y;
  const int *tokens, *n_tokens, *n_prompt, *bias_ids;
  const float *repetition, *presence, *frequency, *bias;
  const uint32_t *allowed;
  int64_t x_stride, y_stride, token_stride, bias_stride, allowed_stride;
  int vocab, max_tokens, n_bias;
};

// One workgroup: a span of 4096 logits of one row. Every workgroup of a row reads all of the
// row's tokens (from L2 but for the first) and counts those that fall into its span with integer
// LDS atomics, whose order changes nothing; so the row needs neither a second launch nor counters
// in memory. A count is the tokens at and past n_prompt in the low 31 bits, and in the top bit
// whether any token of the row is this one.
// Biases: an id may come twice; the first entry of an id adds all of its entries, in list order,
// so the sum does not depend on which thread came first.
__global__ __launch_bounds__(kLogitThreads) void adjust_logits_kernel(LogitArgs a) {
  __shared__ uint32_t count[kLogitSpan];
  __shared__ float extra[kLogitSpan];
  __shared__ int ids[kMaxBiases];
  const int row = blockIdx.y, v0 = blockIdx.x * kLogitSpan, tid = threadIdx.x;
  const int span = min(kLogitSpan, a.vocab - v0);
  for (int i = tid; i < kLogitSpan; i += kLogitThreads) {
    count[i] = 0;
    extra[i] = 0.0f;
  }
  if (a.n_bias) {
    for (int i = tid; i < a.n_bias; i += kLogitThreads) ids[i] = a.bias_ids[row * a.bias_stride + i] - v0;
  }
  __syncthreads();
  if (a.max_tokens) {
    const int n = max(0, min(a.n_tokens ? a.n_tokens[row] : a.max_tokens, a.max_tokens));
    const int made = a.n_prompt ? a.n_prompt[row] : 0;
    const int *tok = a.tokens + row * a.token_stride;
    for (int i = tid; i < n; i += kLogitThreads) {
      const uint32_t v = (uint32_t)tok[i] - (uint32_t)v0;
      if (v < (uint32_t)span) {
        atomicOr(&count[v], 0x80000000u);
        if (i >= made) atomicAdd(&count[v], 1u);
      }
    }
  }
  for (int i = tid; i < a.n_bias; i += kLogitThreads) {
    const int v = ids[i];
    if (v < 0 || v >= span) continue;
    bool first = true;
    for (int j = 0; j < i; ++j) first = first && ids[j] != v;
    if (!first) continue;
    float sum = 0.0f;
    for (int j = i; j < a.n_bias; ++j)
      if (ids[j] == v) sum += a.bias[row * a.bias_stride + j];
    extra[v] = sum;
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : 1.0f, pres = a.presence ? a.presence[row] : 0.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;
  const float *x = a.x + row * a.x_stride + v0;
  float *y = a.y + row * a.y_stride + v0;
  for (int i = tid; i < span; i += kLogitThreads) {
    float l = x[i];
    const uint32_t c = count[i];
    if (c) {
      l = l > 0.0f ? l / rep : l * rep;
      const uint32_t made = c & 0x7FFFFFFFu;
      if (made) l = l - freq * (float)made - pres;
    }
    l += extra[i];
    if (a.allowed) {
      const int v = v0 + i;
      if (!(a.allowed[row * a.allowed_stride + (v >> 5)] >> (v & 31) & 1u)) l = -__builtin_inff();
    }
    y[i] = l;
  }
}

}  // namespace
}  // namespace rlq

extern "C" int rlq_adjust_logits(const float *logits, int64_t stride, int rows, int vocab, const int *tokens,
                                 int64_t token_stride, int max_tokens, const int *n_tokens, const int *n_prompt,
                                 const float *repetition, const float *presence, const float *frequency,
                                 const int *bias_ids, const float *bias, int n_bias, int64_t bias_stride,
                                 const uint32_t *allowed, int64_t allowed_stride, float *out, int64_t out_stride,
                                 void *stream) {
  RLQ_REQUIRE(rows >= 0 && rows <= 65535 && vocab >= 0 && max_tokens >= 0,
              "rlq_adjust_logits: rows=%d, vocab=%d, max_tokens=%d", rows, vocab, max_tokens);
  RLQ_REQUIRE(n_bias >= 0 && n_bias <= rlq::kMaxBiases, "rlq_adjust_logits: n_bias=%d is not in 0 .. %d", n_bias,
              rlq::kMaxBiases);
  if (rows == 0 || vocab == 0) return 0;
  RLQ_REQUIRE(logits && out, "rlq_adjust_logits: null pointer");
  RLQ_REQUIRE(stride >= vocab && out_stride >= vocab, "rlq_adjust_logits: row strides (%lld, %lld) < %d logits",
              (long long)stride, (long long)out_stride, vocab);
  RLQ_REQUIRE(max_tokens == 0 || (tokens && token_stride >= 0), "rlq_adjust_logits: null tokens");
  RLQ_REQUIRE(n_bias == 0 || (bias_ids && bias && bias_stride >= 0), "rlq_adjust_logits: null biases");
  RLQ_REQUIRE(!allowed || allowed_stride == 0 || allowed_stride >= ((int64_t)vocab + 31) / 32,
              "rlq_adjust_logits: a mask row of %lld words is shorter than the vocabulary", (long long)allowed_stride);
  rlq::LogitArgs a{logits, out, tokens, n_tokens, n_prompt, bias_ids, repetition, presence, frequency, bias, allowed,
                   stride, out_stride, token_stride, bias_stride, allowed_stride, vocab, max_tokens, n_bias};
  const dim3 grid((unsigned)((vocab + rlq::kLogitSpan - 1) / rlq::kLogitSpan), (unsigned)rows);
  rlq::adjust_logits_kernel<<<grid, rlq::kLogitThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}
