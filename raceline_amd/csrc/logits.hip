// Adjustments of a row of logits before a token is chosen from it: penalties for tokens that
// were said already, biases, and a mask of the tokens that may follow. Stands between rl_head
// and rl_top_k_device.
#include "rlq_common.h"
#include "../../include/rlq.h"

namespace rlq {
namespace {

constexpr int kLogitThreads = 512, kLogitSpan = 4096, kLogitPer = kLogitSpan / kLogitThreads / 4, kMaxBiases = 1024;
constexpr int kTokenSteps = 4;   // tokens read ahead: 4 a thread and step

struct LogitArgs {
  const float *x;
  float *y;
  const int *tokens, *n_tokens, *n_prompt, *bias_ids;
  const float *repetition, *presence, *frequency, *bias;
  const uint32_t *allowed;
  int64_t x_stride, y_stride, token_stride, bias_stride, allowed_stride;
  int vocab, max_tokens, n_bias;
  int wide, wide_tokens;   // rows of logits (of tokens) start on 16 bytes
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

// One workgroup: a span of 4096 logits of one row. Every workgroup of a row reads all of the row's
// tokens (from L2 but for the first) and counts those that fall into its span with integer LDS
// atomics, whose order changes nothing; so the row needs neither a second launch nor counters in
// memory. A count is the tokens from n_prompt on in the low 31 bits; the top bit is set by the
// tokens before.
// Loads return in the order in which they were issued: biases and the first 8192 tokens come
// before the logits, four neighbours a thread and step, which arrive while the tokens are counted.
// Bound by HBM without tokens and biases (16 rows of 248,320 in 6.7 us), by the span that most of
// them fall into with them (8000 tokens and 200 biases a row 14.4 us, half of the tokens and a quarter of
// the biases in one span).
// Biases: an id may come twice. Its first entry (found by an integer atomic, whose order changes
// nothing) adds up all of its entries in list order, so the sum does not depend on which thread
// came first; the list is looked through only for ids that do come twice.
__global__ __launch_bounds__(kLogitThreads) void adjust_logits_kernel(LogitArgs a) {
  __shared__ uint32_t count[kLogitSpan];
  __shared__ uint32_t extra[kLogitSpan];   // while the biases are sorted out: n_bias - first entry; then their sum's bits
  __shared__ i32x4 ids[kMaxBiases / 4];
  __shared__ f32x4 biases[kMaxBiases / 4];
  const int row = blockIdx.y, v0 = blockIdx.x * kLogitSpan, tid = threadIdx.x;
  const int span = min(kLogitSpan, a.vocab - v0);
  const float *x = a.x + row * a.x_stride + v0;
  float *y = a.y + row * a.y_stride + v0;
  const int *tok = a.tokens + row * a.token_stride;
  const int n = a.max_tokens ? max(0, min(a.n_tokens ? a.n_tokens[row] : a.max_tokens, a.max_tokens)) : 0;
  const int made = a.n_prompt ? a.n_prompt[row] : 0, whole = a.wide_tokens ? n & ~3 : 0;
  int id0 = -1;
  float bias0 = 0.0f;
  if (tid < a.n_bias) {
    id0 = a.bias_ids[row * a.bias_stride + tid] - v0;
    bias0 = a.bias[row * a.bias_stride + tid];
  }
  i32x4 t0[kTokenSteps];
#pragma unroll
  for (int k = 0; k < kTokenSteps; ++k) {
    const int i = (k * kLogitThreads + tid) * 4;
    if (i < whole) t0[k] = *reinterpret_cast<const i32x4 *>(tok + i);
  }
  f32x4 l[kLogitPer];
  uint32_t bits[kLogitPer];
#pragma unroll
  for (int k = 0; k < kLogitPer; ++k) {
    const int v = (k * kLogitThreads + tid) * 4;
    bits[k] = ~0u;
    if (v >= span) continue;
    if (a.wide && v + 4 <= span) {
      l[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(x + v));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) l[k][e] = v + e < span ? x[v + e] : 0.0f;
    }
    if (a.allowed) bits[k] = a.allowed[row * a.allowed_stride + ((v0 + v) >> 5)] >> (v & 31);
  }
  if (n) {
    for (int i = tid; i < kLogitSpan / 4; i += kLogitThreads) reinterpret_cast<u32x4 *>(count)[i] = u32x4{0, 0, 0, 0};
  }
  if (a.n_bias) {
    for (int i = tid; i < kLogitSpan / 4; i += kLogitThreads) reinterpret_cast<u32x4 *>(extra)[i] = u32x4{0, 0, 0, 0};
  }
  if (n || a.n_bias) lds_barrier();
  for (int i = tid; i < ((a.n_bias + 3) & ~3); i += kLogitThreads) {
    const bool more = i >= kLogitThreads && i < a.n_bias;   // the first entry of a thread is there already
    int v = i < kLogitThreads ? id0 : more ? a.bias_ids[row * a.bias_stride + i] - v0 : -1;
    if (v >= span) v = -1;
    reinterpret_cast<int *>(ids)[i] = max(v, -1);
    reinterpret_cast<float *>(biases)[i] = i < kLogitThreads ? bias0 : more ? a.bias[row * a.bias_stride + i] : 0.0f;
    if (v >= 0) atomicMax(&extra[v], (uint32_t)(a.n_bias - i));
  }
  if (n) {
    auto add = [&](int i, int t) {
      const uint32_t v = (uint32_t)t - (uint32_t)v0;
      if (v >= (uint32_t)span) return;
      if (i >= made) atomicAdd(&count[v], 1u);
      else atomicOr(&count[v], 0x80000000u);
    };
#pragma unroll
    for (int k = 0; k < kTokenSteps; ++k) {
      const int i = (k * kLogitThreads + tid) * 4;
      if (i >= whole) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) add(i + e, t0[k][e]);
    }
#pragma unroll 4
    for (int i = (kTokenSteps * kLogitThreads + tid) * 4; i < whole; i += kLogitThreads * 4) {
      const i32x4 t = *reinterpret_cast<const i32x4 *>(tok + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) add(i + e, t[e]);
    }
#pragma unroll 4
    for (int i = whole + tid; i < n; i += kLogitThreads) add(i, tok[i]);
  }
  if (a.n_bias) {
    lds_barrier();
    for (int i = tid; i < a.n_bias; i += kLogitThreads) {
      const int v = reinterpret_cast<const int *>(ids)[i];
      if (v >= 0 && (extra[v] & 0xFFFFu) != (uint32_t)(a.n_bias - i)) {
        atomicOr(&extra[v], 0x80000000u);           // the id comes twice
        reinterpret_cast<int *>(ids)[i] = -2 - v;   // still v's, and not its first
      }
    }
    lds_barrier();
    for (int i = tid; i < a.n_bias; i += kLogitThreads) {
      const int v = reinterpret_cast<const int *>(ids)[i];
      if (v < 0) continue;
      float sum = reinterpret_cast<const float *>(biases)[i];
      if (extra[v] >> 31) {
        for (int j = i / 4; j < (a.n_bias + 3) / 4; ++j) {
          const i32x4 id = ids[j];
          const f32x4 b = biases[j];
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += id[e] == -2 - v ? b[e] : 0.0f;
        }
      }
      extra[v] = __float_as_uint(sum);
    }
  }
  if (n || a.n_bias) lds_barrier();
  const float rep = a.repetition ? a.repetition[row] : 1.0f, pres = a.presence ? a.presence[row] : 0.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;
#pragma unroll
  for (int k = 0; k < kLogitPer; ++k) {
    const int v = (k * kLogitThreads + tid) * 4;
    if (v >= span) continue;
    if (n) {
      const u32x4 c = *reinterpret_cast<const u32x4 *>(count + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!c[e]) continue;
        l[k][e] = l[k][e] > 0.0f ? l[k][e] / rep : l[k][e] * rep;
        const uint32_t made = c[e] & 0x7FFFFFFFu;
        if (made) l[k][e] = l[k][e] - freq * (float)made - pres;
      }
    }
    if (a.n_bias) l[k] += __builtin_bit_cast(f32x4, *reinterpret_cast<const u32x4 *>(extra + v));
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(bits[k] >> e & 1u)) l[k][e] = -__builtin_inff();
    if (a.wide && v + 4 <= span) {
      *reinterpret_cast<f32x4 *>(y + v) = l[k];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v + e < span) y[v + e] = l[k][e];
    }
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
                   stride, out_stride, token_stride, bias_stride, allowed_stride, vocab, max_tokens, n_bias,
                   rlq::aligned(logits, 16) && rlq::aligned(out, 16) && stride % 4 == 0 && out_stride % 4 == 0,
                   rlq::aligned(tokens, 16) && token_stride % 4 == 0};
  const dim3 grid((unsigned)((vocab + rlq::kLogitSpan - 1) / rlq::kLogitSpan), (unsigned)rows);
  rlq::adjust_logits_kernel<<<grid, rlq::kLogitThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}
