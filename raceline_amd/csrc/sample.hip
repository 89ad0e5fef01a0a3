// A token from each row of logits, by temperature, top-k, top-p and min-p and a random number given for
// the row: what follows rl_head and rlq_adjust_logits where the most likely token is not simply taken.
#include "rlq_common.h"
#include "../../include/rlq.h"

namespace rlq {
namespace {

constexpr int kSampleThreads = 1024, kSampleTile = 4 * kSampleThreads, kMaxVocab = 1 << 22;
constexpr int kMaxTiles = kMaxVocab / kSampleTile;

struct SampleArgs {
  const float *logits;
  int64_t stride;
  const double *uniform;
  const float *temperature, *top_p, *min_p;
  const int *top_k;
  int *tokens;
  float *probs;
  int vocab, shift;   // weights are held in steps of 2^-shift of the largest
};

// Logits in their order as whole numbers; both zeros are one, NaN lies below -inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr uint32_t kNothing = 0x007FFFFFu;   // order_of(-inf)

__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7FFFFFFFu : ~key);
}

// The weight of a logit, exp((x - top) / T), in 64 bits, and rounded to steps of 2^-shift: sums of the steps
// are whole numbers, so they depend neither on the order of the sums nor on how a row is cut. With
// 2^18 tokens a step is 2^-44 of the largest weight.
struct Weight {
  double top, inverse;
  float top_logit;
  int shift;
  __device__ double operator()(float x) const {
    if (x == top_logit) return 1.0;
    const double below = static_cast<double>(x) - top;     // -inf beside an infinite top too
    return below > -__builtin_inf() ? exp(below * inverse) : 0.0;
  }
  __device__ uint64_t steps(double w) const { return static_cast<uint64_t>(rint(ldexp(w, shift))); }
};

template <typename V>
__device__ V block_sum(V x, V *scratch) {
  for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  V sum = 0;
  for (int i = 0; i < kSampleThreads / 64; ++i) sum += scratch[i];
  return sum;
}

// One workgroup a row. The kept tokens are a prefix of the row in the order of its logits (equal ones by
// index), told by a logit and how many of those equal to it are kept; a search by digits of eight bits finds it,
// with counts for top-k and with weights for top-p.
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ unsigned long long hist[256], scratch[kSampleThreads / 64], tile_sum[kMaxTiles];
  __shared__ int tile_equal[kMaxTiles];
  __shared__ unsigned long long found_sum, found_left;
  __shared__ uint32_t found_key;
  const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
  const float *x = a.logits + row * a.stride;

  uint32_t most = 0;
  for (int i = tid; i < V; i += kSampleThreads) most = max(most, order_of(x[i]));
  for (int off = 32; off; off >>= 1) most = max(most, __shfl_xor(most, off));
  if ((tid & 63) == 0) scratch[tid >> 6] = most;
  __syncthreads();
  for (int i = 0; i < kSampleThreads / 64; ++i) most = max(most, (uint32_t)scratch[i]);
  if (most <= kNothing) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = 0.0f;
    }
    return;
  }
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  const bool greedy = !(t > 0.0f);
  Weight weight;
  weight.top_logit = logit_of(most), weight.top = weight.top_logit, weight.shift = a.shift;
  weight.inverse = greedy ? 1.0 : 1.0 / static_cast<double>(t);
  int k = greedy ? 1 : a.top_k ? a.top_k[row] : 0;
  if (k <= 0 || k > V) k = V;
  const float p = a.top_p ? fminf(fmaxf(a.top_p[row], 0.0f), 1.0f) : 1.0f;   // NaN: 0 .. below
  const bool all_p = a.top_p ? !(a.top_p[row] < 1.0f) : true;
  const double least = a.min_p && a.min_p[row] > 0.0f ? fminf(a.min_p[row], 1.0f) : 0.0;

  // The smallest prefix whose measure (a count, or steps of weight) reaches `target`: sets found_key, and
  // found_left: what the tokens equal to it have to give.
  auto search = [&](uint64_t target, uint32_t floor, bool by_weight) {
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kSampleThreads) {
        const uint32_t key = order_of(x[i]);
        if (key < floor || (shift < 24 && key >> (shift + 8) != prefix)) continue;
        const uint64_t w = by_weight ? weight.steps(weight(x[i])) : 1;
        if (w) atomicAdd(&hist[key >> shift & 255], (unsigned long long)w);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        for (; d > 0 && above + hist[d] < target; --d) above += hist[d];
        found_key = d, found_sum = above;
      }
      __syncthreads();
      prefix = prefix << 8 | found_key;
      above = found_sum;
    }
    __syncthreads();
    if (tid == 0) found_key = prefix, found_left = target - above;
    __syncthreads();
  };

  uint32_t cut = 0;      // kept: keys above, and the first `equal` of those equal to it
  uint64_t equal = 0;
  if (k < V) {
    search(k, 0, false);
    cut = found_key, equal = found_left;
  }
  if (!all_p) {
    uint64_t sum = 0;
    for (int i = tid; i < V; i += kSampleThreads)
      if (order_of(x[i]) > cut) sum += weight.steps(weight(x[i]));
    sum = block_sum(sum, reinterpret_cast<uint64_t *>(scratch));
    if (equal) sum += equal * weight.steps(weight(logit_of(cut)));
    const uint64_t target = max((uint64_t)1, (uint64_t)ceil(p * static_cast<double>(sum)));
    search(target, cut, true);
    const uint64_t each = weight.steps(weight(logit_of(found_key)));
    const uint64_t need = (found_left + each - 1) / each;
    if (found_key != cut || need < equal) equal = need;
    cut = found_key;
  }

  // steps of the kept tokens, tile by tile
  const int tiles = (V + kSampleTile - 1) / kSampleTile;
  auto kept_steps = [&](uint32_t key) -> uint64_t {
    if (key <= kNothing) return 0;
    const double w = weight(logit_of(key));
    return w >= least ? weight.steps(w) : 0;
  };
  const uint64_t each = equal ? kept_steps(cut) : 0;
  for (int tile = 0; tile < tiles; ++tile) {
    uint64_t sum = 0;
    int same = 0;
    for (int i = tile * kSampleTile + tid; i < min(V, (tile + 1) * kSampleTile); i += kSampleThreads) {
      const uint32_t key = order_of(x[i]);
      if (key > cut) sum += kept_steps(key);
      same += key == cut;
    }
    sum = block_sum(sum, reinterpret_cast<uint64_t *>(scratch));
    same = block_sum(same, reinterpret_cast<int *>(scratch));
    if (tid == 0) tile_sum[tile] = sum, tile_equal[tile] = same;
  }
  __syncthreads();
  uint64_t total = 0, seen = 0;
  for (int tile = 0; tile < tiles; ++tile) {
    const uint64_t same = min((uint64_t)tile_equal[tile], equal - min(equal, seen));
    total += tile_sum[tile] + same * each;
    seen += tile_equal[tile];
  }
  const double u = fmin(fmax(a.uniform[row], 0.0), 1.0);
  const uint64_t mark = min(total - 1, (uint64_t)(u * static_cast<double>(total)));
  uint64_t before = 0;
  seen = 0;
  int tile = 0;
  for (;; ++tile) {
    const uint64_t same = min((uint64_t)tile_equal[tile], equal - min(equal, seen));
    const uint64_t sum = tile_sum[tile] + same * each;
    if (before + sum > mark || tile == tiles - 1) break;
    before += sum;
    seen += tile_equal[tile];
  }
  // inside the tile: four neighbouring tokens a thread
  const int i0 = tile * kSampleTile + tid * 4;
  uint32_t key[4];
  int same = 0;
  for (int e = 0; e < 4; ++e) {
    key[e] = i0 + e < V ? order_of(x[i0 + e]) : 0;
    same += i0 + e < V && key[e] == cut;
  }
  auto scan = [&](auto mine) {     // sum over the threads in front
    auto upto = mine;
    for (int off = 1; off < 64; off <<= 1) {
      const auto o = __shfl_up(upto, off);
      if ((tid & 63) >= off) upto += o;
    }
    __syncthreads();
    if ((tid & 63) == 63) scratch[tid >> 6] = upto;
    __syncthreads();
    for (int w = 0; w < tid >> 6; ++w) upto += scratch[w];
    return upto - mine;
  };
  uint64_t rank = seen + scan((unsigned long long)same), mine[4], sum = 0;
  for (int e = 0; e < 4; ++e) {
    mine[e] = i0 + e < V && key[e] > cut ? kept_steps(key[e]) : 0;
    if (i0 + e < V && key[e] == cut) mine[e] = rank++ < equal ? each : 0;
    sum += mine[e];
  }
  uint64_t at = before + scan((unsigned long long)sum);
  for (int e = 0; e < 4; ++e) {
    if (at <= mark && mark < at + mine[e]) {
      a.tokens[row] = i0 + e;
      if (a.probs) a.probs[row] = static_cast<float>(static_cast<double>(mine[e]) / static_cast<double>(total));
    }
    at += mine[e];
  }
}

}  // namespace
}  // namespace rlq

extern "C" {

size_t rlq_sample_workspace_bytes(int rows, int vocab) {
  return 0;
}

int rlq_sample(const float *logits, int64_t stride, int rows, int vocab, const double *uniform,
               const float *temperature, const int *top_k, const float *top_p, const float *min_p, int *tokens,
               float *probs, void *workspace, size_t workspace_bytes, void *stream) {
  RLQ_REQUIRE(rows >= 0 && rows <= 65535, "rlq_sample: rows=%d is not in 0 .. 65535", rows);
  RLQ_REQUIRE(vocab >= 1 && vocab <= rlq::kMaxVocab, "rlq_sample: vocab=%d is not in 1 .. %d", vocab, rlq::kMaxVocab);
  if (rows == 0) return 0;
  RLQ_REQUIRE(logits && uniform && tokens, "rlq_sample: null pointer");
  RLQ_REQUIRE(stride >= vocab, "rlq_sample: row stride %lld < %d logits", (long long)stride, vocab);
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  rlq::SampleArgs a{logits, stride, uniform, temperature, top_p, min_p, top_k, tokens, probs, vocab, 62 - bits};
  rlq::sample_row_kernel<<<rows, rlq::kSampleThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}

}  // extern "C"
