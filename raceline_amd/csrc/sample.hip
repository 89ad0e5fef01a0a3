// A token from each row of logits, by temperature, top-k, top-p and min-p and a random number given for
// the row: what follows rl_head and rlq_adjust_logits where the most likely token is not simply taken.
//
// The kept tokens are a prefix of the row in the falling order of its logits, equal ones by index; the
// choice goes through them in order of index. Weights are whole numbers (steps of 2^-44 of the largest), so
// that every sum below is exact and depends neither on the order of its terms nor on how the row is cut.
// Four launches, in which a row's tiles of 4096 logits go side by side:
//   top      the largest logit of each tile;
//   bins     counts and weights of the row in 1024 bins by the distance from the largest logit, 32 a factor
//            of e; what lies past the last one weighs nothing;
//   gather   the bins that hold the cuts of top-k and top-p; the weights of what is surely kept, by tile, and
//            the tokens of those bins, as a list;
//   choose   the cut inside the list, the tile in which the weights reach the number, and the token there.
#include "rlq_common.h"
#include "../../include/rlq.h"

#include <algorithm>

namespace rlq {
namespace {

constexpr int kSampleThreads = 1024, kSampleTile = 4 * kSampleThreads, kMaxVocab = 1 << 22;
constexpr int kMaxTiles = kMaxVocab / kSampleTile, kBins = kSampleThreads, kBinsPer = 32;
constexpr int kDigit = 11, kDigits = 1 << kDigit;

struct SampleArgs {
  const float *logits;
  int64_t stride;
  const double *uniform;
  const float *temperature, *top_p, *min_p;
  const int *top_k;
  int *tokens;
  float *probs;
  int vocab, tiles, shift, wide;   // weights are held in steps of 2^-shift of the largest
  char *scratch;
};

// A row's scratch.
struct RowScratch {
  uint64_t *tile_sum, *bin_sum;
  uint32_t *tile_top, *bin_count, *listed, *list;
};

__host__ __device__ inline int64_t row_bytes(int vocab, int tiles) {
  return ((int64_t)tiles * 12 + kBins * 12 + 16 + (int64_t)vocab * 4 + 15) / 16 * 16;
}

__device__ __forceinline__ RowScratch row_scratch(const SampleArgs &a, int row) {
  char *at = a.scratch + row * row_bytes(a.vocab, a.tiles);
  RowScratch r;
  r.tile_sum = reinterpret_cast<uint64_t *>(at);
  r.bin_sum = r.tile_sum + a.tiles;
  r.tile_top = reinterpret_cast<uint32_t *>(r.bin_sum + kBins);
  r.bin_count = r.tile_top + a.tiles;
  r.listed = r.bin_count + kBins;
  r.list = r.listed + 4;
  return r;
}

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

// A token's place in the row's order: larger comes first.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int token) {
  return static_cast<uint64_t>(key) << 32 | ~static_cast<uint32_t>(token);
}

// What a row asks for.
struct Filter {
  double top, inverse, least, unit;   // unit: 2^shift
  float top_logit, p;
  int k;
  bool by_count, by_weight;

  // exp((x - top) / T)
  __device__ double weight(uint32_t key) const {
    const float x = logit_of(key);
    if (x == top_logit) return 1.0;
    const double below = static_cast<double>(x) - top;     // -inf beside an infinite top too
    return below > -__builtin_inf() ? exp(below * inverse) : 0.0;
  }
  __device__ uint64_t steps(double w) const { return static_cast<uint64_t>(rint(w * unit)); }
  __device__ uint64_t kept_steps(uint32_t key) const {
    const double w = weight(key);
    return w >= least ? steps(w) : 0;
  }
  // Falls as the logit rises, in every step of its rounding. The last bin begins at e^-31.97, a quarter of a
  // step of 2^-44.
  __device__ int bin(uint32_t key) const {
    const float x = logit_of(key);
    if (key <= kNothing) return kBins - 1;
    if (x == top_logit) return 0;
    const double d = (top - static_cast<double>(x)) * inverse * kBinsPer;
    return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
  }
};

__device__ __forceinline__ Filter filter_of(const SampleArgs &a, int row, uint32_t most) {
  Filter f;
  const float t = a.temperature ? a.temperature[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f;
  const float m = a.min_p ? a.min_p[row] : 0.0f;
  const int k = !(t > 0.0f) ? 1 : a.top_k ? a.top_k[row] : 0;
  f.top_logit = logit_of(most), f.top = f.top_logit, f.unit = static_cast<double>((uint64_t)1 << a.shift);
  f.inverse = t > 0.0f ? 1.0 / static_cast<double>(t) : 1.0;
  f.by_count = k > 0 && k < a.vocab, f.k = f.by_count ? k : a.vocab;
  f.by_weight = p < 1.0f, f.p = fmaxf(p, 0.0f);
  f.least = m > 0.0f ? fminf(m, 1.0f) : 0.0;
  return f;
}

// A thread's four neighbouring logits of a tile, in their order; 0 behind the row.
__device__ __forceinline__ void load_keys(const SampleArgs &a, int row, int i0, uint32_t (&key)[4]) {
  const float *x = a.logits + row * a.stride + i0;
  if (a.wide && i0 + 4 <= a.vocab) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(x);
#pragma unroll
    for (int e = 0; e < 4; ++e) key[e] = order_of(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) key[e] = i0 + e < a.vocab ? order_of(x[e]) : 0;
  }
}

template <typename V>
__device__ __forceinline__ V wave_sum(V x) {
#pragma unroll
  for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

// Sum over the threads up to this one. Begins and ends with a barrier.
template <typename V>
__device__ __forceinline__ V scan_block(V x, V *scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const V o = __shfl_up(x, off);
    if (lane >= off) x += o;
  }
  __syncthreads();
  if (lane == 63) scratch[wave] = x;
  __syncthreads();
  V t = lane < kSampleThreads / 64 ? scratch[lane] : 0;
  V front = lane < wave ? t : 0;
  front = wave_sum(front);
  __syncthreads();
  return x + front;
}

__device__ __forceinline__ uint32_t top_of_row(const RowScratch &s, int tiles) {
  uint32_t most = 0;
  for (int i = threadIdx.x & 63; i < tiles; i += 64) most = max(most, s.tile_top[i]);
#pragma unroll
  for (int off = 32; off; off >>= 1) most = max(most, __shfl_xor(most, off));
  return most;
}

__global__ __launch_bounds__(kSampleThreads) void sample_top_kernel(SampleArgs a) {
  __shared__ uint32_t waves[kSampleThreads / 64];
  const int row = blockIdx.y, tid = threadIdx.x;
  const RowScratch s = row_scratch(a, row);
  for (int i = blockIdx.x * kSampleThreads + tid; i < kBins; i += gridDim.x * kSampleThreads) s.bin_sum[i] = 0, s.bin_count[i] = 0;
  if (blockIdx.x == 0 && tid == 0) *s.listed = 0;
  uint32_t key[4];
  load_keys(a, row, blockIdx.x * kSampleTile + tid * 4, key);
  uint32_t most = max(max(key[0], key[1]), max(key[2], key[3]));
#pragma unroll
  for (int off = 32; off; off >>= 1) most = max(most, __shfl_xor(most, off));
  if ((tid & 63) == 0) waves[tid >> 6] = most;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSampleThreads / 64; ++i) most = max(most, waves[i]);
    s.tile_top[blockIdx.x] = most;
  }
}

__global__ __launch_bounds__(kSampleThreads) void sample_bins_kernel(SampleArgs a) {
  __shared__ unsigned long long sums[kBins];
  __shared__ uint32_t counts[kBins];
  const int row = blockIdx.y, tid = threadIdx.x;
  const RowScratch s = row_scratch(a, row);
  uint32_t key[4];
  load_keys(a, row, blockIdx.x * kSampleTile + tid * 4, key);
  const uint32_t most = top_of_row(s, a.tiles);
  const Filter f = filter_of(a, row, most);
  if (most <= kNothing || !(f.by_count || f.by_weight)) return;
  sums[tid] = 0, counts[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int bin = f.bin(key[e]);
    if (bin == kBins - 1) continue;
    atomicAdd(&sums[bin], static_cast<unsigned long long>(f.steps(f.weight(key[e]))));
    atomicAdd(&counts[bin], 1u);
  }
  __syncthreads();
  if (counts[tid]) {
    atomicAdd(reinterpret_cast<unsigned long long *>(s.bin_sum) + tid, sums[tid]);
    atomicAdd(s.bin_count + tid, counts[tid]);
  }
}

// Where the cuts lie, from the bins: the same in every thread.
struct Cuts {
  int count_bin;              // that of top-k's last token; kBins: none
  int first, last;            // those that can hold top-p's last token; without top-p: top-k's
  uint64_t before_count, sum_before_count;   // tokens and weight in front of count_bin
  uint64_t sum_before_first, sum;            // weight in front of `first`, and of all bins
  __device__ bool listed(int bin) const { return (bin >= first && bin <= last) || bin == count_bin; }
};

__device__ __forceinline__ uint64_t share_of(float p, uint64_t sum) {
  return max((uint64_t)1, static_cast<uint64_t>(ceil(p * static_cast<double>(sum))));
}

__device__ Cuts find_cuts(const Filter &f, const RowScratch &s) {
  __shared__ unsigned long long scratch[kSampleThreads / 64], shared[6];
  const int tid = threadIdx.x;
  const uint64_t count = s.bin_count[tid], sum = s.bin_sum[tid];
  const uint64_t upto = scan_block<unsigned long long>(count, scratch), sums = scan_block<unsigned long long>(sum, scratch);
  if (tid == kBins - 1) shared[0] = kBins, shared[1] = 0, shared[2] = sums, shared[3] = sums, shared[4] = shared[5] = kBins;
  __syncthreads();
  if (f.by_count && upto >= (uint64_t)f.k && upto - count < (uint64_t)f.k)
    shared[0] = tid, shared[1] = upto - count, shared[2] = sums - sum, shared[3] = sums;
  __syncthreads();
  Cuts c;
  c.count_bin = (int)shared[0], c.before_count = shared[1], c.sum_before_count = shared[2], c.sum = sums;
  c.first = c.last = c.count_bin;
  if (f.by_weight) {
    const uint64_t low = share_of(f.p, shared[2]), high = share_of(f.p, shared[3]);
    if (sums >= low && sums - sum < low) shared[4] = tid;
    if (sums >= high && sums - sum < high) shared[5] = tid;
    __syncthreads();
    c.first = (int)shared[4], c.last = (int)shared[5];
  }
  __syncthreads();
  if (tid == 0) shared[0] = 0;
  __syncthreads();
  if (tid == c.first) shared[0] = sums - sum;
  if (tid == kBins - 1) shared[1] = sums;
  __syncthreads();
  c.sum_before_first = shared[0], c.sum = shared[1];
  return c;
}

__global__ __launch_bounds__(kSampleThreads) void sample_gather_kernel(SampleArgs a) {
  __shared__ unsigned long long waves[kSampleThreads / 64];
  __shared__ uint32_t found, place;
  const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * kSampleTile + tid * 4;
  const RowScratch s = row_scratch(a, row);
  uint32_t key[4];
  load_keys(a, row, i0, key);
  const uint32_t most = top_of_row(s, a.tiles);
  if (most <= kNothing) return;
  const Filter f = filter_of(a, row, most);
  if (tid == 0) found = 0;
  Cuts c;
  c.first = c.last = c.count_bin = kBins;
  if (f.by_count || f.by_weight) c = find_cuts(f, s);
  else __syncthreads();
  uint64_t sum = 0;
  uint32_t at[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int bin = f.bin(key[e]);
    at[e] = ~0u;
    if (bin == kBins - 1) continue;
    if (c.listed(bin)) at[e] = atomicAdd(&found, 1u);
    else if (bin < c.first) sum += f.kept_steps(key[e]);
  }
  sum = wave_sum(sum);
  if ((tid & 63) == 0) waves[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSampleThreads / 64; ++i) sum += waves[i];
    s.tile_sum[blockIdx.x] = sum;
    if (found) place = atomicAdd(s.listed, found);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (at[e] != ~0u) s.list[place + at[e]] = i0 + e;
}

// Of the list's tokens that `take` admits, the place of the last one of the shortest prefix that measures
// `target` (steps of weight, or tokens): by digits of eleven bits, from the top.
template <bool WEIGHT, typename Take>
__device__ uint64_t cut_list(const SampleArgs &a, int row, const Filter &f, const uint32_t *list, int n, uint64_t target,
                             unsigned long long *hist, unsigned long long *scratch, Take take) {
  __shared__ unsigned long long found[2];
  const int tid = threadIdx.x;
  const float *x = a.logits + row * a.stride;
  uint64_t prefix = 0;
  for (int shift = 55; shift >= 0; shift -= kDigit) {   // 64 bits: six digits, the first of nine bits
    hist[tid] = 0, hist[tid + kSampleThreads] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const uint32_t key = order_of(x[list[i]]);
      const uint64_t at = place_of(key, list[i]);
      if ((shift < 55 && at >> (shift + kDigit) != prefix) || !take(key, at)) continue;
      const uint64_t w = WEIGHT ? f.steps(f.weight(key)) : 1;
      atomicAdd(&hist[at >> shift & (kDigits - 1)], static_cast<unsigned long long>(w));
    }
    __syncthreads();
    // from the largest digit down, two a thread
    const int d = kDigits - 1 - 2 * tid;
    const uint64_t one = hist[d], two = hist[d - 1];
    const uint64_t upto = scan_block<unsigned long long>(one + two, scratch);
    const uint64_t before = upto - one - two;
    if (before < target && upto >= target) {
      const bool first = before + one >= target;
      found[0] = first ? d : d - 1;
      found[1] = target - before - (first ? 0 : one);
    }
    __syncthreads();
    prefix = prefix << kDigit | found[0];
    target = found[1];
    __syncthreads();
  }
  return prefix;
}

__global__ __launch_bounds__(kSampleThreads) void sample_choose_kernel(SampleArgs a) {
  __shared__ unsigned long long tile_sum[kMaxTiles], hist[kDigits], scratch[kSampleThreads / 64], chosen[2];
  const int row = blockIdx.x, tid = threadIdx.x;
  const RowScratch s = row_scratch(a, row);
  const uint32_t most = top_of_row(s, a.tiles);
  if (most <= kNothing) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = 0.0f;
    }
    return;
  }
  const Filter f = filter_of(a, row, most);
  const float *x = a.logits + row * a.stride;
  const int n = *s.listed;
  uint64_t cut = 0;        // kept: what lies here or in front
  if (f.by_count || f.by_weight) {
    const Cuts c = find_cuts(f, s);
    uint64_t sum = c.sum;
    if (c.count_bin < kBins) {
      cut = cut_list<false>(a, row, f, s.list, n, f.k - c.before_count, hist, scratch,
                            [&](uint32_t key, uint64_t) { return f.bin(key) == c.count_bin; });
      if (f.by_weight) {
        uint64_t part = 0;
        for (int i = tid; i < n; i += kSampleThreads) {
          const uint32_t key = order_of(x[s.list[i]]);
          if (f.bin(key) == c.count_bin && place_of(key, s.list[i]) >= cut) part += f.steps(f.weight(key));
        }
        const uint64_t upto = scan_block<unsigned long long>(part, scratch);
        if (tid == kSampleThreads - 1) chosen[0] = upto;
        __syncthreads();
        sum = c.sum_before_count + chosen[0];
      }
    }
    if (f.by_weight) {
      const uint64_t least = cut;
      cut = cut_list<true>(a, row, f, s.list, n, share_of(f.p, sum) - c.sum_before_first, hist, scratch,
                           [&](uint32_t key, uint64_t at) {
                             const int bin = f.bin(key);
                             return at >= least && bin >= c.first && bin <= c.last;
                           });
    }
  }
  for (int i = tid; i < a.tiles; i += kSampleThreads) tile_sum[i] = s.tile_sum[i];
  __syncthreads();
  for (int i = tid; i < n; i += kSampleThreads) {
    const uint32_t key = order_of(x[s.list[i]]);
    if (place_of(key, s.list[i]) < cut) continue;
    const uint64_t w = f.kept_steps(key);
    if (w) atomicAdd(&tile_sum[s.list[i] / kSampleTile], static_cast<unsigned long long>(w));
  }
  __syncthreads();
  const uint64_t mine = tid < a.tiles ? tile_sum[tid] : 0;
  const uint64_t upto = scan_block<unsigned long long>(mine, scratch);
  if (tid == kSampleThreads - 1) chosen[0] = upto;
  __syncthreads();
  const uint64_t total = chosen[0];
  const double u = fmin(fmax(a.uniform[row], 0.0), 1.0);
  const uint64_t mark = min(total - 1, static_cast<uint64_t>(u * static_cast<double>(total)));
  __syncthreads();
  if (upto > mark && upto - mine <= mark) chosen[0] = tid, chosen[1] = upto - mine;
  __syncthreads();
  const int i0 = static_cast<int>(chosen[0]) * kSampleTile + tid * 4;
  uint32_t key[4];
  load_keys(a, row, i0, key);
  uint64_t each[4], sum = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    each[e] = key[e] > kNothing && place_of(key[e], i0 + e) >= cut ? f.kept_steps(key[e]) : 0;
    sum += each[e];
  }
  uint64_t at = chosen[1] + scan_block<unsigned long long>(sum, scratch) - sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (at <= mark && mark < at + each[e]) {
      a.tokens[row] = i0 + e;
      if (a.probs) a.probs[row] = static_cast<float>(static_cast<double>(each[e]) / static_cast<double>(total));
    }
    at += each[e];
  }
}

}  // namespace
}  // namespace rlq

extern "C" {

size_t rlq_sample_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > rlq::kMaxVocab) return 0;
  return (size_t)rows * rlq::row_bytes(vocab, (vocab + rlq::kSampleTile - 1) / rlq::kSampleTile);
}

int rlq_sample(const float *logits, int64_t stride, int rows, int vocab, const double *uniform,
               const float *temperature, const int *top_k, const float *top_p, const float *min_p, int *tokens,
               float *probs, void *workspace, size_t workspace_bytes, void *stream) {
  RLQ_REQUIRE(rows >= 0 && rows <= 65535, "rlq_sample: rows=%d is not in 0 .. 65535", rows);
  RLQ_REQUIRE(vocab >= 1 && vocab <= rlq::kMaxVocab, "rlq_sample: vocab=%d is not in 1 .. %d", vocab, rlq::kMaxVocab);
  if (rows == 0) return 0;
  RLQ_REQUIRE(logits && uniform && tokens, "rlq_sample: null pointer");
  RLQ_REQUIRE(stride >= vocab, "rlq_sample: row stride %lld < %d logits", (long long)stride, vocab);
  const size_t need = rlq_sample_workspace_bytes(rows, vocab);
  RLQ_REQUIRE(workspace && rlq::aligned(workspace, 16) && workspace_bytes >= need,
              "rlq_sample: needs %zu bytes of 16-byte aligned workspace, got %zu", need, workspace_bytes);
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  const int tiles = (vocab + rlq::kSampleTile - 1) / rlq::kSampleTile;
  rlq::SampleArgs a{logits, stride, uniform, temperature, top_p, min_p, top_k, tokens, probs, vocab, tiles,
                    std::min(44, 62 - bits), rlq::aligned(logits, 16) && stride % 4 == 0, static_cast<char *>(workspace)};
  const dim3 grid((unsigned)tiles, (unsigned)rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  rlq::sample_top_kernel<<<grid, rlq::kSampleThreads, 0, st>>>(a);
  RLQ_HIP(hipGetLastError());
  if (top_k || top_p || temperature) {
    rlq::sample_bins_kernel<<<grid, rlq::kSampleThreads, 0, st>>>(a);
    RLQ_HIP(hipGetLastError());
  }
  rlq::sample_gather_kernel<<<grid, rlq::kSampleThreads, 0, st>>>(a);
  RLQ_HIP(hipGetLastError());
  rlq::sample_choose_kernel<<<rows, rlq::kSampleThreads, 0, st>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}

}  // extern "C"
