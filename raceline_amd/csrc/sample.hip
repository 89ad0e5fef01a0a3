// A token from each row of logits, by temperature, top-k, top-p and min-p and a random number given for
// the row: what follows rl_head and rlq_adjust_logits where the most likely token is not simply taken.
//
// The kept tokens are a prefix of the row in the falling order of its logits, equal ones by index; the
// choice goes through them in order of index. Weights are whole numbers (steps of 2^-44 of the largest), so
// that every sum below is exact and depends neither on the order of its terms nor on how the row is cut.
// Four launches, in which a row's tiles of 8192 logits go side by side:
//   top      the largest logit of each tile;
//   bins     counts and weights of the row in 1024 bins by the distance from the largest logit, 32 a factor
//            of e; what lies past the last one weighs nothing;
//   gather   the bins that hold the cuts of top-k and top-p; the weights of what is surely kept, by tile, and
//            the tokens of those bins, as a list;
//   choose   the cut inside the list, the tile in which the weights reach the number, and the token there.
// Small calls are bound by the four launches and the chain of scans and barriers in the last (one row of 248320: 30 us,
// of which top 2.8, bins 7.8, gather 7.7, choose 11.6), large ones by the VALU: 64-bit weights, 16 rows under top-p
// 44.7 us, 45 rows under min-p 34.6 (45 MB; VALU share of gather 0.69). Rows that ask for nothing take 21 us, a temperature alone 23,
// temperature 0 28 (one row each). The list is short where logits spread as a model's do; where a cut lies among many alike one
// workgroup goes through all of them again and again: a constant row of 248320 1.4 ms, a normal one of spread 0.025 0.7 ms, 16 of them the same.
// Tiles of 4096 were slower in all but one row (16 rows 54 for 50, 45 rows 42 for 38, one row 31 for 33, before the weights' series).
#include "lanes.h"
#include "../../include/rlq.h"

#include <algorithm>

namespace rlq {
namespace {

constexpr int kSampleThreads = 1024, kPer = 8, kSampleTile = kPer * kSampleThreads, kMaxVocab = 1 << 22;
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

__device__ __forceinline__ void add(uint64_t *p, uint64_t x) { atomicAdd(reinterpret_cast<unsigned long long *>(p), static_cast<unsigned long long>(x)); }

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
constexpr double kNoStep = -46.0;            // 2^-46 is a quarter of a step at most: rounds to none

__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7FFFFFFFu : ~key);
}

// A token's place in the row's order: larger comes first.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int token) {
  return static_cast<uint64_t>(key) << 32 | ~static_cast<uint32_t>(token);
}

// What a row asks for.
//
// Weights, exp((x - top) / T) = 2^d with d = (x - top) log2(e) / T: d = n + j/16 + r with |r| <= 1/32, so 2^d is
// 2^n times an entry of a table times the series of e^(r ln 2) to its sixth power, whose next term lies below
// 2^-55. Off by a few 2^-53, where a step is 2^-44; a third of the operations of a 64-bit exponential
// with its special cases.
struct Filter {
  double top, inverse, least, least_exponent, unit;   // surely below `least` under least_exponent; inverse: log2(e) / T; unit: 2^shift
  float top_logit, p;
  int k;
  bool by_count, by_weight;

  // d, or where that is nothing -inf
  __device__ double exponent(uint32_t key) const {
    const float x = logit_of(key);
    if (x == top_logit) return 0.0;
    const double below = static_cast<double>(x) - top;     // -inf beside an infinite top too
    return below > -__builtin_inf() ? below * inverse : below;
  }
  __device__ double weight_of(double d, const double *table) const {
    if (!(d > -1000.0)) return 0.0;
    const double m = rint(d * 16.0), r = (d - m * 0.0625) * 0.6931471805599453;
    const int i = static_cast<int>(m);
    double e = 1.0 / 720;
    e = __builtin_fma(e, r, 1.0 / 120);
    e = __builtin_fma(e, r, 1.0 / 24);
    e = __builtin_fma(e, r, 1.0 / 6);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    return ldexp(table[i & 15] * e, i >> 4);
  }
  __device__ uint64_t steps(double w) const { return static_cast<uint64_t>(rint(w * unit)); }
  __device__ uint64_t steps_of(uint32_t key, const double *table) const { return steps(weight_of(exponent(key), table)); }
  __device__ uint64_t kept_steps(uint32_t key, const double *table) const {
    const double d = exponent(key);
    if (d < least_exponent) return 0;
    const double w = weight_of(d, table);
    return w >= least ? steps(w) : 0;
  }
  // Falls as the logit rises, in every step of its rounding. The last bin begins at 2^-46.1, a quarter of a step
  // of 2^-44.
  __device__ int bin(uint32_t key) const {
    if (key <= kNothing) return kBins - 1;
    const double d = exponent(key) * -(kBinsPer * 0.6931471805599453);
    return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
  }
};

// 2^(j/16).
__constant__ double kSixteenths[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0};

// What top-k asks for (a temperature of 0: one token), 0 for all.
__device__ __forceinline__ int count_of(const SampleArgs &a, int row) {
  const int k = a.temperature && !(a.temperature[row] > 0.0f) ? 1 : a.top_k ? a.top_k[row] : 0;
  return k > 0 && k < a.vocab ? k : 0;
}

__device__ __forceinline__ Filter filter_of(const SampleArgs &a, int row, uint32_t most) {
  Filter f;
  const float t = a.temperature ? a.temperature[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f;
  const float m = a.min_p ? a.min_p[row] : 0.0f;
  const int k = count_of(a, row);
  f.top_logit = logit_of(most), f.top = f.top_logit, f.unit = static_cast<double>((uint64_t)1 << a.shift);
  f.inverse = 1.4426950408889634 / (t > 0.0f ? static_cast<double>(t) : 1.0);
  f.by_count = k > 0, f.k = k;
  f.by_weight = p < 1.0f, f.p = fmaxf(p, 0.0f);
  f.least = m > 0.0f ? fminf(m, 1.0f) : 0.0;
  f.least_exponent = m > 0.0f ? fmax(static_cast<double>(__log2f(fminf(m, 1.0f))) - 1e-4, kNoStep) : kNoStep;
  return f;
}

// A thread's eight neighbouring logits of a tile, in their order; 0 behind the row.
__device__ __forceinline__ void load_keys(const SampleArgs &a, int row, int i0, uint32_t (&key)[kPer]) {
  const float *x = a.logits + row * a.stride + i0;
  if (a.wide && i0 + kPer <= a.vocab) {
#pragma unroll
    for (int e = 0; e < kPer; e += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4 *>(x + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) key[e + i] = order_of(v[i]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) key[e] = i0 + e < a.vocab ? order_of(x[e]) : 0;
  }
}

// Sum over the threads up to this one. Begins and ends with a barrier.
template <typename V>
__device__ __forceinline__ V scan_block(V x, V *scratch) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  x = scan_wave(x);
  lds_barrier();
  if (lane == 63) scratch[wave] = x;
  lds_barrier();
  const V waves = scan_wave<V>(lane < kSampleThreads / 64 ? scratch[lane] : 0);
  lds_barrier();
  return wave ? x + of_lane(waves, wave - 1) : x;
}

__device__ __forceinline__ uint32_t top_of_row(const RowScratch &s, int tiles) {
  uint32_t most = 0;
  for (int i = threadIdx.x & 63; i < tiles; i += 64) most = max(most, s.tile_top[i]);
  return most_of_wave(most);
}

// What a row asks for, formed by one wave for the workgroup, and the table; a barrier has to follow.
__device__ __forceinline__ void set_up(const SampleArgs &a, const RowScratch &s, int row, Filter *f, double *table, uint32_t *most) {
  if (threadIdx.x < 64) {
    const uint32_t top = top_of_row(s, a.tiles);
    const Filter x = filter_of(a, row, top);
    if (threadIdx.x == 0) *f = x, *most = top;
  }
  if (threadIdx.x >= 64 && threadIdx.x < 80) table[threadIdx.x - 64] = kSixteenths[threadIdx.x - 64];
}

__global__ __launch_bounds__(kSampleThreads) void sample_top_kernel(SampleArgs a) {
  __shared__ uint32_t waves[kSampleThreads / 64];
  const int row = blockIdx.y, tid = threadIdx.x;
  const RowScratch s = row_scratch(a, row);
  for (int i = blockIdx.x * kSampleThreads + tid; i < kBins; i += gridDim.x * kSampleThreads) s.bin_sum[i] = 0, s.bin_count[i] = 0;
  if (blockIdx.x == 0 && tid == 0) *s.listed = 0;
  uint32_t key[kPer];
  load_keys(a, row, blockIdx.x * kSampleTile + tid * kPer, key);
  uint32_t most = key[0];
#pragma unroll
  for (int e = 1; e < kPer; ++e) most = max(most, key[e]);
  most = most_of_wave(most);
  if ((tid & 63) == 0) waves[tid >> 6] = most;
  lds_barrier();
  if (tid < 64) {
    most = most_of_wave(tid < kSampleThreads / 64 ? waves[tid] : 0);
    if (tid == 0) s.tile_top[blockIdx.x] = most;
  }
}

__global__ __launch_bounds__(kSampleThreads) void sample_bins_kernel(SampleArgs a) {
  __shared__ uint64_t sums[kBins];
  __shared__ uint32_t counts[kBins], most;
  __shared__ double table[16];
  __shared__ Filter f;
  const int row = blockIdx.y, tid = threadIdx.x;
  if (!count_of(a, row) && !(a.top_p && a.top_p[row] < 1.0f)) return;      // nothing is cut
  const RowScratch s = row_scratch(a, row);
  uint32_t key[kPer];
  load_keys(a, row, blockIdx.x * kSampleTile + tid * kPer, key);
  set_up(a, s, row, &f, table, &most);
  sums[tid] = 0, counts[tid] = 0;
  lds_barrier();
  if (most <= kNothing) return;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int bin = f.bin(key[e]);
    if (bin == kBins - 1) continue;
    if (f.by_weight) add(&sums[bin], f.steps_of(key[e], table));
    if (f.by_count) atomicAdd(&counts[bin], 1u);
  }
  lds_barrier();
  if (sums[tid]) add(s.bin_sum + tid, sums[tid]);
  if (counts[tid]) atomicAdd(s.bin_count + tid, counts[tid]);
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

// count and sum: those of the thread's bin.
__device__ Cuts find_cuts(const Filter &f, uint64_t count, uint64_t sum) {
  __shared__ uint64_t scratch[kSampleThreads / 64], shared[6];
  const int tid = threadIdx.x;
  const uint64_t upto = scan_block<uint64_t>(count, scratch), sums = scan_block<uint64_t>(sum, scratch);
  if (tid == kBins - 1) shared[0] = kBins, shared[1] = 0, shared[2] = sums, shared[3] = sums, shared[4] = shared[5] = kBins;
  lds_barrier();
  if (f.by_count && upto >= (uint64_t)f.k && upto - count < (uint64_t)f.k)
    shared[0] = tid, shared[1] = upto - count, shared[2] = sums - sum, shared[3] = sums;
  lds_barrier();
  Cuts c;
  c.count_bin = (int)shared[0], c.before_count = shared[1], c.sum_before_count = shared[2], c.sum = sums;
  c.first = c.last = c.count_bin;
  if (f.by_weight) {
    const uint64_t low = share_of(f.p, shared[2]), high = share_of(f.p, shared[3]);
    if (sums >= low && sums - sum < low) shared[4] = tid;
    if (sums >= high && sums - sum < high) shared[5] = tid;
    lds_barrier();
    c.first = (int)shared[4], c.last = (int)shared[5];
  }
  lds_barrier();
  if (tid == 0) shared[0] = 0;
  lds_barrier();
  if (tid == c.first) shared[0] = sums - sum;
  if (tid == kBins - 1) shared[1] = sums;
  lds_barrier();
  c.sum_before_first = shared[0], c.sum = shared[1];
  return c;
}

__global__ __launch_bounds__(kSampleThreads) void sample_gather_kernel(SampleArgs a) {
  __shared__ uint64_t waves[kSampleThreads / 64];
  __shared__ uint32_t found, place, most;
  __shared__ double table[16];
  __shared__ Filter f;
  const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * kSampleTile + tid * kPer;
  const RowScratch s = row_scratch(a, row);
  uint32_t key[kPer];
  load_keys(a, row, i0, key);
  const uint64_t bin_count = s.bin_count[tid], bin_sum = s.bin_sum[tid];
  set_up(a, s, row, &f, table, &most);
  if (tid == 0) found = 0;
  lds_barrier();
  if (most <= kNothing) return;
  Cuts c;
  c.first = c.last = c.count_bin = kBins;
  if (f.by_count || f.by_weight) c = find_cuts(f, bin_count, bin_sum);
  uint64_t sum = 0;
  uint32_t at[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) at[e] = ~0u;
  if (c.first == kBins) {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (key[e] > kNothing) sum += f.kept_steps(key[e], table);
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int bin = f.bin(key[e]);
      if (bin == kBins - 1) continue;
      if (c.listed(bin)) at[e] = atomicAdd(&found, 1u);
      else if (bin < c.first) sum += f.kept_steps(key[e], table);
    }
  }
  sum = sum_wave(sum);
  if ((tid & 63) == 0) waves[tid >> 6] = sum;
  lds_barrier();
  if (tid < 64) {
    sum = sum_wave<uint64_t>(tid < kSampleThreads / 64 ? waves[tid] : 0);
    if (tid == 0) {
      s.tile_sum[blockIdx.x] = sum;
      if (found) place = atomicAdd(s.listed, found);
    }
  }
  lds_barrier();
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    if (at[e] != ~0u) s.list[place + at[e]] = i0 + e;
}

// A thread's tokens of the list: those of one round of kListed, in registers where the list is no longer.
constexpr int kEach = 4, kListed = kEach * kSampleThreads;

struct Listed {
  uint64_t place[kEach], steps[kEach];   // place 0: none
  int bin[kEach], token[kEach];
  uint32_t key[kEach];
};

// The tokens and their logits; their weights need the row's filter.
__device__ __forceinline__ void load_tokens(const SampleArgs &a, const RowScratch &s, int row, int round, int n, Listed &x) {
  const float *logits = a.logits + row * a.stride;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = round * kListed + e * kSampleThreads + threadIdx.x;
    x.token[e] = static_cast<int>(s.list[min(i, a.vocab - 1)]);         // asked for beside n
    if (i >= n) x.token[e] = -1;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) x.key[e] = x.token[e] >= 0 ? order_of(logits[x.token[e]]) : 0;
}

__device__ __forceinline__ void weigh(const Filter &f, const double *table, Listed &x) {
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    x.place[e] = x.steps[e] = 0, x.bin[e] = kBins;
    if (x.token[e] < 0) continue;
    x.place[e] = place_of(x.key[e], x.token[e]);
    x.steps[e] = f.steps_of(x.key[e], table);
    x.bin[e] = f.bin(x.key[e]);
  }
}

// Of the list's tokens in bins first .. last and not behind `from`, the place of the last one of the shortest prefix
// that measures `target` (steps of weight, or tokens). By digits of eleven bits, from the highest in which
// two of them differ, until one token is left.
template <bool WEIGHT, typename Load>
__device__ uint64_t cut_list(Load load, Listed &x, int rounds, int first, int last, uint64_t from, uint64_t target,
                             uint64_t *hist, uint64_t *scratch) {
  __shared__ uint64_t found[4];
  const int tid = threadIdx.x;
  auto taken = [&](int e) { return x.place[e] && x.bin[e] >= first && x.bin[e] <= last && x.place[e] >= from; };
  if (tid == 0) found[0] = found[2] = found[3] = 0;
  lds_barrier();
  uint32_t high = 0, low = 0;              // of the logits; low: the largest complement
  int count = 0;
  for (int round = 0; round < rounds; ++round) {
    if (rounds > 1) load(round);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const bool one = taken(e);
      count += __popcll(__ballot(one));
      if (!one) continue;
      high = max(high, x.key[e]), low = max(low, ~x.key[e]);
      found[1] = x.place[e];
    }
  }
  high = most_of_wave(high), low = most_of_wave(low);
  if ((tid & 63) == 0 && count) {
    atomicMax(reinterpret_cast<uint32_t *>(&found[2]), low);
    atomicMax(reinterpret_cast<uint32_t *>(&found[3]), high);
    add(&found[0], count);
  }
  lds_barrier();
  if (found[0] == 1) return found[1];      // a bin of its own, as the likeliest tokens have
  low = ~static_cast<uint32_t>(found[2]), high = static_cast<uint32_t>(found[3]);
  int open = 32 + (low == high ? 0 : 32 - __builtin_clz(low ^ high));     // bits that are not known
  uint64_t prefix = static_cast<uint64_t>(high) << 32;
  prefix = open < 64 ? prefix >> open : 0;
  lds_barrier();
  while (open) {
    const int width = min(open, kDigit), shift = open - width;
    hist[tid] = 0, hist[tid + kSampleThreads] = 0;
    if (tid == 0) found[2] = 0;
    lds_barrier();
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load(round);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (!taken(e) || (open < 64 && x.place[e] >> open != prefix)) continue;
        add(&hist[x.place[e] >> shift & ((1u << width) - 1)], WEIGHT ? x.steps[e] : 1);
      }
    }
    lds_barrier();
    // from the largest digit down, two a thread
    const int d = kDigits - 1 - 2 * tid;
    const uint64_t one = hist[d], two = hist[d - 1];
    const uint64_t upto = scan_block<uint64_t>(one + two, scratch), before = upto - one - two;
    if (before < target && upto >= target) {
      const bool in_one = before + one >= target;
      found[0] = in_one ? d : d - 1;
      found[1] = target - before - (in_one ? 0 : one);
    }
    lds_barrier();
    prefix = prefix << width | found[0];
    target = found[1];
    open = shift;
    if (open) {      // one token left is the one
      for (int round = 0; round < rounds; ++round) {
        if (rounds > 1) load(round);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (taken(e) && x.place[e] >> open == prefix) {
            add(&found[2], 1);
            found[3] = x.place[e];
          }
      }
      lds_barrier();
      if (found[2] == 1) return found[3];
    }
    lds_barrier();
  }
  return prefix;
}

__global__ __launch_bounds__(kSampleThreads) void sample_choose_kernel(SampleArgs a) {
  __shared__ uint64_t tile_sum[kMaxTiles], hist[kDigits], scratch[kSampleThreads / 64], chosen[2];
  __shared__ double table[16];
  __shared__ Filter f;
  __shared__ uint32_t most;
  const int row = blockIdx.x, tid = threadIdx.x;
  const RowScratch s = row_scratch(a, row);
  const uint64_t bin_count = s.bin_count[tid], bin_sum = s.bin_sum[tid];
  const int n = *s.listed, rounds = (n + kListed - 1) / kListed;
  Listed x;
  load_tokens(a, s, row, 0, n, x);
  set_up(a, s, row, &f, table, &most);
  for (int i = tid; i < a.tiles; i += kSampleThreads) tile_sum[i] = s.tile_sum[i];
  lds_barrier();
  if (most <= kNothing) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = 0.0f;
    }
    return;
  }
  weigh(f, table, x);
  auto load = [&](int round) {
    load_tokens(a, s, row, round, n, x);
    weigh(f, table, x);
  };
  uint64_t cut = 0;        // kept: what lies here or in front
  if (f.by_count || f.by_weight) {
    const Cuts c = find_cuts(f, bin_count, bin_sum);
    uint64_t sum = c.sum;
    if (c.count_bin < kBins) {
      cut = cut_list<false>(load, x, rounds, c.count_bin, c.count_bin, 0, f.k - c.before_count, hist, scratch);
      if (f.by_weight) {
        uint64_t part = 0;
        for (int round = 0; round < rounds; ++round) {
          if (rounds > 1) load(round);
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            if (x.bin[e] == c.count_bin && x.place[e] >= cut) part += x.steps[e];
        }
        const uint64_t upto = scan_block<uint64_t>(part, scratch);
        if (tid == kSampleThreads - 1) chosen[0] = upto;
        lds_barrier();
        sum = c.sum_before_count + chosen[0];
      }
    }
    if (f.by_weight)
      cut = cut_list<true>(load, x, rounds, c.first, c.last, cut, share_of(f.p, sum) - c.sum_before_first, hist, scratch);
  }
  for (int round = 0; round < rounds; ++round) {
    if (rounds > 1) load(round);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (!x.place[e] || x.place[e] < cut || !x.steps[e]) continue;
      const uint64_t w = f.kept_steps(x.key[e], table);
      if (w) add(&tile_sum[x.token[e] / kSampleTile], w);
    }
  }
  lds_barrier();
  const uint64_t mine = tid < a.tiles ? tile_sum[tid] : 0;
  const uint64_t upto = scan_block<uint64_t>(mine, scratch);
  if (tid == kSampleThreads - 1) chosen[0] = upto;
  lds_barrier();
  const uint64_t total = chosen[0];
  const double u = fmin(fmax(a.uniform[row], 0.0), 1.0);
  const uint64_t mark = min(total - 1, static_cast<uint64_t>(u * static_cast<double>(total)));
  lds_barrier();
  if (upto > mark && upto - mine <= mark) chosen[0] = tid, chosen[1] = upto - mine;
  lds_barrier();
  const int i0 = static_cast<int>(chosen[0]) * kSampleTile + tid * kPer;
  uint32_t key[kPer];
  load_keys(a, row, i0, key);
  uint64_t each[kPer], sum = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    each[e] = key[e] > kNothing && place_of(key[e], i0 + e) >= cut ? f.kept_steps(key[e], table) : 0;
    sum += each[e];
  }
  uint64_t at = chosen[1] + scan_block<uint64_t>(sum, scratch) - sum;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
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
