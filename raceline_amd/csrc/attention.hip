// Attention of new tokens over the paged cache: the step between rope_append and the o linear.
// Plays the part of attn_flash and attn_combine (kernels/flash.metal:132,339).
//
//   s = scale * q . k            (a cap: s = cap * tanh(s / cap))
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)   over the keys j a row sees:
//       pos - window < j <= pos, pos = kv_len - q_len + i for row i of its sequence
//
// One pass over the keys with a running reference m and running sums in fp32. Rows are (token,
// query head) pairs of one key/value head, row r = (token r / G, head r % G): the G heads that
// share a key/value head read it once, and a tile of rows spans few positions.
// Two kernels: few_rows_kernel (a sequence with at most 32 rows a head: decoding, drafts) is bound
// by the stream of keys and values, many_rows_kernel by the matrix cores and the exponentials.
#include "paged.h"
#include "../../include/rlq.h"

#include <algorithm>
#include <cmath>

namespace rlq {
namespace {

constexpr int kThreads = 256;
constexpr int kFewRows = 32;      // rows of a few_rows_kernel tile
constexpr int kManyRows = 128;    // rows of a many_rows_kernel tile
constexpr float kLog2e = 1.44269504088896340736f;

// Weights are exp2(x - ref) with x the score in base-2 units. ref follows the largest score
// seen, kBelow under it, and moves only when a score passes ref + kBelow + kRefSlack: most
// steps then leave the accumulators alone. For fp16 (kBelow 7) a weight is at most 2^15, inside fp16, and
// 2^-14, where fp16 loses bits, lies 2^21 under the largest: what is lost there does not show in the sum.
// bf16 has no such bound but values up to 2^128: a weight is at most 2^-12 (kBelow -20), so that the sums
// of thousands of such values stay in range.
constexpr float kRefSlack = 8.0f;

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  const void *q;
  void *out;
  PagedCache c;
  int64_t q_stride, out_stride;
  // Sums of tiles whose keys are split: of few_rows_kernel, then of many_rows_kernel. A unit is one of the
  // split tiles of one key/value head.
  float *part;                // [unit][run][row of the tile][D]: a run's sums, not divided
  float2 *part_stat;          // [unit][run][row of the tile]: (ref, sum of weights)
  int4 *units;                // [unit]: (first row of the sequence, first row of the tile in it, rows of the sequence, runs)
  int few_units, many_units;
  int heads, group, window, out_bf16, q_wide, out_wide;
  // of a head's tiles, longest first, the first `whole` are not split, the keys of the next `cut` are, in at
  // most `splits` runs of `span` (a multiple of 32), and what is left is not
  int whole, cut, splits, span;
  int few_splits, few_span, few_rows;   // few_rows_kernel: all tiles, of few_rows rows
  int few, many;              // which kernels this call launches
  float unit;                 // base-2 units of a score as the product gives it, or of a capped one (1)
  float cap_log2;             // the cap in base-2 units, 0 for none
  float over_cap, exp_cap;    // score / cap, and the same in the power of tanh's exponential
  float near_cap[6];          // a capped score in base-2 units over the score, in powers of (score / cap)^2
};

template <typename T>
struct Mfma;
template <>
struct Mfma<_Float16> {
  typedef half8 op;
  static __device__ __forceinline__ f32x4 mul16(op a, op b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mul32(op a, op b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static constexpr unsigned kExp = 0x7C00u;
  static constexpr float kBelow = 7.0f;
};
template <>
struct Mfma<__bf16> {
  typedef bf16x8 op;
  static __device__ __forceinline__ f32x4 mul16(op a, op b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mul32(op a, op b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static constexpr unsigned kExp = 0x7F80u;
  static constexpr float kBelow = -20.0f;
};

// Capped scores in base-2 units, cap tanh(y) with y = score / cap. 1 - 2 / (1 + e^2y) is off by 2^-21.5
// times the cap wherever y lies, so that a cap of 10^4 would cost the weights of small scores their
// bits and one of 10^7 all of them. It serves for caps up to 88 (128 in base 2), where that is 2^-15 of a
// weight, an eighth of what an fp16 row is rounded by. Under larger ones tanh(y) / y is a polynomial
// in y^2 up to |y| = 0.6 (fitted to the least relative error, 2^-24.4), so that a score is off by its
// own roundings; past 0.6 the form above is off by 2^-20.6 of what it gives, and a wave with no
// such score skips it. The polynomial alone would take longer (six prompts capped at 30: 89 to 92 us against
// 85): two exponential-class operations cost less than its eight others.
constexpr float kFarCap = 0.6f, kSmallCap = 128.0f;   // of a score over the cap, of a cap in base 2

__device__ __forceinline__ float far_capped(const AttnArgs &a, float s) {
  const float e = __builtin_amdgcn_exp2f(s * a.exp_cap);
  return a.cap_log2 - 2.0f * a.cap_log2 * __builtin_amdgcn_rcpf(1.0f + e);
}

__device__ __forceinline__ float near_capped(const AttnArgs &a, float s, float y) {
  const float z = y * y;
  float r = a.near_cap[5];
#pragma unroll
  for (int i = 4; i >= 0; --i) r = __builtin_fmaf(r, z, a.near_cap[i]);
  return s * r;
}

template <int N, typename Scores>
__device__ __forceinline__ void cap_scores(const AttnArgs &a, Scores &x) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = far_capped(a, x[i]);
}

template <int N, typename Scores>
__device__ __forceinline__ void large_cap_scores(const AttnArgs &a, Scores &x) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(x[i]));
  if (__any(most * a.over_cap > kFarCap)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = x[i] * a.over_cap;
      x[i] = fabsf(y) <= kFarCap ? near_capped(a, x[i], y) : far_capped(a, x[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = near_capped(a, x[i], x[i] * a.over_cap);
  }
}

__device__ __forceinline__ float max_halves(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Eight weights as a matrix operand. TERMS 2: the rounding's remainder as a second operand, 16 bits
// of a weight for bf16 and 22 for fp16. few_rows_kernel always has it, since it waits for memory (32
// sequences of up to 16384 tokens 218 us with one term and with two, off by 2.8e-4 of the rows and by
// 2.07e-4, which is the rows' own rounding to fp16). many_rows_kernel has it where one term would have
// fewer bits than the rows that leave (bf16 keys, fp16 rows) and where the caller asks for it; elsewhere its
// rounding is as large as the rows' own (2.9e-4 against 2.07e-4, bf16 2.07e-3 against 1.63e-3), and half
// of the matrix products more cost 27 to 37% (a 27B layer's chunk 332 us against 439, six capped
// prompts 84 against 111, a chunk of 333 tokens in heads of 64 49 against 63).
template <typename T, int TERMS>
__device__ __forceinline__ void weights(const float (&p)[8], typename Mfma<T>::op (&w)[TERMS]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const T hi = static_cast<T>(p[e]);
    w[0][e] = hi;
    if constexpr (TERMS == 2) w[1][e] = static_cast<T>(p[e] - static_cast<float>(hi));
  }
}

// Infinities and NaN among values that some row does not see would reach it as 0 * inf. In blocks
// that are masked for some row the product is therefore formed without them (finite8), and whether
// some row does see one is noted. `seen`: bit e, whether any row sees the run's key e; what lies
// behind a sequence's end is never read into a result. In blocks that every row sees the product is
// formed with them, and is NaN where a weight, or its second term, rounds to 0 or below. In both
// cases they are added at the end to the rows that see them (add_odd), whose sums they alone
// decide: an infinity makes the rows that see it infinite, wherever it lies. (NaN that finite values made, by
// sums past fp32 of both signs, stays: it is kMade until then, which nothing is added to.)
template <typename T>
__device__ __forceinline__ u32x4 finite8(u32x4 v, unsigned seen, bool &odd) {
  constexpr unsigned E = Mfma<T>::kExp;
  u32x4 r;
  unsigned found = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (v[i] & E) == E, hi = (v[i] & (E << 16)) == E << 16;
    found |= (lo ? 1u << 2 * i : 0u) | (hi ? 2u << 2 * i : 0u);
    r[i] = (lo ? 0u : v[i] & 0xFFFFu) | (hi ? 0u : v[i] & 0xFFFF0000u);
  }
  odd |= (found & seen) != 0;
  return r;
}

// Which kernel takes a sequence: few_rows where both run and its rows fit one tile of it.
__device__ __forceinline__ bool is_few(const AttnArgs &a, const Sequence &s) {
  return a.few && (!a.many || s.tokens * a.group <= kFewRows);
}

// First position that any row of the sequence sees, to the block below; the runs of `span` keys
// begin there.
__device__ __forceinline__ int first_key(const AttnArgs &a, const Sequence &s) {
  return a.window ? max(0, s.kv - s.tokens + 1 - a.window) & ~(kBlockKeys - 1) : 0;
}

// Runs that hold keys of the sequence; where there is one, its workgroup finishes the rows itself.
__device__ __forceinline__ int runs_of(const AttnArgs &a, const Sequence &s, int splits, int span) {
  return max(1, min(splits, (s.kv - first_key(a, s) + span - 1) / span));
}

// many_rows_kernel's tile of a rank, longest first: a chip that is given its last long tile late
// waits for it (six prompts of up to 1537 tokens in the order of the batch, the longest last:
// 87 us, in this order 77). Tile d of a sequence counts as long as the sequence before the
// call's rows and (d + 1) * 128 / group of them; 64 lanes try 64 lengths at a time for the one past
// which lie as many tiles as the rank says. The search goes through the sequences, seven times or so:
// more than kRanked go in the order of the batch, last tile first. (Searched and in order, heads of 128: 63 prompts of
// 300 tokens 340 us and 131, 32 of up to 900 216 and 142, 20 of up to 1500 188 and 157; but 20 chunks of up to
// 500 tokens over up to 8000 482 and 606.) Up to 63 by a prefix sum of their tiles, so that no number is
// without one; more as find_sequence numbers them.
constexpr int kRanked = 16;

__device__ __forceinline__ Sequence find_tile(const AttnArgs &a, int rank, int slots) {
  if (a.c.batch > 63) return find_sequence(a.c, slots - 1 - rank, a.group, kManyRows, 1);
  const int lane = threadIdx.x & 63, batch = a.c.batch;
  const int row = row_start(a.c, min(lane, batch)), kv = cached(a.c, min(lane, batch - 1));
  const int tokens = max(0, __shfl(row, lane + 1) - row);
  int tiles = lane < batch ? (tokens * a.group + kManyRows - 1) / kManyRows : 0;
  if (a.few && tokens * a.group <= kFewRows) tiles = 0;   // few_rows_kernel's
  if (batch > kRanked) {
    int upto = tiles;                                      // of the sequences up to this lane's
    for (int off = 1; off < 64; off <<= 1) {
      const int left = __shfl_up(upto, off);               // by every lane: one that is masked off gives 0
      upto += lane >= off ? left : 0;
    }
    const int at = __builtin_amdgcn_readlane(upto, 63) - 1 - rank;
    const int b = __popcll(__ballot(upto <= at));
    Sequence s = {-1, 0, 0, 0, 0};
    if (at < 0) return s;
    s.b = b;
    s.item = at - __builtin_amdgcn_readlane(upto, b) + __builtin_amdgcn_readlane(tiles, b);
    s.row0 = __builtin_amdgcn_readlane(row, b);
    s.tokens = __builtin_amdgcn_readlane(tokens, b);
    s.kv = __builtin_amdgcn_readlane(kv, b);
    return s;
  }
  const int before = kv - tokens;
  auto shorter = [&](int length, int b) {                  // tiles of sequence b no longer than that
    const int64_t x = static_cast<int64_t>(length - __builtin_amdgcn_readlane(before, b)) * a.group;
    const int most = __builtin_amdgcn_readlane(tiles, b);
    return static_cast<int>(max<int64_t>(0, min<int64_t>(x / kManyRows, most)));
  };
  auto longer = [&](int length) {                          // of all sequences, longer
    int n = 0;
    for (int b = 0; b < batch; ++b) n += __builtin_amdgcn_readlane(tiles, b) - shorter(length, b);
    return n;
  };
  Sequence s = {-1, 0, 0, 0, 0};
  // no tile is longer than `most`, and none is as short as `least`
  int least = kMaxPositions, most = 0;
  for (int b = 0; b < batch; ++b) {
    const int from = __builtin_amdgcn_readlane(before, b), n = __builtin_amdgcn_readlane(tiles, b);
    if (!n) continue;
    least = min(least, from);
    most = max(most, from + static_cast<int>((static_cast<int64_t>(n) * kManyRows + a.group - 1) / a.group));
  }
  if (rank >= longer(least)) return s;
  while (most - least > 1) {                               // longer(most) <= rank < longer(least)
    const int step = (most - least + 63) / 64, at = min(most, least + (lane + 1) * step);
    const uint64_t low = __ballot(longer(at) <= rank);
    const int first = __builtin_ctzll(low);                // the last lane's length is `most`
    most = min(most, least + (first + 1) * step);
    least = least + first * step;
  }
  int left = rank - __builtin_amdgcn_readfirstlane(longer(most));
  for (int b = 0; b < batch; ++b) {
    const int upto = __builtin_amdgcn_readfirstlane(shorter(most, b));
    const int n = upto - __builtin_amdgcn_readfirstlane(shorter(most - 1, b));
    if (left < n) {
      s.b = b;
      s.item = upto - 1 - left;
      s.row0 = __builtin_amdgcn_readlane(row, b);
      s.tokens = __builtin_amdgcn_readlane(tokens, b);
      s.kv = __builtin_amdgcn_readlane(kv, b);
      break;
    }
    left -= n;
  }
  return s;
}

// Row r of a tile's run among the partial sums.
__device__ __forceinline__ int few_part(const AttnArgs &a, int unit, int run, int r) {
  return (unit * a.few_splits + run) * a.few_rows + r;
}

__device__ __forceinline__ int many_part(const AttnArgs &a, int unit, int run, int r) {
  return few_part(a, a.few_units, 0, 0) + (unit * a.splits + run) * kManyRows + r;
}

// A sum x over one reference, times the factor f to another's. An infinity stays one where f is 0.
__device__ __forceinline__ float scaled(float x, float f) {
  const float y = x * f;
  return __builtin_isnan(y) ? x : y;
}

constexpr unsigned kMade = 1;   // bits of a sum that was NaN beside a sum of weights that is not

__device__ __forceinline__ float marked(float o, float sum) {
  return __builtin_isnan(o) && !__builtin_isnan(sum) ? __uint_as_float(kMade) : o;
}

__device__ __forceinline__ float unmarked(float o) { return __float_as_uint(o) == kMade ? __builtin_nanf("") : o; }

// Whether a block holds any infinity or NaN; a wave looks at it a kilobyte at a time.
template <typename T, int D>
__device__ __forceinline__ bool block_odd(const AttnArgs &a, int at) {
  constexpr unsigned E = Mfma<T>::kExp;
  const u32x4 *v = reinterpret_cast<const u32x4 *>(static_cast<const T *>(a.c.v) + static_cast<int64_t>(at) * (kBlockKeys * D));
  bool odd = false;
#pragma unroll 4
  for (int i = 0; i < D / 16; ++i) {
    const u32x4 x = v[i * 64 + (threadIdx.x & 63)];
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= (x[e] & E) == E || (x[e] & (E << 16)) == E << 16;
  }
  return __any(odd);
}

// Adds the infinities and NaN among the values of block `at` (its first key `first`) to o (o[i]:
// dimension dim(i)) for the keys that a row sees.
template <typename T, int D, int N, typename Dim>
__device__ __forceinline__ void add_odd(const AttnArgs &a, int at, int first, int lo, int hi, Dim dim, float (&o)[N]) {
  const unsigned short *v = static_cast<const unsigned short *>(a.c.v) + static_cast<int64_t>(at) * (kBlockKeys * D);
  for (int key = 0; key < kBlockKeys; ++key) {
    const bool seen = first + key >= lo && first + key <= hi;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned x = v[value_run(dim(i), key >> 4, key >> 2 & 1) + (key >> 3 & 1) * 4 + (key & 3)];
      if (seen && (x & Mfma<T>::kExp) == Mfma<T>::kExp)
        o[i] += static_cast<float>(__builtin_bit_cast(T, static_cast<unsigned short>(x)));
    }
  }
}

// What a finished row is multiplied by. A row that found no score above -inf has a sum of 0 and is
// zero; what it saw being NaN shows in the sum alone (a maximum passes NaN over).
__device__ __forceinline__ float over_sum(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

// Four neighbouring dimensions of a finished row.
__device__ __forceinline__ void store4(const AttnArgs &a, int row, int col, f32x4 o) {
  if (a.out_bf16) {
    __bf16 *p = static_cast<__bf16 *>(a.out) + row * a.out_stride + col;
    const bf16x4 y = __builtin_convertvector(o, bf16x4);
    if (a.out_wide) {
      *reinterpret_cast<bf16x4 *>(p) = y;
    } else {
      for (int i = 0; i < 4; ++i) p[i] = y[i];
    }
  } else {
    _Float16 *p = static_cast<_Float16 *>(a.out) + row * a.out_stride + col;
    const half4 y = __builtin_convertvector(o, half4);
    if (a.out_wide) {
      *reinterpret_cast<half4 *>(p) = y;
    } else {
      for (int i = 0; i < 4; ++i) p[i] = y[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ typename Mfma<T>::op load_q(const AttnArgs &a, int row, int col) {
  typedef typename Mfma<T>::op op;
  const T *p = static_cast<const T *>(a.q) + row * a.q_stride + col;
  if (a.q_wide) return *reinterpret_cast<const op *>(p);
  op r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = p[i];
  return r;
}

// ----------------------------------------------------------------------------- few rows

// One workgroup: up to 16 * NT rows of one sequence and key/value head over one run of its keys.
// Its four waves take blocks of 32 keys in turn, straight from memory into registers, each with
// its own running sums, which meet in LDS at the end: nothing is shared until then, so a wave
// never waits for another, and 8 waves a CU keep their next keys and values in flight.
// v_mfma_f32_16x16x32: S^T (keys x rows) = K Q^T with the operand's row r standing for key
// 16 (r / 8) + r % 8 (then + 8), so that a lane's eight weights belong to one 16-byte run of V.
// Bound by the stream of keys and values, read past the caches: 32 sequences of up to 16384 tokens, 4
// heads of 256, 1.21 GB in 210 us, 5.8 TB/s (229 us through the L2; a plain read gets 6.9 TB/s).
// LARGE_CAP: a cap over kSmallCap, whose code would cost the other calls (one token of 1024 keys in heads
// of 64 9.0 us with it, 8.7 without).
template <typename T, int D, int NT, bool LARGE_CAP>
__global__ __launch_bounds__(kThreads, D * NT > 256 ? 1 : 2) void few_rows_kernel(AttnArgs a) {
  constexpr int KS = D / 32, DT = D / 16, ROWS = 16 * NT, TERMS = 2;
  typedef typename Mfma<T>::op op;
  __shared__ float stat[4][ROWS][2];
  __shared__ float sums[2][ROWS][D + 4];
  __shared__ op queries[NT][KS][64];

  const int KV = a.c.kv_heads, head = blockIdx.x % KV, split = (blockIdx.x / KV) % a.few_splits;
  const int64_t slot = blockIdx.x / KV / a.few_splits;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, r = lane & 15;
  // beside many_rows_kernel a sequence of few rows is one tile: items are the sequences
  const Sequence s = find_sequence(a.c, slot, a.many ? 0 : a.group, ROWS, 1);
  const int b = s.b, tile = s.item * ROWS, rows = s.tokens * a.group;
  const int unit = static_cast<int>(blockIdx.x / (KV * a.few_splits)) * KV + head;
  const bool none = b < 0 || tile < 0 || tile >= rows || !is_few(a, s);
  const int runs = none ? 0 : runs_of(a, s, a.few_splits, a.few_span);
  if (a.few_splits > 1 && split == 0 && tid == 0) a.units[unit] = make_int4(s.row0, tile, rows, runs);
  if (split >= runs) return;

  // rows of this lane's columns, and what they see
  int lo[NT], hi[NT], row[NT], col[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int R = tile + n * 16 + r, tok = R / a.group;
    const bool here = R < rows;
    row[n] = here ? s.row0 + tok : -1;
    col[n] = (head * a.group + R - tok * a.group) * D;
    hi[n] = here ? s.kv - s.tokens + tok : -1;                       // last key seen
    lo[n] = a.window ? max(0, hi[n] - a.window + 1) : 0;             // first
    for (int k = wave; k < KS; k += 4)
      queries[n][k][lane] = here ? load_q<T>(a, row[n], col[n] + 32 * k + 8 * g) : op{};
  }
  __syncthreads();
  const int last = min(rows, tile + ROWS) - 1;
  const int lo_any = a.window ? max(0, s.kv - s.tokens + tile / a.group - a.window + 1) : 0;
  const int lo_all = a.window ? max(0, s.kv - s.tokens + last / a.group - a.window + 1) : 0;
  const int hi_any = s.kv - s.tokens + last / a.group, hi_all = s.kv - s.tokens + tile / a.group;
  const int base = first_key(a, s) + split * a.few_span;
  const int end = min(hi_any + 1, split == a.few_splits - 1 ? hi_any + 1 : base + a.few_span);
  const int blk0 = max(base, lo_any & ~(kBlockKeys - 1)) / kBlockKeys, blk1 = (end + kBlockKeys - 1) / kBlockKeys;

  f32x4 o[NT][DT];
  float ref[NT], sum[NT];
  bool odd = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    ref[n] = -__builtin_inff(), sum[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[n][d] = f32x4{0, 0, 0, 0};
  }

  const T *kc = static_cast<const T *>(a.c.k), *vc = static_cast<const T *>(a.c.v);
  // key 16 (r / 8) + r % 8 of a step of 32 dimensions: two operand steps of 16
  const int koff = (g >> 1) * 512 + (g & 1) * 256 + (16 * (r >> 3) + (r & 7)) * 8;
  const int voff = (g >> 1) * 512 + (g & 1) * 256 + r * 8;
  const int key0 = 16 * (g >> 1) + 4 * (g & 1);   // this lane's keys: key0 + 8 j + i
  op kr[KS][2];
  u32x4 vr[DT];
  int pages = -1;                                  // lane i: this wave's block from + i, by its number in the cache
  int from = 0;
  const int nblk = max(0, blk1 - blk0), mine = nblk > wave ? (nblk - wave + 3) / 4 : 0;
  auto page_at = [&](int i) {
    if (i >= mine) return -1;
    if (i - from >= 64 || i == 0) {
      from = i;
      const int blk = blk0 + wave + 4 * (i + lane);
      pages = i + lane < mine ? block_at(a.c, b, head, blk) : -1;
    }
    return __builtin_amdgcn_readlane(pages, i - from);
  };
  auto load_k = [&](int at) {
    const T *p = kc + static_cast<int64_t>(at) * (kBlockKeys * D) + koff;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      kr[k][0] = __builtin_nontemporal_load(reinterpret_cast<const op *>(p + k * 1024));
      kr[k][1] = __builtin_nontemporal_load(reinterpret_cast<const op *>(p + k * 1024 + 64));
    }
  };
  int page = page_at(0);
  if (page >= 0) load_k(page);
  for (int i = 0; i < mine; ++i) {
    const int blk = blk0 + wave + 4 * i, first = blk * kBlockKeys;
    const int next = page_at(i + 1);
    if (page < 0) {
      page = next;
      if (page >= 0) load_k(page);
      continue;
    }
    const T *vp = vc + static_cast<int64_t>(page) * (kBlockKeys * D) + voff;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      vr[d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vp + (d >> 1) * 1024 + (d & 1) * 128));

    f32x4 sc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sc[n][j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KS; ++k) sc[n][j] = Mfma<T>::mul16(kr[k][j], queries[n][k][lane], sc[n][j]);
      }
    if (next >= 0) load_k(next);
    page = next;

    const bool masked = first < lo_all || first + kBlockKeys - 1 > hi_all || first + kBlockKeys > end;
    op w[NT][TERMS];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[8], top = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = sc[n][e >> 2][e & 3];
      if constexpr (LARGE_CAP) large_cap_scores<8>(a, x);
      else if (a.cap_log2 != 0.0f) cap_scores<8>(a, x);
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = first + key0 + 8 * (e >> 2) + (e & 3);
          x[e] = key >= lo[n] && key <= hi[n] ? x[e] : -__builtin_inff();
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = max_halves(top) * a.unit;
      if (__any(top > ref[n] + (Mfma<T>::kBelow + kRefSlack))) {
        const float to = top > ref[n] + (Mfma<T>::kBelow + kRefSlack) ? top - Mfma<T>::kBelow : ref[n];
        const float f = ref[n] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref[n] - to);
        ref[n] = to;
        sum[n] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] *= f;
      }
      const float m = ref[n] == -__builtin_inff() ? 0.0f : ref[n];
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.unit, -m));
        sum[n] += p[e];
      }
      weights<T, TERMS>(p, w[n]);
    }
    if (masked) {
      unsigned seen = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = first + key0 + 8 * (e >> 2) + (e & 3);
        seen |= key >= lo_any && key <= hi_any ? 1u << e : 0u;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) vr[d] = finite8<T>(vr[d], seen, odd);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
          o[n][d] = Mfma<T>::mul16(__builtin_bit_cast(op, vr[d]), w[n][t], o[n][d]);
  }

  // Sums that are not finite beside a sum of weights that is: values made them so, and are added once
  // the waves' shares are scaled.
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sum[n] += __shfl_xor(sum[n], 16);
    sum[n] += __shfl_xor(sum[n], 32);
    float t[2] = {};
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i & 1] = __builtin_fmaf(o[n][d][i], 0.0f, t[i & 1]);
    odd |= row[n] >= 0 && !__builtin_isnan(sum[n]) && __builtin_isnan(t[0] + t[1]);
  }
  const bool any_odd = __any(odd);

  // the waves' sums: the largest reference first, then each wave's share scaled to it (where the wave
  // found no score, its sums are 0, or NaN where what it saw was)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (g == 0) stat[wave][n * 16 + r][0] = ref[n], stat[wave][n * 16 + r][1] = sum[n];
  }
  __syncthreads();
  float total[NT], top[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    top[n] = -__builtin_inff(), total[n] = 0.0f;
    for (int w2 = 0; w2 < 4; ++w2) top[n] = fmaxf(top[n], stat[w2][n * 16 + r][0]);
    const float m = top[n] == -__builtin_inff() ? 0.0f : top[n];
    for (int w2 = 0; w2 < 4; ++w2)
      total[n] += stat[w2][n * 16 + r][1] * __builtin_amdgcn_exp2f(stat[w2][n * 16 + r][0] - m);
    const float f = __builtin_amdgcn_exp2f(ref[n] - m);
    if (__builtin_expect(any_odd, 0)) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][d][i] = marked(scaled(o[n][d][i], f), sum[n]);
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d) o[n][d] *= f;
    }
  }
  if (__builtin_expect(any_odd, 0)) {
    for (int i = 0; i < mine; ++i) {
      const int blk = blk0 + wave + 4 * i, first = blk * kBlockKeys;
      const int at = block_at(a.c, b, head, blk);
      if (at < 0 || !block_odd<T, D>(a, at)) continue;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          float part[4] = {o[n][d][0], o[n][d][1], o[n][d][2], o[n][d][3]};
          add_odd<T, D, 4>(a, at, first, lo[n], min(hi[n], end - 1), [&](int j) { return 16 * d + 4 * g + j; }, part);
          o[n][d] = f32x4{part[0], part[1], part[2], part[3]};
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][d][i] = unmarked(o[n][d][i]);
  }
  // waves 2 and 3 hand theirs to waves 0 and 1, then wave 1 to wave 0
  for (int step = 2; step; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          *reinterpret_cast<f32x4 *>(&sums[wave - step][n * 16 + r][d * 16 + 4 * g]) = o[n][d];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[n][d] += *reinterpret_cast<const f32x4 *>(&sums[wave][n * 16 + r][d * 16 + 4 * g]);
    }
    __syncthreads();
  }
  if (wave) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (row[n] < 0) continue;
    if (runs == 1) {
      const float f = over_sum(total[n]);
#pragma unroll
      for (int d = 0; d < DT; ++d) store4(a, row[n], col[n] + d * 16 + 4 * g, o[n][d] * f);
    } else {
      const int64_t at = few_part(a, unit, split, n * 16 + r);
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(a.part + at * D + d * 16 + 4 * g) = o[n][d];
      if (g == 0) a.part_stat[at] = make_float2(top[n], total[n]);
    }
  }
}

// ----------------------------------------------------------------------------- many rows

__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_rsrc(const void *p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, bytes, 0x00020000);
}

// One LDS-DMA: 16 bytes a lane into the kilobyte at lds + at. (Not a template: in one, the host
// pass refuses the 16-byte size.)
__device__ __forceinline__ void dma_kb(__amdgpu_buffer_rsrc_t r, unsigned char *lds, int at, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + at), 16, voff, soff, 0, 0);
}

template <int N, int AHEAD, int READS, int PER, int VALU>
__device__ __forceinline__ void feed_step() {
  if constexpr (N < READS * PER) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (VALU > 0) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    if constexpr (N % PER == 0 && N / PER + AHEAD < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    feed_step<N + 1, AHEAD, READS, PER, VALU>();
  }
}

// The order of a run of products whose A operands come from LDS: AHEAD reads first, then
// after each operand's PER products the next read, VALU operations of the softmax between
// them. Left to itself the compiler reads two operands, waits for both, and multiplies.
template <int AHEAD, int READS, int PER, int VALU>
__device__ __forceinline__ void feed_products() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
  feed_step<0, AHEAD, READS, PER, VALU>();
}

constexpr int kAhead = 4;

template <int D>
constexpr int kTileKeys = D >= 128 ? 32 : 64;

// Workgroups of many_rows_kernel that a CU holds, by its registers.
template <int D, int TERMS>
constexpr int kManyHeld = D == 64 ? (TERMS == 1 ? 4 : 3) : D == 128 && TERMS == 1 ? 3 : 2;

// LARGE_CAP as above: 1 to 3% of the other calls.
template <typename T, int D, int TERMS, bool LARGE_CAP>
__global__ __launch_bounds__(kThreads, (kManyHeld<D, TERMS>)) void many_rows_kernel(AttnArgs a) {
  constexpr int KB = kTileKeys<D>, NB = KB / kBlockKeys, KS = D / 16, DT = D / 32, ROWS = kManyRows;
  constexpr int kBlockBytes = kBlockKeys * D * 2, kStage = 2 * NB * kBlockBytes, kPieces = kBlockBytes / 1024;
  typedef typename Mfma<T>::op op;
  extern __shared__ unsigned char lds[];   // two stages, then a flag
  int *odd = reinterpret_cast<int *>(lds + 2 * kStage);

  const int KV = a.c.kv_heads, head = blockIdx.x % KV, item = blockIdx.x / KV, slots = a.c.rows * a.group / kManyRows + a.c.batch;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  const int past = item - a.whole;   // items of the split tiles and behind them
  const bool whole = past < 0 || past >= a.cut * a.splits;
  const int splits = whole ? 1 : a.splits, split = whole ? 0 : past % splits, nth = past / splits;
  const Sequence s = find_tile(a, past < 0 ? item : whole ? item - a.cut * (a.splits - 1) : a.whole + nth, slots);
  const int b = s.b, tile = s.item * kManyRows, rows = s.tokens * a.group;
  const bool none = b < 0 || tile < 0 || tile >= rows || is_few(a, s);
  const int runs = none ? 0 : runs_of(a, s, splits, a.span), unit = nth * KV + head;
  if (!whole && split == 0 && tid == 0) a.units[a.few_units + unit] = make_int4(s.row0, tile, rows, runs);
  if (split >= runs) return;

  // this lane's rows and what they see
  const int p0 = s.kv - s.tokens;
  const int R = tile + wave * 32 + n32, tok = R / a.group;
  const bool here = R < rows;
  const int row = here ? s.row0 + tok : -1, col = (head * a.group + R - tok * a.group) * D;
  const int hi = here ? p0 + tok : -1, lo = a.window ? max(0, hi - a.window + 1) : 0;
  op q[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) q[k] = here ? load_q<T>(a, row, col + 16 * k + 8 * h) : op{};
  // keys that any row of the tile sees, and that all of its rows see
  const int last = min(rows, tile + ROWS) - 1;
  const int lo_any = a.window ? max(0, p0 + tile / a.group - a.window + 1) : 0, hi_any = p0 + last / a.group;
  const int lo_all = a.window ? max(0, p0 + last / a.group - a.window + 1) : 0, hi_all = p0 + tile / a.group;
  const int base = first_key(a, s) + split * a.span;
  const int end = min(hi_any + 1, split == splits - 1 ? hi_any + 1 : base + a.span);
  const int blk0 = max(base, lo_any & ~(kBlockKeys - 1)) / kBlockKeys, blk1 = (end + kBlockKeys - 1) / kBlockKeys;
  const int nblk = max(0, blk1 - blk0), tiles = (nblk + NB - 1) / NB;

  f32x16 o[DT];
  float ref = -__builtin_inff(), sum = 0.0f;
  if (tid == 0) *odd = 0;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

  const char *kc = static_cast<const char *>(a.c.k), *vc = static_cast<const char *>(a.c.v);
  int pages = -1, from = 0;   // lane i: block from + i of the run, by its number in the cache
  auto page_at = [&](int i) {
    if (i >= nblk) return -1;
    if (i - from >= 64 || i == 0) {
      from = i;
      pages = i + lane < nblk ? block_at(a.c, b, head, blk0 + i + lane) : -1;
    }
    return __builtin_amdgcn_readlane(pages, i - from);
  };
  auto stage = [&](int kt, int buf, int (&page)[NB]) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      page[j] = page_at(kt * NB + j);
      if (page[j] < 0) continue;
      const int64_t at = static_cast<int64_t>(page[j]) * kBlockBytes;
      const int to = buf * kStage + j * kBlockBytes + wave * 1024;
      const __amdgpu_buffer_rsrc_t kr = block_rsrc(kc + at, kBlockBytes), vr = block_rsrc(vc + at, kBlockBytes);
#pragma unroll
      for (int i = 0; i < kPieces / 4; ++i) dma_kb(kr, lds, to + i * 4096, 16 * lane, wave * 1024 + i * 4096);
#pragma unroll
      for (int i = 0; i < kPieces / 4; ++i)
        dma_kb(vr, lds, to + NB * kBlockBytes + i * 4096, 16 * lane, wave * 1024 + i * 4096);
    }
  };

  int page[NB], next[NB];
  if (tiles) stage(0, 0, page);
  for (int kt = 0; kt < tiles; ++kt) {
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's pieces of the tile have landed
    __syncthreads();                      // and every wave's; the other stage's readers are done
    if (kt + 1 < tiles) stage(kt + 1, (kt + 1) & 1, next);
    unsigned char *kl = lds + (kt & 1) * kStage + lane * 16, *vl = kl + NB * kBlockBytes;
    const int first = (blk0 + kt * NB) * kBlockKeys;

    bool masked = first < lo_all || first + KB - 1 > hi_all || first + KB > end;
#pragma unroll
    for (int j = 0; j < NB; ++j) masked |= page[j] < 0;   // also the blocks behind the last
    if (masked) {   // for the workgroup as a whole: take out what finite8 takes out, once for all waves
#pragma unroll
      for (int j = 0; j < NB; ++j)
        for (int i = wave; i < kPieces; i += 4) {
          unsigned seen = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = first + 32 * j + 16 * (i & 1) + 8 * (e >> 2) + 4 * h + (e & 3);
            seen |= key >= lo_any && key <= hi_any && page[j] >= 0 ? 1u << e : 0u;
          }
          bool here = false;
          u32x4 *v = reinterpret_cast<u32x4 *>(vl + j * kBlockBytes + i * 1024);
          *v = finite8<T>(*v, seen, here);
          if (here) *odd = 1;
        }
      __syncthreads();
    }
    f32x16 sc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[j][i] = 0.0f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const op key = *reinterpret_cast<const op *>(kl + j * kBlockBytes + k * 1024);
        sc[j] = Mfma<T>::mul32(key, q[k], sc[j]);
      }
    feed_products<kAhead, NB * KS, 1, 0>();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (LARGE_CAP) {
#pragma unroll
      for (int j = 0; j < NB; ++j) large_cap_scores<16>(a, sc[j]);
    } else if (a.cap_log2 != 0.0f) {
#pragma unroll
      for (int j = 0; j < NB; ++j) cap_scores<16>(a, sc[j]);
    }
    if (masked) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = first + 32 * j + 8 * (i >> 2) + 4 * h + (i & 3);
          sc[j][i] = key >= lo && key <= hi && page[j] >= 0 ? sc[j][i] : -__builtin_inff();
        }
    }
    op va[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) va[i] = *reinterpret_cast<const op *>(vl + i * 1024);
    __builtin_amdgcn_sched_barrier(0);
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[j][i]);
    top = max_halves(top) * a.unit;
    if (__any(top > ref + (Mfma<T>::kBelow + kRefSlack))) {
      const float to = top > ref + (Mfma<T>::kBelow + kRefSlack) ? top - Mfma<T>::kBelow : ref;
      const float f = ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref - to);
      ref = to;
      sum *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    const float m = ref == -__builtin_inff() ? 0.0f : ref;
    // weights of block j, and the products of block j - 1 between them
    __builtin_amdgcn_sched_barrier(0);
    op w[NB][2][TERMS];
#pragma unroll
    for (int j = 0; j <= NB; ++j) {
      if (j < NB) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][8 * t + e], a.unit, -m));
            sum += p[e];
          }
          weights<T, TERMS>(p, w[j][t]);
        }
      }
      if (j > 0) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const op v = j == 1 && 2 * d + t < kAhead ? va[(2 * d + t) % kAhead] : *reinterpret_cast<const op *>(vl + (j - 1) * kBlockBytes + (2 * d + t) * 1024);
#pragma unroll
            for (int x = 0; x < TERMS; ++x) o[d] = Mfma<T>::mul32(v, w[j - 1][t][x], o[d]);
          }
        if (j < NB) feed_products<0, 2 * DT, TERMS, 32 / (DT * TERMS) + 1>();
        else if (NB == 1) feed_products<0, 2 * DT, TERMS, 0>();
        else feed_products<kAhead, 2 * DT, TERMS, 0>();
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) page[j] = next[j];
  }

  const float total = sum + __shfl_xor(sum, 32);
  __syncthreads();
  // sums that are not finite beside a sum of weights that is: values made them so
  const bool plain = row >= 0 && !__builtin_isnan(total);
  float t[4] = {};
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i & 3] = __builtin_fmaf(o[d][i], 0.0f, t[i & 3]);
  const bool found = *odd || (plain && __builtin_isnan(t[0] + t[1] + (t[2] + t[3])));
  if (__builtin_expect(__any(found), 0)) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = marked(o[d][i], total);
    for (int i = 0; i < nblk; ++i) {
      const int at = block_at(a.c, b, head, blk0 + i);
      if (at < 0 || !block_odd<T, D>(a, at)) continue;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        float part[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) part[e] = o[d][e];
        add_odd<T, D, 16>(a, at, (blk0 + i) * kBlockKeys, lo, min(hi, end - 1),
                          [&](int e) { return 32 * d + 8 * (e >> 2) + 4 * h + (e & 3); }, part);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = part[e];
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = unmarked(o[d][i]);
  }
  if (row < 0) return;
  if (runs == 1) {
    const float f = over_sum(total);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(a, row, col + 32 * d + 8 * i + 4 * h,
               f32x4{o[d][4 * i] * f, o[d][4 * i + 1] * f, o[d][4 * i + 2] * f, o[d][4 * i + 3] * f});
  } else {
    const int64_t at = many_part(a, unit, split, wave * 32 + n32);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4 *>(a.part + at * D + 32 * d + 8 * i + 4 * h) =
            f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (h == 0) a.part_stat[at] = make_float2(ref, total);
  }
}

// ----------------------------------------------------------------------------- the runs' sums

template <int N, int D, typename Row>
__device__ __forceinline__ void add_runs(Row row, int first, int runs, float mine, float (&o)[D / 64]) {
  constexpr int PER = D / 64;
  typedef float fvec __attribute__((ext_vector_type(PER)));
  fvec p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = *reinterpret_cast<const fvec *>(row(min(first + i, runs - 1)));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float f = __shfl(mine, first + i);
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] += first + i < runs ? scaled(p[i][e], f) : 0.0f;
  }
}

// One wave: one row of a unit; adds its runs' sums, always in the same order. Where the row is and
// how many runs it has its tile's first workgroup wrote; the statistics of all runs come with one load (at
// most 64 runs), the sums eight runs at a time (four where there are no more). Neighbouring workgroups
// are neighbouring heads, as in the kernels that stored the sums: where the heads are a multiple of the 8
// XCDs, a row is joined from the L2 that holds it (nine sequences' drafts with 8 heads 32.3 -> 30.6 us).
template <int D>
__global__ __launch_bounds__(kThreads) void join_runs_kernel(AttnArgs a) {
  constexpr int PER = D / 64;
  constexpr int kWaves = kThreads / 64;
  const int few = a.few_units * a.few_rows / kWaves, lane = threadIdx.x & 63, KV = a.c.kv_heads;   // few: workgroups
  const bool is_few = static_cast<int>(blockIdx.x) < few;
  const int rows = is_few ? a.few_rows : kManyRows, most = is_few ? a.few_splits : a.splits;
  const int block = is_few ? blockIdx.x : blockIdx.x - few, head = block % KV, nth = block / KV * kWaves;
  const int unit = (nth >> __builtin_ctz(rows)) * KV + head;
  const int r = (nth & (rows - 1)) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = is_few ? few_part(a, unit, 0, r) : many_part(a, unit, 0, r);   // run i: at + i * rows
  const float2 stat = a.part_stat[at + min(lane, most - 1) * rows];
  const int4 u = a.units[(is_few ? 0 : a.few_units) + unit];
  const int runs = __builtin_amdgcn_readfirstlane(u.w), R = __builtin_amdgcn_readfirstlane(u.y) + r;
  if (runs <= 1 || R >= __builtin_amdgcn_readfirstlane(u.z)) return;   // finished by its workgroup, or no row
  float top = lane < runs ? stat.x : -__builtin_inff();
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float mine = lane < runs ? __builtin_amdgcn_exp2f(stat.x - (top == -__builtin_inff() ? 0.0f : top)) : 0.0f;
  float total = lane < runs ? stat.y * mine : 0.0f;
  for (int off = 32; off; off >>= 1) total += __shfl_xor(total, off);
  float o[PER] = {};
  const float *p = a.part + at * D + lane * PER;
  auto row = [&](int i) { return p + static_cast<int64_t>(i) * rows * D; };
  if (runs <= 4) {
    add_runs<4, D>(row, 0, runs, mine, o);
  } else {
    for (int i = 0; i < runs; i += 8) add_runs<8, D>(row, i, runs, mine, o);
  }
  const float f = over_sum(total);
  const int tok = R / a.group;
  const int64_t to = static_cast<int64_t>(u.x + tok) * a.out_stride + (head * a.group + R - tok * a.group) * D + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (a.out_bf16) static_cast<__bf16 *>(a.out)[to + e] = static_cast<__bf16>(o[e] * f);
    else static_cast<_Float16 *>(a.out)[to + e] = static_cast<_Float16>(o[e] * f);
  }
}

// ----------------------------------------------------------------------------- host

// How a call is launched, from its sizes alone (max_q and max_kv bound the sequences' new and
// cached tokens; they choose, they do not limit what is computed).
struct Plan {
  int few, many, whole, cut, splits, span, few_splits, few_span, few_tiles;
  int64_t few_slots, slots;     // a head's tiles at most, of few_rows_kernel and of many_rows_kernel
  int few_units, many_units;    // of the partial sums
  int64_t part_rows;
  size_t bytes;
};

constexpr int64_t kMaxGrid = (int64_t)UINT32_MAX / kThreads;   // a launch counts its threads in 32 bits

// few_rows_kernel: how the keys are split into runs (of whole blocks for the four waves, 64 at most).
// Where the keys and values take 8 us or more at 5.5 TB/s, as many runs as give 512 workgroups, two a
// CU: fewer leave memory idle and sequences of different lengths uneven (nine sequences' drafts 29.6
// us with 576 workgroups, 35 with 288). (Heads of 256 with more than 16 rows hold one workgroup a CU; 256
// workgroups were from 31% faster, 4 sequences of up to 16000 tokens, to 22% slower, 16 of up to 8000, as their
// lengths fall.) Below that a call is a chain of latencies: a run of 128 keys (a block a wave)
// takes `first`, each further 128 keys `step`, joining 2.1 us and 0.13 a run, and the least sum is taken. So
// one token of 512 keys in heads of 64 is one run (6.2 us, four runs 7.3), of 1024 keys eight (7.7, one
// run 9.3), in heads of 256 eight as well (10.6, one run 22.9), and of 4096 keys 16 (13.9, 32 runs 13.3, eight 18.1).
void split_few(int64_t tiles, int kv, int D, int *splits, int *span) {
  const double first = D == 256 ? 7.5 : D == 128 ? 5.5 : 4.6, step = D == 256 ? 1.9 : D == 128 ? 1.0 : 0.75;
  const bool streams = (double)tiles * kv * D * 4 / 5.5e6 >= 8;
  const int block = 4 * kBlockKeys, most = (int)std::min<int64_t>(64, (511 + tiles) / tiles);
  double best = 0;
  for (int n = streams ? most : 1; n <= most; ++n) {
    const int run = (int)(((int64_t)kv + (int64_t)n * block - 1) / ((int64_t)n * block) * block), runs = (kv + run - 1) / run;
    const double us = first + step * (run / block - 1) + (runs > 1 ? 2.1 + 0.13 * runs : 0);
    if (best == 0 || us < best) best = us, *splits = runs, *span = run;
  }
}

// many_rows_kernel's microseconds a key for one of 1, 2, .. workgroups that share a CU (measured over
// 8192 keys, whole chips of them); as many as its registers let in. With weights of one term: with two a
// key takes a third longer and heads of 64 and 128 hold one workgroup less, but the plan is the same, since
// the scratch's size is asked for without the types (a 27B chunk 423 us, 332 with one term).
struct Rates {
  int most;
  double key[4];
};
const Rates &rates(int D) {
  static const Rates r64 = {4, {0.0163, 0.0232, 0.0319, 0.0404}}, r128 = {3, {0.0256, 0.0344, 0.0496}},
                     r256 = {2, {0.0403, 0.0644}};
  return D == 64 ? r64 : D == 128 ? r128 : r256;
}

// Microseconds of a CU that gets `whole` tiles of `keys` keys and then `pieces` of `run` keys, as
// they come to an end.
double cu_time(const Rates &r, int whole, int keys, int pieces, int run) {
  double left[4] = {}, t = 0;
  int held = 0;
  for (;;) {
    while (held < r.most && whole + pieces > 0) left[held++] = whole > 0 ? (--whole, keys) : (--pieces, run);
    if (!held) return t;
    const double least = *std::min_element(left, left + held);
    t += least * r.key[held - 1];
    int kept = 0;
    for (int i = 0; i < held; ++i)
      if (left[i] > least) left[kept++] = left[i] - least;
    held = kept;
  }
}

constexpr int64_t kMaxParts = 256 << 20;   // bytes of many_rows_kernel's partial sums

// many_rows_kernel: which tiles are split into how many runs, by the least estimated time of a CU
// (256 of them). Not all tiles alike: 320 tiles leave a quarter of the CUs with two, so 256 stay
// whole and the other 64 are split in four; splitting writes and reads the runs' sums once, and
// joining costs a launch. What is left for splitting are the shortest tiles: `step` keys fewer for
// every `alike` tiles of a head, the sequences being taken for alike. (A prompt's last tiles hold its first
// keys, and are not worth splitting.) Up to twice as many tiles are split as the estimate has, for calls
// whose sequences are not alike; the scratch is for those, kMaxParts at most. Where a sequence has no more than two
// tiles a head, its keys come from memory for each: a lone workgroup takes 1.25 times as long, two
// of a CU 1.12 (32 sequences of 40 tokens over 4000 keys in heads of 256: 256 tiles, whole 202 us, in two 170).
void split_many(int64_t per_head, int kv_heads, int kv, int all, int64_t alike, double step, int D, Plan *p) {
  Rates r = rates(D);
  if (per_head <= 2 * alike) r.key[0] *= 1.25, r.key[1] *= 1.12;
  const int64_t tiles = per_head * kv_heads;
  p->whole = (int)std::min<int64_t>(per_head, INT32_MAX), p->cut = 0, p->splits = 1;
  p->span = (kv + kBlockKeys - 1) / kBlockKeys * kBlockKeys;
  if (tiles > 256 * r.most * 3) return;          // the last round is short beside the others
  auto keys_of = [&](int64_t tile) { return (int)std::max(1.0, std::min<double>(kv, all - (double)(tile / alike) * step)); };
  const int64_t most = kMaxParts / ((int64_t)kv_heads * kManyRows * (D + 2) * 4);   // runs of a head's tiles in the scratch
  const int64_t full = tiles / 256, over = tiles - full * 256;
  double best = cu_time(r, (int)full, kv, over ? 1 : 0, keys_of(full * 256 / kv_heads));
  for (int pass = 0; pass < 2; ++pass) {
    const int64_t keep = pass ? full * 256 / kv_heads : 0, rest = tiles - keep * kv_heads;
    if ((pass && !keep) || rest <= 0) continue;
    const int left = keys_of(keep);
    for (int pieces = 1; pieces <= 12; ++pieces) {   // of a CU; as many runs as make no CU have more
      const int64_t n = std::min<int64_t>({64, pieces * 256 / rest, left / 128});
      if (n < 2) continue;
      const int run = (int)((left + n * kBlockKeys - 1) / (n * kBlockKeys) * kBlockKeys), runs = (left + run - 1) / run;
      if ((per_head - keep) * runs > most) continue;
      const double us = cu_time(r, (int)((keep * kv_heads + 255) / 256), kv, (int)((rest * runs + 255) / 256), run) + 5 +
                        (double)rest * runs * kManyRows * D * 8 / 4.2e6;
      if (us < best) best = us, p->whole = (int)keep, p->splits = runs, p->span = run;
    }
  }
  if (p->splits > 1) p->cut = (int)std::min({2 * (per_head - p->whole), p->slots - p->whole, most / p->splits});
}

Plan plan_of(int T, int B, int heads, int kv_heads, int D, int max_q, int max_kv, int window) {
  Plan p{};
  const int group = heads / kv_heads;
  const int64_t rows = (int64_t)max_q * group, all_rows = (int64_t)T * group;
  p.many = rows > kFewRows;
  // sequences of few rows beside long ones: their own kernel where they may be long in keys; up to
  // 2048, a tile of them takes no longer than its neighbours, and the launches it saves (the kernel's
  // and the join's) are 8 us. (One kernel and two, a chunk of 512 tokens beside 32 single ones of up to
  // 2000 keys, 27B heads: 94 us and 104, of up to 4000 230 and 158, heads of 128 93 and 82, 176 and 138;
  // beside 8 of up to 4000 91 and 111, a chunk of 2048 beside 32 of them 229 and 274: the keys alone do not decide.)
  p.few = !p.many || (B > 1 && (int64_t)B * max_q > T && max_kv > 2048);
  p.few_tiles = !p.many && rows <= 16 ? 1 : 2;
  const int few_rows = 16 * p.few_tiles;
  int kv = std::max(1, max_kv);
  if (window && window < kMaxPositions && window < kv) kv = (int)std::min<int64_t>(kv, (int64_t)window + max_q + kBlockKeys);
  p.splits = p.few_splits = 1;
  p.span = p.few_span = (kv + 127) / 128 * 128;
  if (p.few) {
    p.few_slots = (p.many ? 0 : all_rows / few_rows) + B;
    const int64_t per = std::max<int64_t>(1, (rows + few_rows - 1) / few_rows);
    split_few((p.many ? B : std::max(B * per, all_rows / few_rows)) * kv_heads, kv, D, &p.few_splits, &p.few_span);
  }
  if (p.many) {
    p.slots = all_rows / kManyRows + B;
    // tiles of a head, as if as many sequences as can had max_q new tokens
    const int64_t longest = std::min<int64_t>(max_q, T), alike = T / longest, tail = T - alike * longest;
    const int64_t per_head = alike * ((longest * group + kManyRows - 1) / kManyRows) + (tail * group + kManyRows - 1) / kManyRows;
    split_many(std::min(per_head, p.slots), kv_heads, kv, std::max(1, max_kv), alike, (double)kManyRows / group, D, &p);
  }
  // under 2^21 and 2^20 rows: split_few gives at most 511 workgroups and one a tile, split_many 2^20 rows of 64
  p.few_units = p.few_splits > 1 ? (int)(p.few_slots * kv_heads) : 0;
  p.many_units = p.cut * kv_heads;
  p.part_rows = (int64_t)p.few_units * p.few_splits * few_rows + (int64_t)p.many_units * p.splits * kManyRows;
  p.bytes = (size_t)p.part_rows * (D + 2) * sizeof(float) + (size_t)(p.few_units + p.many_units) * sizeof(int4);
  return p;
}

template <typename T, int D, int TERMS>
int launch_attn(const AttnArgs &a, const Plan &p, hipStream_t st) {
  const bool large_cap = a.cap_log2 > kSmallCap;
  if (p.few) {
    const int64_t grid = p.few_slots * a.c.kv_heads * p.few_splits;
    RLQ_REQUIRE(grid <= kMaxGrid, "rlq_attention: %lld workgroups are too many for a launch", (long long)grid);
    auto fn = p.few_tiles == 1 ? (large_cap ? few_rows_kernel<T, D, 1, true> : few_rows_kernel<T, D, 1, false>)
                               : (large_cap ? few_rows_kernel<T, D, 2, true> : few_rows_kernel<T, D, 2, false>);
    fn<<<(unsigned)grid, kThreads, 0, st>>>(a);
    RLQ_HIP(hipGetLastError());
  }
  if (p.many) {
    constexpr int lds = 2 * 2 * kTileKeys<D> * D * 2 + 64;
    const int64_t grid = (p.slots + (int64_t)p.cut * (p.splits - 1)) * a.c.kv_heads;
    RLQ_REQUIRE(grid <= kMaxGrid, "rlq_attention: %lld workgroups are too many for a launch", (long long)grid);
    static LdsOptIn opt[2];
    auto fn = large_cap ? many_rows_kernel<T, D, TERMS, true> : many_rows_kernel<T, D, TERMS, false>;
    if (int rc = allow_large_lds(reinterpret_cast<const void *>(fn), opt[large_cap])) return rc;
    fn<<<(unsigned)grid, kThreads, lds, st>>>(a);
    RLQ_HIP(hipGetLastError());
  }
  if (p.bytes) {
    const int64_t grid = ((int64_t)p.few_units * a.few_rows + (int64_t)p.many_units * kManyRows) / (kThreads / 64);
    RLQ_REQUIRE(grid <= kMaxGrid, "rlq_attention: %lld workgroups are too many for a launch", (long long)grid);
    join_runs_kernel<D><<<(unsigned)grid, kThreads, 0, st>>>(a);
    RLQ_HIP(hipGetLastError());
  }
  return 0;
}

template <typename T, int TERMS>
int launch_size(const AttnArgs &a, const Plan &p, int D, hipStream_t st) {
  if (D == 64) return launch_attn<T, 64, TERMS>(a, p, st);
  if (D == 128) return launch_attn<T, 128, TERMS>(a, p, st);
  return launch_attn<T, 256, TERMS>(a, p, st);
}

bool sizes_ok(int T, int B, int heads, int kv_heads, int D, int max_q, int max_kv, int window) {
  return T >= 0 && T <= (1 << 26) && B >= 0 && B <= (1 << 20) && kv_heads >= 1 && heads >= kv_heads &&
         heads % kv_heads == 0 && heads <= (1 << 20) && (int64_t)heads * D <= INT32_MAX && (int64_t)T * heads <= INT32_MAX / 2 && (D == 64 || D == 128 || D == 256) && max_q >= 0 &&
         max_kv >= 0 && max_kv <= kMaxPositions && window >= 0;
}

}  // namespace
}  // namespace rlq

extern "C" {

size_t rlq_attention_workspace_bytes(int T, int heads, int kv_heads, int D, int B, int max_q, int max_kv, int window) {
  if (!rlq::sizes_ok(T, B, heads, kv_heads, D, max_q, max_kv, window) || T == 0 || B == 0) return 0;
  return rlq::plan_of(T, B, heads, kv_heads, D, max_q, max_kv, window).bytes;
}

int rlq_attention(const void *q, int q_stride, int T, int heads, int kv_heads, int D, int dtype, const void *k_cache,
                  const void *v_cache, int n_pages, int page_size, const int *cu_q, const int *kv_len,
                  const int *table, int table_stride, int table_width, int B, int max_q, int max_kv, float scale,
                  int window, float softcap, void *out, int out_stride, int out_dtype, void *workspace,
                  size_t workspace_bytes, void *stream) {
  using namespace rlq;
  RLQ_REQUIRE(D == 64 || D == 128 || D == 256, "rlq_attention: head size %d is not 64, 128 or 256", D);
  RLQ_REQUIRE(dtype == RLQ_F16 || dtype == RLQ_BF16, "rlq_attention: unknown dtype %d", dtype);
  const bool full_weights = (out_dtype & RLQ_FULL_WEIGHTS) != 0;
  out_dtype &= ~RLQ_FULL_WEIGHTS;
  RLQ_REQUIRE(out_dtype == RLQ_F16 || out_dtype == RLQ_BF16, "rlq_attention: unknown output dtype %d", out_dtype);
  RLQ_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0,
              "rlq_attention: %d heads do not share %d key/value heads evenly", heads, kv_heads);
  RLQ_REQUIRE(page_size >= 32 && page_size % 32 == 0, "rlq_attention: page_size=%d is not a multiple of 32", page_size);
  RLQ_REQUIRE(n_pages >= 0 && table_width >= 0 && table_stride >= table_width,
              "rlq_attention: n_pages=%d, table_width=%d, table_stride=%d", n_pages, table_width, table_stride);
  RLQ_REQUIRE((int64_t)n_pages * kv_heads * (page_size / 32) <= INT32_MAX,
              "rlq_attention: a cache of %d pages of %d holds more than 2^31 blocks", n_pages, page_size);
  RLQ_REQUIRE((int64_t)table_width * page_size <= kMaxPositions,
              "rlq_attention: a table of %d pages of %d holds more than 2^29 positions", table_width, page_size);
  RLQ_REQUIRE(scale > 0 && scale * kLog2e < __builtin_inff(), "rlq_attention: scale=%g must be positive and under 2.3e38", scale);
  RLQ_REQUIRE(softcap >= 0 && softcap < __builtin_inff(), "rlq_attention: softcap=%g must be 0 or positive", softcap);
  RLQ_REQUIRE(sizes_ok(T, B, heads, kv_heads, D, max_q, max_kv, window),
              "rlq_attention: T=%d, B=%d, heads=%d, max_q=%d, max_kv=%d or window=%d is out of range", T, B, heads, max_q,
              max_kv, window);
  const float exp_cap = softcap > 0 ? 2.0f * kLog2e * scale / softcap : 0.0f;
  RLQ_REQUIRE(exp_cap < __builtin_inff(), "rlq_attention: scale=%g over softcap=%g passes fp32", scale, softcap);
  if (T == 0 || B == 0) return 0;
  RLQ_REQUIRE(q && out && cu_q && kv_len, "rlq_attention: null pointer");
  RLQ_REQUIRE((k_cache && v_cache) || n_pages == 0, "rlq_attention: null cache");
  RLQ_REQUIRE(table || table_width == 0, "rlq_attention: null table");
  RLQ_REQUIRE(q_stride >= heads * D && out_stride >= heads * D,
              "rlq_attention: a row stride (q %d, out %d) is shorter than %d heads of %d", q_stride, out_stride, heads, D);
  RLQ_REQUIRE(aligned(k_cache, 16) && aligned(v_cache, 16), "rlq_attention: the cache must be 16-byte aligned");
  const Plan p = plan_of(T, B, heads, kv_heads, D, max_q, max_kv, window);
  RLQ_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 16)),
              "rlq_attention: needs %zu bytes of 16-byte aligned workspace (got %zu)", p.bytes, workspace_bytes);
  AttnArgs a{};
  a.q = q, a.out = out;
  a.c = {const_cast<void *>(k_cache), const_cast<void *>(v_cache), cu_q, kv_len, table, n_pages, page_size / kBlockKeys,
         kv_heads, B, T, table_stride, table_width};
  a.q_stride = q_stride, a.out_stride = out_stride;
  if (p.bytes) {
    a.part = static_cast<float *>(workspace);
    a.part_stat = reinterpret_cast<float2 *>(a.part + p.part_rows * D);
    a.units = reinterpret_cast<int4 *>(a.part_stat + p.part_rows);
    a.few_units = p.few_units, a.many_units = p.many_units;
  }
  a.heads = heads, a.group = heads / kv_heads, a.window = window < kMaxPositions ? window : 0, a.out_bf16 = out_dtype == RLQ_BF16;
  a.q_wide = aligned(q, 16) && q_stride % 8 == 0;
  a.out_wide = aligned(out, 8) && out_stride % 4 == 0;
  a.whole = p.cut ? p.whole : INT32_MAX, a.cut = p.cut, a.splits = p.splits, a.span = p.span;
  a.few_splits = p.few_splits, a.few_span = p.few_span, a.few_rows = 16 * p.few_tiles;
  a.few = p.few, a.many = p.many;
  a.unit = softcap > 0 ? 1.0f : scale * kLog2e;
  if (softcap > 0) {
    constexpr float tanh_over_y[6] = {1.0f, -0.33333284f, 0.13331689f, -0.053768702f, 0.020753626f, -0.0058521652f};
    a.cap_log2 = std::min(softcap, 1e38f) * kLog2e;   // twice that is finite
    a.over_cap = scale / softcap, a.exp_cap = exp_cap;
    for (int i = 0; i < 6; ++i) a.near_cap[i] = tanh_over_y[i] * (scale * kLog2e);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool two = full_weights || (dtype == RLQ_BF16 && out_dtype == RLQ_F16);
  if (dtype == RLQ_F16) return two ? launch_size<_Float16, 2>(a, p, D, st) : launch_size<_Float16, 1>(a, p, D, st);
  return two ? launch_size<__bf16, 2>(a, p, D, st) : launch_size<__bf16, 1>(a, p, D, st);
}

}  // extern "C"
