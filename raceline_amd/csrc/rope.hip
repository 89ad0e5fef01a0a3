// Rotary positions and the write into the paged cache: what stands between a layer's stacked
// q/k/v linear (fp32 rows) and its attention. Plays the part of attn_prep
// (kernels/ops.metal:468-519: q/k RMS norm, RoPE, cache write) with both pair layouts, any number of
// rotated dimensions and frequencies scaled for long contexts.
#include "paged.h"
#include "../../include/rlq.h"

#include <cmath>

namespace rlq {
namespace {

constexpr int kRopeThreads = 256;

struct RopeArgs {
  const float *q, *k, *v;
  const double *freq;
  const float *q_norm, *k_norm;
  void *q_out;
  PagedCache c;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int heads, rot, interleaved, wide;   // wide: every row starts on 16 bytes
  int heads_per;                       // of a key/value head's query heads and its key, those of one workgroup
  float mscale, eps;
};

template <typename T>
struct Pack8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

template <typename T>
__device__ __forceinline__ typename Pack8<T>::type narrow8(const float (&x)[8]) {
  typename Pack8<T>::type r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = static_cast<T>(x[i]);
  return r;
}

__device__ __forceinline__ void load8(const float *p, bool wide, float (&x)[8]) {
  if (wide) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}

// One workgroup: the tokens of one sequence that fall into one block of 32 positions, and some (in
// small calls one, in large ones all) of the heads of one key/value head: the query heads that
// share it, then its key, with which go its values.
//   angle   a = pos * f, reduced to a fraction of a turn in 64 bits (a far position times a
//           32-bit frequency would be off by more than the rounding of the result), then
//           sincospi in 32; once per token and pair, kept in LDS for all heads.
//   values  transposed through LDS into runs of eight keys; a run that is only partly new is
//           written element by element, so that the other tokens' values stay.
// Bound by HBM for the most part: 2048 tokens of 20 + 2 * 4 heads of 256 (88 MB) in 19.7 us, where a plain
// conversion of as many numbers takes 16.7; 37 chunks of up to 300 tokens in heads of 128, all of them turned
// (213 MB), in 56 us and 38: a workgroup forms 2048 angles ahead of its stores there. Small calls take
// one head a workgroup, in the two cases measured 6.7 us against 9.4 with all heads (5 tokens of
// 16 + 2 * 4 heads) and 21.5 against 33 (that chunk, before a thread's items were stepped through
// without divisions); large ones all, so that angles are formed once (those 37 chunks 57.7 us, one head a
// workgroup 71.6).
template <typename T, int D>
__global__ __launch_bounds__(kRopeThreads) void rope_append_kernel(RopeArgs a) {
  constexpr int kChunks = D / 8, kRowStep = kRopeThreads / kChunks, kPad = D + 8;
  extern __shared__ float2 turn[];   // [32][rot / 2], then the values, [32][kPad]
  typedef typename Pack8<T>::type pack8;

  const int slot = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const Sequence s = find_sequence(a.c, slot, 1, kBlockKeys, 2);
  const int p0 = s.kv - s.tokens, block = (p0 >> 5) + s.item;
  const int first = max(p0, block * kBlockKeys), tokens = min(s.kv, (block + 1) * kBlockKeys) - first;
  if (s.b < 0 || tokens <= 0) return;
  const int row = s.row0 + first - p0, lane_key = first - block * kBlockKeys;
  const int at = block_at(a.c, s.b, head, block);

  const int group = a.heads / a.c.kv_heads, half = a.rot >> 1, chunk = tid % kChunks, d0 = chunk * 8;
  const int head0 = blockIdx.z * a.heads_per, heads = min(a.heads_per, group + 1 - head0);
  const bool with_key = head0 + heads == group + 1;
  T *vals = reinterpret_cast<T *>(turn + kBlockKeys * half);
  // a thread's items: head h (group: the key) of token t, kRowStep tokens on each time
  auto source = [&](int h, int t) {
    return h < group ? a.q + (row + t) * a.q_stride + (head * group + h) * D : a.k + (row + t) * a.k_stride + head * D;
  };
  int h = head0 + tid / kChunks / tokens, t = tid / kChunks % tokens;
  const float *src = source(h, t);
  float next[8] = {};
  if (h < head0 + heads) load8(src + d0, a.wide, next);
  for (int i = tid; i < tokens * half; i += kRopeThreads) {
    const int t = i / half, p = i - t * half;
    double x = (first + t) * (a.freq[p] * 0.15915494309189533577);   // turns
    x -= rint(x);
    float sin, cos;
    sincospif(2.0f * static_cast<float>(x), &sin, &cos);
    turn[t * half + p] = make_float2(cos * a.mscale, sin * a.mscale);
  }
  if (with_key) {
    for (int t = tid / kChunks; t < tokens; t += kRowStep) {
      float x[8];
      load8(a.v + (row + t) * a.v_stride + head * D + d0, a.wide, x);
      *reinterpret_cast<pack8 *>(vals + (lane_key + t) * kPad + d0) = narrow8<T>(x);
    }
  }
  __syncthreads();

  T *kb = at < 0 ? nullptr : static_cast<T *>(a.c.k) + static_cast<int64_t>(at) * (kBlockKeys * D);
  T *vb = at < 0 ? nullptr : static_cast<T *>(a.c.v) + static_cast<int64_t>(at) * (kBlockKeys * D);
  while (h < head0 + heads) {
    const bool is_q = h < group;
    const float *w = is_q ? a.q_norm : a.k_norm, *from = src;
    const int token = t, q_head = head * group + h;
    float x[8], r = 1.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = next[j];
    for (t += kRowStep; t >= tokens; t -= tokens) ++h;
    src = source(h, t);
    if (h < head0 + heads) load8(src + d0, a.wide, next);
    if (w) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
      for (int off = kChunks / 2; off; off >>= 1) ss += __shfl_xor(ss, off);
      r = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= r * w[d0 + j];
    }
    if (a.interleaved) {
      if (d0 < a.rot) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          if (d0 + j >= a.rot) break;
          const float2 cs = turn[token * half + ((d0 + j) >> 1)];
          const float u = x[j], v = x[j + 1];
          x[j] = u * cs.x - v * cs.y;
          x[j + 1] = u * cs.y + v * cs.x;
        }
      }
    } else if (d0 < a.rot) {
      const int step = half % 8 == 0 ? (d0 < half ? half / 8 : -(half / 8)) : 0;
      float o[8];
      if (step) {   // the partners are a whole chunk of another lane of this row
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = __shfl(x[j], (tid & 63) + step);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = d0 + j, e = d < half ? d + half : d - half;
          o[j] = d < a.rot ? from[e] * (w ? r * w[e] : 1.0f) : 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        if (d >= a.rot) break;
        const float2 cs = turn[token * half + (d < half ? d : d - half)];
        x[j] = d < half ? x[j] * cs.x - o[j] * cs.y : o[j] * cs.y + x[j] * cs.x;
      }
    }
    const pack8 y = narrow8<T>(x);
    if (is_q) {
      T *dst = static_cast<T *>(a.q_out) + (row + token) * a.out_stride + q_head * D + d0;
      if (a.wide) {
        *reinterpret_cast<pack8 *>(dst) = y;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[j] = y[j];
      }
    } else if (kb) {
      *reinterpret_cast<pack8 *>(kb + key_offset(lane_key + token, d0)) = y;
    }
  }
  if (!vb || !with_key) return;
  for (int i = tid; i < D * 4; i += kRopeThreads) {
    const int d = (i & 31) | ((i >> 7) << 5), t = (i >> 6) & 1, h = (i >> 5) & 1;
    T *dst = vb + value_run(d, t, h);
    pack8 y = {};
    int held = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = 16 * t + 8 * (e >> 2) + 4 * h + (e & 3);
      if (key >= lane_key && key < lane_key + tokens) {
        y[e] = vals[key * kPad + d];
        held |= 1 << e;
      }
    }
    if (held == 255) {
      *reinterpret_cast<pack8 *>(dst) = y;
    } else if (held) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (held >> e & 1) dst[e] = y[e];
    }
  }
}

template <typename T, int D>
int launch_size(RopeArgs a, hipStream_t st) {
  const int64_t blocks = a.c.rows / kBlockKeys + 2 * (int64_t)a.c.batch;
  const int group = a.heads / a.c.kv_heads;
  a.heads_per = blocks * a.c.kv_heads < 1024 ? 1 : group + 1;
  const dim3 grid((unsigned)blocks, (unsigned)a.c.kv_heads, (unsigned)((group + a.heads_per) / a.heads_per));
  const int lds = kBlockKeys * ((a.rot / 2) * (int)sizeof(float2) + (D + 8) * (int)sizeof(T));
  RLQ_REQUIRE(grid.z <= 65535, "rlq_rope_append: %d heads share a key/value head, more than 65534", group);
  rope_append_kernel<T, D><<<grid, kRopeThreads, lds, st>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}

template <typename T>
int launch_rope(const RopeArgs &a, int D, hipStream_t st) {
  if (D == 64) return launch_size<T, 64>(a, st);
  if (D == 128) return launch_size<T, 128>(a, st);
  return launch_size<T, 256>(a, st);
}

}  // namespace
}  // namespace rlq

extern "C" {

int rlq_rope_frequencies(int scaling, int rot, double base, double factor, double low, double high, double original,
                         double *freq) {
  RLQ_REQUIRE(freq && rot >= 0 && rot % 2 == 0, "rlq_rope_frequencies: rot=%d must be even, freq set", rot);
  RLQ_REQUIRE(scaling >= RLQ_ROPE_PLAIN && scaling <= RLQ_ROPE_PARTS, "rlq_rope_frequencies: unknown scaling %d",
              scaling);
  RLQ_REQUIRE(base > 1 && std::isfinite(base), "rlq_rope_frequencies: base=%g must be above 1", base);
  RLQ_REQUIRE(scaling == RLQ_ROPE_PLAIN || (factor >= 1 && std::isfinite(factor)),
              "rlq_rope_frequencies: factor=%g must be at least 1", factor);
  RLQ_REQUIRE(scaling != RLQ_ROPE_NTK || rot > 2 || rot == 0, "rlq_rope_frequencies: NTK scaling needs rot > 2");
  RLQ_REQUIRE(scaling != RLQ_ROPE_PARTS || (low >= 0 && high > low && std::isfinite(high) && original > 0 &&
                                            std::isfinite(original)),
              "rlq_rope_frequencies: parts needs 0 <= low < high and original > 0 (got %g, %g, %g)", low, high, original);
  const double b = scaling == RLQ_ROPE_NTK ? base * std::pow(factor, rot / (rot - 2.0)) : base;
  for (int i = 0; i < rot / 2; ++i) {
    double f = std::pow(b, -2.0 * i / rot);
    if (scaling == RLQ_ROPE_LINEAR) f /= factor;
    if (scaling == RLQ_ROPE_PARTS) {
      const double turns = original * f / (2 * M_PI);
      const double keep = std::fmin(1.0, std::fmax(0.0, (turns - low) / (high - low)));
      f = (1 - keep) * f / factor + keep * f;
    }
    freq[i] = f;
  }
  return 0;
}

int rlq_rope_append(const float *q, int q_stride, const float *k, int k_stride, const float *v, int v_stride, int T,
                    const double *freq, int rot, int interleaved, float mscale, const float *q_norm,
                    const float *k_norm, float eps, int heads, int kv_heads, int D, int dtype, void *q_out,
                    int q_out_stride, void *k_cache, void *v_cache, int n_pages, int page_size, const int *cu_q,
                    const int *kv_len, const int *table, int table_stride, int table_width, int B, void *stream) {
  RLQ_REQUIRE(T >= 0 && B >= 0, "rlq_rope_append: T=%d and B=%d must not be negative", T, B);
  RLQ_REQUIRE(D == 64 || D == 128 || D == 256, "rlq_rope_append: head size %d is not 64, 128 or 256", D);
  RLQ_REQUIRE(dtype == RLQ_F16 || dtype == RLQ_BF16, "rlq_rope_append: unknown dtype %d", dtype);
  RLQ_REQUIRE(kv_heads >= 1 && kv_heads <= 65535 && heads >= kv_heads && heads % kv_heads == 0,
              "rlq_rope_append: %d heads do not share %d key/value heads evenly", heads, kv_heads);
  RLQ_REQUIRE((int64_t)heads * D <= INT32_MAX, "rlq_rope_append: %d heads of %d are too many", heads, D);
  RLQ_REQUIRE(rot >= 0 && rot <= D && rot % 2 == 0, "rlq_rope_append: rot=%d must be even and at most %d", rot, D);
  RLQ_REQUIRE(page_size >= 32 && page_size % 32 == 0, "rlq_rope_append: page_size=%d is not a multiple of 32",
              page_size);
  RLQ_REQUIRE(n_pages >= 0 && table_width >= 0 && table_stride >= table_width,
              "rlq_rope_append: n_pages=%d, table_width=%d, table_stride=%d", n_pages, table_width, table_stride);
  RLQ_REQUIRE((int64_t)n_pages * kv_heads * (page_size / 32) <= INT32_MAX,
              "rlq_rope_append: a cache of %d pages of %d holds more than 2^31 blocks", n_pages, page_size);
  RLQ_REQUIRE((int64_t)table_width * page_size <= rlq::kMaxPositions,
              "rlq_rope_append: a table of %d pages of %d holds more than 2^29 positions", table_width, page_size);
  RLQ_REQUIRE(T <= (1 << 26) && B <= (1 << 20), "rlq_rope_append: T=%d or B=%d is too large", T, B);
  if (T == 0 || B == 0) return 0;
  RLQ_REQUIRE(q && k && v && q_out && cu_q && kv_len && (rot == 0 || freq), "rlq_rope_append: null pointer");
  RLQ_REQUIRE((k_cache && v_cache) || n_pages == 0, "rlq_rope_append: null cache");
  RLQ_REQUIRE(table || table_width == 0, "rlq_rope_append: null table");
  RLQ_REQUIRE(q_stride >= heads * D && q_out_stride >= heads * D && k_stride >= kv_heads * D &&
                  v_stride >= kv_heads * D,
              "rlq_rope_append: a row stride is shorter than the row (q %d, k %d, v %d, q_out %d)", q_stride, k_stride,
              v_stride, q_out_stride);
  RLQ_REQUIRE(rlq::aligned(k_cache, 16) && rlq::aligned(v_cache, 16), "rlq_rope_append: the cache must be 16-byte aligned");
  rlq::RopeArgs a{};
  a.q = q, a.k = k, a.v = v, a.freq = freq, a.q_norm = q_norm, a.k_norm = k_norm, a.q_out = q_out;
  a.c = {k_cache, v_cache, cu_q, kv_len, table, n_pages, page_size / 32, kv_heads, B, T, table_stride, table_width};
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.out_stride = q_out_stride;
  a.heads = heads, a.rot = rot, a.interleaved = interleaved, a.mscale = mscale, a.eps = eps;
  a.wide = rlq::aligned(q, 16) && rlq::aligned(k, 16) && rlq::aligned(v, 16) && rlq::aligned(q_out, 16) &&
           q_stride % 4 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0 && q_out_stride % 8 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == RLQ_F16 ? rlq::launch_rope<_Float16>(a, D, st) : rlq::launch_rope<__bf16>(a, D, st);
}

}  // extern "C"
