// The short causal convolution of a linear-attention layer: every channel of the in projection's fp32
// rows with its own few taps, a SiLU, and the last inputs of each sequence kept as its state. Plays the
// part of lin_conv (kernels/ops.metal:281, dispatched by src/engine.mm:1086-1154).
#include "paged.h"
#include "../../include/rlq.h"

namespace rlq {
namespace {

constexpr int kConvThreads = 64, kMaxTaps = 4, kLongRun = 16, kShortRun = 4, kManyWaves = 2048;

struct ConvArgs {
  const float *x, *w, *bias;
  float *state;
  void *out;
  const int *slots, *keep;
  PagedCache c;   // rows and sequences alone
  int64_t x_stride, out_stride;
  int channels, silu, n_slots;
};

template <int VEC>
struct Floats {
  float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Floats<VEC> load_floats(const float *p) {
  Floats<VEC> r;
  if constexpr (VEC == 4) {
    const f32x4 x = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = x[e];
  } else {
    r.v[0] = *p;
  }
  return r;
}

template <int VEC>
__device__ __forceinline__ void store_floats(float *p, const Floats<VEC> &x) {
  if constexpr (VEC == 4) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{x.v[0], x.v[1], x.v[2], x.v[3]};
  } else {
    *p = x.v[0];
  }
}

// y_t = act(bias + sum_j w[j] x_{t - (TAPS-1) + j}), summed in fp32 in the order of the taps.
// A thread takes VEC neighbouring channels of one sequence over a run of tokens, whose inputs slide
// through its registers; the run in front is read again for TAPS - 1 rows. The state is read and
// written by the threads of a sequence's first run alone, so no other has to be waited for.
// Bound by HBM in long calls (2048 rows of 8192 channels, 101 MB, in 21 us, 4.8 TB/s; a plain conversion of as many
// numbers takes 14.8), by a launch and two dependent loads in small ones (one token 3.1 us).
template <typename T, int TAPS, int VEC, int RUN>
__global__ __launch_bounds__(kConvThreads) void causal_conv_kernel(ConvArgs a) {
  const Sequence s = find_sequence(a.c, blockIdx.x, 1, RUN, 1);
  const int t0 = s.item * RUN, tokens = min(s.tokens - t0, RUN);
  const int c0 = (blockIdx.y * kConvThreads + threadIdx.x) * VEC;
  if (s.b < 0 || tokens <= 0 || c0 >= a.channels) return;
  const float *x = a.x + s.row0 * a.x_stride + c0;
  const int slot = a.slots[s.b];
  const bool has_state = slot >= 0 && slot < a.n_slots;
  float *state = a.state + (has_state ? static_cast<int64_t>(slot) * (TAPS - 1) * a.channels + c0 : 0);

  // no branch stands between the loads, so all are on their way at once: behind a short run its last row comes
  // again, in front of a sequence without a state its first
  Floats<VEC> in[TAPS - 1 + RUN];
  const bool begins = t0 == 0, from_state = begins && has_state && s.kv > s.tokens;
  const float *before = from_state ? state : begins ? x : x + (t0 - (TAPS - 1)) * a.x_stride;   // a run is longer than the taps
  const int64_t step = from_state ? a.channels : begins ? 0 : a.x_stride;
#pragma unroll
  for (int j = 0; j < TAPS - 1; ++j) in[j] = load_floats<VEC>(before + j * step);
#pragma unroll
  for (int i = 0; i < RUN; ++i) in[TAPS - 1 + i] = load_floats<VEC>(x + (t0 + min(i, tokens - 1)) * a.x_stride);
  float w[VEC][TAPS], bias[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    bias[e] = a.bias ? a.bias[c0 + e] : 0.0f;
    if constexpr (TAPS == 4 && VEC == 4) {
      const f32x4 v = *reinterpret_cast<const f32x4 *>(a.w + (c0 + e) * static_cast<int64_t>(TAPS));
#pragma unroll
      for (int j = 0; j < TAPS; ++j) w[e][j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < TAPS; ++j) w[e][j] = a.w[(c0 + e) * static_cast<int64_t>(TAPS) + j];
    }
  }
  __builtin_amdgcn_sched_barrier(0);   // the compiler would put each load in front of its use
  if (begins && !from_state) {
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) in[j] = {};
  }
  if (begins && has_state) {
    // after `end` tokens: inputs end - (TAPS-1) .. end - 1, from the old state where that is negative
    const int end = a.keep ? max(0, min(a.keep[s.b], s.tokens)) : s.tokens;
    if (end) {
      Floats<VEC> now[TAPS - 1];
#pragma unroll
      for (int j = 0; j < TAPS - 1; ++j) {
        const int at = end - (TAPS - 1) + j;
        if (at >= 0) {
          now[j] = load_floats<VEC>(x + at * a.x_stride);
        } else {
#pragma unroll
          for (int i = 0; i < TAPS - 1; ++i)
            if (at + TAPS - 1 == i) now[j] = in[i];
        }
      }
#pragma unroll
      for (int j = 0; j < TAPS - 1; ++j) store_floats<VEC>(state + static_cast<int64_t>(j) * a.channels, now[j]);
    }
  }
  const bool silu = a.silu;
  T *out = static_cast<T *>(a.out) + (s.row0 + t0) * a.out_stride + c0;
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    T y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float sum = bias[e];
#pragma unroll
      for (int j = 0; j < TAPS; ++j) sum += w[e][j] * in[i + j].v[e];
      // at most 1: no overflow on either side; formed for every row, so that no branch stands between them
      const float t = __expf(-fabsf(sum)), f = (sum >= 0.0f ? 1.0f : t) * __builtin_amdgcn_rcpf(1.0f + t);
      y[e] = static_cast<T>(sum * (silu ? f : 1.0f));
    }
    if (i >= tokens) continue;
    if constexpr (VEC == 4) {
      typedef T pack4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<pack4 *>(out + i * a.out_stride) = pack4{y[0], y[1], y[2], y[3]};
    } else {
      out[i * a.out_stride] = y[0];
    }
  }
}

template <typename T, int TAPS, int VEC, int RUN>
int launch_run(const ConvArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(a.c.rows / RUN + a.c.batch), (unsigned)((a.channels + kConvThreads * VEC - 1) / (kConvThreads * VEC)));
  RLQ_REQUIRE(grid.y <= 65535, "rlq_causal_conv: %d channels are too many", a.channels);
  causal_conv_kernel<T, TAPS, VEC, RUN><<<grid, kConvThreads, 0, st>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}

// A run reads the taps - 1 rows in front again, so longer ones read less: 16 tokens (2048 rows: 56 us where a wave's loads
// waited for one another, 20.9 with all on their way; runs of 8 21.6, of 32 22.1, their registers). Where runs of 16 are
// fewer than 2048 waves, 4 tokens: 24 drafts of five rows 5.2 us, 10.3 in runs of 16.
template <typename T, int TAPS, int VEC>
int launch_conv(const ConvArgs &a, hipStream_t st) {
  const int64_t waves = (int64_t)a.c.rows / kLongRun * ((a.channels + kConvThreads * VEC - 1) / (kConvThreads * VEC));
  return waves >= kManyWaves ? launch_run<T, TAPS, VEC, kLongRun>(a, st) : launch_run<T, TAPS, VEC, kShortRun>(a, st);
}

template <typename T>
int launch_taps(const ConvArgs &a, int taps, bool wide, hipStream_t st) {
  if (taps == 2) return wide ? launch_conv<T, 2, 4>(a, st) : launch_conv<T, 2, 1>(a, st);
  if (taps == 3) return wide ? launch_conv<T, 3, 4>(a, st) : launch_conv<T, 3, 1>(a, st);
  return wide ? launch_conv<T, 4, 4>(a, st) : launch_conv<T, 4, 1>(a, st);
}

}  // namespace
}  // namespace rlq

extern "C" int rlq_causal_conv(const float *x, int x_stride, int T, int channels, int taps, const float *w,
                               const float *bias, int silu, float *state, int n_slots, const int *cu_q,
                               const int *kv_len, const int *slots, const int *keep, int B, void *out, int out_stride,
                               int out_dtype, void *stream) {
  RLQ_REQUIRE(T >= 0 && B >= 0, "rlq_causal_conv: T=%d and B=%d must not be negative", T, B);
  RLQ_REQUIRE(T <= (1 << 26) && B <= (1 << 20), "rlq_causal_conv: T=%d or B=%d is too large", T, B);
  RLQ_REQUIRE(channels >= 1, "rlq_causal_conv: channels=%d", channels);
  RLQ_REQUIRE(taps >= 2 && taps <= rlq::kMaxTaps, "rlq_causal_conv: taps=%d is not in 2 .. %d", taps, rlq::kMaxTaps);
  RLQ_REQUIRE(out_dtype == RLQ_F16 || out_dtype == RLQ_BF16, "rlq_causal_conv: unknown output dtype %d", out_dtype);
  RLQ_REQUIRE(n_slots >= 0, "rlq_causal_conv: n_slots=%d", n_slots);
  if (T == 0 || B == 0) return 0;
  RLQ_REQUIRE(x && w && out && cu_q && kv_len && slots, "rlq_causal_conv: null pointer");
  RLQ_REQUIRE(state || n_slots == 0, "rlq_causal_conv: null state");
  RLQ_REQUIRE(x_stride >= channels && out_stride >= channels,
              "rlq_causal_conv: a row stride is shorter than the row (x %d, out %d)", x_stride, out_stride);
  rlq::ConvArgs a{};
  a.x = x, a.w = w, a.bias = bias, a.state = state, a.out = out, a.slots = slots, a.keep = keep;
  a.c.cu_q = cu_q, a.c.kv_len = kv_len, a.c.batch = B, a.c.rows = T;
  a.x_stride = x_stride, a.out_stride = out_stride, a.channels = channels, a.silu = silu, a.n_slots = n_slots;
  const bool wide = rlq::aligned(x, 16) && rlq::aligned(w, 16) && rlq::aligned(state, 16) && rlq::aligned(out, 8) &&
                    x_stride % 4 == 0 && out_stride % 4 == 0 && channels % 4 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return out_dtype == RLQ_F16 ? rlq::launch_taps<_Float16>(a, taps, wide, st) : rlq::launch_taps<__bf16>(a, taps, wide, st);
}
