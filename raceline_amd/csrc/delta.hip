// The gated delta rule of a linear-attention layer: a state of Dk x Dv fp32 per sequence and value head,
// faded by each token and corrected towards its value at its key, and read at its query; the rows
// normalised and gated for the out projection. Plays the parts of lin_prep_qk, lin_gates, gated_delta and
// lin_out_norm (kernels/ops.metal:320,338,362,424, dispatched by src/engine.mm:1086-1154).
#include "paged.h"
#include "../../include/rlq.h"

#include <cmath>

namespace rlq {
namespace {

struct DeltaArgs {
  const void *q, *k, *v;
  const float *a, *b, *a_log, *dt_bias, *z, *norm;
  float *state;
  void *out;
  const int *slots, *keep;
  PagedCache c;   // rows and sequences alone
  int64_t q_stride, k_stride, v_stride, a_stride, b_stride, z_stride, out_stride;
  int k_heads, v_heads, dv, n_slots, wide;
  float eps, scale, norm_eps;
};

// log of a token's fade, -exp(a_log) softplus(a + dt_bias), and its weight, sigmoid(b).
__device__ __forceinline__ float log_fade(float a, float dt_bias, float rate) {
  const float x = a + dt_bias;
  return -rate * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
}

__device__ __forceinline__ float sigmoid(float x) {
  const float t = expf(-fabsf(x));
  return (x >= 0.0f ? 1.0f : t) / (1.0f + t);
}

// Sums over the lanes that differ in bits 3 to 5 (0 to 2) of their number; every lane gets the sum.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

__device__ __forceinline__ float sum_high(float x) {
  x += dpp<0x128>(x);   // row_ror:8
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float sum_low(float x) {
  x += dpp<0xB1>(x);    // quad_perm 1 0 3 2
  x += dpp<0x4E>(x);    // quad_perm 2 3 0 1
  return x + dpp<0x141>(x);   // row_half_mirror
}

template <typename T, int N>
__device__ __forceinline__ void load_narrow(const T *p, bool wide, float (&x)[N]) {
  typedef T pack __attribute__((ext_vector_type(N < 8 ? N : 8)));
  if (wide) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const pack v = *reinterpret_cast<const pack *>(p + i);
#pragma unroll
      for (int j = 0; j < 8 && j < N; ++j) x[i + j] = static_cast<float>(v[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = static_cast<float>(p[i]);
  }
}

// Token by token: S <- g S, d = beta (v - S^T k), S <- S + k d^T, o = S^T q, which is
//   p = S^T k, r = S^T q,  d = beta (v - g p),  o = g r + (k.q) d,  S <- g S + k d^T,
// so that both reads of the state go side by side. A workgroup takes one value head of one sequence, a
// wave 32 columns of its state: lane 8 i + c the rows i DK/8 .. and the columns 4 c .. 4 c + 3, in registers
// for all of the call's tokens. Sums over the rows go over the lanes of a column without LDS; only the norm of
// the output needs the other waves.
template <typename T, typename TO, int DK>
__global__ __launch_bounds__(512) void delta_tokens_kernel(DeltaArgs a) {
  constexpr int kRows = DK / 8;
  __shared__ float squares[2][8];
  const int b = blockIdx.x / a.v_heads, head = blockIdx.x - b * a.v_heads;
  const int row0 = row_start(a.c, b), n = row_start(a.c, b + 1) - row0;
  if (n <= 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k0 = (lane >> 3) * kRows, col = wave * 32 + (lane & 7) * 4;
  const int k_head = head / (a.v_heads / a.k_heads), slot = a.slots[b];
  const bool has_state = slot >= 0 && slot < a.n_slots;
  float *state = a.state + (has_state ? (static_cast<int64_t>(slot) * a.v_heads + head) * DK * a.dv + k0 * a.dv + col : 0);
  const int end = has_state ? (a.keep ? max(0, min(a.keep[b], n)) : n) : 0;

  float s[kRows][4];
  if (has_state && cached(a.c, b) > n) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const f32x4 x = *reinterpret_cast<const f32x4 *>(state + i * a.dv);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = x[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.0f;
  }
  const T *qp = static_cast<const T *>(a.q) + row0 * a.q_stride + k_head * DK + k0;
  const T *kp = static_cast<const T *>(a.k) + row0 * a.k_stride + k_head * DK + k0;
  const T *vp = static_cast<const T *>(a.v) + row0 * a.v_stride + head * a.dv + col;
  const float *ap = a.a + row0 * a.a_stride + head, *bp = a.b + row0 * a.b_stride + head;
  const float *zp = a.z ? a.z + row0 * a.z_stride + head * a.dv + col : nullptr;
  TO *op = static_cast<TO *>(a.out) + row0 * a.out_stride + head * a.dv + col;
  const float rate = expf(a.a_log[head]), dt_bias = a.dt_bias[head];
  float w[4] = {};
  if (zp) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = a.norm[col + e];
  }
  for (int t = 0; t < n; ++t) {
    float q[kRows], k[kRows], v[4], z[4];
    load_narrow<T, kRows>(qp + t * a.q_stride, a.wide, q);
    load_narrow<T, kRows>(kp + t * a.k_stride, a.wide, k);
    load_narrow<T, 4>(vp + t * a.v_stride, a.wide, v);
    if (zp) {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = zp[t * a.z_stride + e];
    }
    const float fade = expf(log_fade(ap[t * a.a_stride], dt_bias, rate)), beta = sigmoid(bp[t * a.b_stride]);
    // to length 1 before the products: those of raw rows with a state could pass fp32
    float kk = 0.0f, qq = 0.0f, kq = 0.0f, p[4] = {}, r[4] = {};
#pragma unroll
    for (int i = 0; i < kRows; ++i) kk += k[i] * k[i], qq += q[i] * q[i];
    const float rk = 1.0f / sqrtf(sum_high(kk) + a.eps), rq = a.scale / sqrtf(sum_high(qq) + a.eps);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      k[i] *= rk;
      q[i] *= rq;
      kq += k[i] * q[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] += s[i][e] * k[i];
        r[e] += s[i][e] * q[i];
      }
    }
    kq = sum_high(kq);
    float o[4], d[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[e] = beta * (v[e] - fade * sum_high(p[e]));
      o[e] = fade * sum_high(r[e]) + kq * d[e];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = fade * s[i][e] + k[i] * d[e];
    if (t + 1 == end) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        *reinterpret_cast<f32x4 *>(state + i * a.dv) = f32x4{s[i][0], s[i][1], s[i][2], s[i][3]};
    }
    if (zp) {
      const float mine = sum_low(o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3]);
      if (lane == 0) squares[t & 1][wave] = mine;
      __syncthreads();          // the other half is free: its last readers are past the barrier before
      float sum = 0.0f;
      for (int i = 0; i < a.dv / 32; ++i) sum += squares[t & 1][i];
      const float r = 1.0f / sqrtf(sum / a.dv + a.norm_eps);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o[e] * r * w[e] * (z[e] * sigmoid(z[e]));
    }
    if (lane < 8) {
      if (a.wide) {
        typedef TO pack4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<pack4 *>(op + t * a.out_stride) =
            pack4{static_cast<TO>(o[0]), static_cast<TO>(o[1]), static_cast<TO>(o[2]), static_cast<TO>(o[3])};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) op[t * a.out_stride + e] = static_cast<TO>(o[e]);
      }
    }
  }
}

template <typename T, typename TO>
int launch_delta(const DeltaArgs &a, int DK, hipStream_t st) {
  const unsigned grid = (unsigned)a.c.batch * (unsigned)a.v_heads;
  if (DK == 64) delta_tokens_kernel<T, TO, 64><<<grid, a.dv * 2, 0, st>>>(a);
  else delta_tokens_kernel<T, TO, 128><<<grid, a.dv * 2, 0, st>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace rlq

extern "C" {

size_t rlq_gated_delta_workspace_bytes(int T, int k_heads, int v_heads, int Dk, int Dv, int B, int max_q) {
  return 0;
}

int rlq_gated_delta(const void *q, int q_stride, const void *k, int k_stride, const void *v, int v_stride, int T,
                    int k_heads, int v_heads, int Dk, int Dv, int dtype, const float *a, int a_stride, const float *b,
                    int b_stride, const float *a_log, const float *dt_bias, float eps, float scale, const float *z,
                    int z_stride, const float *norm, float norm_eps, float *state, int n_slots, const int *cu_q,
                    const int *kv_len, const int *slots, const int *keep, int B, int max_q, void *out, int out_stride,
                    int out_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  RLQ_REQUIRE(T >= 0 && B >= 0, "rlq_gated_delta: T=%d and B=%d must not be negative", T, B);
  RLQ_REQUIRE(T <= (1 << 26) && B <= (1 << 20), "rlq_gated_delta: T=%d or B=%d is too large", T, B);
  RLQ_REQUIRE(Dk == 64 || Dk == 128, "rlq_gated_delta: key size %d is not 64 or 128", Dk);
  RLQ_REQUIRE(Dv == 64 || Dv == 128 || Dv == 256, "rlq_gated_delta: value size %d is not 64, 128 or 256", Dv);
  RLQ_REQUIRE(dtype == RLQ_F16 || dtype == RLQ_BF16, "rlq_gated_delta: unknown dtype %d", dtype);
  RLQ_REQUIRE(out_dtype == RLQ_F16 || out_dtype == RLQ_BF16, "rlq_gated_delta: unknown output dtype %d", out_dtype);
  RLQ_REQUIRE(k_heads >= 1 && v_heads >= k_heads && v_heads % k_heads == 0 && v_heads <= 65535,
              "rlq_gated_delta: %d value heads do not share %d key heads evenly", v_heads, k_heads);
  RLQ_REQUIRE((int64_t)v_heads * Dv <= INT32_MAX && (int64_t)B * v_heads <= INT32_MAX,
              "rlq_gated_delta: %d heads of %d sequences are too many", v_heads, B);
  RLQ_REQUIRE(eps > 0 && std::isfinite(eps), "rlq_gated_delta: eps=%g must be above 0", eps);
  RLQ_REQUIRE(std::isfinite(scale), "rlq_gated_delta: scale=%g", scale);
  RLQ_REQUIRE((z == nullptr) == (norm == nullptr), "rlq_gated_delta: z and norm come together");
  RLQ_REQUIRE(!norm || (norm_eps > 0 && std::isfinite(norm_eps)), "rlq_gated_delta: norm_eps=%g must be above 0", norm_eps);
  RLQ_REQUIRE(n_slots >= 0 && max_q >= 0, "rlq_gated_delta: n_slots=%d, max_q=%d", n_slots, max_q);
  if (T == 0 || B == 0) return 0;
  RLQ_REQUIRE(q && k && v && a && b && a_log && dt_bias && out && cu_q && kv_len && slots, "rlq_gated_delta: null pointer");
  RLQ_REQUIRE((state && rlq::aligned(state, 16)) || n_slots == 0, "rlq_gated_delta: the state must be set and 16-byte aligned");
  RLQ_REQUIRE(q_stride >= k_heads * Dk && k_stride >= k_heads * Dk && v_stride >= v_heads * Dv && a_stride >= v_heads &&
                  b_stride >= v_heads && out_stride >= v_heads * Dv && (!z || z_stride >= v_heads * Dv),
              "rlq_gated_delta: a row stride is shorter than the row (q %d, k %d, v %d, a %d, b %d, z %d, out %d)", q_stride,
              k_stride, v_stride, a_stride, b_stride, z_stride, out_stride);
  rlq::DeltaArgs x{};
  x.q = q, x.k = k, x.v = v, x.a = a, x.b = b, x.a_log = a_log, x.dt_bias = dt_bias, x.z = z, x.norm = norm;
  x.state = state, x.out = out, x.slots = slots, x.keep = keep;
  x.c.cu_q = cu_q, x.c.kv_len = kv_len, x.c.batch = B, x.c.rows = T;
  x.q_stride = q_stride, x.k_stride = k_stride, x.v_stride = v_stride, x.a_stride = a_stride, x.b_stride = b_stride;
  x.z_stride = z_stride, x.out_stride = out_stride;
  x.k_heads = k_heads, x.v_heads = v_heads, x.dv = Dv, x.n_slots = n_slots;
  x.eps = eps, x.scale = scale, x.norm_eps = norm_eps;
  x.wide = rlq::aligned(q, 16) && rlq::aligned(k, 16) && rlq::aligned(v, 16) && rlq::aligned(out, 8) &&
           q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && out_stride % 4 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == RLQ_F16) {
    return out_dtype == RLQ_F16 ? rlq::launch_delta<_Float16, _Float16>(x, Dk, st) : rlq::launch_delta<_Float16, __bf16>(x, Dk, st);
  }
  return out_dtype == RLQ_F16 ? rlq::launch_delta<__bf16, _Float16>(x, Dk, st) : rlq::launch_delta<__bf16, __bf16>(x, Dk, st);
}

}  // extern "C"
