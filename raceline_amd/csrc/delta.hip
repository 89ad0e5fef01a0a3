// The gated delta rule of a linear-attention layer: a state of Dk x Dv fp32 per sequence and value head,
// faded by each token and corrected towards its value at its key, and read at its query; the rows
// normalised and gated for the out projection. Plays the parts of lin_prep_qk, lin_gates, gated_delta and
// lin_out_norm (kernels/ops.metal:320,338,362,424, dispatched by src/engine.mm:1086-1154).
#include "lanes.h"
#include "paged.h"
#include "../../include/rlq.h"

#include <algorithm>
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
  int k_heads, v_heads, dv, n_slots, wide, wide_z;
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

// z sigmoid(z), to a few roundings of fp32: the rows it gates are rounded to 16 bits.
__device__ __forceinline__ float gate_of(float z) {
  const float t = __expf(-fabsf(z));
  return z * ((z >= 0.0f ? 1.0f : t) * __builtin_amdgcn_rcpf(1.0f + t));
}

// The squares of a row of 2^64 pass fp32: where their mean and eps did, they are formed again of the row made smaller by this
// (and eps by its square, which is no float).
constexpr float kSmaller = 0x1p-96f;

template <typename T, int N>
__device__ __forceinline__ void load_row(const T *p, bool wide, T (&x)[N]) {
  constexpr int kPack = N < 8 ? N : 8;
  typedef T pack __attribute__((ext_vector_type(kPack)));
  if (wide) {
#pragma unroll
    for (int i = 0; i < N; i += kPack) {
      const pack v = *reinterpret_cast<const pack *>(p + i);
#pragma unroll
      for (int j = 0; j < kPack; ++j) x[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = p[i];
  }
}

// Token by token: S <- g S, d = beta (v - S^T k), S <- S + k d^T, o = S^T q, which is
//   p = S^T k, r = S^T q,  d = beta (v - g p),  o = g r + (k.q) d,  S <- g S + k d^T,
// so that both reads of the state go side by side. A workgroup takes one value head of one sequence, a
// wave 32 columns of its state: lane 8 i + c the rows i DK/8 .. and the columns 4 c .. 4 c + 3, in registers
// for all of the call's tokens; sums over the rows go over the lanes of a column without LDS. What does not depend on
// the state goes beside it, eight tokens at a time: keys and queries to length 1, a token a wave, before; the norm of
// the rows and their gate, four values a thread, behind.
// Bound by HBM for many sequences (48 of 32 heads of 128 x 128: 203 MB in 43.9 us, 4.6 TB/s), else by a token's 1 us, of which
// half is the issue of its work on 64 elements a lane (VALU share 0.45 at one wave a SIMD) and half the chain of its sums (one token
// 6.8 us, nine drafts of five 10.5).
template <typename T, typename TO, int DK>
__global__ __launch_bounds__(512) void delta_tokens_kernel(DeltaArgs a) {
  constexpr int kRows = DK / 8, kOf = DK / 64, kBatch = 8, kMostDv = 256;
  __shared__ __align__(16) float ks[kBatch][DK], qs[kBatch][DK], vs[kBatch][kMostDv], os[kBatch][kMostDv];
  __shared__ float squares[kBatch][kMostDv / 32], kqs[kBatch];
  const int b = blockIdx.x / a.v_heads, head = blockIdx.x - b * a.v_heads;
  const int row0 = row_start(a.c, b), n = row_start(a.c, b + 1) - row0;
  if (n <= 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = a.dv / 32;
  const int k0 = (lane >> 3) * kRows, col = wave * 32 + (lane & 7) * 4;
  const int k_head = head / (a.v_heads / a.k_heads), slot = a.slots[b];
  const bool has_state = slot >= 0 && slot < a.n_slots;
  float *state = a.state + (has_state ? (static_cast<int64_t>(slot) * a.v_heads + head) * DK * a.dv + k0 * a.dv + col : 0);
  const int end = has_state ? (a.keep ? max(0, min(a.keep[b], n)) : n) : 0;

  const float *ap = a.a + row0 * a.a_stride + head, *bp = a.b + row0 * a.b_stride + head;
  float fades = ap[min(lane, n - 1) * a.a_stride], betas = bp[min(lane, n - 1) * a.b_stride];   // of 64 tokens, one a lane
  float s[kRows][4];
  const T *qp = static_cast<const T *>(a.q) + row0 * a.q_stride + k_head * DK;
  const T *kp = static_cast<const T *>(a.k) + row0 * a.k_stride + k_head * DK;
  const float rate = expf(a.a_log[head]), dt_bias = a.dt_bias[head];
  // a thread's token of eight, and four of its values
  const int quads = a.dv / 4, mine = tid / quads, at = (tid - mine * quads) * 4;
  const T *vp = static_cast<const T *>(a.v) + row0 * a.v_stride + head * a.dv + at;
  const float *zp = a.z ? a.z + row0 * a.z_stride + head * a.dv + at : nullptr;
  TO *op = static_cast<TO *>(a.out) + row0 * a.out_stride + head * a.dv + at;
  f32x4 w = {};
  if (zp) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = a.norm[at + e];
  }
  for (int t0 = 0; t0 < n; t0 += kBatch) {
    const int m = min(kBatch, n - t0);
    if (t0) lds_barrier();               // the rows in front have been read
    // loads return in order: the rows first, whose work then goes beside the state's arrival
    const int token = t0 + min(mine, m - 1);
    f32x4 z = {};
    T v[4], qr[kOf], kr[kOf];
    auto fetch = [&](int t) {
      load_row<T, kOf>(qp + (t0 + t) * a.q_stride + lane * kOf, a.wide, qr);
      load_row<T, kOf>(kp + (t0 + t) * a.k_stride + lane * kOf, a.wide, kr);
    };
    fetch(min(wave, m - 1));
    load_row<T, 4>(vp + token * a.v_stride, a.wide, v);
    if (zp) {
      const float *from = zp + token * a.z_stride;
      if (a.wide_z) z = *reinterpret_cast<const f32x4 *>(from);
      else z = f32x4{from[0], from[1], from[2], from[3]};
    }
    if (t0 == 0) {
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
    }
    if (mine < m) {
      *reinterpret_cast<f32x4 *>(&vs[mine][at]) = f32x4{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]),
                                                        static_cast<float>(v[3])};
    }
    for (int t = wave; t < m; t += waves) {
      if (t != wave) fetch(t);
      float kk = 0.0f, qq = 0.0f, kq = 0.0f, k[kOf], q[kOf];
#pragma unroll
      for (int i = 0; i < kOf; ++i) {
        k[i] = static_cast<float>(kr[i]), q[i] = static_cast<float>(qr[i]);
        kk += k[i] * k[i], qq += q[i] * q[i];
      }
      // to length 1 before the products: those of raw rows could pass fp32
      const float rk = __builtin_amdgcn_rsqf(sum_high(sum_low(kk)) + a.eps);
      const float rq = a.scale * __builtin_amdgcn_rsqf(sum_high(sum_low(qq)) + a.eps);
#pragma unroll
      for (int i = 0; i < kOf; ++i) {
        k[i] *= rk, q[i] *= rq;
        kq += k[i] * q[i];
        ks[t][lane * kOf + i] = k[i];
        qs[t][lane * kOf + i] = q[i];
      }
      kq = sum_high(sum_low(kq));
      if (lane == 0) kqs[t] = kq;
    }
    if ((t0 & 63) == 0) {
      if (t0) fades = ap[min(t0 + lane, n - 1) * a.a_stride], betas = bp[min(t0 + lane, n - 1) * a.b_stride];
      fades = expf(log_fade(fades, dt_bias, rate));
      betas = sigmoid(betas);
    }
    lds_barrier();
    for (int t = 0; t < m; ++t) {
      const float fade = __uint_as_float(of_lane(__float_as_uint(fades), t0 + t & 63));
      const float beta = __uint_as_float(of_lane(__float_as_uint(betas), t0 + t & 63));
      float k[kRows], q[kRows], p[4] = {}, r[4] = {};
#pragma unroll
      for (int i = 0; i < kRows; i += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(&ks[t][k0 + i]), y = *reinterpret_cast<const f32x4 *>(&qs[t][k0 + i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) k[i + e] = x[e], q[i + e] = y[e];
      }
      const f32x4 v = *reinterpret_cast<const f32x4 *>(&vs[t][col]);
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] += s[i][e] * k[i];
          r[e] += s[i][e] * q[i];
        }
      const float kq = kqs[t];
      f32x4 o;
      float d[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d[e] = beta * (v[e] - fade * sum_high(p[e]));
        o[e] = fade * sum_high(r[e]) + kq * d[e];
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = fade * s[i][e] + k[i] * d[e];
      if (lane < 8) *reinterpret_cast<f32x4 *>(&os[t][col]) = o;
      const float sum = sum_low(o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3]);
      if (lane == 0) squares[t][wave] = sum;
      if (t0 + t + 1 == end) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          *reinterpret_cast<f32x4 *>(state + i * a.dv) = f32x4{s[i][0], s[i][1], s[i][2], s[i][3]};
      }
    }
    lds_barrier();
    if (mine < m) {
      f32x4 o = *reinterpret_cast<const f32x4 *>(&os[mine][at]);
      if (zp) {
        float sum = 0.0f;
        for (int i = 0; i < waves; ++i) sum += squares[mine][i];
        float square = sum * (1.0f / a.dv) + a.norm_eps;
        if (square == __builtin_inff()) {
          sum = 0.0f, o *= kSmaller;
          for (int i = 0; i < a.dv; ++i) {
            const float x = os[mine][i] * kSmaller;
            sum += x * x;
          }
          square = sum * (1.0f / a.dv) + a.norm_eps * kSmaller * kSmaller;
        }
        const float r = __builtin_amdgcn_rsqf(square);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * r * w[e] * gate_of(z[e]);
      }
      TO *to = op + (t0 + mine) * a.out_stride;
      if (a.wide) {
        typedef TO pack4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<pack4 *>(to) =
            pack4{static_cast<TO>(o[0]), static_cast<TO>(o[1]), static_cast<TO>(o[2]), static_cast<TO>(o[3])};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = static_cast<TO>(o[e]);
      }
    }
  }
}

// ------------------------------------------------------------------ chunks of 64 tokens

// The published triangular (WY) form of the rule. With G_i the sum of log g up to row i of a chunk,
// L_ij = beta_i e^(G_i - G_j) k_i.k_j below the diagonal and S the state in front of the chunk, the rule over the chunk's rows is
//   R = beta (V - e^G (K S)),   U = (I + L)^-1 R,
//   O = e^G (Q S) + P U,        P_ij = e^(G_i - G_j) q_i.k_j on and below the diagonal,
//   S <- e^(G_64) S + (e^(G_64 - G) K)^T U.
// delta_chunks_kernel forms what does not depend on S, of all chunks at once: T = (I + L)^-1, P, and the rows
// as operands. delta_chain_kernel goes through a sequence's chunks with S. A 2048-token chunk of a prompt, 16 key and 32
// value heads of 128: 24 + 50 us, and 17 for the rows' norm and gate; token by token it took 5870.
//
// The products are to keep the state to fp32: rows of q and k, brought to a length of 2^13 .. 2^14 by a power of
// two, are exact in fp16 (what bf16 loses there lies 2^-38 below the length); T, P, R, U and S are two fp16
// terms (2^-22), T, at most 1, times 2^14, and P before the length of q is taken out, so that what has faded
// keeps its bits. Operands stand in the order in which sums leave the matrix cores: slot 8 h + 4 a + b of a step of
// 32 is row 16 a + 4 h + b, so that what a lane holds of a result is what it holds of the next product.

constexpr int kChunk = 64, kGateThreads = 256, kHeadsPer = 2, kPrepareThreads = 256 * kHeadsPer, kMatPad = 68;
constexpr int kBlock = 64 * 8;                       // halves of a 16 x 32 operand
constexpr float kUnit = 16384.0f, kLength = 8192.0f; // T is held times kUnit, rows of q and k at this length or twice it
// Under the last-level cache (256 MB) beside the rows that come and go, in runs of even length: a 32768-token prompt of
// 32 heads takes 1465 us with 256 MB at a time, 1339 with 192, 1351 with 160; one of 8192 374, 342 and 362.
constexpr int64_t kMostScratch = 192 << 20;

// What a chunk leaves for the chain, in bytes from its place.
struct ChunkLayout {
  int dk, k_heads, v_heads, dv;
  __host__ __device__ int64_t k_head() const { return 3 * kChunk * dk * 2; }       // K, Q, K^T
  __host__ __device__ int64_t v_head() const { return 4 * 8 * kBlock * 2 + 6 * kChunk * 4; }   // T, P (two terms), factors
  __host__ __device__ int64_t rows_at() const { return k_heads * k_head() + v_heads * v_head(); }
  __host__ __device__ int64_t bytes() const { return rows_at() + (int64_t)kChunk * v_heads * dv * 4; }
  __host__ __device__ int64_t state() const { return (int64_t)v_heads * dk * dv * 4; }
};

struct ChunkArgs {
  DeltaArgs d;
  ChunkLayout at;
  char *chunks;       // of the chunks first .. first + count - 1
  float *carry[2];    // states that go from one run of chunks to the next
  int first, count, run;
  int sequences;      // that a run can touch
};

struct Chunk {
  int start, rows;
};

// A sequence's rows up to the kept ones, then the others, in chunks.
__device__ __forceinline__ int kept_rows(const DeltaArgs &a, int b, int n) {
  const int slot = a.slots[b], kept = a.keep ? a.keep[b] : n;
  return slot >= 0 && slot < a.n_slots && kept > 0 && kept < n ? kept : n;
}

__device__ __forceinline__ int chunks_of(int n, int kept) {
  return (kept + kChunk - 1) / kChunk + (n - kept + kChunk - 1) / kChunk;
}

__device__ __forceinline__ Chunk chunk_of(int n, int kept, int item) {
  const int head = (kept + kChunk - 1) / kChunk;
  const int start = item < head ? item * kChunk : kept + (item - head) * kChunk;
  return {start, min(kChunk, (item < head ? kept : n) - start)};
}

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// x as two fp16 terms. The barrier keeps the product that x may come from out of the conversion: fused, it
// is rounded once, and where that differs the second term was that of another first one (one value in
// ten thousand was off by 2^-11).
__device__ __forceinline__ void split(const float (&x)[4], half4 &high, half4 &low) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    f32x2 v = {x[i], x[i + 1]};
    asm("" : "+v"(v[0]), "+v"(v[1]));
    const half2v h = __builtin_convertvector(v, half2v);
    const f32x2 rest = {__builtin_fmaf(static_cast<float>(h[0]), -1.0f, v[0]), __builtin_fmaf(static_cast<float>(h[1]), -1.0f, v[1])};
    const half2v l = __builtin_convertvector(rest, half2v);
    high[i] = h[0], high[i + 1] = h[1];
    low[i] = l[0], low[i + 1] = l[1];
  }
}

// An infinity or NaN stays in its own column, so it has no part in a size that other columns are held by.
__device__ __forceinline__ float finite_size(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.0f; }

// 2^x; what x loses in fp32 is nothing beside 2^x where x is large.
__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x)); }

// A workgroup forms what the chain needs of one chunk and one key head: the rows of q and k as operands, and of
// two of the value heads that share it, four waves each, T, P and the rows' factors.
// T = (I + L)^-1 in fp32: the inverses of the four 16 x 16 blocks on the diagonal, a lane a column, joined by
// -T22 (L21 T11) to blocks of 32 and of 64 with fp32 matrix products, whose result is the next one's operand.
// Bound by VALU work (share 0.5, MFMA 0.07, 3.6 waves a SIMD) between short phases with a barrier each: 22 us for 512
// chunks and key heads (two rounds of the chip). One value head a workgroup formed K K^T twice; the blocks' inverses
// by lane broadcasts were slower (23.3 for 21.9), and so was asking for values and gates ahead (24 for 23).
template <typename T, int DK>
__global__ __launch_bounds__(kPrepareThreads, 2) void delta_chunks_kernel(ChunkArgs p) {
  constexpr int kPad = DK + 8, kSteps = DK / 32, kPer = DK / 8;
  const DeltaArgs &a = p.d;
  // rows of k and q, then, when they have been read, L and its inverse of both heads
  __shared__ __align__(16) char pool[kHeadsPer * kChunk * kMatPad * 4];
  __shared__ __align__(16) float kk[kChunk][kMatPad], qk[kChunk][kMatPad];
  __shared__ __align__(16) double totals[kHeadsPer][kChunk];
  __shared__ __align__(16) float rk[kChunk], rq[kChunk], betas[kHeadsPer][kChunk], most[kHeadsPer][4];
  static_assert(2 * kChunk * kPad * 2 <= (int)sizeof(pool), "the rows fit");
  _Float16(*ks)[kPad] = reinterpret_cast<_Float16(*)[kPad]>(pool), (*qs)[kPad] = ks + kChunk;

  const Sequence s = find_sequence(a.c, p.first + blockIdx.x, 1, kChunk, 2);
  if (s.b < 0 || s.tokens <= 0) return;
  const int kept = kept_rows(a, s.b, s.tokens);
  if (s.item >= chunks_of(s.tokens, kept)) return;
  const Chunk c = chunk_of(s.tokens, kept, s.item);
  const int group = a.v_heads / a.k_heads, parts = (group + kHeadsPer - 1) / kHeadsPer;
  const int k_head = blockIdx.y / parts, part = blockIdx.y - k_head * parts;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave >> 2, mine = wave & 3, own = tid & 255;
  const int head = k_head * group + min(part * kHeadsPer + half, group - 1);
  const bool there = part * kHeadsPer + half < group;      // an odd group's last pair has one head
  const int64_t row0 = s.row0 + c.start;
  char *place = p.chunks + blockIdx.x * p.at.bytes();
  char *head_place = place + p.at.k_heads * p.at.k_head() + head * p.at.v_head();
  float *factors = reinterpret_cast<float *>(head_place + 4 * 8 * kBlock * 2);

  {  // rows to lengths of 2^13 .. 2^14, in fp16; eight threads a row
    const int row = tid >> 3, d0 = (tid & 7) * kPer;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      T y[kPer];
      float x[kPer], sum = 0.0f, largest = 0.0f;
      const T *from = which ? static_cast<const T *>(a.q) + (row0 + min(row, c.rows - 1)) * a.q_stride
                            : static_cast<const T *>(a.k) + (row0 + min(row, c.rows - 1)) * a.k_stride;
      load_row<T, kPer>(from + k_head * DK + d0, a.wide, y);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        x[i] = row < c.rows ? static_cast<float>(y[i]) : 0.0f;
        largest = fmaxf(largest, fabsf(x[i]));
      }
      largest = fmaxf(largest, dpp<kQuadSwap1>(largest));
      largest = fmaxf(largest, dpp<kQuadSwap2>(largest));
      largest = fmaxf(largest, dpp<kHalfMirror>(largest));
      // to 1 .. 2 by the largest, so that no square passes fp32, then to the length
      const int ex = max(1, min(253, (int)(__float_as_uint(largest) >> 23)));
      const float unit = __uint_as_float(ex << 23);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        x[i] *= __uint_as_float((254 - ex) << 23);
        sum += x[i] * x[i];
      }
      sum = sum_low(sum);
      const int length = max(127, (int)(__float_as_uint(sqrtf(sum)) >> 23));
      const float up = __uint_as_float((267 - min(length, 254)) << 23), down = unit * __uint_as_float((min(length, 254) - 13) << 23);
      _Float16 *to = which ? &qs[row][d0] : &ks[row][d0];
#pragma unroll
      for (int i = 0; i < kPer; i += 8) {
        half8 z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = static_cast<_Float16>(x[i + j] * up);
        *reinterpret_cast<half8 *>(to + i) = z;
      }
      if ((tid & 7) == 0) (which ? rq : rk)[row] = down / sqrtf(sum * unit * unit + a.eps);
    }
  }
  {  // the largest finite value of the head
    const T *from = static_cast<const T *>(a.v) + row0 * a.v_stride + head * a.dv;
    const int per = a.dv / 8;
    float x = 0.0f;
    for (int i = own; i < c.rows * per; i += 256) {
      T y[8];
      load_row<T, 8>(from + i / per * a.v_stride + i % per * 8, a.wide, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fmaxf(x, finite_size(static_cast<float>(y[e])));
    }
    x = most_of_wave(x);
    if (lane == 0) most[half][mine] = x;
  }
  lds_barrier();
  if (mine == 0) {
    // sums of logarithms (base 2) in 64 bits: what they differ by between rows that forget little is to be exact
    // beside rows that forget all (2^-184 is nothing in fp32)
    double sum = 0.0;
    float w = 0.0f;
    if (lane < c.rows) {
      const float x = log_fade(a.a[(row0 + lane) * a.a_stride + head], a.dt_bias[head], expf(a.a_log[head]));
      sum = (x < -128.0f ? -128.0f : x) * 1.4426950408889634;
      w = sigmoid(a.b[(row0 + lane) * a.b_stride + head]);
    }
    for (int off = 1; off < 64; off <<= 1) {
      const double o = __shfl_up(sum, off);
      if (lane >= off) sum += o;
    }
    totals[half][lane] = sum;
    betas[half][lane] = w;
    const double last = __shfl(sum, 63);
    const float fade = exp2_of(sum);
    if (there) {
      factors[lane] = w;
      factors[kChunk + lane] = w * fade * rk[lane];
      factors[2 * kChunk + lane] = rk[lane] * (kLength / kUnit) * exp2_of(last - sum);
      factors[3 * kChunk + lane] = fade;
      factors[4 * kChunk + lane] = rq[lane];
      if (lane == 0) {
        factors[5 * kChunk] = exp2_of(last);
        factors[5 * kChunk + 1] = fmaxf(fmaxf(most[half][0], most[half][1]), fmaxf(most[half][2], most[half][3]));
      }
    }
  }
  {  // K K^T of one half, Q K^T of the other, 16 rows a wave, on and below the diagonal
    f32x4 x[4] = {};
    const _Float16(*rows)[kPad] = half ? qs : ks;
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      const half8 left = *reinterpret_cast<const half8 *>(&rows[mine * 16 + r][t * 32 + h * 8]);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n <= mine) x[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(left, *reinterpret_cast<const half8 *>(&ks[n * 16 + r][t * 32 + h * 8]), x[n], 0, 0, 0);
    }
    float(*to)[kMatPad] = half ? qk : kk;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n <= mine) to[mine * 16 + h * 4 + i][n * 16 + r] = x[n][i];
  }
  if (part == 0) {  // the rows as operands
    _Float16 *to = reinterpret_cast<_Float16 *>(place + k_head * p.at.k_head());
    for (int i = tid; i < 4 * kSteps * 64; i += kPrepareThreads) {
      const int l = i & 63, t = (i >> 6) % kSteps, tile = (i >> 6) / kSteps, row = tile * 16 + (l & 15);
      const int d = t * 32 + (l >> 4) * 4;
      const half4 k0 = *reinterpret_cast<const half4 *>(&ks[row][d]), k1 = *reinterpret_cast<const half4 *>(&ks[row][d + 16]);
      const half4 q0 = *reinterpret_cast<const half4 *>(&qs[row][d]), q1 = *reinterpret_cast<const half4 *>(&qs[row][d + 16]);
      *reinterpret_cast<half8 *>(to + i * 8) = __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7);
      *reinterpret_cast<half8 *>(to + kChunk * DK + i * 8) = __builtin_shufflevector(q0, q1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    for (int i = tid; i < (DK / 16) * 2 * 64; i += kPrepareThreads) {
      const int l = i & 63, t = (i >> 6) & 1, d = (i >> 7) * 16 + (l & 15), row = t * 32 + (l >> 4) * 4;
      half8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = ks[row + (e >> 2) * 16 + (e & 3)][d];
      *reinterpret_cast<half8 *>(to + 2 * kChunk * DK + i * 8) = y;
    }
  }
  lds_barrier();

  float(*m)[kMatPad] = reinterpret_cast<float(*)[kMatPad]>(pool) + half * kChunk;
  const double *total = totals[half];
  const int i = own >> 2, m0 = (own & 3) * 16;              // sixteen columns of one row a thread
  // its place in operands of T and P: the row's tile, the step of 32 columns, and the half of its slots
  _Float16 *block = reinterpret_cast<_Float16 *>(head_place) + ((i >> 4) * 2 + (m0 >> 5)) * kBlock + (i & 15) * 8 + (m0 >> 4 & 1) * 4;
  const bool used = there && (i >= 32 || m0 < 32);           // above the diagonal nothing is read
  auto put_operand = [&](const float (&x)[4], int which, int g) {
    half4 high, low;
    split(x, high, low);
    *reinterpret_cast<half4 *>(block + which * 16 * kBlock + g * 128) = high;
    *reinterpret_cast<half4 *>(block + (which * 16 + 8) * kBlock + g * 128) = low;
  };
  {  // L, and P as operands
    const double ti = total[i];
    const float bi = betas[half][i] * rk[i];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      // without branches: above the diagonal what was read is thrown away
      const int j0 = m0 + g * 4;
      const f32x4 kr = *reinterpret_cast<const f32x4 *>(&kk[i][j0]), qr = *reinterpret_cast<const f32x4 *>(&qk[i][j0]);
      const f32x4 r4 = *reinterpret_cast<const f32x4 *>(&rk[j0]);
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = exp2_of(ti - total[j0 + e]) * r4[e], l = bi * f * kr[e], m = f * qr[e];
        x[e] = j0 + e < i ? l : 0.0f;
        y[e] = j0 + e <= i ? m : 0.0f;
      }
      *reinterpret_cast<f32x4 *>(&m[i][m0 + g * 4]) = f32x4{x[0], x[1], x[2], x[3]};
      if (used) put_operand(y, 1, g);
    }
  }
  lds_barrier();
  {  // a lane solves for column r of its wave's block
    float x[16];
    const int at = mine * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float sum = i == r ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) sum -= m[at + i][at + j] * x[j];
      x[i] = sum;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (h == i >> 2) m[at + i][at + r] = x[i];
  }
  lds_barrier();
  auto times = [&](int row, int col, const f32x4 &right, f32x4 sum) {
    const f32x4 left = *reinterpret_cast<const f32x4 *>(&m[row * 16 + r][col * 16 + h * 4]);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(left[e], right[e], sum, 0, 0, 0);
    return sum;
  };
  auto block_of = [&](int row, int col) {
    return f32x4{m[row * 16 + h * 4][col * 16 + r], m[row * 16 + h * 4 + 1][col * 16 + r],
                 m[row * 16 + h * 4 + 2][col * 16 + r], m[row * 16 + h * 4 + 3][col * 16 + r]};
  };
  auto put = [&](int row, int col, const f32x4 &x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m[row * 16 + h * 4 + e][col * 16 + r] = -x[e];
  };
  if (mine < 2) {
    const int at = mine * 2;
    const f32x4 x = times(at + 1, at, block_of(at, at), f32x4{});
    put(at + 1, at, times(at + 1, at + 1, x, f32x4{}));
  }
  lds_barrier();
  f32x4 low0 = {}, low1 = {};
  if (mine < 2) {
    const f32x4 t0 = mine ? f32x4{} : block_of(0, 0), t1 = block_of(1, mine);
    const f32x4 x0 = times(2, 1, t1, times(2, 0, t0, f32x4{})), x1 = times(3, 1, t1, times(3, 0, t0, f32x4{}));
    low0 = times(2, 2, x0, f32x4{});
    low1 = times(3, 3, x1, times(3, 2, x0, f32x4{}));
  }
  lds_barrier();
  if (mine < 2) put(2, mine, low0), put(3, mine, low1);
  lds_barrier();
  if (!used) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 y = *reinterpret_cast<const f32x4 *>(&m[i][m0 + g * 4]);
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = m0 + g * 4 + e <= i ? y[e] * kUnit : 0.0f;
    put_operand(x, 0, g);
  }
}

// sqrt(x^2 + y^2) of two that are not negative, by a power of two so that neither square passes fp32. The fused operations are
// spelled out here and in set_scale: all waves have to come to the same bits, in code that the compiler makes more than once.
__device__ __forceinline__ float length_of(float x, float y) {
  const int ex = max(1, min(253, (int)(__float_as_uint(fmaxf(x, y)) >> 23)));
  const float down = __uint_as_float((254 - ex) << 23);
  x *= down, y *= down;
  return __builtin_amdgcn_sqrtf(__builtin_fmaf(x, x, y * y)) * __uint_as_float(ex << 23);
}

constexpr int kChainThreads = 512;
constexpr float kMostSize = 3.0e38f;   // a bound past fp32 has to come back as it fades
constexpr float kFarScale = 0x1p20f;   // 2^33 from one chunk's scale to the next, less the 2^13 of kLength

// A workgroup goes through a sequence's chunks with 16 columns of one head's state. Four waves are the chain: each
// has 16 of a chunk's rows, K S, R and U; four others read the rows out (Q S and, a step later, P U), 16 rows
// each; and every wave has a tile of 16 of the state's rows (64 of them: the chain's waves). S, R and U go between
// the waves as operands in LDS, a barrier after each.
// Values are held times a power of two that keeps them in fp16's range: with keys of length 1 and beta at most 1 the square
// of a column's length in S grows by at most the values' squares (64 of the largest a chunk), and R and U are never
// larger than a column of S and 9 of the largest value. Without a fade that bound is 8 sqrt(n) of the largest value after n chunks
// (lengths added up, not their squares, would be 8 n, and 512 chunks would cost values of 2^-18 of the largest their last bits).
// What a wave reads of the next chunk is asked for as soon as this chunk's has been used, so every load has a whole
// step to arrive; no branch stands between a load and its use, or the wait there would be for all of them. The values
// come by way of the reading waves, which have slack: their loads and addresses cost the chain 3 of 50 us.
// Bound by the chain: a step is 1.5 us, K S, R, U and S with three barriers, each a few dependent products (32 steps 50 us,
// 39 without any load; 256 workgroups of two waves a SIMD, MFMA 0.17, VALU 0.41, LDS 0.29). A 16-column slice fills the chip
// from one sequence of 32 heads of 128; two slices a CU share its cycles. With the reading waves' Q asked for beside the
// state's step 50.7, without loads above T's diagonal 49.2 (branches), at four waves a SIMD 92 (spills).
template <typename T, typename TO, int DK>
__global__ __launch_bounds__(kChainThreads, 2) void delta_chain_kernel(ChunkArgs p) {
  constexpr int kSteps = DK / 32;   // steps over the state's rows
  const DeltaArgs &a = p.d;
  __shared__ __align__(16) _Float16 sb[2][kSteps][64][8], rb[2][2][64][8], ub[2][2][64][8], wb[2][2][64][8];
  __shared__ f32x4 vb[4][64];       // a chunk's values, as the chain's lanes hold its rows
  __shared__ float most[8];

  // workgroups of one head run on one XCD, whose L2 then holds its chunk for all of them
  const int slices = a.dv / 16, xcd = blockIdx.x & 7, rest = blockIdx.x >> 3;
  const int slice = rest % slices;
  const int64_t pair = static_cast<int64_t>(rest / slices) * 8 + xcd;
  if (pair >= static_cast<int64_t>(p.sequences) * a.v_heads) return;
  int b = static_cast<int>(pair / a.v_heads);
  const int head = static_cast<int>(pair - static_cast<int64_t>(b) * a.v_heads);
  if (p.sequences < a.c.batch) {
    b += max(0, find_sequence(a.c, p.first, 1, kChunk, 2).b);
    if (b >= a.c.batch) return;
  }
  const int row0 = row_start(a.c, b), n = row_start(a.c, b + 1) - row0;
  if (n <= 0) return;
  const int kept = kept_rows(a, b, n), chunks = chunks_of(n, kept), kept_chunks = (kept + kChunk - 1) / kChunk;
  const int64_t base = first_item(row0, b, 1, kChunk, 2);
  const int c0 = static_cast<int>(max((int64_t)0, p.first - base));
  const int c1 = static_cast<int>(min((int64_t)chunks, p.first + p.count - base));
  if (c0 >= c1) return;

  const int tid = threadIdx.x, lane = tid & 63, tile = __builtin_amdgcn_readfirstlane(tid >> 6), wave = tile & 3;
  const bool chain = tile < 4, has_tile = DK == 128 || chain;
  const int r = lane & 15, h = lane >> 4, col = slice * 16 + r, row = wave * 16 + h * 4;
  const bool below = wave >= 2;     // rows 32 and on: the second step over a chunk's rows is not above the diagonal
  const int k_head = head / (a.v_heads / a.k_heads), slot = a.slots[b];
  const bool has_state = slot >= 0 && slot < a.n_slots, stored = has_state && has_tile && (!a.keep || a.keep[b] > 0);
  const int64_t in_state = (static_cast<int64_t>(head) * DK + tile * 16 + h * 4) * a.dv + col;
  float *state = has_state ? a.state + static_cast<int64_t>(slot) * a.v_heads * DK * a.dv + in_state : nullptr;

  // the places of this head's data in a chunk's: a uniform place and a lane's offset of 32 bits
  const int64_t step_bytes = p.at.bytes();
  const char *place = p.chunks + (base + c0 - p.first) * step_bytes;
  const int64_t k_at = k_head * p.at.k_head(), rows_at = k_at + (chain ? 0 : kChunk * DK * 2) + wave * kSteps * kBlock * 2;
  const int64_t tile_at = k_at + (2 * kChunk * DK + tile * 2 * kBlock) * 2;
  const int64_t head_at = p.at.k_heads * p.at.k_head() + head * p.at.v_head();
  const int64_t mats_at = head_at + ((chain ? 0 : 16) + wave * 2) * kBlock * 2, factors_at = head_at + 4 * 8 * kBlock * 2;
  const int row_bytes = wave * 16 * 4;          // a wave's rows among 64 factors
  const int second = below ? kBlock * 2 : 0;    // above the diagonal the first step's again, unused
  uint32_t lane_at = lane * 16, row_at = h * 16, zero = 0;
  asm("" : "+v"(zero));             // a vector load, which is waited for with the others
  auto load8 = [&](const char *from) { return *reinterpret_cast<const half8 *>(from + lane_at); };
  auto load4 = [&](const char *from) { return *reinterpret_cast<const f32x4 *>(from + row_at); };
  auto load_pair = [&](const char *from) { return *reinterpret_cast<const f32x2 *>(from + factors_at + 5 * kChunk * 4 + zero); };

  half8 rows[kSteps], mats[2][2], kt[2];      // K and T, or Q and P (term, step); the tile of K^T
  auto load_rows = [&]() {
#pragma unroll
    for (int e = 0; e < kSteps; ++e) rows[e] = load8(place + rows_at + e * kBlock * 2);
  };
  auto load_mats = [&]() {
#pragma unroll
    for (int term = 0; term < 2; ++term)
#pragma unroll
      for (int e = 0; e < 2; ++e) mats[term][e] = load8(place + mats_at + term * 8 * kBlock * 2 + (e ? second : 0));
  };
  auto load_tile = [&]() {
    if (!has_tile) return;
#pragma unroll
    for (int e = 0; e < 2; ++e) kt[e] = load8(place + tile_at + e * kBlock * 2);
  };
  auto operand = [&](const _Float16 (&from)[64][8]) { return *reinterpret_cast<const half8 *>(&from[lane][0]); };
  auto mfma = [](const half8 &x, const half8 &y, const f32x4 &sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, sum, 0, 0, 0);
  };
  // A product's operands are asked for together, and `beside` (the next loads) is issued while they come: the compiler would
  // wait for LDS three times in a row, and issue the loads behind the product, where the others wait for it.
  // This wave's rows times the state:
  auto times_state = [&](auto beside) {
    half8 high[kSteps], low[kSteps];
#pragma unroll
    for (int e = 0; e < kSteps; ++e) high[e] = operand(sb[0][e]), low[e] = operand(sb[1][e]);
    __builtin_amdgcn_sched_barrier(0);
    beside();
    __builtin_amdgcn_sched_barrier(0);
    f32x4 sum = {}, low_sum = {};
#pragma unroll
    for (int e = 0; e < kSteps; ++e) {
      sum = mfma(rows[e], high[e], sum);
      low_sum = mfma(rows[e], low[e], low_sum);
    }
    return sum + low_sum;
  };
  // its rows of a chunk's 64 x 64 matrix in two terms times 64 x 16 values in two
  auto times_mats = [&](const _Float16 (&y)[2][2][64][8], f32x4 sum, auto beside) {
    const half8 high = operand(y[0][0]), low = operand(y[1][0]), high2 = operand(y[0][1]), low2 = operand(y[1][1]);
    __builtin_amdgcn_sched_barrier(0);
    beside();
    __builtin_amdgcn_sched_barrier(0);
    f32x4 low_sum = mfma(mats[0][0], low, f32x4{}), last = mfma(mats[1][0], high, f32x4{});
    sum = mfma(mats[0][0], high, sum);
    if (below) {
      low_sum = mfma(mats[0][1], low2, low_sum);
      last = mfma(mats[1][1], high2, last);
      sum = mfma(mats[0][1], high2, sum);
    }
    return sum + (low_sum + last);
  };
  auto give = [&](_Float16 (&to)[2][2][64][8], const float (&x)[4]) {
    half4 high, low;
    split(x, high, low);
    *reinterpret_cast<half4 *>(&to[0][wave >> 1][lane][(wave & 1) * 4]) = high;
    *reinterpret_cast<half4 *>(&to[1][wave >> 1][lane][(wave & 1) * 4]) = low;
  };
  float s[4];
  auto give_state = [&]() {
    half4 high, low;
    split(s, high, low);
    *reinterpret_cast<half4 *>(&sb[0][tile >> 1][lane][(tile & 1) * 4]) = high;
    *reinterpret_cast<half4 *>(&sb[1][tile >> 1][lane][(tile & 1) * 4]) = low;
  };

  float size = 0.0f, inverse, scale, fade, value;   // size: a bound of the length of a column of S
  // the power of two that brings R, U and S of the next step under 2^15, and its inverse
  auto set_scale = [&]() {
    const int ex = max(15, min(254, (int)(__float_as_uint(__builtin_fmaf(9.0f, value, size)) >> 23)));
    inverse = __uint_as_float((ex - 14) << 23);
    scale = __uint_as_float((268 - ex) << 23);
  };
  // a chunk's fade and its largest value; the next one's give the scale of what this one hands on
  const char *second_place = place + (c0 + 1 < c1 ? step_bytes : 0);
  f32x2 next = load_pair(place);         // then the next chunk's
  fade = next[0], value = next[1];
  Chunk c = chunk_of(n, kept, c0);
  {
    const float *from = !has_tile ? nullptr : c0 ? p.carry[p.run & 1] + in_state : has_state && cached(a.c, b) > n ? state : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = from ? from[i * a.dv] : 0.0f;
      size = fmaxf(size, finite_size(s[i]));
    }
    size = most_of_wave(size);
    if (lane == 0) most[tile] = size;
  }
  load_rows();
  load_mats();
  lds_barrier();
  size = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) size = fmaxf(size, most[i]);
  size *= DK == 128 ? 11.32f : 8.0f;
  set_scale();
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] *= scale;
  if (has_tile) give_state();

  // what the step behind needs for its S
  auto load_update = [&]() {
    load_tile();
    next = load_pair(second_place);
  };
  // the bound behind this chunk: beside a product, as nothing of it waits for one
  auto grow = [&]() { size = fminf(length_of(fade * size, 8.0f * value), kMostSize); };
  // S <- fade S + K^T W, of this wave's tile, and the next chunk's scale
  auto update_state = [&](int at, auto beside) {
    const float faded = fade * kLength, back = inverse * (1.0f / kLength);
    f32x4 sum, low = {};
    half8 w[2][2];
    if (has_tile) {
#pragma unroll
      for (int e = 0; e < 2; ++e) w[0][e] = operand(wb[0][e]), w[1][e] = operand(wb[1][e]);
    }
    __builtin_amdgcn_sched_barrier(0);
    beside();
    __builtin_amdgcn_sched_barrier(0);
    if (has_tile) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = faded * s[i];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum = mfma(kt[e], w[0][e], sum);
        low = mfma(kt[e], w[1][e], low);
      }
    }
    fade = next[0], value = next[1];
    asm("" : "+v"(fade), "+v"(value));     // registers of their own: those of a load stay its own from step to step
    set_scale();
    const float up = back * scale;
    const bool far = __builtin_amdgcn_readfirstlane(__float_as_int(up)) > __float_as_int(kFarScale);   // the same in every lane
    second_place += at + 2 < c1 ? step_bytes : 0;
    if (has_tile) {
      sum += low;
      // To the next scale. What the operands' last bits leave in a state that has faded away, 64 times 2^-25 at most, stays in its
      // range where the scales lie less than 2^33 apart. Past that it is held there, so that it does not grow into an
      // infinity, and the factors come one by one, as their product can pass fp32 (0 times it is NaN, for good).
      if (!far) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = sum[i] * up;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float t = sum[i] * back;
          s[i] = __builtin_fmaf(t, 0.0f, __builtin_amdgcn_fmed3f(t * scale, -2.0f * kUnit, 2.0f * kUnit));   // t: NaN where it is not finite
        }
      }
      give_state();
      if (at + 1 == kept_chunks && stored) {
#pragma unroll
        for (int i = 0; i < 4; ++i) state[i * a.dv] = sum[i] * back;
      }
      if (at + 1 == c1 && at + 1 < chunks) {
        float *to = p.carry[(p.run + 1) & 1] + in_state;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i * a.dv] = sum[i] * back;
      }
    }
  };

  // of the next chunk, by the waves that have slack
  T v[4];
  const T *values = static_cast<const T *>(a.v) + row0 * a.v_stride + head * a.dv + slice * 16;
  int64_t value_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) value_at[i] = (row + i) * a.v_stride + r;
  auto load_values = [&](int start) {                              // behind the chunk's rows its last one again
    const int end = start < kept ? kept : n;
    const T *from = values + start * a.v_stride;
    if (start + kChunk <= end) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = from[value_at[i]];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = values[min(start + row + i, end - 1) * a.v_stride + r];
    }
  };
  auto give_values = [&]() {
    vb[wave][lane] = f32x4{static_cast<float>(v[0]), static_cast<float>(v[1]), static_cast<float>(v[2]), static_cast<float>(v[3])};
  };

  if (chain) {
    f32x4 take, seen, left;            // factors of this wave's rows of V, K S and U
    auto load_factors = [&]() {
      take = load4(place + factors_at + row_bytes);
      seen = load4(place + factors_at + kChunk * 4 + row_bytes);
    };
    load_factors();
    left = load4(place + factors_at + 2 * kChunk * 4 + row_bytes);
    __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt(0): the loop's own waits are then for loads of a step before
    lds_barrier();

    for (int at = c0; at < c1; ++at) {
      f32x4 y;
      const f32x4 ks = times_state([&]() {
        y = vb[wave][lane];
        load_update();
      });
      place += at + 1 < c1 ? step_bytes : 0;             // the last chunk's data come again, unused
      float x[4], w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = take[i] * (y[i] * scale) - seen[i] * ks[i];   // take: 0 behind the rows
      give(rb, x);
      lds_barrier();

      const f32x4 u = times_mats(rb, f32x4{}, [&]() {
        load_rows();
        load_factors();
        grow();
      });
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = u[i] * (1.0f / kUnit);
        w[i] = left[i] * u[i];
      }
      give(wb, w);
      give(ub, x);
      lds_barrier();

      update_state(at, [&]() {
        load_mats();
        left = load4(place + factors_at + 2 * kChunk * 4 + row_bytes);
      });
      lds_barrier();
    }
  } else {
    f32x4 read, length, qs = {};           // factors of this wave's rows of Q S, and of all of them
    auto load_factors = [&]() {
      read = load4(place + factors_at + 3 * kChunk * 4 + row_bytes);
      length = load4(place + factors_at + 4 * kChunk * 4 + row_bytes);
    };
    load_factors();
    const int64_t width = a.z ? static_cast<int64_t>(a.v_heads) * a.dv : a.out_stride;
    float *scratch = reinterpret_cast<float *>(p.chunks + (base + c0 - p.first) * step_bytes + p.at.rows_at()) + row * width +
                     head * a.dv + col;
    TO *out = static_cast<TO *>(a.out) + (static_cast<int64_t>(row0) + c.start + row) * a.out_stride + head * a.dv + col;
    float unit = 0.0f;
    // the rows of the chunk whose U lies in LDS
    auto finish = [&]() {
      // one by one: their product can lie below fp32's last bits where the row does not
      const f32x4 o = times_mats(ub, read * qs, load_update) * length * unit;
      if (a.z) {
        if (c.rows == kChunk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) scratch[i * width] = o[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row + i < c.rows) scratch[i * width] = o[i];
        }
        scratch = reinterpret_cast<float *>(reinterpret_cast<char *>(scratch) + step_bytes);
      } else {
        if (c.rows == kChunk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i * width] = static_cast<TO>(o[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row + i < c.rows) out[i * width] = static_cast<TO>(o[i]);
        }
        out += c.rows * width;
      }
      c.start += c.rows;
      c.rows = min(kChunk, (c.start < kept ? kept : n) - c.start);
    };
    load_update();
    load_values(c.start);
    give_values();
    int ahead = c.start + c.rows;
    auto next_values = [&]() {
      load_values(ahead);
      ahead += min(kChunk, (ahead < kept ? kept : n) - ahead);
    };
    next_values();
    __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt(0), as above
    lds_barrier();

    for (int at = c0; at < c1; ++at) {
      place += at + 1 < c1 ? step_bytes : 0;
      lds_barrier();
      qs = times_state([] {});
      unit = a.scale * inverse;
      load_rows();
      give_values();
      next_values();
      grow();

      lds_barrier();
      update_state(at, [] {});
      lds_barrier();
      finish();              // beside the chain's next K S
      load_mats();
      load_factors();
    }
  }
}

// The chunks' rows, fp32, normalised and gated: a workgroup a row, four neighbouring values a lane. The chain's workgroups
// hold 16 columns of a head, so its norm needs a pass of its own: 2048 rows of 4096 values, 84 MB, 15 us (5.6 TB/s).
template <typename TO>
__global__ __launch_bounds__(kGateThreads) void delta_gate_kernel(ChunkArgs p) {
  const DeltaArgs &a = p.d;
  const Sequence s = find_sequence(a.c, p.first + blockIdx.x, 1, kChunk, 2);
  if (s.b < 0 || s.tokens <= 0) return;
  const int kept = kept_rows(a, s.b, s.tokens), row = blockIdx.y;
  if (s.item >= chunks_of(s.tokens, kept)) return;
  const Chunk c = chunk_of(s.tokens, kept, s.item);
  if (row >= c.rows) return;
  const int width = a.v_heads * a.dv, lanes = a.dv / 4;
  const float *o = reinterpret_cast<const float *>(p.chunks + blockIdx.x * p.at.bytes() + p.at.rows_at()) + static_cast<int64_t>(row) * width;
  const int64_t out_row = static_cast<int64_t>(s.row0) + c.start + row;
  for (int i = threadIdx.x * 4; i < width; i += kGateThreads * 4) {   // whole heads: a head's lanes are of one wave
    f32x4 x = *reinterpret_cast<const f32x4 *>(o + i);
    auto mean = [&]() {
      float sum = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
      for (int off = lanes / 2; off; off >>= 1) sum += __shfl_xor(sum, off);
      return sum * (1.0f / a.dv);
    };
    float square = mean() + a.norm_eps;
    if (square == __builtin_inff()) {    // in all lanes of a head
      x *= kSmaller;
      square = mean() + a.norm_eps * kSmaller * kSmaller;
    }
    const float f = __builtin_amdgcn_rsqf(square);
    const float *z = a.z + out_row * a.z_stride + i, *w = a.norm + i % a.dv;
    TO *to = static_cast<TO *>(a.out) + out_row * a.out_stride + i;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = static_cast<TO>(x[e] * f * w[e] * gate_of(z[e]));
  }
}

// Whether a call goes token by token. Heads of 128 x 128, 16 key and 32 value heads, kernels alone (us, tokens and
// chunks): one sequence of 16 rows 21 and 22.6, of 24 rows 29 and 22.8; four of 32 rows 38 and 42, of 48 rows 55 and
// 44; sixteen of 48 rows 85 and 106, of 64 rows 110 and 107; 32 of 64 rows 211 and 217, of 100 318 and 289; 64 of 64 rows 400 and
// 483, of 100 604 and 645; 128 of 100 rows 1173 and 1273, of 200 2266 and 1829; 512 of 100 rows 4551 and 5754. A token takes its 1 us
// in all heads at once as long as they find room; the chunks of one sequence fill the chip, those of many short ones are half empty.
// The rule gives 64 of 100 rows to the chunks (7% lost). It goes by these heads for all: of 150 sizes in five geometries (12 to 160
// rows, 1 to 256 sequences) it is within 3% of the better form in all but eight, which lose 14 to 41% (256 of 112 rows, 8 heads of 64 x 128:
// 392 and 552; heads of 128 x 256 1.3 times in 12 rows of one sequence, 23 and 18).
// Batches of 2^27 columns and more (32768 sequences of 32 heads of 128) are past what the chunks are for, whatever max_q says: each run's
// workgroups look through all sequences. 32700 of 32 heads of 64 x 128, a row each: 13 ms and 2386; with one of 20000 rows
// beside them 26 and 2395.
constexpr int64_t kMostColumns = 1 << 27, kMostHeads = 1 << 24;
bool by_tokens(int B, int v_heads, int dv, int max_q) {
  const int64_t heads = (int64_t)B * v_heads;
  return max_q <= std::min<int64_t>({112, 50 + heads / 48, 12 + heads / 6}) || ((heads + 7) / 8 * 8 * dv >= kMostColumns && heads < kMostHeads);
}

struct ChunkPlan {
  int64_t slots;
  int most, count;      // chunks that the scratch holds at a time; those of a run
  int64_t bytes;
};

ChunkPlan plan_chunks(const ChunkLayout &at, int T, int B) {
  ChunkPlan r;
  r.slots = T / kChunk + 2 * (int64_t)B;
  r.most = (int)std::min<int64_t>(r.slots, std::max<int64_t>(1, kMostScratch / at.bytes()));
  const int64_t runs = (r.slots + r.most - 1) / r.most;
  r.count = (int)((r.slots + runs - 1) / runs);
  r.bytes = r.most * at.bytes() + (r.most < r.slots ? 2 * at.state() : 0);
  return r;
}

template <typename T, typename TO, int DK>
int launch_chunks(const DeltaArgs &a, void *workspace, hipStream_t st) {
  ChunkArgs p{};
  p.d = a;
  p.at = {DK, a.k_heads, a.v_heads, a.dv};
  const ChunkPlan plan = plan_chunks(p.at, a.c.rows, a.c.batch);
  p.chunks = static_cast<char *>(workspace);
  p.carry[0] = reinterpret_cast<float *>(p.chunks + plan.most * p.at.bytes());
  p.carry[1] = reinterpret_cast<float *>(reinterpret_cast<char *>(p.carry[0]) + p.at.state());
  const int parts = (a.v_heads / a.k_heads + kHeadsPer - 1) / kHeadsPer;
  // a sequence has two chunks' places or more, so the chain of a run need not look at all of many sequences
  p.sequences = (int)std::min<int64_t>(a.c.batch, plan.count / 2 + 2);
  const int64_t chain_grid = ((int64_t)p.sequences * a.v_heads + 7) / 8 * 8 * (a.dv / 16);
  RLQ_REQUIRE((int64_t)a.c.batch * a.v_heads < kMostHeads && a.k_heads * (int64_t)parts <= 65535 && chain_grid * kChainThreads <= UINT32_MAX,
              "rlq_gated_delta: %d heads of %d sequences are too many for chunks", a.v_heads, a.c.batch);
  for (int64_t first = 0; first < plan.slots; first += plan.count, ++p.run) {
    p.first = (int)first;
    p.count = (int)std::min<int64_t>(plan.count, plan.slots - first);
    delta_chunks_kernel<T, DK><<<dim3(p.count, a.k_heads * parts), kPrepareThreads, 0, st>>>(p);
    RLQ_HIP(hipGetLastError());
    delta_chain_kernel<T, TO, DK><<<(unsigned)chain_grid, kChainThreads, 0, st>>>(p);
    RLQ_HIP(hipGetLastError());
    if (a.z) {
      delta_gate_kernel<TO><<<dim3(p.count, kChunk), kGateThreads, 0, st>>>(p);
      RLQ_HIP(hipGetLastError());
    }
  }
  return 0;
}

template <typename T, typename TO>
int launch_delta(const DeltaArgs &a, int DK, int max_q, void *workspace, hipStream_t st) {
  if (!by_tokens(a.c.batch, a.v_heads, a.dv, max_q)) return DK == 64 ? launch_chunks<T, TO, 64>(a, workspace, st) : launch_chunks<T, TO, 128>(a, workspace, st);
  const unsigned grid = (unsigned)a.c.batch * (unsigned)a.v_heads;
  RLQ_REQUIRE(a.c.batch * (int64_t)a.v_heads * a.dv * 2 <= UINT32_MAX, "rlq_gated_delta: %d heads of %d sequences are too many",
              a.v_heads, a.c.batch);
  if (DK == 64) delta_tokens_kernel<T, TO, 64><<<grid, a.dv * 2, 0, st>>>(a);
  else delta_tokens_kernel<T, TO, 128><<<grid, a.dv * 2, 0, st>>>(a);
  RLQ_HIP(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace rlq

extern "C" {

size_t rlq_gated_delta_workspace_bytes(int T, int k_heads, int v_heads, int Dk, int Dv, int B, int max_q) {
  if (T <= 0 || B <= 0 || rlq::by_tokens(B, v_heads, Dv, max_q) || k_heads < 1 || v_heads < k_heads || Dk <= 0 || Dv <= 0) return 0;
  return (size_t)rlq::plan_chunks({Dk, k_heads, v_heads, Dv}, T, B).bytes;
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
  RLQ_REQUIRE(eps >= 1e-37f && std::isfinite(eps), "rlq_gated_delta: eps=%g must be at least 1e-37", eps);
  RLQ_REQUIRE(std::isfinite(scale), "rlq_gated_delta: scale=%g", scale);
  RLQ_REQUIRE((z == nullptr) == (norm == nullptr), "rlq_gated_delta: z and norm come together");
  RLQ_REQUIRE(!norm || (norm_eps >= 1e-37f && std::isfinite(norm_eps)), "rlq_gated_delta: norm_eps=%g must be at least 1e-37",
              norm_eps);
  RLQ_REQUIRE(n_slots >= 0 && max_q >= 0, "rlq_gated_delta: n_slots=%d, max_q=%d", n_slots, max_q);
  if (T == 0 || B == 0) return 0;
  RLQ_REQUIRE(q && k && v && a && b && a_log && dt_bias && out && cu_q && kv_len && slots, "rlq_gated_delta: null pointer");
  RLQ_REQUIRE((state && rlq::aligned(state, 16)) || n_slots == 0, "rlq_gated_delta: the state must be set and 16-byte aligned");
  RLQ_REQUIRE(q_stride >= k_heads * Dk && k_stride >= k_heads * Dk && v_stride >= v_heads * Dv && a_stride >= v_heads &&
                  b_stride >= v_heads && out_stride >= v_heads * Dv && (!z || z_stride >= v_heads * Dv),
              "rlq_gated_delta: a row stride is shorter than the row (q %d, k %d, v %d, a %d, b %d, z %d, out %d)", q_stride,
              k_stride, v_stride, a_stride, b_stride, z_stride, out_stride);
  const size_t need = rlq_gated_delta_workspace_bytes(T, k_heads, v_heads, Dk, Dv, B, max_q);
  RLQ_REQUIRE(need == 0 || (workspace && rlq::aligned(workspace, 16) && workspace_bytes >= need),
              "rlq_gated_delta: needs %zu bytes of 16-byte aligned workspace, got %zu", need, workspace_bytes);
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
  x.wide_z = rlq::aligned(z, 16) && z_stride % 4 == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == RLQ_F16) {
    return out_dtype == RLQ_F16 ? rlq::launch_delta<_Float16, _Float16>(x, Dk, max_q, workspace, st) : rlq::launch_delta<_Float16, __bf16>(x, Dk, max_q, workspace, st);
  }
  return out_dtype == RLQ_F16 ? rlq::launch_delta<__bf16, _Float16>(x, Dk, max_q, workspace, st) : rlq::launch_delta<__bf16, __bf16>(x, Dk, max_q, workspace, st);
}

}  // extern "C"
