// Sums, maxima and prefix sums over the lanes of a wave without LDS: DPP moves inside rows of 16 lanes, swaps of
// rows and halves between them.
#pragma once

#include "rlq_common.h"

namespace rlq {

// The value of the lane that CTRL names (row_shr, row_ror, quad_perm, mirrors, broadcasts of a row's last lane); 0 where
// it names none or ROWS leaves the lane's row out.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false);
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(x)));
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint64_t dpp(uint64_t x) {
  return static_cast<uint64_t>(dpp<CTRL, ROWS>(static_cast<uint32_t>(x >> 32))) << 32 | dpp<CTRL, ROWS>(static_cast<uint32_t>(x));
}

constexpr int kQuadSwap1 = 0xB1, kQuadSwap2 = 0x4E, kHalfMirror = 0x141, kRowRor8 = 0x128;

// Sum over the lanes that differ in bits 3 to 5 of their number; every lane gets it.
__device__ __forceinline__ float sum_high(float x) {
  x += dpp<kRowRor8>(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Over those that differ in bits 0 to 2.
__device__ __forceinline__ float sum_low(float x) {
  x += dpp<kQuadSwap1>(x);
  x += dpp<kQuadSwap2>(x);
  return x + dpp<kHalfMirror>(x);
}

// The largest of a wave, none below 0, in every lane; NaN is passed over.
__device__ __forceinline__ float most_of_wave(float x) {
  x = fmaxf(x, dpp<kQuadSwap1>(x));
  x = fmaxf(x, dpp<kQuadSwap2>(x));
  x = fmaxf(x, dpp<kHalfMirror>(x));
  x = fmaxf(x, dpp<kRowRor8>(x));
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ uint32_t most_of_wave(uint32_t x) {
  x = max(x, dpp<kQuadSwap1>(x));
  x = max(x, dpp<kQuadSwap2>(x));
  x = max(x, dpp<kHalfMirror>(x));
  x = max(x, dpp<kRowRor8>(x));
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(r[0], r[1]);
}

// Sum over the lanes up to this one, itself among them (whole numbers).
template <typename V>
__device__ __forceinline__ V scan_wave(V x) {
  x += dpp<0x111>(x);          // row_shr 1, 2, 4, 8
  x += dpp<0x112>(x);
  x += dpp<0x114>(x);
  x += dpp<0x118>(x);
  x += dpp<0x142, 0xa>(x);     // the last lane of rows 0 and 2 to rows 1 and 3
  return x + dpp<0x143, 0xc>(x);   // the last lane of the lower half to the upper
}

__device__ __forceinline__ uint32_t of_lane(uint32_t x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ uint64_t of_lane(uint64_t x, int lane) {
  return static_cast<uint64_t>(of_lane(static_cast<uint32_t>(x >> 32), lane)) << 32 | of_lane(static_cast<uint32_t>(x), lane);
}

template <typename V>
__device__ __forceinline__ V sum_wave(V x) {
  return of_lane(scan_wave(x), 63);
}

}  // namespace rlq
