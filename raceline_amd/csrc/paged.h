// The paged key/value cache: layout, and how a kernel finds its sequence, shared by the
// operator that writes it (rope.hip) and the one that reads it (attention.hip).
//
// A page holds page_size positions (a multiple of 32) of every key/value head; a block is 32
// positions of one head, 32 * D 16-bit elements, contiguous. Inside a block the elements lie in
// the order in which the matrix cores take them as A operands, so that a wave's 16-byte loads
// are a contiguous kilobyte and need no transpose:
//   keys    [D/16][2][32][8]        step of 16 dimensions, half, key, dimension: the 32 x 16
//                                   operand of v_mfma_f32_32x32x16 (lane l: row l % 32, k 8 (l / 32) ..)
//   values  [D/32][2][2][32][2][4]  tile of 32 dimensions, t, h, dimension, a, b: the same operand of
//                                   V transposed, whose k slot 8 h + 4 a + b is key 16 t + 8 a + 4 h + b.
// That order of the keys is the one in which a lane holds a column of S = K Q^T (its accumulator
// rows are 8 (i / 4) + 4 (l / 32) + i % 4), so the weights go from the softmax into the second
// product without leaving their lane.
#pragma once

#include "rlq_common.h"

namespace rlq {

constexpr int kBlockKeys = 32;

struct PagedCache {
  void *k, *v;
  const int *cu_q, *kv_len, *table;
  int n_pages, blocks_per_page, kv_heads, batch, rows, table_stride, table_width;
};

__device__ __forceinline__ int key_offset(int key, int d) {
  return (d >> 4) * 512 + ((d >> 3) & 1) * 256 + key * 8 + (d & 7);
}

// Element of the 16-byte run that holds, for dimension d, the keys 16 t + 8 a + 4 h + b.
__device__ __forceinline__ int value_run(int d, int t, int h) {
  return (d >> 5) * 1024 + t * 512 + h * 256 + (d & 31) * 8;
}

// First element of a block.
__device__ __forceinline__ int64_t block_base(const PagedCache &c, int page, int head, int block, int D) {
  return ((static_cast<int64_t>(page) * c.kv_heads + head) * c.blocks_per_page + block % c.blocks_per_page) *
         (kBlockKeys * D);
}

// The page of a sequence's block, or -1: a block past the table's row, or an entry that names no
// page (its keys are then seen by nobody, and nothing is written there).
__device__ __forceinline__ int page_of(const PagedCache &c, int seq, int block) {
  const int at = block / c.blocks_per_page;
  if (block < 0 || at >= c.table_width) return -1;
  const int page = c.table[static_cast<int64_t>(seq) * c.table_stride + at];
  return page >= 0 && page < c.n_pages ? page : -1;
}

// First row of a sequence, inside the call's rows whatever the array holds.
__device__ __forceinline__ int row_start(const PagedCache &c, int seq) {
  return max(0, min(c.cu_q[seq], c.rows));
}

// Tokens of a sequence in the cache, the call's own among them; inside what positions can hold
// whatever the array holds.
constexpr int kMaxPositions = 1 << 29;

__device__ __forceinline__ int cached(const PagedCache &c, int seq) {
  return max(0, min(c.kv_len[seq], kMaxPositions));
}

// Work items are numbered without a prefix sum over the sequences' own counts: sequence b begins
// at (first row * mul) / div + extra * b, which leaves room for its items (a sequence of n rows
// takes at most ceil(n * mul / div) + extra - 1), and a few numbers without an item. Every
// thread takes part; returns the sequence whose range holds `slot`, or -1. One round trip to
// memory for up to blockDim.x sequences, against log2(batch) for a binary search.
__device__ __forceinline__ int64_t slot_base(const PagedCache &c, int seq, int mul, int div, int extra) {
  return static_cast<int64_t>(row_start(c, seq)) * mul / div + static_cast<int64_t>(extra) * seq;
}

template <int THREADS>
__device__ __forceinline__ int find_sequence(const PagedCache &c, int64_t slot, int mul, int div, int extra,
                                             int *shared) {
  int below = 0;
  for (int i = threadIdx.x; i < c.batch; i += THREADS) below += slot_base(c, i, mul, div, extra) <= slot ? 1 : 0;
  for (int off = 32; off; off >>= 1) below += __shfl_xor(below, off);
  if (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = below;
    __syncthreads();
    below = 0;
    for (int i = 0; i < THREADS / 64; ++i) below += shared[i];
  }
  return below - 1;
}

}  // namespace rlq
