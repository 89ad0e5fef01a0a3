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

// Number of a sequence's block of one head among all blocks of the cache, or -1 where it names no
// page: a block past the table's row, or an entry outside the cache (nobody sees its keys, and
// nothing is written there).
__device__ __forceinline__ int block_at(const PagedCache &c, int seq, int head, int block) {
  const int at = block / c.blocks_per_page;
  if (block < 0 || at >= c.table_width) return -1;
  const int page = c.table[static_cast<int64_t>(seq) * c.table_stride + at];
  if (page < 0 || page >= c.n_pages) return -1;
  return (page * c.kv_heads + head) * c.blocks_per_page + block - at * c.blocks_per_page;
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
// takes at most ceil(n * mul / div) + extra - 1), and a few numbers without an item.
struct Sequence {
  int b, row0, tokens, kv;   // b < 0: none; kv: tokens in the cache, the call's own among them
  int item;                  // number of the item among the sequence's
};

__device__ __forceinline__ int64_t first_item(int row0, int seq, int mul, int div, int extra) {
  return static_cast<int64_t>(row0) * mul / div + static_cast<int64_t>(extra) * seq;
}

// The sequence whose range holds item `slot`; the same in every lane of a wave. A wave looks over
// 64 sequences with one load of a lane (one round trip to memory, against log2(batch) for a
// binary search), and up to 63 sequences take the rest of what it returns from the same loads.
__device__ __forceinline__ Sequence find_sequence(const PagedCache &c, int64_t slot, int mul, int div, int extra) {
  const int lane = threadIdx.x & 63;
  Sequence s;
  if (c.batch < 64) {
    const int row = row_start(c, min(lane, c.batch)), kv = cached(c, min(lane, c.batch - 1));
    const bool below = lane < c.batch && first_item(row, lane, mul, div, extra) <= slot;
    s.b = __popcll(__ballot(below)) - 1;
    const int at = max(s.b, 0);
    s.row0 = __builtin_amdgcn_readlane(row, at);
    s.tokens = __builtin_amdgcn_readlane(row, at + 1) - s.row0;
    s.kv = __builtin_amdgcn_readlane(kv, at);
  } else {
    int below = 0;
    for (int i = lane; i < c.batch; i += 64) below += first_item(row_start(c, i), i, mul, div, extra) <= slot ? 1 : 0;
    for (int off = 32; off; off >>= 1) below += __shfl_xor(below, off);
    s.b = __builtin_amdgcn_readfirstlane(below) - 1;
    const int at = max(s.b, 0);
    s.row0 = row_start(c, at);
    s.tokens = row_start(c, at + 1) - s.row0;
    s.kv = cached(c, at);
  }
  // in scalar registers: what follows from them (page ids, addresses of copies) has to stay there
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.row0 = __builtin_amdgcn_readfirstlane(s.row0);
  s.tokens = max(0, __builtin_amdgcn_readfirstlane(s.tokens));
  s.kv = __builtin_amdgcn_readfirstlane(s.kv);
  s.item = __builtin_amdgcn_readfirstlane(static_cast<int>(slot - first_item(s.row0, max(s.b, 0), mul, div, extra)));
  return s;
}

}  // namespace rlq
