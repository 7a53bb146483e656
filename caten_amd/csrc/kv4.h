// The KV cache of a batch of sequences in 4 bits, in one pool of pages (kv4.hip, kv4_attn.hip): how a page is laid out.
// A page holds kKvPageRows rows of every key / value head; (n_pages, kv_heads, kv4_head_bytes) bytes for the keys and as
// many for the values.  A block of 32 channels of a row is one fp16 scale d and 32 numbers -8 .. 7 (GGUF's Q4_0 block with
// the numbers as two's complement nibbles).  A head's part of a page: 32 Dh bytes of quants, then 4 Dh bytes of scales.
//   keys    [row][8-channel group g of a block][block][4 bytes]: a lane that holds one row and one g finds its 8 channels
//           of every block side by side, and one group's 4 x 8 channels are what one matrix instruction takes per block.
//           Low nibbles: channels 0 .. 3 of the group, high ones 4 .. 7.
//   values  [block][channel % 16][row, reordered]: transposed, since the product over rows wants many rows of one channel in
//           a lane.  Low nibbles: channels 0 .. 15 of the block, high ones 16 .. 31.  Row 16 s + 4 g + i lies at 16 g + 4 s + i:
//           the rows whose probabilities lane group g holds after the product with the keys are then 16 bytes in a row.
//   scales  [row / 4][block][row % 4] in both.
// No byte is shared by two rows, so rows may be written by different threads in any order.
#pragma once
#include "common.h"

namespace cthip {

constexpr int kKv4MaxSeqs = 4096;  // sequences of one call (their starts are kept in LDS)
static_assert(kKvPageRows == 64, "the reordering of a value page's rows");
__host__ __device__ inline int kv4_head_bytes(int dh) { return 36 * dh; }
__host__ __device__ inline int kv4_key_offset(int row, int g, int b, int dh) { return row * (dh >> 1) + g * (dh >> 3) + 4 * b; }
__host__ __device__ inline int kv4_value_place(int row) { return ((row >> 2) & 3) * 16 + (row >> 4) * 4 + (row & 3); }
__host__ __device__ inline int kv4_value_offset(int row, int b, int c) { return (b * 16 + c) * kKvPageRows + kv4_value_place(row); }
__host__ __device__ inline int kv4_scale_offset(int row, int b, int dh) { return 32 * dh + (((row >> 2) * (dh >> 5) + b) * 4 + (row & 3)) * 2; }
inline bool kv4_shape_ok(int kv_heads, int head_dim) {
  return kv_heads > 0 && kv_heads <= 65535 && (head_dim == 32 || head_dim == 64 || head_dim == 128);
}

}  // namespace cthip
