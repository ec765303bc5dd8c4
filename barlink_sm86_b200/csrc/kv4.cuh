// SPDX-License-Identifier: MIT
//
// The 4-bit key/value cache: what a tile of it looks like.
//
// A cache is [blocks][KV heads][block_size / 16] tiles; a tile holds 16 tokens of one head, 20 * hd bytes:
//
//   K codes   16 rows of hd/2 bytes.  The 8 codes of dims 32 a + 8 t + e (e = nibble of a 32-bit word) are word
//             t * NA + a of the row, NA = hd / 32 groups: lane t of a quad finds its share of every group in one load.
//   V codes   8 token pairs of hd bytes.  Dims 4 (8 a + g) + i of the pair's tokens are word g * NA + a: nibbles 0..3 the
//             first token's, 4..7 the second's, so that one mask leaves two tokens of a dim in the halves of a register.
//   K params  16 rows: step[NA], low[NA], bf16.
//   V params  the same.
//
// A code c of 0..15 stands for low + step * c.  A byte belongs to one token, so tokens are written without reading.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace bl {

constexpr int kQ4Tokens = 16;  // of a tile
constexpr int kQ4Group = 32;   // dims that share step and low

__host__ __device__ constexpr int q4_tile_bytes(int hd) { return 20 * hd; }
__host__ __device__ constexpr int q4_v_codes(int hd) { return 8 * hd; }
__host__ __device__ constexpr int q4_k_params(int hd) { return 16 * hd; }
__host__ __device__ constexpr int q4_v_params(int hd) { return 18 * hd; }

// one head's tile of token slot % block_size of block slot / block_size
__device__ __forceinline__ size_t q4_tile_offset(int blk, int in_block, int h, int nkv, int block_size, int hd) {
  return ((size_t(blk) * nkv + h) * (block_size / kQ4Tokens) + in_block / kQ4Tokens) * q4_tile_bytes(hd);
}

}  // namespace bl
