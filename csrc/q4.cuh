// Format of the 4-bit key / value cache, shared by the kernels that write, read and attend over it.
//
// A page of one kv head is block_size / 16 tiles; a tile holds 16 tokens in 18 * head size bytes:
//   [keys: 8 hd][values: 8 hd][scales: 16 tokens x (ng of the keys, ng of the values) fp16],  ng = hd / 32.
// A code n stands for scale * (n - 8), one scale per token and 32 neighbouring elements.
//
// The order of the codes is that of the mma.sync fragments of the attention kernel, so that a lane loads its operands with
// 16-byte accesses, a warp's access is 512 neighbouring bytes, and no code moves between lanes. Lane 4 r + c, word
// i = j * ng + g (at byte (i / 4) * 512 + lane * 16 + (i % 4) * 4 of its half):
//   keys    token 8 j + r, elements 32 g + 8 c + (0..7), lowest nibble first: a row of the A operand of K Q^T;
//   values  tokens 8 j + 2 c (low 16 bits) and 8 j + 2 c + 1 (high), elements 32 g + 4 r + (0..3): four rows of V^T, two
//           neighbours of the contraction in one register.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace icb {

constexpr int kQ4Tile = 16;                                   // tokens of a tile

__host__ __device__ constexpr int q4_tile_bytes(int hd) { return 18 * hd; }

__device__ __forceinline__ int q4_word_at(int i, int lane) { return (i >> 2) * 512 + lane * 16 + (i & 3) * 4; }

// Word of token t (0..15) and elements 8 * chunk + (0..7) of the keys.
__device__ __forceinline__ int q4_key_at(int ng, int t, int chunk) {
  return q4_word_at((t >> 3) * ng + (chunk >> 2), (t & 7) * 4 + (chunk & 3));
}
// Half word of token t and elements 4 * quad + (0..3) of the values (from the start of the values' half).
__device__ __forceinline__ int q4_value_at(int ng, int t, int quad) {
  return q4_word_at((t >> 3) * ng + (quad >> 3), (quad & 7) * 4 + ((t & 7) >> 1)) + (t & 1) * 2;
}

// A slot (block * block_size + offset) of kv head h as its tile's first byte.
__device__ __forceinline__ long long q4_tile_of(long long slot, int h, int hkv, int tiles, int tile_bytes) {
  const long long block = slot / (tiles * kQ4Tile);
  const int inside = (int)(slot - block * (tiles * kQ4Tile));
  return ((block * hkv + h) * tiles + (inside >> 4)) * tile_bytes;
}

}  // namespace icb
