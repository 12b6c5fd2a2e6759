// The 4-bit key/value cache: where a token's codes and a group's two numbers lie in a page.
//
// Each group of 32 features of a token of a key/value head keeps mn = bfloat16(min) and sc = bfloat16((max - mn) / 15) as the word
// sc << 16 | mn, and a code of 4 bits per feature; a feature stands for mn + sc * code.  A pool is [page][kv head][bytes]: a page
// of 64 tokens of one head is HD / 64 tiles of 5,120 bytes, each of 4096 / HD tokens (64 tokens of a head of 64, 32 of a head of 128):
//
//   2,048 bytes  key codes: per token the words (t, group), t = 0..3, features 32 group + 8 t + e in nibble e / 2 + 4 (e % 2)
//     512 bytes  the keys' words, per token and group
//   2,048 bytes  value codes: per 16 tokens, 64 features (half) and g = 0..7 the words (t, u), t, u = 0..3, of token 8 (u / 2) + 2 t + u % 2,
//                features 64 half + 4 g + n in nibble n, 64 half + 32 + 4 g + n in nibble 4 + n
//     512 bytes  the values' words
//
// That is the order in which mma.m16n8k16 wants its operands: a lane of a warp reads its part of 16 keys (as the 16 x 16 operand) or of the
// values of 16 tokens (transposed) with one conflict-free vector load, and a tile is one contiguous copy.
#pragma once

#include "common.cuh"

namespace exl3 {
namespace kv4 {

constexpr int PAGE = 64;
constexpr int TILE = 5120;
constexpr int K_WORDS = 2048, V_CODES = 2560, V_WORDS = 4608;      // byte offsets in a tile
constexpr float SC_MIN = 1e-30f;                                    // scales not above it count as zero: all codes are 0

__host__ __device__ constexpr int tile_tokens(int hd) { return 4096 / hd; }
__host__ __device__ constexpr int page_bytes(int hd) { return hd / 64 * TILE; }

// Byte of the value word (half, g) of token tok (of the tile's) in the tile.
template <int HD> __device__ inline int v_word(int tok, int half, int g) {
  const int u = tok & 15;
  return V_CODES + ((((tok >> 4) * (HD / 64) + half) * 8 + g) * 4 + ((u & 7) >> 1)) * 16 + ((u >> 3) * 2 + (u & 1)) * 4;
}
// Byte of the key word (t, group).
template <int HD> __device__ inline int k_word(int tok, int t, int group) { return tok * (HD / 2) + (t * (HD / 32) + group) * 4; }

__device__ inline float word_sc(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ inline float word_mn(uint32_t w) { return __uint_as_float(w << 16); }

}  // namespace kv4
}  // namespace exl3
