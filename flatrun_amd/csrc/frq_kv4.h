// The 4-bit paged cache: how a tile of 32 tokens of one key head lies in
// memory, shared by the kernels that write, read and attend to it.
//
// A block is 32 channels of one head of one token: e its element of largest
// magnitude (the first of equals), d = fp16(-e / 8) held to +-65504, code =
// round_even(x / d) + 8 held to [0, 15], value d (code - 8): the values of a
// Q4_0 block. A block that holds an inf or a NaN has d = NaN.
//
// The cache is [page][head][tile]; a page holds a multiple of 32 tokens. A
// tile of NG = head_dim / 32 blocks a token is 1152 NG bytes,
//   K codes 512 NG | K scales 64 NG | V codes 512 NG | V scales 64 NG
// with the codes in the order in which the matrix instructions
// (v_mfma_f32_16x16x32_f16) take them, so that a lane of the attention kernel
// has its operands after 16-byte loads, a mask and an offset, and no code
// passes through LDS or another lane:
//   K  token t = 16u + m, channel 32g + 8j + c: lane 16j + m, word u NG + g,
//      nibble c/2 + 4 (c%2). Lane l's column m = l%16 of the product q K^T,
//      its eight k-slots the channels 8j .. 8j + 7 of group g.
//   V  token t = 16u + 4j + i, channels 32g + n (low nibble) and 32g + 16 + n
//      (high): lane 16j + n, word 2g + u, byte {0, 2, 1, 3}[i]. The eight
//      k-slots of lane group j in P V are the tokens 4j .. 4j + 3 and
//      16 + 4j .. 16 + 4j + 3.
// Word p of lane l is at 16 (64 (p / 4) + l) + 4 (p % 4). The scale of token t
// and group g is number (2 (t % 16) + t / 16) NG + g: both tokens of a lane of
// the first product in one load.
#pragma once

#include "frq_vals.h"

namespace frq {

constexpr int kKvTile = 32;           // tokens
constexpr int kKvBlock = 32;          // channels that share a scale

constexpr int kv_tile_bytes(int ng) { return 1152 * ng; }
constexpr int kv_ks_off(int ng) { return 512 * ng; }
constexpr int kv_vc_off(int ng) { return 576 * ng; }
constexpr int kv_vs_off(int ng) { return 1088 * ng; }

// Byte offset of word p of lane l within a tile's K or V codes.
__host__ __device__ constexpr int kv_word(int p, int lane) { return 16 * (64 * (p >> 2) + lane) + 4 * (p & 3); }

// Byte offset of the scale of token t (of the tile), group g.
__host__ __device__ constexpr int kv_scale(int t, int g, int ng) { return 2 * ((2 * (t & 15) + (t >> 4)) * ng + g); }

}  // namespace frq
