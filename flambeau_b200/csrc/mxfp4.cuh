// Four-bit weights: blocks of 32 numbers along a row share one power-of-two scale (a byte S, the scale is 2^(S - 127); 255: the
// block is not a number), each number is a sign, two bits of exponent and one of mantissa (magnitudes 0, 1/2, 1, 3/2, 2, 3, 4, 6).
//
// Two layouts.  Rows: codes [rows][16 bytes a block], element 2 i of a block in the low half of byte i, and scales
// [rows][blocks].  Tiles, what the product reads: 128 rows x 128 columns in MX_TILE_BYTES contiguous bytes, zeros beyond the
// matrix, row tile by row tile, within one along the columns: [block of 32 columns][row][16 bytes], then [row][4 scales].  One bulk
// copy fetches a tile, and the 32 threads of a warp, a row each, read 512 contiguous bytes of shared memory.
#pragma once

#include "common.cuh"

constexpr int MX_BLOCK = 32;                                             // numbers that share a scale
constexpr int MX_LAST_SCALE = 252;                                       // the largest that quantising writes: 6 x 2^125 is a float32
constexpr int MX_ROWS = 128, MX_COLS = 128;                              // a tile
constexpr int MX_CODE_BYTES = MX_ROWS * MX_COLS / 2;
constexpr int MX_TILE_BYTES = MX_CODE_BYTES + MX_ROWS * MX_COLS / MX_BLOCK;
// Scales up to 2^1 are multiplied in as they are (see mx_decode); a matrix with larger ones carries a shift that its scales are
// lowered by in the tiles, and that the product's results are raised by.
constexpr int MX_TOP_SCALE = 128;

// Eight codes in a 32-bit word of a tile: columns 2 j and 2 j + 1 (j = 0..3) in the lower and upper half, their bits where one
// shift and one mask (for j = 3 three of each) bring the sign to bit 15 and the three magnitude bits to bits 8..6 of a
// bfloat16: as the end of its exponent and the first bit of its mantissa they are the number times 2^-126, subnormal ones
// included, which one multiplication by 2^(S - 1) puts right.
//   j = 0: bits 15, 8, 7, 6    j = 1: 12, 5, 4, 3    j = 2: 9, 2, 1, 0    j = 3: 14, 13, 11, 10
__host__ __device__ __forceinline__ uint32_t mx_place(uint32_t code, int j) {       // one code's bits within its half
    const uint32_t s = code >> 3, m = code & 7u;
    if (j == 3) return s << 14 | (m >> 2) << 13 | (m & 3u) << 10;
    return (s << 15 | m << 6) >> (3 * j);
}
__device__ __forceinline__ uint32_t mx_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// The four pairs of a word, times `scale` (a bfloat16 pair of 2^(S - 1)).
__device__ __forceinline__ void mx_decode(uint32_t w, uint32_t scale, uint32_t* out) {
    constexpr uint32_t MASK = 0x81C081C0u;
    out[0] = mx_mul(w & MASK, scale);
    out[1] = mx_mul((w << 3) & MASK, scale);
    out[2] = mx_mul((w << 6) & MASK, scale);
    out[3] = mx_mul(((w << 1) & 0x80008000u) | ((w >> 5) & 0x01000100u) | ((w >> 4) & 0x00C000C0u), scale);
}
// 2^(S - 1) twice, for scales of a tile (0 .. MX_TOP_SCALE, 255: not a number).
__device__ __forceinline__ uint32_t mx_scale(uint32_t s) {
    const uint32_t one = s == 255u ? 0x7FC0u : (s + 126u) << 7;
    return one | one << 16;
}
