// Four-bit weights: blocks of 32 numbers along a row share one power-of-two scale (a byte S, the scale is 2^(S - 127); 255: the
// block is not a number), each number is a sign, two bits of exponent and one of mantissa (magnitudes 0, 1/2, 1, 3/2, 2, 3, 4, 6).
//
// Two layouts.  Rows: codes [rows][16 bytes a block], element 2 i of a block in the low half of byte i, and scales
// [rows][blocks].  Tiles, what the product reads: 128 rows x 128 columns in MX_TILE_BYTES contiguous bytes, zeros beyond the
// matrix, row tile by row tile, within one along the columns: [block of 32 columns][row][16 bytes of codes], then the scales as
// tcgen05.mma wants them in tensor memory, [lane i][j] words of the four scales of row 32 j + i.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

constexpr int MX_BLOCK = 32;                                             // numbers that share a scale
constexpr int MX_LAST_SCALE = 252;                                       // the largest that quantising writes: 6 x 2^125 is a float32
constexpr int MX_ROWS = 128, MX_COLS = 128;                              // a tile
constexpr int MX_CODE_BYTES = MX_ROWS * MX_COLS / 2;
constexpr int MX_TILE_BYTES = MX_CODE_BYTES + MX_ROWS * MX_COLS / MX_BLOCK;

// tcgen05.mma takes such numbers (e2m1) from tensor memory in bytes, the code in bits 5 to 2, zeros around it.  Eight codes in a
// 32-bit word of a tile: columns 0..3 where they are wanted, columns 4..7 in the bits between, four places further in a word that turns.
__host__ __device__ __forceinline__ uint32_t mx_place(uint32_t code, int column) {
    const int to = 8 * (column & 3) + (column < 4 ? 2 : 30) & 31;
    return code << to | (to > 28 ? code >> (32 - to) : 0u);
}
// The bytes of columns 0..3 and 4..7.
__device__ __forceinline__ void mx_decode(uint32_t w, uint32_t& first, uint32_t& second) {
    first = w & 0x3C3C3C3Cu;
    second = __funnelshift_l(w, w, 4) & 0x3C3C3C3Cu;
}
// 2^(S - 127) in float32.
__device__ __forceinline__ float mx_scale_f32(uint32_t s) {
    return __uint_as_float(s == 255u ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
}

// ---- rows of bfloat16 numbers as two e4m3 numbers each ----
// With 2^e <= amax < 2^(e + 1) the largest magnitude of a block of 32, y = x 2^(7 - e) lies below 2^8; its first part is y rounded
// to e4m3, its second what that left, times 2^5.  Eight bits of mantissa go into four and four where |y| >= 2^-7: such numbers, down to
// 2^-14 of 2^e, are held exactly.  Below, the second part's last place, 2^-14, rounds them: what is lost is at most 2^-15, or 2^-22 of
// amax.  That is a rounding to fewer bits than bfloat16 has, of numbers that stand beside one 2^14 times as large.
// Scales: MX_FIRST less than the exponent's field for the first part, 5 less again for the second; blocks below 2^-115 use that
// exponent's, and lose 2^-137 at most (nothing of a bfloat16 number).  A block with an infinity or a NaN gets scales of 255, and so do
// the sums that it is part of.
constexpr int MX_LEAST_FIELD = 12, MX_FIRST = 7, MX_SECOND_LESS = 5;
// `top`: the largest magnitude's 15 bits of the block.
__device__ __forceinline__ uint32_t mx_row_scale(uint32_t top) {
    const uint32_t field = top >> 7;
    return field == 255u ? 255u : max(field, (uint32_t)MX_LEAST_FIELD) - MX_FIRST;
}
// Eight numbers (pairs in four words) under the block's scale: bytes of the first and the second parts.  y goes through half precision,
// which holds eight bits of mantissa from 2^-14 on and is off by at most 2^-25 below.
__device__ __forceinline__ void mx_split8(const uint4& eight, uint32_t scale, uint2& first, uint2& second) {
    const uint32_t w[4] = {eight.x, eight.y, eight.z, eight.w};
    const float inv = __uint_as_float((scale == 255u ? 127u : 254u - scale) << 23);
    const __half2 by = __float2half2_rn(32.0f);
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 y = __floats2half2_rn(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);
        uint16_t p, q;
        uint32_t back;
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(p) : "r"(*reinterpret_cast<const uint32_t*>(&y)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(p));
        const __half2 left = __hmul2(__hsub2(y, *reinterpret_cast<const __half2*>(&back)), by);
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(q) : "r"(*reinterpret_cast<const uint32_t*>(&left)));
        h[i] = p;
        l[i] = q;
    }
    first = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    second = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
}
__device__ __forceinline__ uint32_t mx_second_scales(uint32_t four) {       // of four first ones (255 stays; a sum is NaN by the first)
    return __vsubus4(four, 0x01010101u * MX_SECOND_LESS);
}
// Eight numbers of a row from column k on: zeros from K on.  `aligned`: the row starts on a 16-byte border.
__device__ __forceinline__ uint4 mx_load8(const __nv_bfloat16* row, int k, int K, bool aligned) {
    if (aligned && k + 8 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < K ? (uint32_t)__bfloat16_as_ushort(row[k + i]) : 0u;
    return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}
// The largest magnitudes' bits among eight numbers, of the even and of the odd ones.
__device__ __forceinline__ uint32_t mx_top8(const uint4& v) {
    constexpr uint32_t MAGNITUDES = 0x7fff7fffu;
    return __vmaxu2(__vmaxu2(v.x & MAGNITUDES, v.y & MAGNITUDES), __vmaxu2(v.z & MAGNITUDES, v.w & MAGNITUDES));
}

// A block of 32 numbers of a row, of which four neighbouring lanes have the four of 128 columns: its parts, and for the first of the
// four lanes their scales.
__device__ __forceinline__ uint32_t mx_split_block(const uint4 (&v)[4], uint2 (&one)[4], uint2 (&two)[4]) {
    const uint32_t top = __vmaxu2(__vmaxu2(mx_top8(v[0]), mx_top8(v[1])), __vmaxu2(mx_top8(v[2]), mx_top8(v[3])));
    const uint32_t scale = mx_row_scale(max(top & 0xffffu, top >> 16));
    const uint32_t half = scale | __shfl_down_sync(0xffffffffu, scale, 1) << 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) mx_split8(v[i], scale, one[i], two[i]);
    return half | __shfl_down_sync(0xffffffffu, half, 2) << 16;
}
// Where a row's word of scales lies among those of a tile.
__device__ __forceinline__ int mx_scale_place(int row) { return (row >> 7) * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4; }

// Rows that a product reads: row m is x[m], or x[index[m]] (zeros where that is none of x's `count`), times share[pair[m]] (rounded
// to bfloat16) where there are shares.
struct MxRows {
    const __nv_bfloat16* x; long ld; int count, aligned;
    const int* index; const float* share; const int* pair;
};
// Eight numbers times f, rounded to bfloat16.
__device__ __forceinline__ uint4 mx_times(uint4 v, float f) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return v;
}
// Where the rows' scales go: [K / 128][token tile][tile_bytes], for a tile of n tokens the first parts as rows 0 .. and the second ones
// up to 64 tokens as rows n .., else from the next multiple of 128 on, by 128 rows as [lane i][j] words of row 32 j + i.  A tile is
// `tokens` rows; grouped: up to `most` neighbouring row tiles of `tile` rows of one group, in the place of the first of them.
// Rows of a tile whose group is none of the `groups` get scales of 255.
struct MxScaleLayout { int tokens, tile_bytes; const int* tile_group; int tile, most, n_tiles, groups; };
int fb_mxfp4_split_rows(const MxRows& rows, int M, int K, void* parts, void* scales, const MxScaleLayout& layout, cudaStream_t stream);
