// Rows into four bits and back, and the tiles that the product reads (formats in mxfp4.cuh).
//
// A block's scale is the smallest power of two, not below 2^-127, under which its largest magnitude stays below 7, where rounding
// still ends at 6: with amax = m 2^e, 1 <= m < 2, it is 2^(e - 2), or 2^(e - 1) where m >= 1.75.  Scales end at 2^125, so that every
// number of a block is a finite float32; magnitudes above 6 times that become it.  Codes are the nearest of the grid, ties to the even
// code.  Both follow from bits and from products with powers of two, so they are the same on any machine.  A block with an infinity or
// a NaN gets scale 255 and decodes to NaN.
//
// Bound by memory: 2 or 4 bytes in, 17/32 out.  Four threads share a block, eight numbers each; a warp reads 512 bytes (bfloat16) in
// a row.
#include "mxfp4.cuh"

#include <cuda_fp16.h>

namespace {

// Eight numbers of a row from column c on; zeros beyond K.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// One quarter of a block: eight numbers into codes; the lanes of a block are neighbours.  Every lane of the warp.
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], uint32_t& scale) {
    uint32_t top = 0;                                                    // the largest magnitude's bits (NaN above infinity)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int s = min(MX_LAST_SCALE, max(0, (int)(top >> 23) - 2 + ((top & 0x7fffffu) >= 0x600000u ? 1 : 0)));
    const float inv = __uint_as_float((uint32_t)(254 - s) << 23);        // 2^(127 - s)
    uint32_t out;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(out)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv), "f"(v[6] * inv),
          "f"(v[7] * inv));
    const bool finite = top < 0x7f800000u;
    scale = finite ? (uint32_t)s : 255u;
    return finite ? out : 0u;
}

// Rows of whole blocks, one behind the other on 16-byte borders: UNROLL quarters a thread, all fetched before the first is used.
// (28,672 x 4,096 bfloat16 with the form below: 94 us, of which 45 are memory's; like this 49.)
constexpr int UNROLL = 4;
template <typename T>
__global__ void __launch_bounds__(256)
quantize_flat_kernel(const T* __restrict__ x, long quarters, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    fb_pdl_launch_dependents();
    fb_pdl_wait();
    const long first = (long)blockIdx.x * (256 * UNROLL) + threadIdx.x;
    float v[UNROLL][8];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long q = first + 256 * u;
        if (q < quarters) load8(x + 8 * q, v[u]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long q = first + 256 * u;
        uint32_t scale;
        const uint32_t out = quantize8(v[u], scale);
        if (q < quarters) {
            reinterpret_cast<uint32_t*>(codes)[q] = out;
            if ((q & 3) == 0) scales[q >> 2] = (uint8_t)scale;
        }
    }
}

// Any rows.  VEC: they start on 16-byte borders.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
quantize_kernel(const T* __restrict__ x, long ldx, long rows, int K, int blocks, uint8_t* __restrict__ codes,
                uint8_t* __restrict__ scales) {
    fb_pdl_launch_dependents();
    fb_pdl_wait();
    const long quarters = rows * blocks * 4;                             // a quarter: eight numbers
    const long step = (long)gridDim.x * 256;
    for (long base = (long)blockIdx.x * 256; base < quarters; base += step) {     // (whole warps stay together for the shuffles)
        const long q = base + threadIdx.x;
        const bool mine = q < quarters;
        const long row = mine ? q / (blocks * 4) : 0;
        const int c = mine ? 8 * (int)(q - row * (blocks * 4)) : 0;
        float v[8];
        const T* p = x + row * ldx + c;
        if (VEC && mine && c + 8 <= K) {
            load8(p, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = mine && c + i < K ? fb_to_float(p[i]) : 0.0f;
        }
        uint32_t scale;
        const uint32_t out = quantize8(v, scale);
        if (mine) {
            reinterpret_cast<uint32_t*>(codes)[q] = out;                 // (quarters of a row follow one another)
            if ((q & 3) == 0) scales[q >> 2] = (uint8_t)scale;
        }
    }
}

// Eight codes into the numbers that they stand for.
template <typename T>
__device__ __forceinline__ void dequantize8(uint32_t w, float scale, T (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t pair;                                                   // (two codes of a byte in float16)
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}" : "=r"(pair) : "r"(w >> (8 * i)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        v[2 * i] = fb_from_float<T>(f.x * scale);
        v[2 * i + 1] = fb_from_float<T>(f.y * scale);
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
dequantize_flat_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, long quarters, T* __restrict__ out) {
    fb_pdl_launch_dependents();
    fb_pdl_wait();
    const long first = (long)blockIdx.x * (256 * UNROLL) + threadIdx.x;
    uint32_t w[UNROLL], s[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long q = first + 256 * u;
        w[u] = q < quarters ? reinterpret_cast<const uint32_t*>(codes)[q] : 0u;
        s[u] = q < quarters ? scales[q >> 2] : 0u;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long q = first + 256 * u;
        alignas(16) T v[8];
        dequantize8(w[u], mx_scale_f32(s[u]), v);
        if (q < quarters) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4*>(out + 8 * q)[i] = reinterpret_cast<const uint4*>(v)[i];
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, long rows, int K, int blocks,
                  T* __restrict__ out, long ldo) {
    fb_pdl_launch_dependents();
    fb_pdl_wait();
    const long quarters = rows * blocks * 4, step = (long)gridDim.x * 256;
    for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < quarters; q += step) {
        const long row = q / (blocks * 4);
        const int c = 8 * (int)(q - row * (blocks * 4));
        alignas(16) T v[8];
        dequantize8(reinterpret_cast<const uint32_t*>(codes)[q], mx_scale_f32(scales[q >> 2]), v);
        T* p = out + row * ldo + c;
        if (VEC && c + 8 <= K) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < K) p[i] = v[i];
        }
    }
}

// The kernel that writes the tiles lets no kernel behind it in before it ends: the product asks for its first weights ahead of its
// wait for the kernel before it, and that kernel may have come in early itself.
// A thread a row and block of 32 columns: its 16 bytes of codes in the tiles' order, its scale.
__global__ void __launch_bounds__(128)
tiles_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int N, int blocks, int tiles_k, uint8_t* __restrict__ tiles) {
    fb_pdl_wait();
    const int row = threadIdx.x, b = blockIdx.x, n = blockIdx.y * MX_ROWS + row, group = blockIdx.z;
    const size_t tile = ((size_t)group * gridDim.y + blockIdx.y) * tiles_k + b / 4;
    uint8_t* dst = tiles + tile * MX_TILE_BYTES;
    uint32_t w[4] = {0, 0, 0, 0};
    int s = 0;
    if (n < N && b < blocks) {
        const size_t at = ((size_t)group * N + n) * blocks + b;
        const uint4 c = reinterpret_cast<const uint4*>(codes)[at];
        const uint32_t in[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[i] |= mx_place(in[i] >> (4 * j) & 15u, j);
        s = scales[at];
    }
    reinterpret_cast<uint4*>(dst)[(b & 3) * MX_ROWS + row] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[MX_CODE_BYTES + ((row & 31) * 4 + (row >> 5)) * 4 + (b & 3)] = (uint8_t)s;
}

// A thread a block of 32 numbers, SPLIT_ROWS rows (of one tile) a group of blocks: parts[p][m][k] (bytes, rows of Kp, a multiple of 128,
// zeros behind K), their scales as `layout` says.  (14,336 x 4,096 numbers, 117 MB in and out each: 45 us, memory's 36; a thread eight
// numbers, where what is not conversion outweighs it, took 61.)
constexpr int SPLIT_ROWS = 4;
template <bool GROUPED>
__global__ void __launch_bounds__(256)
split_kernel(const __grid_constant__ MxRows rows, int M, int K, int Kp, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales,
             const __grid_constant__ MxScaleLayout layout) {
    // (grouped: the product comes in behind the wait, and so behind the kernels that order the rows: it looks up its weights and asks
    // for them while the rows are split)
    if constexpr (!GROUPED) fb_pdl_launch_dependents();
    fb_pdl_wait();
    if constexpr (GROUPED) fb_pdl_launch_dependents();
    const int blocks = Kp / MX_BLOCK, lane = threadIdx.x & 31, first = blockIdx.x * SPLIT_ROWS;
    const int item = blockIdx.y * 256 + threadIdx.x, q = item / blocks, m = first + q, k = (item - q * blocks) * MX_BLOCK;
    int unit, tokens, at, tiles;                         // the scales' tile, its tokens, the first row's place in it, all tiles
    bool no_group = false;                               // (the tile's group is beyond the weights: its sums are to be NaN)
    if constexpr (GROUPED) {
        const int t = first / layout.tile, g = layout.tile_group[t];
        if (g < 0) return;                               // (rows of tiles without a group are not multiplied, whatever they hold)
        no_group = g >= layout.groups;
        unit = t;
        int n = 1;
        if (layout.most > 1) {
            // where the run of tiles of this group begins, 32 at a time, and so where the unit of up to `most` that holds t does
            int begin = 0;
            for (int t0 = t; t0 > 0; t0 -= 32) {
                const int left = t0 - 1 - lane;
                const uint32_t other = __ballot_sync(0xffffffffu, left < 0 || layout.tile_group[left] != g);
                if (other) {
                    begin = t0 - (__ffs((int)other) - 1);
                    break;
                }
            }
            unit = begin + (t - begin) / layout.most * layout.most;
            while (n < layout.most && unit + n < layout.n_tiles && layout.tile_group[unit + n] == g) ++n;
        }
        tokens = n * layout.tile;
        at = first - unit * layout.tile;
        tiles = layout.n_tiles;
    } else {
        unit = first / layout.tokens;
        tokens = layout.tokens;
        at = first - unit * layout.tokens;
        tiles = (M + layout.tokens - 1) / layout.tokens;
    }
    const bool mine = q < SPLIT_ROWS && m < M;           // (of the four lanes that share 128 columns all or none)
    const int from = mine ? rows.index ? rows.index[m] : m : -1;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_uint4(0, 0, 0, 0);
    if (from >= 0 && from < rows.count) {
        const __nv_bfloat16* row = rows.x + (size_t)from * rows.ld;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = mx_load8(row, k + 8 * i, K, rows.aligned != 0);
        if (rows.share) {
            const float share = rows.share[rows.pair[m]];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = mx_times(v[i], share);
        }
    }
    uint2 one[4], two[4];
    uint32_t word = mx_split_block(v, one, two);
    if (GROUPED && no_group) word = 0xffffffffu;
    if (!mine) return;
    uint4* to_first = reinterpret_cast<uint4*>(parts + (size_t)m * Kp + k);
    uint4* to_second = reinterpret_cast<uint4*>(parts + ((size_t)M + m) * Kp + k);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        to_first[h] = make_uint4(one[2 * h].x, one[2 * h].y, one[2 * h + 1].x, one[2 * h + 1].y);
        to_second[h] = make_uint4(two[2 * h].x, two[2 * h].y, two[2 * h + 1].x, two[2 * h + 1].y);
    }
    if ((lane & 3) == 0) {
        const int apart = tokens <= 64 ? tokens : (tokens + 127) / 128 * 128;
        uint8_t* to = scales + ((size_t)(k >> 7) * tiles + unit) * layout.tile_bytes;
        *reinterpret_cast<uint32_t*>(to + mx_scale_place(at + q)) = word;
        *reinterpret_cast<uint32_t*>(to + mx_scale_place(apart + at + q)) = mx_second_scales(word);
    }
}

int grid_of(long threads, int per_block) {
    const long blocks = (threads + per_block - 1) / per_block, most = 8L * fb_sm_count();
    return (int)(blocks < most ? blocks : most);
}

}  // namespace

// codes [rows, 16 ceil(K / 32)] and scales [rows, ceil(K / 32)] (contiguous) of x [rows, K], float32 or bfloat16 with rows ldx
// elements apart; the columns behind K of a row's last block count as zeros.
FB_API int fb_quantize_mxfp4(const void* x, int dtype, long long ldx, long long rows, int K, void* codes, void* scales,
                             cudaStream_t stream) {
    FB_REQUIRE(rows >= 0 && K > 0 && K <= (1 << 30), "quantize_mxfp4: bad sizes");
    FB_REQUIRE(ldx >= K || rows <= 1, "quantize_mxfp4: a row stride is shorter than its row");
    FB_REQUIRE(((uintptr_t)codes & 15) == 0, "quantize_mxfp4: codes must be 16-byte aligned");
    if (rows == 0) return 0;
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    FB_DISPATCH_DTYPE(dtype, T, {
        const bool vec = ((uintptr_t)x & 15) == 0 && (rows == 1 || ldx * sizeof(T) % 16 == 0);
        if (vec && K % MX_BLOCK == 0 && (rows == 1 || ldx == K) && rows * blocks < (1LL << 36)) {
            const long quarters = (long)rows * blocks * 4, per = 256 * UNROLL;
            fb_launch((quantize_flat_kernel<T>), dim3((unsigned)((quarters + per - 1) / per)), dim3(256), 0, stream, (const T*)x, quarters,
                      (uint8_t*)codes, (uint8_t*)scales);
            return fb_check_launch("quantize_mxfp4");
        }
        auto kernel = vec ? quantize_kernel<T, true> : quantize_kernel<T, false>;
        fb_launch(kernel, dim3(grid_of((long)rows * blocks * 4, 256)), dim3(256), 0, stream, (const T*)x, (long)ldx, (long)rows, K,
                  blocks, (uint8_t*)codes, (uint8_t*)scales);
    });
    return fb_check_launch("quantize_mxfp4");
}

// out [rows, K], float32 or bfloat16: the numbers that codes and scales stand for (bfloat16 holds them exactly;
// 4 and 6 times 2^127, which fb_quantize_mxfp4 never writes, are infinite in both).
FB_API int fb_dequantize_mxfp4(const void* codes, const void* scales, long long rows, int K, void* out, int dtype, long long ldo,
                               cudaStream_t stream) {
    FB_REQUIRE(rows >= 0 && K > 0 && K <= (1 << 30), "dequantize_mxfp4: bad sizes");
    FB_REQUIRE(ldo >= K || rows <= 1, "dequantize_mxfp4: a row stride is shorter than its row");
    FB_REQUIRE(((uintptr_t)codes & 15) == 0, "dequantize_mxfp4: codes must be 16-byte aligned");
    if (rows == 0) return 0;
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK;
    FB_DISPATCH_DTYPE(dtype, T, {
        const bool vec = ((uintptr_t)out & 15) == 0 && (rows == 1 || ldo * sizeof(T) % 16 == 0);
        if (vec && K % MX_BLOCK == 0 && (rows == 1 || ldo == K) && rows * blocks < (1LL << 36)) {
            const long quarters = (long)rows * blocks * 4, per = 256 * UNROLL;
            fb_launch((dequantize_flat_kernel<T>), dim3((unsigned)((quarters + per - 1) / per)), dim3(256), 0, stream, (const uint8_t*)codes,
                      (const uint8_t*)scales, quarters, (T*)out);
            return fb_check_launch("dequantize_mxfp4");
        }
        auto kernel = vec ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
        fb_launch(kernel, dim3(grid_of((long)rows * blocks * 4, 256)), dim3(256), 0, stream, (const uint8_t*)codes,
                  (const uint8_t*)scales, (long)rows, K, blocks, (T*)out, (long)ldo);
    });
    return fb_check_launch("dequantize_mxfp4");
}

// Bytes of one matrix [N, K] in tiles.
FB_API long long fb_mxfp4_tile_bytes(int N, int K) {
    return ((long long)N + MX_ROWS - 1) / MX_ROWS * (((long long)K + MX_COLS - 1) / MX_COLS) * MX_TILE_BYTES;
}

// `groups` matrices [N, K] from rows (codes, scales as fb_quantize_mxfp4 writes them) into tiles.
FB_API int fb_mxfp4_tiles(const void* codes, const void* scales, int groups, int N, int K, void* tiles, cudaStream_t stream) {
    FB_REQUIRE(groups > 0 && N > 0 && K > 0 && groups <= 65535 && N <= 65535 * MX_ROWS && K <= (1 << 30), "mxfp4_tiles: bad sizes");
    FB_REQUIRE(((uintptr_t)codes & 15) == 0 && ((uintptr_t)tiles & 15) == 0, "mxfp4_tiles: operands must be 16-byte aligned");
    const int blocks = (K + MX_BLOCK - 1) / MX_BLOCK, tiles_k = (K + MX_COLS - 1) / MX_COLS;
    fb_launch(tiles_kernel, dim3(4 * tiles_k, (N + MX_ROWS - 1) / MX_ROWS, groups), dim3(128), 0, stream, (const uint8_t*)codes,
              (const uint8_t*)scales, N, blocks, tiles_k, (uint8_t*)tiles);
    return fb_check_launch("mxfp4_tiles");
}

// The rows of a product with four-bit weights as two e4m3 numbers each (mxfp4.cuh): `parts` takes 2 M Kp bytes (Kp: K rounded up to
// a multiple of 128), `scales` what `layout` says, both 16-byte aligned.
int fb_mxfp4_split_rows(const MxRows& rows, int M, int K, void* parts, void* scales, const MxScaleLayout& layout, cudaStream_t stream) {
    const int Kp = (K + MX_COLS - 1) / MX_COLS * MX_COLS;
    const dim3 grid((unsigned)((M + SPLIT_ROWS - 1) / SPLIT_ROWS), (unsigned)((SPLIT_ROWS * (Kp / MX_BLOCK) + 255) / 256));
    fb_launch(layout.tile_group ? split_kernel<true> : split_kernel<false>, grid, dim3(256), 0, stream, rows, M, K, Kp, (uint8_t*)parts,
              (uint8_t*)scales, layout);
    return fb_check_launch("mxfp4_split_rows");
}
