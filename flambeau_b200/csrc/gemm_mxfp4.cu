// out[M,N] = X[M,K] * W[N,K]^T with X in bfloat16 and W in four bits (mxfp4.cuh) on the 5th-generation tensor cores.
//
// tcgen05.mma.kind::mxf8f6f4 multiplies numbers of up to 8 bits whose blocks of 32 along K carry power-of-two scales, and sums in
// float32.  A four-bit weight is such a number as it is.  A row's bfloat16 numbers become two e4m3 numbers each, the second what the
// first left, under one scale a block of 32 (mxfp4.cuh): numbers down to 2^-14 of the block's largest are held exactly, smaller ones to
// 2^-22 of it.  So the product is that of bfloat16 rows with the weights' numbers, summed in float32, but for rows with numbers so far
// above their neighbours: what those lose is what a float32 sum with the largest among its terms loses, and shows where the largest meets a
// weight of zero (one of 2^13 in every block: 8e-4 of such sums).  A third part would be half as many MMAs again.  An infinity or a NaN
// among a row's numbers makes all its sums NaN.
//
// Why this instruction, on one SM, for 128 features x 128 of K (a tile of 8,704 bytes, which HBM brings every 370 cycles): kind::f16
// takes 8 instructions of 70 cycles at least, whatever the number of tokens up to 128, and its weights have to be decoded to
// bfloat16 (19 instructions for eight: shifts, masks, multiplications); this kind takes 4 of 35 cycles up to 32 tokens (N = 64: both
// parts side by side), and decoding is moving bits (3 instructions for eight), since the scales go to the tensor core as they are.
//
// Layout.  A CTA owns 128 output features x a tile of tokens ("swap-AB": the weight is the 128-row operand, the tokens are N).  A stage
// is 128 of K (256 up to 32 tokens): one bulk copy brings a weight tile as it lies in memory, groups of four warps take the stages in
// turn and decode, a thread a feature, into tensor memory, where the MMA takes its A operand and both operands' scales from; the rows'
// parts, made once for all CTAs by a kernel of their own, come by TMA (K-major, 128-byte swizzle), their scales by tcgen05.cp.  Up to
// 64 tokens the two parts are N's two halves, which the epilogue adds; with more they are two instructions into one accumulator.
//
// Forms.  Few (up to 8 tokens, the CTA splits the rows itself) and narrow (up to 32): the tiles of all row tiles form one line that the
// CTAs cut into equal stretches.  Wide: token tiles of up to 64 or 128, the output through shared memory.  Shares of K go to slabs
// that the next kernel adds, or meet in scratch, where the CTA that arrives last (a counter a row tile, no waiting) adds them in
// order.  Grouped (routed experts): row tiles of one group each; a unit is a run of neighbouring ones.
//
// full[s]: a stage's rows (by bytes) and its decoded weights (by arrivals) are there; done[s]: its MMAs are.  Two accumulators, so that
// the epilogue of one unit overlaps the products of the next.  Every mbarrier wait is bounded as in gemm_tc.cu.
//
// What bounds it.  A few rows: a stage's way through waits, decoding, barriers and MMAs.  A tile takes 166 of a scheduler's issue
// slots in all, 40% of those of the SMs at work (profiled), where HBM has it under way for 370 cycles; before that a launch and the way
// from the first weights to the first MMA, 3 to 4 us (8 x 28,672 x 4,096: 13.9 us in a graph, 69% of HBM's rate).  Many rows: the MMAs,
// 512 cycles for 128 x 128 x 128 in two parts, at the clock that the power limit leaves (2,048 x 28,672 x 4,096: 355 us in bursts at
// 1.63 GHz, 413 at 1.35).
#include "group_units.cuh"
#include "mxfp4.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <limits.h>

namespace {

constexpr int A_COLS = MX_COLS / 4;               // tensor-memory columns of a stage's weights, then of their scales
constexpr int SFA_COLS = 4;
constexpr int MAX_W = 24, MAX_R = 8;              // most stages of packed weights / of rows and decoded weights
constexpr int LIST = 512;                         // units of the grouped form that are kept in shared memory
constexpr int CHUNK = 16;                         // tokens that a group of four epilogue warps takes at a time
constexpr int OUT_BYTES = 4096, OUT_BUFFERS = 3;  // a staged box of the output: 16 tokens, 8 of ungated float32
constexpr int FLAGS = 640;                        // bytes of barriers and flags
constexpr int CONTROL = FLAGS + 4 * LIST;         // and the list
constexpr int FEW_TOKENS = 8, NARROW_TOKENS = 32, WIDE_TOKENS = 128;      // most tokens of a tile of each form
constexpr int SPLITTERS = 8;                      // warps that make the parts of few rows
constexpr int SIDE_BY_SIDE = 64;                  // most tokens whose two parts are one operand
constexpr int ATOM = 512;                         // scales of 128 rows for a stage, as tcgen05.cp brings them to tensor memory
constexpr int TMEM = 512, SMEM = 227 * 1024;

// TOK: most tokens of a tile.  R stages of KT tiles of rows and decoded weights, GROUPS of four decoding warps: a stage of one tile is
// 1,500 cycles on its way from the first look at its weights to the end of its MMAs, of which a group works on it for half.  Where
// the MMAs are short, instructions are the bound, and two tiles a stage spare half of its waits and barriers.
// PAIR: a unit is two neighbouring feature tiles, which share the stages of rows; their accumulators are the two that are otherwise
// those of successive units, and sixteen warps store them.  It halves the reading of rows, and one round of pairs can replace two
// of single tiles (128 x 28,672 x 4,096: 30 us, 34 single; 64 rows 21.1 and 22.2); see plan_wide.
template <int TOK, bool PAIR> struct Form {
    static constexpr bool WIDE = TOK > NARROW_TOKENS;                    // (the narrow forms cut the line of tiles, and store directly)
    static constexpr bool FEW = TOK <= FEW_TOKENS;
    static constexpr int TILES = PAIR ? 2 : 1;
    static constexpr int KT = WIDE ? 1 : 2;                              // tiles along K of a stage
    static constexpr int R = TOK <= NARROW_TOKENS ? 4 : PAIR ? 3 : TOK <= SIDE_BY_SIDE ? 6 : 4;
    static constexpr int GROUPS = FEW ? 3 : TOK <= NARROW_TOKENS ? 4 : PAIR ? 2 : 3;
    static constexpr int EPI_GROUPS = FEW ? 1 : PAIR ? 4 : 2, EPI = 128 * EPI_GROUPS;   // groups of four warps, threads of the epilogue
    static constexpr int TURNS = GROUPS / TILES;                         // groups that take a feature tile's stages in turn
    static constexpr int EPI_WARP = 4 + 4 * GROUPS, SPLIT_WARP = EPI_WARP + EPI / 32, THREADS = 32 * (SPLIT_WARP + (FEW ? SPLITTERS : 0));
    static constexpr int ATOMS = TOK <= SIDE_BY_SIDE ? 1 : 2 * ((TOK + 127) / 128);
    static constexpr int ACC_COLS = TOK <= SIDE_BY_SIDE ? 2 * TOK : TOK;
    static constexpr int W_COLS = A_COLS + SFA_COLS;
    static constexpr int TILE_COLS = (TILES * W_COLS + 4 * ATOMS + 7) / 8 * 8;  // [weights | their scales] a feature tile, rows' scales
    static constexpr int TILE_BYTES = (TOK * 256 + ATOMS * ATOM + 1023) / 1024 * 1024; // the rows' parts, their scales
    static constexpr int RING_COLS = KT * TILE_COLS, STAGE_BYTES = KT * TILE_BYTES;
    static constexpr int OUT = WIDE ? EPI_GROUPS * OUT_BUFFERS * OUT_BYTES : 0;
    static constexpr int RING = SMEM - 1024 - CONTROL - OUT;             // for the rings of stages
    static constexpr int FIT = (RING - R * STAGE_BYTES) / MX_TILE_BYTES;
    static constexpr int PRODUCERS = WIDE ? 1 : 2;                       // threads that ask for weights, each for places of its own
    static constexpr int WS = (FIT < MAX_W ? FIT : MAX_W) / PRODUCERS * PRODUCERS;
    // Threads that ask for rows, each for places of its own.  (Groups of 64 rows at most, 180 tokens on 6 of 64 experts, 3,584 x 4,096: one
    // 114 us, two 104.)
    static constexpr int ROW_PRODUCERS = WIDE && TOK <= SIDE_BY_SIDE && !PAIR ? 2 : 1;
    static_assert(R % ROW_PRODUCERS == 0 && PRODUCERS + ROW_PRODUCERS <= 3, "places of their own, warps 0, 2 and 3");
    static constexpr int ARRIVALS = 4 * TILES + (FEW ? KT : 1);          // at full[s]: of the decoding warps, and of who brings the rows
    static_assert(2 * ACC_COLS + R * RING_COLS <= TMEM, "tensor memory");
    static_assert(TURNS <= R && WS % KT == 0 && WS >= KT * (GROUPS + TILES * R) && (!FEW || SPLITTERS / KT <= R),
                  "a wait names a phase by its parity: see the decoding warps");
    static_assert(PRODUCERS == 1 || KT == 2, "each has places of its own");
};

// Atoms of scales that the rows of a tile have: of both parts side by side, or of either part.
__host__ __device__ constexpr int atoms_of(int tokens) { return tokens <= SIDE_BY_SIDE ? 1 : 2 * ((tokens + 127) / 128); }

struct MxArgs {
    const uint8_t* W; long w_group; int groups;           // tiles, bytes of one group's
    MxRows rows;                                          // what X's parts, which come by map_x, are made from
    const uint8_t* x_scales; int scale_bytes;             // their scales, bytes of a tile's
    void* out; long ldo, slab_stride;
    int o_bf16, accumulate, boxed, slabs;                 // boxed: tokens of a box, 0: stored directly
    float* partials; int* counters; int max_segments;
    int M, N, K, kb, bn, tiles_m, tiles_n, units_n, splits;      // units_n: feature tiles, or pairs of them
    uint32_t items;                                       // narrow, not grouped: tiles_n * kb; wide, not grouped: units
    const int* tile_group; int tile, n_tiles;
    FbGate gate; int plain_act;
    int* status;
};

// What a CTA works on at a time: row tile nt (and the one behind it) of a group's matrix, tiles kb0 .. kb0 + n_kb along K, over n_tok
// rows from m0 on.
struct Unit { int m0, n_tok, nt, group, kb0, n_kb, share, shares, id; };

__device__ __forceinline__ void mma_mx(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], [%1], %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
}
// e2m1 x e4m3 -> f32 under E8M0 scales, M = 128; the k-th block of 32 of a stage takes byte k of the scales' words.
__device__ __forceinline__ uint32_t mx_idesc(int n) { return (5u << 7) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (8u << 24); }
__device__ __forceinline__ constexpr uint32_t mx_block(int k) { return ((uint32_t)k << 4) | ((uint32_t)k << 29); }
// 512 bytes of scales, [lane i][j] words of row 32 j + i, into four columns, the same in every quarter of the lanes; in order with the
// MMAs of the same thread.
__device__ __forceinline__ uint64_t scales_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)8 << 16 | (uint64_t)8 << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint4& v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// mbar_wait whose tries may sleep for long: twenty warps that ask again and again take issue slots from those that work.
__device__ __forceinline__ bool wait_long(uint32_t bar, uint32_t parity, int* status) {
    constexpr uint32_t HINT_NS = 1000000;
    unsigned long long t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity), "r"(HINT_NS) : "memory");
        if (ok) return true;
        if (t0 == 0) t0 = global_ns();
        else if (global_ns() - t0 > FB_WAIT_LIMIT_NS) {
            atomicOr(status, FB_STATUS_WAIT_TIMEOUT);
            return false;
        }
    }
}

__device__ __forceinline__ void store_box(const void* map, uint32_t src, int x, int y, int z, bool add) {
    if (add)
        asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                     ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                     ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// g sigmoid(g) u with h = e^(-|g| / 2): g u / (1 + h h), below zero with h h above the line, one h a factor, so that nothing
// overflows and nothing vanishes before the result does (g < -174: zero).  The exponential and the reciprocal are the approximate ones
// (2^-22 and 2^-23 of themselves); what the exponential's argument -|g| log2(e) / 2 loses by rounding is computed with the constant in
// two parts, as Cody and Waite reduce arguments, and comes back as the first term of e^x.  17 x 2^-24 of the result at most, whatever g.
// expf and a division made the epilogue of 160 tokens longer than the products of K = 4,096.
__device__ __forceinline__ float silu_times(float g, float u) {
    constexpr double HALF_LOG2E = 0.72134752044448170368, LN2 = 0.69314718055994530942;
    constexpr float HI = (float)HALF_LOG2E, LO = (float)(HALF_LOG2E - (double)HI);
    const float m = fminf(fabsf(g), 512.0f), t = -HI * m;                  // (an infinity would make a NaN of what t loses)
    const float rest = fmaf(-LO, m, fmaf(-HI, m, -t)) * (float)LN2;
    float h, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(t));
    h = fmaf(h, rest, h);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.0f)));
    const float p = g < 0.0f ? h : 1.0f;
    return g * p * u * (p * r);
}

// The epilogue's code is walked a few times a tile only, so that its instructions come from far: every 128 bytes of them cost
// about as much as ten of the instructions.  What is seldom wanted is kept out of its straight way.
__device__ __noinline__ void let_end() { fb_settle(); }
__device__ __noinline__ float gate_slowly(const FbGate& gate, float g, float u) { return fb_gate_times(gate, g, u); }
__device__ __noinline__ float act_slowly(int act, float z) { return fb_plain_act(act, z); }
template <int N> __device__ __forceinline__ void gate_all(const FbGate& gate, float (&g)[N], const float (&u)[N]) {
    if (__builtin_expect(gate.act == FB_ACT_SILU, 1)) {
#pragma unroll
        for (int q = 0; q < N; ++q) g[q] = silu_times(g[q], u[q]);
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) g[q] = gate_slowly(gate, g[q], u[q]);
    }
}
__device__ __forceinline__ void st_shared(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void st_shared(uint32_t addr, __nv_bfloat16 v) {
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(__bfloat16_as_ushort(v)) : "memory");
}

// The shares of a row tile, `step` float4 apart, added in order; a thread has four neighbouring features of a token, n .. n + 3 of row
// m0 + e / 32.  (What it needs comes by value: read through a reference behind every store, it made this ten times as long.)
template <int EPI>
__device__ __noinline__ void join_shares(const float4* __restrict__ base, size_t step, int shares, int all, int tid, void* out,
                                         long ldo, int m0, int n0, int N, int act, float limit, float slope, int plain_act, int o_bf16,
                                         int accumulate) {
    constexpr int U = 4;                         // sums of a thread at a time, two shares of each on their way
    const FbGate gate = {act, limit, slope};
    for (int e0 = tid; e0 < all; e0 += U * EPI) {
        float4 sum[U];
#pragma unroll
        for (int q = 0; q < U; ++q) sum[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4* p = base + e0;
        for (int s = 0; s < shares; s += 2, p += 2 * step) {
            float4 t[2][U];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < U; ++q)
                    t[h][q] = s + h < shares && e0 + q * EPI < all ? __ldcg(p + h * step + q * EPI) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    sum[q].x += t[h][q].x; sum[q].y += t[h][q].y; sum[q].z += t[h][q].z; sum[q].w += t[h][q].w;
                }
        }
#pragma unroll
        for (int q = 0; q < U; ++q) {
            const int e = e0 + q * EPI;
            if (e >= all) break;
            const int m = m0 + e / (MX_ROWS / 4), n = n0 + 4 * (e % (MX_ROWS / 4));
            float v[4] = {sum[q].x, sum[q].y, sum[q].z, sum[q].w};
            int count = 4, columns = N, col = n;
            if (act) {                           // features alternate gate, up
                float g[2] = {v[0], v[2]};
                const float u[2] = {v[1], v[3]};
                gate_all(gate, g, u);
                v[0] = g[0];
                v[1] = g[1];
                count = 2; columns = N / 2; col = n / 2;
            } else if (plain_act) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = act_slowly(plain_act, v[i]);
            }
            const size_t at = (size_t)m * ldo + col;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= count || col + i >= columns) break;
                if (o_bf16) {
                    reinterpret_cast<__nv_bfloat16*>(out)[at + i] = __float2bfloat16_rn(v[i]);
                } else {
                    float* o = reinterpret_cast<float*>(out) + at + i;
                    *o = accumulate ? *o + v[i] : v[i];
                }
            }
        }
    }
}

template <int TOK, bool GROUPED, bool PAIR>
__global__ void __launch_bounds__(Form<TOK, PAIR>::THREADS, 1)
gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_o,
                  const __grid_constant__ MxArgs a) {
    using F = Form<TOK, PAIR>;
    constexpr bool WIDE = F::WIDE;
    constexpr int WS = F::WS, R = F::R, G = F::GROUPS, KT = F::KT, EPI = F::EPI, EPI_WARP = F::EPI_WARP, TILES = F::TILES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* w_base = smem + R * F::STAGE_BYTES;                         // [stages of rows | weight stages | output boxes | control]
    uint8_t* out_stage = smem + F::RING;
    uint64_t* bars = (uint64_t*)(out_stage + F::OUT);
    uint64_t *w_full = bars, *w_empty = w_full + MAX_W, *full = w_empty + MAX_W, *done = full + MAX_R,
             *acc_full = done + MAX_R, *acc_empty = acc_full + 2;
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
    int* flag = (int*)(tmem_slot + 1);           // what the epilogue decided together
    int* bail = flag + 1;                        // a bounded wait ran out somewhere in this CTA
    int* unit_count = bail + 1;
    int* group_failed = unit_count + 1;          // [group][round]
    uint32_t* list = (uint32_t*)((uint8_t*)bars + FLAGS);
    static_assert(8 * (2 * MAX_W + 2 * MAX_R + 4) + 4 * (4 + 2 * G) <= FLAGS, "barriers and flags");
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_long(smem_u32(bar), parity, a.status); };
    auto bailed = [&]() { return *(volatile int*)bail != 0; };
    const int most = GROUPED ? a.bn / a.tile : 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_W; ++s) { mbar_init(smem_u32(&w_full[s]), 1); mbar_init(smem_u32(&w_empty[s]), 4); }
        for (int s = 0; s < R; ++s) {
            mbar_init(smem_u32(&full[s]), F::ARRIVALS);
            mbar_init(smem_u32(&done[s]), 1);
        }
        for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&acc_full[s]), 1); mbar_init(smem_u32(&acc_empty[s]), EPI); }
        *bail = 0;
        for (int g = 0; g < 2 * G; ++g) group_failed[g] = 0;
        mbar_fence_init();
    }
    if (warp == 3) tmem_alloc(tmem_slot, TMEM);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    fb_pdl_launch_dependents();                  // (behind the allocation: see umma.cuh)
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const uint32_t ring = tmem + 2 * F::ACC_COLS;

    // The CTA's part of the work: items first .. last of the line.  Narrow, not grouped: an item is a tile along K of a row tile; else a
    // unit, and the CTAs take turns.
    constexpr bool LINE = !WIDE && !GROUPED;
    // (32 bits hold items x CTAs: a matrix of 2^38 weights fills the memory.  Twenty warps divide for every unit.)
    uint32_t first = blockIdx.x, last = a.items;
    if constexpr (GROUPED) {
        if (warp == EPI_WARP) {
            // (Which weights a tile wants is the work of kernels that have ended: the one that splits the rows lets this one in behind
            // its own wait.  8 tokens on 6 of 64 experts, 3,584 x 4,096, with a wait here: 60 us, like this 57.)
            const int found = group_units<LIST>(a.tile_group, a.n_tiles, most, list);
            if (lane == 0) *unit_count = found;
        }
        __syncthreads();
        last = (uint32_t)*unit_count * a.units_n;
    } else if constexpr (LINE) {
        first = blockIdx.x * a.items / gridDim.x;
        last = (blockIdx.x + 1) * a.items / gridDim.x;
    }
    GroupWalk walk = {0, 0u};
    auto unit_at = [&](uint32_t item) {              // (asked for ascending items only)
        Unit w;
        if constexpr (GROUPED) {                 // feature tiles vary fastest: the CTAs that run together share few units' rows
            const int i = (int)(item / (uint32_t)a.units_n);
            const uint32_t entry = group_unit<LIST>(a.tile_group, a.n_tiles, most, list, i, walk);
            const int t = (int)(entry & 0xffffffu);
            w.m0 = t * a.tile;
            w.n_tok = (int)(entry >> 24) * a.tile;
            w.group = min(a.tile_group[t], a.groups - 1);            // (none lie beyond the last group's: such a tile's rows are NaN)
            w.nt = TILES * ((int)item - i * a.units_n);
            w.kb0 = 0; w.n_kb = a.kb; w.share = 0; w.shares = 1; w.id = 0;
        } else if constexpr (WIDE) {             // token tiles vary fastest: the CTAs that run together share weight tiles
            const uint32_t units = (uint32_t)a.tiles_m * a.units_n;
            w.share = (int)(item / units);
            w.shares = a.splits;
            const uint32_t u = item - w.share * units, mt = u % (uint32_t)a.tiles_m;
            w.m0 = (int)mt * a.bn;
            w.nt = TILES * (int)(u / (uint32_t)a.tiles_m);
            w.id = (int)mt * a.tiles_n + w.nt;
            w.n_tok = a.bn;
            w.group = 0;
            w.kb0 = (int)((uint32_t)(w.share * a.kb) / (uint32_t)a.splits);
            w.n_kb = (int)((uint32_t)((w.share + 1) * a.kb) / (uint32_t)a.splits) - w.kb0;
        } else {
            w.nt = (int)(item / (uint32_t)a.kb);
            w.kb0 = (int)item - w.nt * a.kb;
            w.n_kb = min((int)(last - item), a.kb - w.kb0);
            w.m0 = 0; w.n_tok = a.bn; w.group = 0; w.id = w.nt;
            const uint32_t from = (uint32_t)(w.nt * a.kb), begin = ((from + 1) * gridDim.x - 1) / a.items;
            w.share = (int)(blockIdx.x - begin);
            w.shares = (int)(((from + a.kb) * gridDim.x - 1) / a.items - begin) + 1;
        }
        return w;
    };
    // CTAs of neighbouring row tiles of a group want the same rows: each begins at another place along K, or they would all ask for the
    // same few lines of L2 at once (8 tokens on 6 of 64 experts, 3,584 x 4,096: 68 us, like this 64).
    auto first_tile = [&](const Unit& w) { return GROUPED ? w.nt % w.n_kb : 0; };
    auto stages_of = [&](const Unit& w) { return (w.n_kb + KT - 1) / KT; };
    auto after = [&](uint32_t item, const Unit& w) { return LINE ? item + w.n_kb : item + gridDim.x; };

    if (warp == 0 || (F::PRODUCERS == 2 && warp == 3)) {
        // ---------------- weights: no other kernel writes them, so they are requested at once ----------------
        if (elect_one()) {
            const int turn = warp == 0 ? 0 : 1;
            int s = turn, i = turn;                  // i: the thread's first tile of the unit
            uint32_t phase = 1;
            for (uint32_t u = first; u < last && !bailed();) {
                const Unit w = unit_at(u);
                const uint8_t* src = a.W + (size_t)w.group * a.w_group + ((size_t)w.nt * a.kb + w.kb0) * MX_TILE_BYTES;
                // (a pair's second tile that is none of the matrix is its first one again: nobody stores what comes of it)
                const size_t next = w.nt + 1 < a.tiles_n ? (size_t)a.kb * MX_TILE_BYTES : 0;
                const int begin = first_tile(w), tiles = TILES * stages_of(w) * KT;
                bool ok = true;
                for (; i < tiles; i += F::PRODUCERS) {
                    ok = wait(&w_empty[s], phase);
                    if (!ok) break;
                    // (a stage's second tile that is none of the unit is the first one again: nothing is multiplied with it)
                    const int k = begin + min(i / TILES, w.n_kb - 1);
                    mbar_expect_tx(smem_u32(&w_full[s]), MX_TILE_BYTES);
                    const uint8_t* from = src + (size_t)(k < w.n_kb ? k : k - w.n_kb) * MX_TILE_BYTES + (i % TILES) * next;
                    bulk_copy_g2s(smem_u32(w_base + (size_t)s * MX_TILE_BYTES), from, MX_TILE_BYTES, smem_u32(&w_full[s]));
                    if ((s += F::PRODUCERS) >= WS) { s -= WS; phase ^= 1u; }
                }
                if (!ok) *bail = 1;
                i -= tiles;
                u = after(u, w);
            }
        }
        __syncwarp();
    } else if (warp == 2 || (F::ROW_PRODUCERS == 2 && warp == 3)) {
        // ---------------- the rows' parts and their scales (of few rows: see the last warps) ----------------
        if (!F::FEW && elect_one()) {
            fb_pdl_wait();
            const int turn = warp == 2 ? 0 : 1;
            int s = turn, i = turn;                  // i: the thread's first stage of the unit
            uint32_t phase = 1;
            for (uint32_t u = first; u < last && !bailed();) {
                const Unit w = unit_at(u);
                const int boxes = GROUPED ? w.n_tok / a.tile : 1, box = GROUPED ? a.tile : a.bn, stages = stages_of(w), begin = first_tile(w);
                const uint32_t scale_bytes = (uint32_t)(atoms_of(w.n_tok) * ATOM);
                const size_t step = (size_t)(GROUPED ? a.n_tiles : a.tiles_m) * a.scale_bytes;       // scales of a tile along K
                const uint8_t* scales = a.x_scales + (size_t)(w.m0 / (GROUPED ? a.tile : a.bn)) * a.scale_bytes + w.kb0 * step;
                int k = begin + KT * i;
                if (k >= w.n_kb) k -= w.n_kb;
                for (; i < stages; i += F::ROW_PRODUCERS) {
                    if (!wait(&done[s], phase)) { *bail = 1; break; }
                    const uint32_t bar = smem_u32(&full[s]);
                    mbar_expect_tx(bar, min(KT, w.n_kb - KT * i) * ((uint32_t)w.n_tok * 2 * 128 + scale_bytes));
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
                        if (t && KT * i + t >= w.n_kb) break;
                        const uint32_t dst = smem_u32(smem) + (uint32_t)(s * F::STAGE_BYTES + t * F::TILE_BYTES);
                        for (int b = 0; b < boxes; ++b) {
#pragma unroll
                            for (int p = 0; p < 2; ++p)      // (rows beyond M are the other part's, or zeros: nobody stores them)
                                tma_load_2d(dst + (uint32_t)(p * w.n_tok + b * box) * 128, &map_x, bar, (w.kb0 + k) * 64, p * a.M + w.m0 + b * box);
                        }
                        bulk_copy_g2s(dst + TOK * 256, scales + k * step, scale_bytes, bar);
                        if (++k == w.n_kb) k = 0;
                    }
                    if (F::ROW_PRODUCERS == 2 && ++k == w.n_kb) k = 0;                       // (the other thread's)
                    if ((s += F::ROW_PRODUCERS) >= R) { s -= R; phase ^= 1u; }
                }
                i -= stages;
                u = after(u, w);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA ----------------
        // (What an instruction's operands are made of is brought to uniform registers first.  Where a stage's place in the ring is counted
        // out, that takes 300 cycles a stage of four instructions; with three or four places as constants it is done once, and a
        // stage takes 140 with its wait and commit, 57 to 260 of them MMAs.)
        if (elect_one()) {
            int s = 0, j = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t x_base = smem_u32(smem), full_base = smem_u32(full), done_base = smem_u32(done);
            const uint64_t desc = umma_desc(x_base), desc_scales = scales_desc(x_base + TOK * 256);
            for (uint32_t u = first; u < last && ok && !bailed(); ++j) {
                const Unit w = unit_at(u);
                const bool both = w.n_tok <= SIDE_BY_SIDE;               // both parts in one operand
                const int b = PAIR ? 0 : j & 1;
                const uint32_t idesc = mx_idesc(both ? 2 * w.n_tok : w.n_tok), second = (uint32_t)w.n_tok * 8;      // (128 bytes, in sixteens)
                const uint32_t sfb_second = (uint32_t)(w.n_tok + 127) / 128 * 4;
                // (the epilogue has drained the accumulator, of two units ago or of the pair before)
                ok = wait(&acc_empty[b], ((uint32_t)(PAIR ? j : j >> 1) & 1u) ^ 1u);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t d = tmem + (uint32_t)(b * F::ACC_COLS);
                auto products = [&](int at, int h, bool fresh) {         // of the tile along K in place `at` of the ring with the h-th feature tile
                    const uint32_t A0 = ring + (uint32_t)(at * F::TILE_COLS), sfb = A0 + TILES * F::W_COLS;
                    const uint64_t x = desc + (uint64_t)(at * (F::TILE_BYTES / 16));
                    const uint32_t A = A0 + h * F::W_COLS, to = d + h * F::ACC_COLS;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_mx(to, A + 8 * k, x + 2 * k, idesc + mx_block(k), A + A_COLS, sfb, fresh && k == 0 ? 0u : 1u);
                    if (TOK > SIDE_BY_SIDE && !both) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_mx(to, A + 8 * k, x + second + 2 * k, idesc + mx_block(k), A + A_COLS, sfb + sfb_second, 1u);
                    }
                };
                auto begin = [&](int at, bool whole) {                   // the stage in place `at`, of KT tiles or of one
                    if (!wait_long(full_base + 8 * at, phase, a.status)) return false;
                    tmem_fence_after();
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        const uint32_t sfb = ring + (uint32_t)((KT * at + k) * F::TILE_COLS) + TILES * F::W_COLS;
#pragma unroll
                        for (int t = 0; t < F::ATOMS; ++t)
                            if ((k == 0 || whole) && (t == 0 || !both))
                                copy_scales(sfb + 4 * t, desc_scales + (uint64_t)(((KT * at + k) * F::TILE_BYTES + t * ATOM) / 16));
                    }
                    return true;
                };
                auto stage = [&](int at, bool fresh, bool whole) {
                    if (!begin(at, whole)) return false;
#pragma unroll
                    for (int k = 0; k < KT; ++k)
                        if (k == 0 || whole) {
#pragma unroll
                            for (int h = 0; h < TILES; ++h) products(KT * at + k, h, fresh && k == 0);
                        }
                    umma_commit(done_base + 8 * at);
                    return true;
                };
                int i = 0;
                const int stages = stages_of(w), whole = w.n_kb / KT;
                if constexpr (PAIR) {
                    // the first tile's products of the stages that the ring holds run ahead, while the epilogue still has the other
                    // accumulator
                    const int s0 = s, ahead = w.n_kb < R ? w.n_kb : R;
                    const uint32_t phase0 = phase;
                    for (; i < ahead && ok; ++i) {
                        ok = begin(s, true);
                        if (ok) products(s, 0, i == 0);
                        if (++s == R) { s = 0; phase ^= 1u; }
                    }
                    if (!ok || !(ok = wait(&acc_empty[1], ((uint32_t)j & 1u) ^ 1u))) break;
                    tmem_fence_after();
                    s = s0;
                    phase = phase0;
                    for (int t = 0; t < ahead; ++t) {
                        products(s, 1, t == 0);
                        umma_commit(done_base + 8 * s);
                        if (++s == R) { s = 0; phase ^= 1u; }
                    }
                }
                while (ok && i < stages) {
                    constexpr int B = R % 4 == 0 ? 4 : 3;
                    static_assert(R % B == 0, "blocks of three or four places");
                    const int before = i;
#pragma unroll
                    for (int p = 0; p < R; p += B) {
                        if (!ok || s != p || i + B > whole) continue;
#pragma unroll
                        for (int q = 0; q < B; ++q) ok = ok && stage(p + q, q == 0 && i == 0, true);
                        s = p + B;
                        i += B;
                    }
                    if (i == before) {
                        ok = stage(s, i == 0, i < whole);
                        ++s; ++i;
                    }
                    if (s == R) { s = 0; phase ^= 1u; }
                }
                if (PAIR && ok) umma_commit(smem_u32(&acc_full[0]));
                if (ok) umma_commit(smem_u32(&acc_full[PAIR ? 1 : b]));
                u = after(u, w);
            }
            if (!ok) *bail = 1;
        }
        __syncwarp();
    } else if (warp >= 4 && warp < EPI_WARP) {
        // ---------------- decode: a thread a feature; weight tiles it = group, group + G, ... (of a pair, always the same one) ----------------
        // (A wait names a phase by its parity alone, and a group does not come to every slot in every round of a ring.  It comes every
        // TURNS stages and has seen the MMAs of the stage TURNS + R ago done, so with TURNS <= R no slot of that ring is two rounds
        // behind, and with WS >= KT (GROUPS + TILES R) none of the weights'.)
        const int quarter = warp & 3, row = quarter * 32 + lane, group = (warp - 4) >> 2;
        const uint32_t lanes = ring + ((uint32_t)(quarter * 32) << 16);
        constexpr int TURNS = F::TURNS;
        const int turn = group / TILES, tile = group % TILES;
        int ws = KT * group, r = turn;
        uint32_t w_phase = 0, r_phase = 0, it = 0;       // it: stages ahead of the unit, modulo TURNS
        int round = 0;
        bool ok = true;
        for (uint32_t u = first; u < last && ok;) {                 // (not `bailed`, which the four warps might see at different times)
            const Unit w = unit_at(u);
            const int stages = stages_of(w);
            int i = turn - (int)it;                                      // the group's first stage of the unit
            if (i < 0) i += TURNS;
            for (; i < stages; i += TURNS) {
                // one of the four warps asks: twenty that ask at every barrier again and again take half of the issue slots
                if (quarter == 0) {
                    ok = wait(&done[r], r_phase ^ 1u);                   // the MMAs that read this place are done
#pragma unroll
                    for (int t = 0; t < KT; ++t)
                        if (ok) ok = wait(&w_full[ws + t], w_phase);
                    if (!ok) group_failed[2 * group + round] = 1;
                }
                asm volatile("bar.sync %0, 128;" ::"r"(6 + group) : "memory");
                ok = *(volatile int*)&group_failed[2 * group + round] == 0;      // (two flags in turn: the next round's is not seen yet)
                round ^= 1;
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tmem_fence_after();
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const uint8_t* src = w_base + (size_t)(ws + t) * MX_TILE_BYTES;
                    const uint4 scales = *reinterpret_cast<const uint4*>(src + MX_CODE_BYTES + lane * 16);
                    uint4 c[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) c[q] = *reinterpret_cast<const uint4*>(src + (q * MX_ROWS + row) * 16);
                    const uint32_t dst = lanes + (uint32_t)(r * F::RING_COLS + t * F::TILE_COLS + tile * F::W_COLS);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t v[16];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const uint32_t in[4] = {c[2 * h + q].x, c[2 * h + q].y, c[2 * h + q].z, c[2 * h + q].w};
#pragma unroll
                            for (int p = 0; p < 4; ++p) mx_decode(in[p], v[8 * q + 2 * p], v[8 * q + 2 * p + 1]);
                        }
                        tmem_st16(dst + 16 * h, v);
                    }
                    tmem_st4(dst + A_COLS, scales);
                    // (behind the stores, which need every number of the row: see gemm_f32_tc.cu)
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&w_empty[ws + t]));
                }
                tmem_wait_st();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full[r]));
                if ((ws += KT * G) >= WS) { ws -= WS; w_phase ^= 1u; }
                if ((r += TURNS) >= R) { r -= R; r_phase ^= 1u; }
            }
            it = (it + (uint32_t)stages) % TURNS;
            u = after(u, w);
        }
        if (!ok) *bail = 1;
    } else if (warp >= EPI_WARP && warp < F::SPLIT_WARP) {
        // ---------------- epilogue: lanes are features, the groups of four warps take 16 tokens in turn ----------------
        fb_pdl_wait();
        const int quarter = warp & 3, half = (warp - EPI_WARP) >> 2, row = quarter * 32 + lane, tid = threadIdx.x - 32 * EPI_WARP;
        const bool leader = quarter == 0 && lane == 0;
        constexpr int STEP = CHUNK * F::EPI_GROUPS;
        const uint32_t box_first = smem_u32(out_stage) + half * (OUT_BUFFERS * OUT_BYTES);       // the group's boxes
        const uint32_t box_last = box_first + (OUT_BUFFERS - 1) * OUT_BYTES;
        uint32_t box_at = box_first;
        int j = 0;
        for (uint32_t u = first; u < last; ++j) {
            Unit w = unit_at(u);
            const uint32_t following = after(u, w);
            bool stop = false;
#pragma unroll 1
            for (int h = 0; h < TILES; ++h, ++w.nt, ++w.id) {
            const bool both = w.n_tok <= SIDE_BY_SIDE, join = !GROUPED && w.shares > 1 && a.slabs == 0;
            const int b = PAIR ? h : j & 1, n0 = w.nt * MX_ROWS, n = n0 + row;
            const int rows = min(w.n_tok, a.M - w.m0);                   // (grouped: whole tiles)
            if (warp == EPI_WARP && (bailed() || !wait(&acc_full[b], (uint32_t)(PAIR ? j : j >> 1) & 1u))) *bail = 1;
            asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
            if (tid == 0) *flag = bailed() ? 2 : 0;                      // one thread decides for all: they meet at barriers below
            asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
            stop = *flag == 2;
            if (stop) break;
            tmem_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * F::ACC_COLS);
            auto sums = [&](int c, float (&v)[16]) {
                tmem_ld16(acc + (uint32_t)c, v);
                if (both) {
                    float second[16];
                    tmem_ld16(acc + (uint32_t)(w.n_tok + c), second);
#pragma unroll
                    for (int q = 0; q < 16; ++q) v[q] += second[q];
                }
            };
            if (PAIR && w.nt >= a.tiles_n) {             // (a pair's second tile that is none of the matrix)
            } else if (join) {
                float* mine = a.partials + ((size_t)w.id * a.max_segments + w.share) * (size_t)(a.bn * MX_ROWS) + row;
                for (int c = half * CHUNK; c < rows; c += STEP) {
                    float v[16];
                    sums(c, v);
#pragma unroll
                    for (int q = 0; q < 16; ++q)
                        if (c + q < rows) mine[(size_t)(c + q) * MX_ROWS] = v[q];
                }
                __threadfence();
                asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
                if (tid == 0) {
                    const bool is_last = atomicAdd(&a.counters[w.id], 1) == w.shares - 1;
                    if (is_last) a.counters[w.id] = 0;                   // ready for the next launch
                    *flag = is_last;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
                if (*flag == 1) {
                    __threadfence();
                    join_shares<EPI>(reinterpret_cast<const float4*>(a.partials) + (size_t)w.id * a.max_segments * (size_t)(a.bn * (MX_ROWS / 4)),
                                     (size_t)a.bn * (MX_ROWS / 4), w.shares, rows * (MX_ROWS / 4), tid, a.out, a.ldo, w.m0, n0, a.N,
                                     a.gate.act, a.gate.limit, a.gate.slope, a.plain_act, a.o_bf16, a.accumulate);
                }
            } else {
                const int slab = a.slabs ? w.share : 0;
#pragma unroll 1
                for (int c = half * CHUNK; c < rows; c += STEP) {
                    float v[16];
                    sums(c, v);
                    if (__builtin_expect(a.plain_act != 0, 0)) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q] = act_slowly(a.plain_act, v[q]);
                    }
                    if (WIDE && a.boxed) {
                        // The values go to shared memory as [token][feature], and one thread sends the box on its way (what lies beyond
                        // the output's edge is not written).  Of three buffers the one that is written was read by the time of the
                        // barrier before: its store is the third last, and the thread that sends waits for all but the last.
                        const int x = a.gate.act ? n0 / 2 : n0;
                        auto send = [&](int token) {
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            if (leader) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                            asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
                            if (leader) store_box(&map_o, box_at, x, w.m0 + token, slab, a.accumulate != 0);
                            box_at = box_at == box_last ? box_first : box_at + OUT_BYTES;
                        };
                        if (a.gate.act) {
                            // features alternate gate, up: the even lane takes the first eight tokens of the pair, the odd one the others
                            float r[8], up[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[q] : v[8 + q], 1);
                                r[q] = lane & 1 ? other : v[q];
                                up[q] = lane & 1 ? v[8 + q] : other;
                            }
                            gate_all(a.gate, r, up);
                            const int at = (lane & 1) * 8 * (MX_ROWS / 2) + (row >> 1);
                            if (a.o_bf16) {
#pragma unroll
                                for (int q = 0; q < 8; ++q) st_shared(box_at + 2 * (at + q * (MX_ROWS / 2)), __float2bfloat16_rn(r[q]));
                            } else {
#pragma unroll
                                for (int q = 0; q < 8; ++q) st_shared(box_at + 4 * (at + q * (MX_ROWS / 2)), r[q]);
                            }
                            send(c);
                        } else if (a.o_bf16) {
#pragma unroll
                            for (int q = 0; q < 16; ++q) st_shared(box_at + 2 * (q * MX_ROWS + row), __float2bfloat16_rn(v[q]));
                            send(c);
                        } else {
#pragma unroll
                            for (int p = 0; p < 2; ++p) {
#pragma unroll
                                for (int q = 0; q < 8; ++q) st_shared(box_at + 4 * (q * MX_ROWS + row), v[8 * p + q]);
                                send(c + 8 * p);
                            }
                        }
                        continue;
                    }
                    // gated: features alternate gate, up; the even lane has act(gate) * up of column n / 2
                    bool writes = n < a.N;
                    int col = n;
                    if (a.gate.act) {
                        float up[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q) up[q] = __shfl_xor_sync(0xffffffffu, v[q], 1);
                        gate_all(a.gate, v, up);
                        writes = !(lane & 1) && n + 1 < a.N;
                        col = n >> 1;
                    }
                    if (writes) {
                        const size_t begin = (size_t)slab * a.slab_stride + (size_t)(w.m0 + c) * a.ldo + col;
                        if (a.o_bf16) {
                            __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(a.out) + begin;
#pragma unroll
                            for (int q = 0; q < 16; ++q)
                                if (c + q < rows) p[(size_t)q * a.ldo] = __float2bfloat16_rn(v[q]);
                        } else {
                            float* p = reinterpret_cast<float*>(a.out) + begin;
#pragma unroll
                            for (int q = 0; q < 16; ++q)
                                if (c + q < rows) p[(size_t)q * a.ldo] = a.accumulate ? p[(size_t)q * a.ldo] + v[q] : v[q];
                            if (!WIDE && a.slabs && w.share == w.shares - 1)         // shares that this row tile does not have
                                for (int s = w.shares; s < a.slabs; ++s) {
                                    p += a.slab_stride;
                                    for (int q = 0; q < 16 && c + q < rows; ++q) p[(size_t)q * a.ldo] = 0.0f;
                                }
                        }
                    }
                }
            }
            tmem_fence_before();
            mbar_arrive(smem_u32(&acc_empty[b]));
            }
            if (stop) {                          // (else the sums of every unit have come, and with them all copies)
                let_end();
                break;
            }
            u = following;
        }
        if (WIDE && leader) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");        // the boxes it sent are in memory
    } else if (F::FEW && warp >= F::SPLIT_WARP) {
        // ---------------- few rows' parts: tiles it = turn, turn + SPLITTERS, ..., a lane a block of 32 of row lane / 4 ----------------
        fb_pdl_wait();
        const int turn = warp - F::SPLIT_WARP, block = lane & 3, r = lane >> 2;
        const __nv_bfloat16* row = r < a.M ? a.rows.x + (size_t)r * a.rows.ld : nullptr;
        int s = turn / KT;
        uint32_t phase = 1, it = 0;              // it: tiles ahead of the unit, modulo SPLITTERS
        bool ok = true;
        for (uint32_t u = first; u < last && ok;) {
            const Unit w = unit_at(u);
            const int tiles = stages_of(w) * KT;
            uint4 raw[4];
            auto load = [&](int i) {                                     // what the lane splits of the unit's i-th tile
                const int k = (w.kb0 + i) * MX_COLS + block * MX_BLOCK;
#pragma unroll
                for (int q = 0; q < 4; ++q) raw[q] = row ? mx_load8(row, k + 8 * q, a.K, a.rows.aligned != 0) : make_uint4(0, 0, 0, 0);
            };
            int i = turn - (int)it;                                      // the warp's first tile of the unit
            if (i < 0) i += SPLITTERS;
            if (i < w.n_kb) load(i);
            for (; i < tiles; i += SPLITTERS) {                          // (of a stage's second tile that is none of the unit nothing is read)
                uint2 one[4], two[4];
                const uint32_t word = mx_split_block(raw, one, two);
                if (i + SPLITTERS < w.n_kb) load(i + SPLITTERS);
                if (lane == 0) ok = wait(&done[s], phase);               // the MMAs that read this place are done
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                uint8_t* stage = smem + s * F::STAGE_BYTES + (turn % KT) * F::TILE_BYTES;
#pragma unroll
                for (int p = 0; p < 2; ++p) {                            // rows of 128 bytes, their sixteens swizzled by the row's place in eight
                    const int at = r + p * w.n_tok;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint2 lo = p ? two[2 * h] : one[2 * h], hi = p ? two[2 * h + 1] : one[2 * h + 1];
                        *reinterpret_cast<uint4*>(stage + at * 128 + (((2 * block + h) ^ (at & 7)) << 4)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    }
                    if (block == 0) *reinterpret_cast<uint32_t*>(stage + TOK * 256 + mx_scale_place(at)) = p ? mx_second_scales(word) : word;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full[s]));
                if ((s += SPLITTERS / KT) >= R) { s -= R; phase ^= 1u; }
            }
            it = (it + (uint32_t)tiles) % SPLITTERS;
            u = after(u, w);
        }
        if (!ok) *bail = 1;
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 3) {
        tmem_fence_after();
        tmem_dealloc(tmem, TMEM);
    }
}

// ---- narrow: how the line of tiles is cut ----
int segments_of(long tiles_n, long kb, long grid) {           // the most stretches that a row tile is cut into
    const long items = tiles_n * kb;
    long most = 1;
    for (long nt = 0; nt < tiles_n; ++nt) {
        const long first = ((nt * kb + 1) * grid - 1) / items, last = ((nt * kb + kb) * grid - 1) / items;
        if (last - first + 1 > most) most = last - first + 1;
    }
    return (int)most;
}
// CTAs, one an SM, each with a few tiles at least or a row tile (32 x 2,048 x 128: 9.3 us where a CTA took four row tiles of one, 5.1
// with one each), and the most stretches that they cut a row tile into: as many CTAs as leave no more than `limit`, or fewer that cut
// every row tile alike, down to two thirds of them: a CTA then has one unit, and SMs are left for the next kernel (32 x 4,096 x 14,336
// to slabs: 148 stretches 16.0 us, 128 quarters 12.2; 8 rows 10.6 and 10.0, added 13.9 and 11.6; 32 x 6,400 x 4,096 12.9 and 7.5 in 100
// halves; with 80 of 148 one row of 10,240 x 8,192 took 13.8 us instead of 12.1).  Where shares have to meet (`join`), row tiles stay
// whole if they come out even and the longest stretch and the meeting take longer (16 x 28,672 x 4,096 gated: 23.0 us in 148 stretches,
// 16.7 in 112 of two whole tiles).  In cycles: STAGE for a tile of an SM, JOIN for the partial sums' way through L2 and back.
constexpr int ANY = 1 << 30, LEAST_ITEMS = 4, STAGE = 370, JOIN = 6000;
struct Cut { int grid, segments; };
// What was last asked for in a place of a thread's table, and the answer to it (neither allocates nor locks).
constexpr int REMEMBERED = 256;
template <int N> constexpr uint32_t place_of(const int (&key)[N]) {
    uint32_t h = 0;                              // (which may wrap; a constant expression, as below, may not overflow an int)
    for (int i = 0; i < N; ++i) h = h * 37u + (uint32_t)key[i];
    return h % REMEMBERED;
}
constexpr int FURTHEST[7] = {INT_MAX, ANY, -ANY, INT_MAX, INT_MIN, 1, INT_MAX};
static_assert(place_of(FURTHEST) < REMEMBERED, "every question has a place");
template <typename Value, int N> struct Remembered {
    int asked[N];
    Value value;
    bool is(const int (&key)[N]) {               // else it is so from now on, and its value wanted
        bool same = true;
        for (int i = 0; i < N; ++i) same = same && asked[i] == key[i];
        if (!same)
            for (int i = 0; i < N; ++i) asked[i] = key[i];
        return same;
    }
};
Cut cut_of(int tiles_n, int kb, int limit, bool join) {
    static thread_local Remembered<Cut, 4> known[REMEMBERED];                // (counting through the tiles takes microseconds)
    const int key[4] = {tiles_n, kb, join ? -limit : limit, fb_sm_count()};
    Remembered<Cut, 4>& was = known[place_of(key)];
    if (was.is(key)) return was.value;
    const long slots = fb_sm_count();
    long grid = ((long)tiles_n * kb + LEAST_ITEMS - 1) / LEAST_ITEMS;
    if (grid < tiles_n) grid = tiles_n;
    if (grid > slots) grid = slots;
    const long even = grid / tiles_n * tiles_n;
    if (even * 3 >= grid * 2) grid = even;
    int segments = segments_of(tiles_n, kb, grid);
    while (segments > limit && grid > 1) segments = segments_of(tiles_n, kb, --grid);
    const long rounds = (tiles_n + slots - 1) / slots;
    if (join && segments > 1 && tiles_n % rounds == 0 && ((long)tiles_n * kb + grid - 1) / grid * STAGE + JOIN >= rounds * kb * STAGE) {
        grid = tiles_n / rounds;
        segments = 1;
    }
    return was.value = Cut{(int)grid, segments};
}
int narrow_tokens(int M) { return (M + 7) / 8 * 8; }

// ---- wide: token tiles and shares of K ----
struct Plan { int bn, splits; bool pair; };
constexpr int MORE_TILES = 2;
constexpr double L2_BYTES = 62.0;                 // what an SM gets from L2 a cycle when all of them ask
// The cheapest of the choices in cycles of an SM.  A stage costs its MMAs (2 cycles a column, twice for two parts of more than 64
// tokens), its way from L2 or its decoding, whichever is most; all CTAs together no less than the weights from HBM.  Decoding's cost
// grows with the CTAs: products that follow one another overlap on the SMs that the first leaves free (67 x 6,144 x 5,120 one after the
// other: 96 CTAs 12.9 us, 144 of fewer tokens 17.2; each by itself about 19.5).  A pair's epilogue overlaps little of the next one's
// products (100 cycles a token for both tiles), of a single tile's only the last one's shows.  Shares of K cost a copy of the output,
// written and read, and where they meet the adding, which nothing overlaps (67 x 6,144 x 5,120: three shares 21 us, whole 15.6 with the
// same tiles).  Where it decides for or against pairs: 301 x 28,672 x 4,096 68 us single, 80 in pairs; 128 x 28,672 x 4,096 34 single,
// 30 in pairs; 1,024 x 6,144 x 4,096 47 single, 55 in pairs.  (Pairs of up to 64 tokens have three stages in flight for the way to L2
// and back, 690 cycles: 64 x 28,672 x 4,096 22.2 single, 21.1 in pairs, 301 in tiles of 64 74.)  What the meeting of shares costs is
// counted as if there were few of them; where there are more than eight, plans come out up to half as long again as the best of their
// neighbours (33 x 1,024 x 14,336: 23.8 us, 64 rows 16.1).
Plan cheapest(long M, long N, int kb, int max_splits, long partial_floats, int n_counters, bool slabs) {
    const long sms = fb_sm_count(), tiles_n = (N + MX_ROWS - 1) / MX_ROWS;
    Plan best = {WIDE_TOKENS, 1, false};
    double best_cost = 1e300;
    const long least = (M + WIDE_TOKENS - 1) / WIDE_TOKENS;
    for (long tiles_m = least; tiles_m <= least + MORE_TILES; ++tiles_m) {
        const int bn = (int)(((M + tiles_m - 1) / tiles_m + 15) / 16 * 16);
        const long tiles = (M + bn - 1) / bn;
        for (int pair = 0; pair <= 1; ++pair) {
            const long units_n = pair ? (tiles_n + 1) / 2 : tiles_n;
            const double l2 = (bn * 256.0 + (pair ? 2 : 1) * (double)MX_TILE_BYTES) / L2_BYTES;
            for (int splits = 1; splits <= max_splits && splits <= kb; ++splits) {
                if (!slabs && splits > 1 && (tiles * tiles_n > n_counters || tiles * tiles_n * splits * bn * MX_ROWS > partial_floats)) break;
                const long units = tiles * units_n * splits, rounds = (units + sms - 1) / sms;
                const double decode = pair ? (bn <= SIDE_BY_SIDE ? 690.0 : 490.0) : 300.0 + (double)(units < sms ? units : sms);
                const double stage = fmax(fmax((pair ? 8.0 : 4.0) * bn, l2), decode) + 30.0;
                double cost = fmax((double)rounds * ((kb + splits - 1) / splits * stage + (pair ? 100.0 * bn : 500.0)) + (pair ? 0.0 : 45.0 * bn),
                                   (double)tiles_n * kb * MX_TILE_BYTES / (23.0 * sms));
                cost += (splits - 1) * (double)M * N * 8.0 / (24.0 * sms);
                if (splits > 1 && !slabs) cost += (double)rounds * (4000.0 + (pair ? 190.0 : 150.0) * bn);
                if (cost < best_cost * (1.0 - 1e-9)) { best_cost = cost; best = Plan{bn, splits, pair != 0}; }
            }
        }
    }
    return best;
}

constexpr long SHARE_FLOATS = 16L << 20;          // most that the shares of one product may take
constexpr int MOST_SPLITS = 16;

Plan plan_wide(int M, int N, int kb, int max_splits, int n_counters, bool slabs) {
    static thread_local Remembered<Plan, 7> known[REMEMBERED];                               // (looking for it takes microseconds)
    const int key[7] = {M, N, kb, max_splits, n_counters, slabs ? 1 : 0, fb_sm_count()};
    Remembered<Plan, 7>& was = known[place_of(key)];
    if (was.is(key)) return was.value;
    return was.value = cheapest(M, N, kb, max_splits, SHARE_FLOATS, n_counters, slabs);
}

template <int TOK, bool GROUPED, bool PAIR>
int launch(const MxArgs& a, const CUtensorMap& mx, const CUtensorMap& mo, long grid, cudaStream_t stream) {
    auto kernel = gemm_mxfp4_kernel<TOK, GROUPED, PAIR>;
    static bool configured[FB_MAX_DEVICES] = {};
    if (fb_needs_setup(configured)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return fb_fail(-2, "gemm_mxfp4: cannot reserve shared memory: %s", cudaGetErrorString(e));
        fb_setup_done(configured);
    }
    fb_launch_class(a.M > 128 && Form<TOK, PAIR>::WIDE ? FB_LAUNCH_GEMM_WIDE : FB_LAUNCH_OTHER, kernel, dim3((unsigned)grid),
                    dim3(Form<TOK, PAIR>::THREADS), SMEM, stream, mx, mo, a);
    return fb_check_launch("gemm_mxfp4");
}

// Whether the form of few rows takes the product (tile: the grouped form's row tile, 0: not grouped).  A CTA splits what it multiplies:
// that spares a kernel that 8 rows spent 4 to 8 us in, behind the weights that the product had on their way by then, and one until the
// first MMA (shares to slabs, 8 x 4,096 x 14,336, 24 stages a CTA: 17.3 us with that kernel, 11.9 without; 8 x 7,168 x 18,432, 55: 21.7
// and 18.2).  But its warps share the issue slots with the decoding: longer stretches are faster with the kernel (8 x 28,672 x 4,096
// gated, 64 stages: 14.9 us, 17.5), and so are 16 rows (15.1 us, 30.8) and products whose row tiles share a group's rows (65 us, 93).
constexpr int FEW_STAGES = 60;
bool few_rows(int M, int N, int K, int tile, bool slabs) {
    if (tile || M > FEW_TOKENS) return false;
    const long tiles_n = (N + MX_ROWS - 1) / MX_ROWS, kb = (K + MX_COLS - 1) / MX_COLS;
    const long grid = slabs ? fb_sm_count() : cut_of((int)tiles_n, (int)kb, ANY, true).grid;
    return tiles_n * kb <= FEW_STAGES * grid;
}

// Bytes of the rows' scales.  (Token tiles are at most MORE_TILES more than the rows need; the grouped form has a place for every row
// tile.)
long long scale_bytes_of(int M, int kb, int tile) {
    const long long tiles = tile ? M / tile : (M + WIDE_TOKENS - 1) / WIDE_TOKENS + MORE_TILES;
    return kb * tiles * ATOM * (tile == 16 || (!tile && M <= SIDE_BY_SIDE) ? 1 : 2);
}

// The rows' parts and scales in `scratch`, their map, the output's map.
int prepare(MxArgs& a, CUtensorMap& mx, CUtensorMap& mo, void* scratch, int box_rows, cudaStream_t stream) {
    const bool grouped = a.tile_group != nullptr;
    if (few_rows(a.M, a.N, a.K, a.tile, a.slabs > 0)) return 0;                 // (the product splits them itself, and stores directly)
    const long Kp = (long)a.kb * MX_COLS, parts = 2L * a.M * Kp;
    a.x_scales = (const uint8_t*)scratch + parts;
    a.scale_bytes = atoms_of(a.bn) * ATOM;
    const int most = grouped ? a.bn / a.tile : 0;
    int rc = fb_mxfp4_split_rows(a.rows, a.M, a.K, scratch, (uint8_t*)scratch + parts,
                                 MxScaleLayout{a.bn, a.scale_bytes, a.tile_group, a.tile, most, a.n_tiles, a.groups}, stream);
    if (rc) return rc;
    rc = fb_tensor_map_bf16(&mx, scratch, 2L * a.M, Kp / 2, Kp / 2, 64, box_rows);       // (bytes, two at a time)
    if (rc) return rc;
    a.boxed = 0;
    if (box_rows <= NARROW_TOKENS && (!grouped || a.tile == 16)) return 0;               // (the narrow form stores directly)
    const int tokens = a.o_bf16 || a.gate.act ? 16 : 8;
    rc = fb_tensor_map_out(&mo, a.out, a.o_bf16 ? 2 : 4, a.M, a.gate.act ? a.N / 2 : a.N, a.ldo, a.slabs ? a.slabs : 1, a.slab_stride,
                           a.gate.act ? MX_ROWS / 2 : MX_ROWS, tokens);
    a.boxed = rc == 0 ? tokens : 0;
    return rc < 0 ? rc : 0;
}

int check_operands(const void* X, long long lda, const void* W, const void* out, int o_dtype, long long ldo, int M, int N,
                   int K, FbGate gate, int plain_act, int* status) {
    FB_REQUIRE(M >= 0 && N > 0 && K > 0, "gemm_mxfp4: bad sizes M=%d N=%d K=%d", M, N, K);
    FB_REQUIRE(o_dtype == FB_F32 || o_dtype == FB_BF16, "gemm_mxfp4: unknown output dtype code %d", o_dtype);
    FB_REQUIRE(!gate.act || (fb_gate_known(gate) && N % 2 == 0 && !plain_act),
               "gemm_mxfp4: a gate needs a known activation, an even number of stacked rows and no plain activation beside it");
    FB_REQUIRE(fb_plain_act_known(plain_act), "gemm_mxfp4: unknown activation code %d", plain_act);
    FB_REQUIRE(((long)N + MX_ROWS - 1) / MX_ROWS * (((long)K + MX_COLS - 1) / MX_COLS) < (1L << 24), "gemm_mxfp4: too many weights, %d x %d", N, K);
    FB_REQUIRE(lda >= K && ldo >= (gate.act ? N / 2 : N), "gemm_mxfp4: a row stride is shorter than its row");
    FB_REQUIRE(((uintptr_t)X & 1) == 0 && W && ((uintptr_t)W & 15) == 0 && status,
               "gemm_mxfp4: unaligned rows or weights, or no status word");
    FB_REQUIRE(((uintptr_t)out & (o_dtype == FB_F32 ? 3 : 1)) == 0, "gemm_mxfp4: unaligned output");
    return 0;
}

}  // namespace

// What the rows' parts and their scales take, a multiple of 256 bytes (tile: the grouped form's row tile, 0: not grouped).
static long long rows_bytes(int M, int N, int K, int tile, bool slabs) {
    if (M <= 0 || N <= 0 || K <= 0 || few_rows(M, N, K, tile, slabs)) return 0;
    const long long kb = (K + MX_COLS - 1) / MX_COLS;
    return (2LL * M * kb * MX_COLS + scale_bytes_of(M, (int)kb, tile) + 255) / 256 * 256;
}

// Floats that shares of K take which meet in scratch: 0 where K is not split.
static long long share_floats(int M, int N, int K, int n_counters) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int tiles_n = (N + MX_ROWS - 1) / MX_ROWS, kb = (K + MX_COLS - 1) / MX_COLS;
    if (M <= NARROW_TOKENS) {
        const int segments = tiles_n <= n_counters ? cut_of(tiles_n, kb, ANY, true).segments : 1;
        return segments > 1 ? (long long)tiles_n * segments * narrow_tokens(M) * MX_ROWS : 0;
    }
    const Plan p = plan_wide(M, N, kb, MOST_SPLITS, n_counters, false);
    return p.splits == 1 ? 0 : (long long)((M + p.bn - 1) / p.bn) * tiles_n * p.splits * p.bn * MX_ROWS;
}

// Bytes of `scratch` that the products below want for M rows, with `n_counters` counters.  slabs: shares of K go to slabs; tile: the
// grouped form's row tile (0: not grouped).
FB_API long long fb_gemm_mxfp4_scratch_bytes(int M, int N, int K, int n_counters, int slabs, int tile) {
    return rows_bytes(M, N, K, tile, slabs != 0) + (slabs || tile ? 0 : 4 * share_floats(M, N, K, n_counters));
}

// X [M,K] bfloat16, W one matrix in tiles (fb_mxfp4_tiles).  `act` (an FbAct code with its constants): W stacks gate
// and up rows alternately and out[m, c] = act(g_c) u_c has N / 2 columns; `plain_act` (an FbPlainAct code): out = act(product);
// `accumulate` (float32): the product is added to what `out` holds.  Shares of K: with slab_stride > 0 (float32, neither activation
// nor accumulate) share s goes to out + s * slab_stride and *splits_used says how many there are (at most max_slabs); else they
// meet in `scratch` and at `counters` (zero before the call and after it).  `scratch`: at least fb_gemm_mxfp4_scratch_bytes on a
// 128-byte border, of calls that run one after the other.
FB_API int fb_gemm_mxfp4(const void* X, long long lda, const void* W, void* out, int o_dtype, long long ldo,
                         long long slab_stride, int max_slabs, int* splits_used, int M, int N, int K, int act, float limit,
                         float slope, int plain_act, int accumulate, int* counters, int n_counters, void* scratch,
                         long long scratch_bytes, int* status, cudaStream_t stream) {
    const FbGate gate = {act, limit, slope};
    if (const int rc = check_operands(X, lda, W, out, o_dtype, ldo, M, N, K, gate, plain_act, status)) return rc;
    FB_REQUIRE(slab_stride == 0 || (o_dtype == FB_F32 && max_slabs >= 1 && slab_stride >= (long long)M * ldo && !act && !plain_act &&
                                    !accumulate),
               "gemm_mxfp4: slabs must be float32, at least one, not overlap, and hold plain shares");
    FB_REQUIRE(!accumulate || (o_dtype == FB_F32 && !act && !plain_act), "gemm_mxfp4: only a float32 product can be added to its output");
    if (splits_used) *splits_used = 1;
    if (M == 0) return 0;
    MxArgs a = {};
    a.W = (const uint8_t*)W; a.out = out; a.ldo = (long)ldo; a.slab_stride = (long)slab_stride;
    a.rows = MxRows{(const __nv_bfloat16*)X, (long)lda, M, lda % 8 == 0 && ((uintptr_t)X & 15) == 0, nullptr, nullptr, nullptr};
    a.o_bf16 = o_dtype == FB_BF16; a.accumulate = accumulate; a.counters = counters;
    a.M = M; a.N = N; a.K = K; a.kb = (K + MX_COLS - 1) / MX_COLS; a.tiles_n = (N + MX_ROWS - 1) / MX_ROWS;
    a.gate = gate; a.plain_act = plain_act; a.status = status;
    const bool slabs = slab_stride > 0;
    const long long need = fb_gemm_mxfp4_scratch_bytes(M, N, K, n_counters, slabs, 0), rows = rows_bytes(M, N, K, 0, slabs);
    FB_REQUIRE((need == 0 || (scratch && ((uintptr_t)scratch & 127) == 0 && scratch_bytes >= need)) && (slabs || (counters && n_counters > 0)),
               "gemm_mxfp4: %lld bytes of scratch wanted, and counters", need);
    a.partials = need > rows ? (float*)((uint8_t*)scratch + rows) : nullptr;
    const bool join = a.partials != nullptr;
    CUtensorMap mx = {}, mo = {};
    if (M <= NARROW_TOKENS) {
        const Cut cut = cut_of(a.tiles_n, a.kb, slabs ? max_slabs : join ? ANY : 1, !slabs);
        a.bn = narrow_tokens(M);
        a.tiles_m = 1; a.splits = 1; a.items = (uint32_t)a.tiles_n * a.kb;
        a.max_segments = cut.segments;
        if (slabs) {
            a.slabs = cut.segments;
            if (splits_used) *splits_used = cut.segments;
        }
        if (const int rc = prepare(a, mx, mo, scratch, a.bn, stream)) return rc;
        return few_rows(M, N, K, 0, slabs) ? launch<FEW_TOKENS, false, false>(a, mx, mo, cut.grid, stream)
                                           : launch<32, false, false>(a, mx, mo, cut.grid, stream);
    }
    const Plan plan = plan_wide(M, N, a.kb, slabs ? (max_slabs < MOST_SPLITS ? max_slabs : MOST_SPLITS) : join ? MOST_SPLITS : 1, n_counters,
                                slabs);
    a.bn = plan.bn;
    a.tiles_m = (M + plan.bn - 1) / plan.bn;
    a.units_n = plan.pair ? (a.tiles_n + 1) / 2 : a.tiles_n;
    a.splits = a.max_segments = plan.splits;
    if (slabs) {
        a.slabs = plan.splits;
        if (splits_used) *splits_used = plan.splits;
    }
    const long items = (long)a.tiles_m * a.units_n * a.splits;
    a.items = (uint32_t)items;
    if (items > 2000000000L) return fb_fail(-1, "gemm_mxfp4: too many tiles (M=%d N=%d)", M, N);
    if (const int rc = prepare(a, mx, mo, scratch, a.bn, stream)) return rc;
    const long grid = items < fb_sm_count() ? items : fb_sm_count();
    if (plan.pair) return a.bn <= 64 ? launch<64, false, true>(a, mx, mo, grid, stream) : launch<128, false, true>(a, mx, mo, grid, stream);
    return a.bn <= 64 ? launch<64, false, false>(a, mx, mo, grid, stream) : launch<128, false, false>(a, mx, mo, grid, stream);
}

// The grouped form: W holds `groups` matrices [N, K] in tiles; the M rows of `out` come in tiles of `tile` (a multiple of 16 up to 128)
// rows of one group each (tile_group, negative: skipped, its rows of `out` stay as they are; beyond the last: its products are NaN, and
// what the activation makes of that).  Row m is X[m], or with row_index X[row_index[m]] (zeros where that is none of the x_rows), with
// row_share times row_share[row_pair[m]].  `scratch`: at least fb_gemm_mxfp4_scratch_bytes on a 128-byte border.
FB_API int fb_gemm_mxfp4_grouped(const void* X, long long lda, int x_rows, const int* row_index, const float* row_share, const int* row_pair,
                                 const void* W, int groups, const int* tile_group, int tile, void* out, int o_dtype,
                                 long long ldo, int M, int N, int K, int act, float limit, float slope, int plain_act, void* scratch,
                                 long long scratch_bytes, int* status, cudaStream_t stream) {
    const FbGate gate = {act, limit, slope};
    if (const int rc = check_operands(X, lda, W, out, o_dtype, ldo, M, N, K, gate, plain_act, status)) return rc;
    FB_REQUIRE(groups > 0 && tile_group, "gemm_mxfp4_grouped: no groups");
    FB_REQUIRE(x_rows >= (row_index ? 0 : M), "gemm_mxfp4_grouped: %d rows are fewer than the %d of the output", x_rows, M);
    FB_REQUIRE(tile >= 16 && tile <= 128 && tile % 16 == 0 && M % tile == 0 && M / tile < (1 << 24),
               "gemm_mxfp4_grouped: the rows must be whole tiles of 16 to 128, not tiles of %d", tile);
    FB_REQUIRE(!row_share || (row_index && row_pair), "gemm_mxfp4_grouped: shares need the rows' index and pairs");
    FB_REQUIRE(scratch && ((uintptr_t)scratch & 127) == 0 && scratch_bytes >= rows_bytes(M, N, K, tile, false), "gemm_mxfp4_grouped: scratch missing");
    if (M == 0) return 0;
    MxArgs a = {};
    a.kb = (K + MX_COLS - 1) / MX_COLS;
    a.tiles_n = (N + MX_ROWS - 1) / MX_ROWS;
    a.W = (const uint8_t*)W; a.w_group = (long)a.tiles_n * a.kb * MX_TILE_BYTES; a.out = out; a.ldo = (long)ldo;
    a.groups = groups;
    a.rows = MxRows{(const __nv_bfloat16*)X, (long)lda, x_rows, lda % 8 == 0 && ((uintptr_t)X & 15) == 0, row_index, row_share, row_pair};
    a.o_bf16 = o_dtype == FB_BF16; a.M = M; a.N = N; a.K = K; a.tiles_m = 1; a.splits = a.max_segments = 1;
    a.gate = gate; a.plain_act = plain_act; a.status = status;
    a.tile_group = tile_group; a.tile = tile; a.n_tiles = M / tile;
    // Tiles of 16 are few rows a group, and stay by themselves: six of one group take as long as six of as many groups (20.5 us, 3,584
    // x 4,096; six tiles of 32 of one group, which are joined, 17.7).  Groups of at most 64 rows have units of 64 (180 tokens on 6 of 64
    // experts, 3,584 x 4,096: 116 us, in units of 128 131), larger ones of 128 (1,024 tokens: 214 us, in units of 64 264).
    const bool narrow = tile == 16, small = M <= (long)SIDE_BY_SIDE * groups && tile <= SIDE_BY_SIDE;
    a.units_n = a.tiles_n;
    const long units = (long)a.n_tiles * a.units_n;
    if (units > 2000000000L) return fb_fail(-1, "gemm_mxfp4_grouped: too many tiles (M=%d N=%d)", M, N);
    CUtensorMap mx = {}, mo = {};
    a.bn = narrow ? tile : (small ? SIDE_BY_SIDE : WIDE_TOKENS) / tile * tile;
    if (const int rc = prepare(a, mx, mo, scratch, tile, stream)) return rc;
    const long grid = units < fb_sm_count() ? units : fb_sm_count();
    if (narrow) return launch<32, true, false>(a, mx, mo, grid, stream);
    return small ? launch<64, true, false>(a, mx, mo, grid, stream) : launch<128, true, false>(a, mx, mo, grid, stream);
}
