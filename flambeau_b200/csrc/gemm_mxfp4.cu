// out[M,N] = X[M,K] * W[N,K]^T with X in bfloat16 and W in four bits (mxfp4.cuh) on the 5th-generation tensor cores.
//
// Every number of W is a bfloat16 number, so the product is that of two bfloat16 matrices, summed in float32: nothing is rounded
// that a bfloat16 weight would not have rounded.  What is gained is memory: 17 bits for every four of a bfloat16 weight.
//
// Layout.  One CTA owns 128 output features x up to 192 tokens ("swap-AB": the weight is the 128-row operand of tcgen05.mma, the
// tokens its N dimension).  A stage is 128 of K: one bulk copy brings a weight tile of 8,704 bytes as it lies in memory, two TMA copies
// (128-byte swizzle) the tokens.  Eight warps decode: a thread a feature, 128 numbers a stage as 64 pairs into tensor memory, where
// the MMA takes its A operand from.  The decoded weights never pass through shared memory: at 88 bytes a cycle for writing and as
// many for reading, which memory speed would ask for, its 128 bytes a cycle would be the bound.  The two groups of four warps
// take the stages in turn.
//
// Warps: 0 weight copies, 1 MMA, 2 token copies, 3 tensor memory, 4..11 decode, 12.. epilogue (a thread a feature; two warps a lane
// quarter in the wide form).  full[s]: the stage's tokens (bytes) and its decoded weights (128 arrivals) are there; done[s]: its
// MMAs are.  Two accumulators, so that the epilogue of one unit overlaps the products of the next.
//
// Shares of K go to slabs that the next kernel adds, or meet in scratch, where the CTA that arrives last (a counter a tile, no
// waiting) adds them in order.  Grouped form (routed experts): a unit is a run of neighbouring row tiles of one group.
//
// Every mbarrier wait is bounded as in gemm_tc.cu.
#include "group_units.cuh"
#include "mxfp4.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

namespace {

constexpr int XBM = MX_ROWS;                      // output features per CTA
constexpr int XBK = MX_COLS;                      // K per stage
constexpr int A_COLS = XBK / 2;                   // tensor-memory columns of a stage's weights
constexpr int MAX_W = 16, MAX_R = 4;              // most stages of packed weights / of tokens and decoded weights
constexpr int X_LIST = 256;                       // units of the grouped form that are kept in shared memory
constexpr int OUT_TOKENS = 16;
constexpr int OUT_BYTES = OUT_TOKENS * XBM * 4;   // a staged box of the output
constexpr int CONTROL = 512 + 4 * X_LIST;         // barriers and flags, the list

// The narrow form (up to 32 tokens: decoding) leaves room for two CTAs an SM, so that one kernel's first weights are on their way
// while the kernel before it drains; the wide form has the SM to itself and sends its output through shared memory.
template <bool WIDE> struct Form {
    static constexpr int EPI_WARPS = WIDE ? 8 : 4;
    static constexpr int THREADS = 32 * (12 + EPI_WARPS);
    static constexpr int MOST_TOKENS = WIDE ? 192 : 32;
    static constexpr int TMEM = WIDE ? 512 : 256;
    static constexpr int SMEM = WIDE ? 227 * 1024 : 113 * 1024;
    static constexpr int OUT = WIDE ? 4 * OUT_BYTES : 0;
    static constexpr int RING = SMEM - 1024 - CONTROL - OUT;          // for both rings of stages
};

struct MxArgs {
    const uint8_t* W; long w_group; const int* shifts;    // tiles, bytes of one group's, what each group's results are raised by
    void* out; long ldo, slab_stride;
    int o_bf16, accumulate, boxed;
    float* partials; int* counters;
    int M, N, K, kb, bn, acc_cols, tiles_m, tiles_n, splits, n_units, ws, ring;
    const int* tile_group; int tile, n_tiles;
    FbGate gate; int plain_act;
    int* status;
};

struct MxUnit { int m0, n_tok, nt, group, split, kb0, n_kb, id; };

__device__ __forceinline__ void store_box(const void* map, uint32_t src, int x, int y, int z, bool add) {
    if (add)
        asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                     ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                     ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <bool WIDE>
__global__ void __launch_bounds__(Form<WIDE>::THREADS, WIDE ? 1 : 2)
gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_o,
                  const __grid_constant__ MxArgs a) {
    using F = Form<WIDE>;
    constexpr int EPI = 32 * F::EPI_WARPS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int WS = a.ws, R = a.ring;
    const uint32_t atom_bytes = (uint32_t)a.bn * 128, x_bytes = 2 * atom_bytes;
    uint8_t* w_base = smem + (size_t)R * x_bytes;                        // [token stages | weight stages | output boxes | control]
    uint8_t* out_stage = smem + F::RING;
    uint64_t* bars = (uint64_t*)(out_stage + F::OUT);
    uint64_t *w_full = bars, *w_empty = w_full + MAX_W, *full = w_empty + MAX_W, *done = full + MAX_R, *acc_full = done + MAX_R,
             *acc_empty = acc_full + 2;
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
    int* flag = (int*)(tmem_slot + 1);           // what the epilogue decided together
    int* bail = flag + 1;                        // a bounded wait ran out somewhere in this CTA
    int* unit_count = bail + 1;
    uint32_t* list = (uint32_t*)((uint8_t*)bars + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(smem_u32(bar), parity, a.status); };
    auto bailed = [&]() { return *(volatile int*)bail != 0; };
    const bool grouped = a.tile_group != nullptr;
    const int most = grouped ? a.bn / a.tile : 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_W; ++s) { mbar_init(smem_u32(&w_full[s]), 1); mbar_init(smem_u32(&w_empty[s]), 128); }
        for (int s = 0; s < MAX_R; ++s) { mbar_init(smem_u32(&full[s]), 129); mbar_init(smem_u32(&done[s]), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&acc_full[s]), 1); mbar_init(smem_u32(&acc_empty[s]), EPI); }
        *bail = 0;
        mbar_fence_init();
    }
    if (warp == 3) tmem_alloc(tmem_slot, F::TMEM);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    fb_pdl_launch_dependents();                  // (behind the allocation: see umma.cuh)
    const uint32_t tmem = *tmem_slot;
    int n_units = a.n_units, stride = gridDim.x;
    if (grouped) {
        if (warp == 12) {
            fb_pdl_wait();                       // which weights a tile wants is the work of the kernels before this one
            const int found = group_units<X_LIST>(a.tile_group, a.n_tiles, most, list);
            if (lane == 0) *unit_count = found;
        }
        __syncthreads();
        n_units = *unit_count * a.tiles_n;
    }
    GroupWalk walk = {0, 0u};
    auto unit_of = [&](int u) {
        MxUnit w;
        if (grouped) {                           // feature tiles vary fastest: the CTAs that run together share few units' rows
            const int i = u / a.tiles_n;
            const uint32_t unit = group_unit<X_LIST>(a.tile_group, a.n_tiles, most, list, i, walk);
            const int t = (int)(unit & 0xffffffu);
            w.m0 = t * a.tile;
            w.n_tok = (int)(unit >> 24) * a.tile;
            w.group = a.tile_group[t];
            w.nt = u - i * a.tiles_n;
            w.id = 0; w.split = 0; w.kb0 = 0; w.n_kb = a.kb;
        } else {                                 // token tiles vary fastest: the CTAs that run together share weight tiles
            const int tiles = a.tiles_m * a.tiles_n;
            w.split = u / tiles;
            w.id = u - w.split * tiles;
            w.m0 = w.id % a.tiles_m * a.bn;
            w.nt = w.id / a.tiles_m;
            w.n_tok = a.bn;
            w.group = 0;
            w.kb0 = (int)((long)w.split * a.kb / a.splits);
            w.n_kb = (int)((long)(w.split + 1) * a.kb / a.splits) - w.kb0;
        }
        return w;
    };

    if (warp == 0) {
        // ---------------- weights: no other kernel writes them, so they are requested at once ----------------
        if (elect_one()) {
            int s = 0;
            uint32_t phase = 1;
            for (int u = blockIdx.x; u < n_units && !bailed(); u += stride) {
                const MxUnit w = unit_of(u);
                const uint8_t* src = a.W + (size_t)w.group * a.w_group + ((size_t)w.nt * a.kb + w.kb0) * MX_TILE_BYTES;
                for (int i = 0; i < w.n_kb; ++i, src += MX_TILE_BYTES) {
                    if (!wait(&w_empty[s], phase)) { *bail = 1; break; }
                    mbar_expect_tx(smem_u32(&w_full[s]), MX_TILE_BYTES);
                    bulk_copy_g2s(smem_u32(w_base + (size_t)s * MX_TILE_BYTES), src, MX_TILE_BYTES, smem_u32(&w_full[s]));
                    if (++s == WS) { s = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---------------- tokens ----------------
        if (elect_one()) {
            fb_pdl_wait();
            int s = 0;
            uint32_t phase = 1;
            for (int u = blockIdx.x; u < n_units && !bailed(); u += stride) {
                const MxUnit w = unit_of(u);
                const int boxes = grouped ? w.n_tok / a.tile : 1, box = grouped ? a.tile : a.bn;
                for (int i = 0; i < w.n_kb; ++i) {
                    if (!wait(&done[s], phase)) { *bail = 1; break; }
                    mbar_expect_tx(smem_u32(&full[s]), (uint32_t)w.n_tok * 256);
                    const uint32_t dst = smem_u32(smem) + (uint32_t)s * x_bytes;
                    for (int b = 0; b < boxes; ++b) {
#pragma unroll
                        for (int h = 0; h < 2; ++h)          // (rows beyond M and columns beyond K arrive as zeros)
                            tma_load_2d(dst + h * atom_bytes + (uint32_t)(b * box) * 128, &map_x, smem_u32(&full[s]),
                                        (w.kb0 + i) * XBK + h * 64, w.m0 + b * box);
                    }
                    if (++s == R) { s = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA ----------------
        if (elect_one()) {
            int s = 0, j = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < n_units && ok && !bailed(); u += stride, ++j) {
                const MxUnit w = unit_of(u);
                const uint32_t idesc = umma_idesc(w.n_tok);
                const int b = j & 1;
                ok = wait(&acc_empty[b], ((uint32_t)(j >> 1) & 1u) ^ 1u);        // (the epilogue has drained it, two units ago)
                if (!ok) break;
                tmem_fence_after();
                const uint32_t d = tmem + (uint32_t)(b * a.acc_cols);
                for (int i = 0; i < w.n_kb; ++i) {
                    ok = wait(&full[s], phase);
                    if (!ok) break;
                    tmem_fence_after();
                    const uint32_t A = tmem + (uint32_t)(2 * a.acc_cols + s * A_COLS);
                    const uint64_t x = umma_desc(smem_u32(smem) + (uint32_t)s * x_bytes);
#pragma unroll
                    for (int k = 0; k < XBK / UMMA_K; ++k)
                        umma_bf16_ts(d, A + (uint32_t)(k * (UMMA_K / 2)), x + (uint64_t)((k >> 2) * (atom_bytes >> 4) + (k & 3) * 2),
                                     idesc, (i > 0 || k > 0) ? 1u : 0u);
                    umma_commit(smem_u32(&done[s]));
                    if (++s == R) { s = 0; phase ^= 1u; }
                }
                if (ok) umma_commit(smem_u32(&acc_full[b]));
            }
            if (!ok) *bail = 1;
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 12) {
        // ---------------- decode: a thread a feature; the group's stages are it = ab, ab + 2, ... ----------------
        // (A wait names a phase by its parity alone.  A group comes to a slot of the rings at every second turn or at every one; it
        // cannot be two turns off: it has seen the MMAs of stage it - 2 - R done, and so every earlier stage decoded, and WS > R + 2.)
        const int quarter = warp & 3, row = quarter * 32 + lane, ab = (warp - 4) >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(2 * a.acc_cols);
        uint32_t it = 0, w_phase = 0, r_phase = 1;
        int ws = 0, r = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < n_units && ok && !bailed(); u += stride) {
            const int n = unit_of(u).n_kb;
            for (int i = 0; i < n; ++i, ++it) {
                if ((int)(it & 1u) == ab) {
                    ok = wait(&w_full[ws], w_phase);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    const uint8_t* src = w_base + (size_t)ws * MX_TILE_BYTES;
                    const uint32_t scales = *reinterpret_cast<const uint32_t*>(src + MX_CODE_BYTES + row * 4);
                    uint4 c[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) c[q] = *reinterpret_cast<const uint4*>(src + (q * MX_ROWS + row) * 16);
                    ok = wait(&done[r], r_phase);                        // the MMAs that read this buffer are done
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tmem_fence_after();
                    const uint32_t dst = lanes + (uint32_t)(r * A_COLS);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t scale = mx_scale(scales >> (8 * q) & 255u);
                        uint32_t v[16];
                        mx_decode(c[q].x, scale, v);
                        mx_decode(c[q].y, scale, v + 4);
                        mx_decode(c[q].z, scale, v + 8);
                        mx_decode(c[q].w, scale, v + 12);
                        tmem_st16(dst + (uint32_t)(q * 16), v);
                    }
                    // (behind the stores, which need every number of the row: see gemm_f32_tc.cu)
                    mbar_arrive(smem_u32(&w_empty[ws]));
                    tmem_wait_st();
                    tmem_fence_before();
                    mbar_arrive(smem_u32(&full[r]));
                }
                if (++ws == WS) { ws = 0; w_phase ^= 1u; }
                if (++r == R) { r = 0; r_phase ^= 1u; }
            }
        }
        if (!ok) *bail = 1;
    } else if (warp >= 12) {
        // ---------------- epilogue: lanes are features ----------------
        fb_pdl_wait();
        const int quarter = warp & 3, half = (warp - 12) >> 2, row = quarter * 32 + lane;
        const bool leader = quarter == 0 && lane == 0;
        constexpr int STEP = OUT_TOKENS * (F::EPI_WARPS / 4);
        const bool join = a.splits > 1 && a.slab_stride == 0;
        uint32_t boxes = 0;                      // boxes this group of warps has staged: the buffers take turns
        int j = 0;
        for (int u = blockIdx.x; u < n_units; u += stride, ++j) {
            const MxUnit w = unit_of(u);
            const int b = j & 1, n0 = w.nt * XBM, n = n0 + row;
            const int rows = min(w.n_tok, a.M - w.m0);                   // (grouped: whole tiles)
            const float* from = nullptr;                                 // where shares are joined: the first one of this tile
            if (bailed() || !wait(&acc_full[b], (uint32_t)(j >> 1) & 1u)) *bail = 1;
            asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
            if (threadIdx.x == 12 * 32) *flag = bailed() ? 2 : 0;        // one thread decides for all: they meet at barriers below
            asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
            if (*flag == 2) break;
            tmem_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * a.acc_cols);
            if (join) {
                float* mine = a.partials + ((size_t)w.id * a.splits + w.split) * (size_t)(a.bn * XBM) + row;
                for (int c = half * OUT_TOKENS; c < rows; c += STEP) {
                    float v[16];
                    tmem_ld16(acc + (uint32_t)c, v);
#pragma unroll
                    for (int q = 0; q < 16; ++q) mine[(size_t)(c + q) * XBM] = v[q];
                }
                __threadfence();
                asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
                if (threadIdx.x == 12 * 32) {
                    const bool last = atomicAdd(&a.counters[w.id], 1) == a.splits - 1;
                    if (last) a.counters[w.id] = 0;                      // ready for the next launch
                    *flag = last;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
                if (*flag == 1) {
                    __threadfence();
                    from = a.partials + (size_t)w.id * a.splits * (size_t)(a.bn * XBM) + row;
                }
            }
            if (!join || from) {
                const int shift = a.shifts[w.group];
                const float raise = shift > 0 ? ldexpf(1.0f, shift) : 1.0f;
#pragma unroll 1
                for (int c = half * OUT_TOKENS; c < rows; c += STEP) {
                    float v[16];
                    if (from) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q] = 0.0f;
                        for (int s = 0; s < a.splits; ++s) {
                            const float* p = from + ((size_t)s * a.bn + c) * XBM;
#pragma unroll
                            for (int q = 0; q < 16; ++q) v[q] += __ldcg(p + q * XBM);
                        }
                    } else {
                        tmem_ld16(acc + (uint32_t)c, v);
                    }
                    if (shift > 0) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q] *= raise;
                    }
                    if (a.plain_act) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q] = fb_plain_act(a.plain_act, v[q]);
                    }
                    // gated: features alternate gate, up; the even lane has act(gate) * up of column n / 2
                    bool writes = n < a.N;
                    int col = n, width = XBM, at = row;
                    if (a.gate.act) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            const float up = __shfl_xor_sync(0xffffffffu, v[q], 1);
                            v[q] = fb_gate_times(a.gate, v[q], up);
                        }
                        writes = !(lane & 1) && n + 1 < a.N;
                        col = n >> 1; width = XBM / 2; at = row >> 1;
                    }
                    if (WIDE && a.boxed) {
                        // the values go to shared memory as [token][feature], and one thread sends the box on its way (what lies
                        // beyond the output's edge is not written)
                        uint8_t* box = out_stage + (half * 2 + (boxes & 1u)) * OUT_BYTES;
                        ++boxes;
                        if (leader) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // it has left this buffer
                        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
                        if (!a.gate.act || !(lane & 1)) {
                            if (a.o_bf16) {
#pragma unroll
                                for (int q = 0; q < 16; ++q) reinterpret_cast<__nv_bfloat16*>(box)[q * width + at] = __float2bfloat16_rn(v[q]);
                            } else {
#pragma unroll
                                for (int q = 0; q < 16; ++q) reinterpret_cast<float*>(box)[q * width + at] = v[q];
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
                        if (leader) store_box(&map_o, smem_u32(box), a.gate.act ? n0 / 2 : n0, w.m0 + c, join ? 0 : w.split, a.accumulate != 0);
                    } else if (writes) {
                        const size_t first = (size_t)w.split * a.slab_stride + (size_t)(w.m0 + c) * a.ldo + col;
                        if (a.o_bf16) {
                            __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(a.out) + first;
#pragma unroll
                            for (int q = 0; q < 16; ++q)
                                if (c + q < rows) p[(size_t)q * a.ldo] = __float2bfloat16_rn(v[q]);
                        } else {
                            float* p = reinterpret_cast<float*>(a.out) + first;
#pragma unroll
                            for (int q = 0; q < 16; ++q)
                                if (c + q < rows) p[(size_t)q * a.ldo] = a.accumulate ? p[(size_t)q * a.ldo] + v[q] : v[q];
                        }
                    }
                }
            }
            tmem_fence_before();
            mbar_arrive(smem_u32(&acc_empty[b]));
        }
        if (WIDE && leader) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");        // the boxes it sent are in memory
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 3) {
        tmem_fence_after();
        tmem_dealloc(tmem, F::TMEM);
    }
}

struct MxPlan { int bn, splits; bool wide; };

// Token tiles and shares of K: the cheapest of the choices in cycles of an SM.  A stage costs its MMAs (4 cycles a token) or its
// decoding, whichever is more; all CTAs together no less than the weights from HBM.  A share of K costs a copy of the output, written
// and read.
MxPlan plan_mxfp4(long M, long N, int kb, int max_splits, long partial_floats, int n_counters, bool slabs) {
    const long sms = fb_sm_count(), tiles_n = (N + XBM - 1) / XBM;
    MxPlan best = {32, 1, false};
    double best_cost = 1e300;
    const bool wide = M > Form<false>::MOST_TOKENS;
    const int most = wide ? Form<true>::MOST_TOKENS : Form<false>::MOST_TOKENS;
    const long least = (M + most - 1) / most, slots = wide ? sms : 2 * sms;
    for (long tiles_m = least; tiles_m <= least + 2; ++tiles_m) {
        const int bn = (int)(((M + tiles_m - 1) / tiles_m + 15) / 16 * 16);
        const double stage = fmax(wide ? 4.0 * bn + 60.0 : 0.0, wide ? 260.0 : 520.0);
        const long tiles = tiles_n * ((M + bn - 1) / bn);
        for (int splits = 1; splits <= max_splits && splits <= kb; ++splits) {
            if (!slabs && splits > 1 && (tiles > n_counters || tiles * splits * bn * XBM > partial_floats)) break;
            const long rounds = (tiles * splits + slots - 1) / slots;
            double cost = fmax((double)rounds * ((kb + splits - 1) / splits * stage + 500.0),
                               (double)tiles_n * kb * MX_TILE_BYTES / (23.0 * sms));
            cost += (splits - 1) * (double)M * N * 8.0 / (24.0 * sms) + (splits > 1 && !slabs ? 1500.0 : 0.0);
            if (cost < best_cost * (1.0 - 1e-9)) { best_cost = cost; best = MxPlan{bn, splits, wide}; }
        }
    }
    return best;
}

constexpr long SHARE_FLOATS = 16L << 20;          // most that the shares of one product may take
constexpr int MOST_SPLITS = 16;

int launch_mxfp4(const MxPlan& plan, MxArgs a, const void* X, long lda, int box_rows, long n_units, cudaStream_t stream) {
    a.bn = plan.bn;
    // tensor memory: two accumulators and `ring` stages of decoded weights
    const int tmem = plan.wide ? Form<true>::TMEM : Form<false>::TMEM;
    a.acc_cols = (a.bn + 31) / 32 * 32;
    a.ring = (tmem - 2 * a.acc_cols) / A_COLS < MAX_R ? (tmem - 2 * a.acc_cols) / A_COLS : MAX_R;
    const int room = (plan.wide ? Form<true>::RING : Form<false>::RING) - a.ring * a.bn * 256;
    a.ws = (room / MX_TILE_BYTES < MAX_W ? room / MX_TILE_BYTES : MAX_W) & ~1;
    if (a.ring < 2 || a.ws < a.ring + 2) return fb_fail(-1, "gemm_mxfp4: no room for the stages of %d tokens", a.bn);
    if (n_units > 2000000000L) return fb_fail(-1, "gemm_mxfp4: too many tiles (M=%d N=%d)", a.M, a.N);
    a.n_units = (int)n_units;
    CUtensorMap mx, mo = {};
    int rc = fb_tensor_map_bf16(&mx, X, a.M, a.K, lda, 64, box_rows);
    if (rc) return rc;
    a.boxed = 0;
    if (plan.wide) {
        rc = fb_tensor_map_out(&mo, a.out, a.o_bf16 ? 2 : 4, a.M, a.gate.act ? a.N / 2 : a.N, a.ldo, a.slab_stride > 0 ? a.splits : 1,
                               a.slab_stride, a.gate.act ? XBM / 2 : XBM, OUT_TOKENS);
        if (rc < 0) return rc;
        a.boxed = rc == 0;
    }
    static bool configured[FB_MAX_DEVICES] = {};
    if (fb_needs_setup(configured)) {
        cudaError_t e = cudaFuncSetAttribute(gemm_mxfp4_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Form<false>::SMEM);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(gemm_mxfp4_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Form<true>::SMEM);
        if (e != cudaSuccess) return fb_fail(-2, "gemm_mxfp4: cannot reserve shared memory: %s", cudaGetErrorString(e));
        fb_setup_done(configured);
    }
    const long slots = plan.wide ? fb_sm_count() : 2L * fb_sm_count();
    const int grid = (int)(n_units < slots ? n_units : slots);
    if (plan.wide)
        fb_launch_class(FB_LAUNCH_GEMM_WIDE, gemm_mxfp4_kernel<true>, dim3(grid), dim3(Form<true>::THREADS), Form<true>::SMEM, stream, mx, mo, a);
    else
        fb_launch_class(FB_LAUNCH_OTHER, gemm_mxfp4_kernel<false>, dim3(grid), dim3(Form<false>::THREADS), Form<false>::SMEM, stream, mx, mo, a);
    return fb_check_launch("gemm_mxfp4");
}

int check_operands(const void* X, long long lda, const void* W, const int* shifts, const void* out, int o_dtype, long long ldo, int M, int N,
                   int K, FbGate gate, int plain_act, int* status) {
    FB_REQUIRE(M >= 0 && N > 0 && K > 0, "gemm_mxfp4: bad sizes M=%d N=%d K=%d", M, N, K);
    FB_REQUIRE(o_dtype == FB_F32 || o_dtype == FB_BF16, "gemm_mxfp4: unknown output dtype code %d", o_dtype);
    FB_REQUIRE(!gate.act || (fb_gate_known(gate) && N % 2 == 0 && !plain_act),
               "gemm_mxfp4: a gate needs a known activation, an even number of stacked rows and no plain activation beside it");
    FB_REQUIRE(fb_plain_act_known(plain_act), "gemm_mxfp4: unknown activation code %d", plain_act);
    FB_REQUIRE(lda >= K && ldo >= (gate.act ? N / 2 : N), "gemm_mxfp4: a row stride is shorter than its row");
    FB_REQUIRE(lda % 8 == 0 && ((uintptr_t)X & 15) == 0, "gemm_mxfp4: rows must start on 16-byte borders");
    FB_REQUIRE(W && ((uintptr_t)W & 15) == 0 && shifts && status, "gemm_mxfp4: unaligned weights, or no shifts, or no status word");
    FB_REQUIRE(((uintptr_t)out & (o_dtype == FB_F32 ? 3 : 1)) == 0, "gemm_mxfp4: unaligned output");
    return 0;
}

}  // namespace

// Floats of `partials` that fb_gemm_mxfp4 wants for the same sizes with `n_counters` counters and without slabs: 0 where K is not
// split.
FB_API long long fb_gemm_mxfp4_scratch_floats(int M, int N, int K, int n_counters) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const MxPlan p = plan_mxfp4(M, N, (K + XBK - 1) / XBK, MOST_SPLITS, SHARE_FLOATS, n_counters, false);
    if (p.splits == 1) return 0;
    return (long long)((M + p.bn - 1) / p.bn) * ((N + XBM - 1) / XBM) * p.splits * p.bn * XBM;
}

// X [M,K] bfloat16, W one matrix in tiles with its shift (fb_mxfp4_tiles).  `act` (an FbAct code with its constants): W stacks gate
// and up rows alternately and out[m, c] = act(g_c) u_c has N / 2 columns; `plain_act` (an FbPlainAct code): out = act(product);
// `accumulate` (float32): the product is added to what `out` holds.  Shares of K: with slab_stride > 0 (float32, neither activation
// nor accumulate) share s goes to out + s * slab_stride and *splits_used says how many there are (at most max_slabs); else they
// meet in `partials` and `counters` (zero before the call and after it), the scratch of calls that run one after the other;
// without it, or with fewer floats than fb_gemm_mxfp4_scratch_floats asks for, K is split less or not at all.
FB_API int fb_gemm_mxfp4(const void* X, long long lda, const void* W, const int* shifts, void* out, int o_dtype, long long ldo,
                         long long slab_stride, int max_slabs, int* splits_used, int M, int N, int K, int act, float limit,
                         float slope, int plain_act, int accumulate, float* partials, long long partial_floats, int* counters,
                         int n_counters, int* status, cudaStream_t stream) {
    const FbGate gate = {act, limit, slope};
    if (const int rc = check_operands(X, lda, W, shifts, out, o_dtype, ldo, M, N, K, gate, plain_act, status)) return rc;
    FB_REQUIRE(slab_stride == 0 || (o_dtype == FB_F32 && max_slabs >= 1 && slab_stride >= (long long)M * ldo && !act && !plain_act && !accumulate),
               "gemm_mxfp4: slabs must be float32, at least one, not overlap, and hold plain shares");
    FB_REQUIRE(!accumulate || (o_dtype == FB_F32 && !act && !plain_act), "gemm_mxfp4: only a float32 product can be added to its output");
    if (splits_used) *splits_used = 1;
    if (M == 0) return 0;
    const bool slabs = slab_stride > 0;
    const MxPlan plan = plan_mxfp4(M, N, (K + XBK - 1) / XBK, slabs ? (max_slabs < MOST_SPLITS ? max_slabs : MOST_SPLITS) : MOST_SPLITS,
                                   partials && counters ? partial_floats : 0, counters ? n_counters : 0, slabs);
    MxArgs a = {};
    a.W = (const uint8_t*)W; a.shifts = shifts; a.out = out; a.ldo = (long)ldo; a.slab_stride = (long)slab_stride;
    a.o_bf16 = o_dtype == FB_BF16; a.accumulate = accumulate; a.partials = partials; a.counters = counters;
    a.M = M; a.N = N; a.K = K; a.kb = (K + XBK - 1) / XBK;
    a.tiles_m = (M + plan.bn - 1) / plan.bn; a.tiles_n = (N + XBM - 1) / XBM; a.splits = plan.splits;
    a.gate = gate; a.plain_act = plain_act; a.status = status;
    if (splits_used) *splits_used = slabs ? plan.splits : 1;
    return launch_mxfp4(plan, a, X, (long)lda, plan.bn, (long)a.tiles_m * a.tiles_n * a.splits, stream);
}

// The grouped form: W holds `groups` matrices [N, K] in tiles with a shift each; the M rows of X and `out` come in tiles of `tile`
// (a multiple of 16 up to 128) rows of one group each (tile_group, negative: skipped, its rows of `out` stay as they are).
FB_API int fb_gemm_mxfp4_grouped(const void* X, long long lda, const void* W, const int* shifts, int groups, const int* tile_group,
                                 int tile, void* out, int o_dtype, long long ldo, int M, int N, int K, int act, float limit,
                                 float slope, int plain_act, int* status, cudaStream_t stream) {
    const FbGate gate = {act, limit, slope};
    if (const int rc = check_operands(X, lda, W, shifts, out, o_dtype, ldo, M, N, K, gate, plain_act, status)) return rc;
    FB_REQUIRE(groups > 0 && tile_group, "gemm_mxfp4_grouped: no groups");
    FB_REQUIRE(tile >= 16 && tile <= 128 && tile % 16 == 0 && M % tile == 0 && M / tile < (1 << 24),
               "gemm_mxfp4_grouped: the rows must be whole tiles of 16 to 128, not tiles of %d", tile);
    if (M == 0) return 0;
    MxArgs a = {};
    a.kb = (K + XBK - 1) / XBK;
    a.tiles_n = (N + XBM - 1) / XBM;
    a.W = (const uint8_t*)W; a.w_group = (long)a.tiles_n * a.kb * MX_TILE_BYTES; a.shifts = shifts; a.out = out; a.ldo = (long)ldo;
    a.o_bf16 = o_dtype == FB_BF16; a.M = M; a.N = N; a.K = K; a.tiles_m = 1; a.splits = 1;
    a.gate = gate; a.plain_act = plain_act; a.status = status;
    a.tile_group = tile_group; a.tile = tile; a.n_tiles = M / tile;
    const bool wide = tile > 16;
    const int most = wide ? Form<true>::MOST_TOKENS : Form<false>::MOST_TOKENS;
    return launch_mxfp4(MxPlan{most / tile * tile, 1, wide}, a, X, (long)lda, tile, (long)a.n_tiles * a.tiles_n, stream);
}
