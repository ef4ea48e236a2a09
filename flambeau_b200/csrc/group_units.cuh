// The units of a grouped product (routed experts): the rows come in tiles that belong to one group each, negative groups are
// skipped, and a unit of tokens is up to `most` neighbouring tiles of one group.  Every CTA lists the units when it starts: one
// warp walks the tiles 32 at a time.  A unit is its first tile and, from bit 24 on, its tiles.
#pragma once

#include "common.cuh"

__device__ __forceinline__ uint32_t group_unit_at(const int* tile_group, int n_tiles, int most, int t) {
    const int g = tile_group[t];
    int c = 1;
    while (c < most && t + c < n_tiles && tile_group[t + c] == g) ++c;
    return (uint32_t)t | (uint32_t)c << 24;
}
// All 32 lanes.  Writes the first LIST units and returns how many there are (most <= 32).  The groups of two stretches of 32 tiles
// are on their way while one is looked at; where the runs of a stretch and of the next begin is a mask of 64 bits.  (With the loads
// of every stretch, and of every unit's eight tiles, waited for where they were wanted, 2,048 tokens on 6 of 64 experts took 8 us
// longer a product of the two-SM kernel, 16,384 on 8 of 512 65.)
template <int LIST>
__device__ __forceinline__ int group_units(const int* tile_group, int n_tiles, int most, uint32_t* list) {
    const int lane = threadIdx.x & 31;
    auto at = [&](int t) { return t < n_tiles ? tile_group[t] : -1; };
    auto begins_of = [&](int g, int before) {
        const int left = __shfl_up_sync(0xffffffffu, g, 1);
        return __ballot_sync(0xffffffffu, g != (lane ? left : before));
    };
    int found = 0, run = 0, g = at(lane), next = at(32 + lane), after = at(64 + lane);      // run: where the one that reaches in began
    uint32_t begins = begins_of(g, -1);
    for (int t0 = 0; t0 < n_tiles; t0 += 32) {
        const int further = at(t0 + 96 + lane);
        const uint32_t begins_next = begins_of(next, __shfl_sync(0xffffffffu, g, 31));
        const uint32_t mine = begins & (0xffffffffu >> (31 - lane));
        const int t = t0 + lane, from = mine ? t0 + 31 - __clz(mine) : run;
        const uint32_t units = __ballot_sync(0xffffffffu, g >= 0 && (t - from) % most == 0);
        const int place = found + __popc(units & ((1u << lane) - 1u));
        const int left = __ffsll((long long)(((unsigned long long)begins_next << 32 | begins) >> (lane + 1)));      // tiles of the run from t on
        if ((units >> lane & 1u) && place < LIST) list[place] = (uint32_t)t | (uint32_t)(left == 0 || left > most ? most : left) << 24;
        found += __popc(units);
        run = __shfl_sync(0xffffffffu, from, 31);
        g = next;
        next = after;
        after = further;
        begins = begins_next;
    }
    return found;
}
// Unit i of the list or, where there are more than it holds, counted on from the last one that this thread asked for: a role asks
// for ascending units, so that it walks the tiles once.  A sort of rows by group makes at most (tiles + (most - 1) groups) / most
// units: with eight tiles a unit 440 hold 3,000 tiles of 64 groups and 1,700 of 256.
struct GroupWalk { int i; uint32_t unit; };
template <int LIST>
__device__ __forceinline__ uint32_t group_unit(const int* tile_group, int n_tiles, int most, const uint32_t* list, int i, GroupWalk& walk) {
    if (i < LIST) return list[i];
    if (walk.i < LIST) walk = GroupWalk{LIST - 1, list[LIST - 1]};
    for (; walk.i < i; ++walk.i) {
        int t = (int)(walk.unit & 0xffffffu) + (int)(walk.unit >> 24);
        while (tile_group[t] < 0) ++t;
        walk.unit = group_unit_at(tile_group, n_tiles, most, t);
    }
    return walk.unit;
}
