// Shared by the dense products (dense.hip, linear_i8.hip, linear_mxfp4.hip): the order of output
// tiles, the swizzle of K chunks in LDS, and the wait for their stages.
#pragma once

#include "pxs_common.h"

namespace pxs {

// Output tile (row tile, column tile) of logical tile t: groups of g row
// tiles share their column tiles, and inside a group consecutive t walk the
// rows, so the tiles one XCD runs at a time cover g row tiles x (32 / g)
// column tiles of operands instead of one row tile x every column tile.
__device__ __forceinline__ void tile_of(int t, int tiles_m, int tiles_n, int g, int & tm, int & tn) {
    if (g <= 1) {
        tm = t / tiles_n;
        tn = t % tiles_n;
        return;
    }
    const int per_group = g * tiles_n;
    const int grp = t / per_group, in = t % per_group;
    const int rows = min(g, tiles_m - grp * g);  // the last group may be short
    tm = grp * g + in % rows;
    tn = in / rows;
}

// Rows of KB = 128 bytes per K chunk in LDS: 8 pieces of 16 bytes,
// XOR-swizzled by row so that the 16 rows one LDS cycle serves (64 banks of
// 4 bytes) read 16 different bank groups.
template <int KB> __device__ __forceinline__ int piece_swz(int row);
template <> __device__ __forceinline__ int piece_swz<128>(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// Waits until at most min(later, MAX) stages of PER instructions each are in
// flight (s_waitcnt's count is a constant, six bits of it vmcnt).
template <int MAX, int PER>
__device__ __forceinline__ void wait_stages(int later) {
    constexpr int n = MAX * PER;
    static_assert(n < 64, "vmcnt has six bits");
    if constexpr (MAX > 0) {
        if (later < MAX) {
            wait_stages<MAX - 1, PER>(later);
            return;
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70 | (n & 15) | ((n >> 4) << 14));
}

} // namespace pxs
