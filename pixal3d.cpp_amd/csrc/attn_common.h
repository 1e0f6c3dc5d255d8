// Shared by the attention kernels (attention.hip, attention_scores.hip,
// attention_tree.hip): the segment of a tile, the LDS layouts of K and V tiles, and sums and maxima over
// the two lanes that share a query.
#pragma once

#include "pxs_common.h"

namespace pxs {

constexpr float kLog2e = 1.4426950408889634f;

// The segment owning query tile t: the largest s with tile_start[s] <= t
// (tile_start is non-decreasing; empty segments repeat a value).  The wave
// samples 64 evenly spaced entries per round and keeps the last interval whose
// start is <= t, so nseg <= 64 takes one dependent load and nseg <= 4096 two.
__device__ __forceinline__ int find_segment(const int64_t * __restrict__ tile_start, int nseg,
                                            int64_t t, int lane) {
    int lo = 0, len = nseg;
    while (len > 1) {
        const int stride = (len + 63) >> 6;
        const int off = lane * stride;
        const bool le = off < len && tile_start[lo + off] <= t;
        const int cnt = max(1, __popcll(__ballot(le)));  // (0 only where tile_start falls)
        lo += (cnt - 1) * stride;
        len = min(stride, len - (cnt - 1) * stride);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// K and V tile rows of 128 bytes (64 bf16) in LDS, XOR-swizzled in 16-byte
// pieces: kswz for the K fragment reads, vswz for the transposed V reads
// (ds_read_b64_tr_b16), so that neither conflicts on LDS banks.
__device__ __forceinline__ int kswz(int row) { return (row & 7) ^ ((row >> 3) & 1); }
__device__ __forceinline__ int vswz(int row) { return (2 * (row & 3)) ^ ((row >> 2) & 1); }

typedef short v4i16 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float lane_pair_max(float v) {
    // max over lanes l and l ^ 32 (v_permlane32_swap exchanges the halves).
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                     false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

__device__ __forceinline__ float lane_pair_sum(float v) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                     false, false);
    return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

} // namespace pxs
