// Attention of drafted tokens over a cache: a sequence's tokens form a tree (several
// continuations that share their beginnings), and a token sees the sequence's cached keys, the
// tokens above it in the tree and itself.
//
//   s(i, j) = scale * q_i . k_j                 with a cap: cap * tanh(s / cap)
//   s = s - slope[head] * |p_i - p_j|           with slopes; a cached key's position is its row
//   o_i = sum_seen exp(s) v_j / sum_seen exp(s)
//
// as the scored attention's (attention_scores.hip).  The tokens' keys and values are rows of
// their own, so that the cache is written only with those that are accepted.
//
// A row is a (query, head) of a key/value head's group, 32 rows a tile.  A tile's work is cut
// into chunks of the cached keys, an item each, the tree's keys with the first.  How long the
// caches are only the device knows: every workgroup takes the chunk's size from the lengths
// (segment_plan), so that a call has about `target` items, whatever the lengths, and a captured
// call follows the cache as it grows.  Chunks write maximum, sum and unnormalised output in fp32,
// which a second launch joins in order.
//
// Who is above a token is walked once per row, from the token up, while the tree's keys are
// taken from the last to the first: no mask is stored, whatever the tree's size.  A parent that
// is no earlier token of the tree ends the walk.

#include "attn_common.h"

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

namespace pxs {
namespace {

struct TreeArgs {
    const void * q;
    const void * k;            // the tokens' own
    const void * v;
    int64_t ldq, ldk, ldv;
    const void * kc;           // the cache's
    const void * vc;
    int64_t ldkc, ldvc;
    const int64_t * cu_q;      // [nseg + 1]
    const int32_t * parents;   // [total_q], within the tree
    const int64_t * start;     // [nseg] first cached row
    const int64_t * len;       // [nseg]
    const int32_t * positions; // [total_q] with slopes
    int nseg;
    int64_t total_q, cache_rows;
    const int64_t * table;     // null: at most 64 segments; or tree_table_kernel's
    int heads, kv_heads, group, d;
    float scale_log2, cap_log2, over_cap;
    const float * slopes;      // [heads] or null
    void * o;
    int64_t ldo;
    int vec;                   // rows of q, k and v in whole 16-byte pieces
    int64_t items;             // launched (bound)
    int64_t slots;             // items with partial results (bound)
    double per_target;         // 1 / items that the chunks add at most
    float * part;              // [slots * kv_heads * kTreeRows][d] unnormalised outputs
    float2 * part_ml;          // [..] maxima (log2 units) and sums
};

constexpr int kTreeRows = 32;
constexpr int kTreeUnit = 128;  // keys that a chunk is a multiple of

// A segment's queries and cached rows, kept within the call's whatever the bounds hold.
struct Tree {
    int q0, nq, nk;
    int64_t k0;
};
__device__ __forceinline__ Tree load_tree(const TreeArgs & a, int s) {
    auto within = [](int64_t v, int64_t lo, int64_t hi) { return max(min(v, hi), lo); };
    const int64_t q0 = within(a.cu_q[s], 0, a.total_q), q1 = within(a.cu_q[s + 1], q0, a.total_q);
    const int64_t k0 = within(a.start[s], 0, a.cache_rows), nk = within(a.len[s], 0, a.cache_rows - k0);
    return {static_cast<int>(q0), static_cast<int>(q1 - q0), static_cast<int>(nk), k0};
}

__device__ __forceinline__ int row_tiles_of(const TreeArgs & a, const Tree & g) {
    return static_cast<int>((static_cast<int64_t>(g.nq) * a.group + kTreeRows - 1) / kTreeRows);
}
// Keys of a chunk, from the sum of row tiles times cached keys: `work` of them over the
// target's items, and one unit more, so that the chunks past a tile's first are at most the target.
__device__ __forceinline__ int chunk_of(const TreeArgs & a, double work) {
    const double units = floor(work * a.per_target * (1.0 / kTreeUnit)) + 1.0;
    return static_cast<int>(min(units * kTreeUnit, static_cast<double>(a.cache_rows + kTreeUnit)));
}
__device__ __forceinline__ int chunks_of(const Tree & g, int chunk) { return g.nk > chunk ? (g.nk - 1) / chunk + 1 : 1; }

// An item: a row tile and the chunk's keys.
struct Item {
    Tree g;
    int kv;
    int row0, rows;       // first row of the tile; rows of the segment
    int key0, key1;       // cached keys
    int chunk, chunks;
    int slot;             // of the item's partial results, where there are more chunks than one
};

__device__ __forceinline__ int tree_sums(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int below = __shfl_up(v, d, 64);
        if (lane >= d) v += below;
    }
    return v;
}

// Of up to 64 segments, one a lane: its bounds, its items and those up to it, the same of
// items with partial results, and the chunk.
struct Plan {
    Tree g;
    int items, end, slots, slots_end, chunk;
};
__device__ __forceinline__ Plan segment_plan(const TreeArgs & a, int lane) {
    Plan p{};
    if (lane < a.nseg) p.g = load_tree(a, lane);
    const int tiles = row_tiles_of(a, p.g);
    double work = static_cast<double>(tiles) * p.g.nk;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) work += __shfl_xor(work, d, 64);
    p.chunk = __builtin_amdgcn_readfirstlane(chunk_of(a, work));
    p.items = tiles * chunks_of(p.g, p.chunk);
    p.end = tree_sums(p.items, lane);
    p.slots = p.items > tiles ? p.items : 0;
    p.slots_end = tree_sums(p.slots, lane);
    return p;
}
__device__ __forceinline__ Tree tree_of(const Tree & g, int from) {
    const int lo = __builtin_amdgcn_readlane(static_cast<int>(g.k0), from);
    return {__builtin_amdgcn_readlane(g.q0, from), __builtin_amdgcn_readlane(g.nq, from), __builtin_amdgcn_readlane(g.nk, from),
            static_cast<int64_t>(static_cast<uint32_t>(lo))};
}

// Item i of a segment whose partial results start at slot0: the row tiles of a chunk next to one
// another, so that an XCD reads it once.
__device__ __forceinline__ bool item_of(const TreeArgs & a, const Tree & g, int i, int chunk, int slot0, Item & w) {
    const int tiles = row_tiles_of(a, g);
    if (tiles == 0 || i < 0) return false;
    w.g = g;
    w.rows = g.nq * a.group;
    w.chunks = chunks_of(g, chunk);
    w.chunk = i / tiles;
    w.row0 = i % tiles * kTreeRows;
    w.key0 = static_cast<int>(min(static_cast<int64_t>(w.chunk) * chunk, static_cast<int64_t>(g.nk)));
    w.key1 = static_cast<int>(min(static_cast<int64_t>(w.key0) + chunk, static_cast<int64_t>(g.nk)));
    w.slot = slot0 + i;
    return w.chunk < w.chunks && (w.chunks == 1 || (w.slot >= 0 && w.slot < a.slots));
}

// Item t; false past the last.
__device__ __forceinline__ bool locate_item(const TreeArgs & a, int t, int lane, Item & w) {
    if (a.table) {
        if (t >= a.table[a.nseg]) return false;
        const int seg = __builtin_amdgcn_readfirstlane(find_segment(a.table, a.nseg, t, lane));
        return item_of(a, load_tree(a, seg), __builtin_amdgcn_readfirstlane(static_cast<int>(t - a.table[seg])),
                       __builtin_amdgcn_readfirstlane(static_cast<int>(a.table[a.nseg + 1])),
                       __builtin_amdgcn_readfirstlane(static_cast<int>(a.table[a.nseg + 2 + seg])), w);
    }
    const Plan p = segment_plan(a, lane);
    const int seg = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < a.nseg && p.end <= t)));
    if (seg >= a.nseg) return false;
    return item_of(a, tree_of(p.g, seg), t - __builtin_amdgcn_readlane(p.end - p.items, seg), p.chunk,
                   __builtin_amdgcn_readlane(p.slots_end - p.slots, seg), w);
}

// Query qi of the call: its segment's first item; false for a row of no segment.
__device__ __forceinline__ bool locate_query(const TreeArgs & a, int qi, int lane, Item & w) {
    if (a.table) {
        if (qi < a.cu_q[0] || qi >= a.cu_q[a.nseg]) return false;
        const int seg = __builtin_amdgcn_readfirstlane(find_segment(a.cu_q, a.nseg, qi, lane));
        const Tree g = load_tree(a, seg);
        if (qi < g.q0 || qi >= g.q0 + g.nq) return false;  // (bounds that fall)
        return item_of(a, g, 0, static_cast<int>(a.table[a.nseg + 1]), static_cast<int>(a.table[a.nseg + 2 + seg]), w);
    }
    const Plan p = segment_plan(a, lane);
    const uint64_t mine = __ballot(lane < a.nseg && qi >= p.g.q0 && qi < p.g.q0 + p.g.nq);
    if (mine == 0) return false;
    const int seg = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(mine)) - 1);
    return item_of(a, tree_of(p.g, seg), 0, p.chunk, __builtin_amdgcn_readlane(p.slots_end - p.slots, seg), w);
}

// The token above token c of the tree whose first row is q0; -1 at the top.
__device__ __forceinline__ int above(const TreeArgs & a, int q0, int c) {
    const int p = a.parents[q0 + c];
    return p >= 0 && p < c ? p : -1;
}

// A score in log2 units, from a product q . k and the distance of the positions.
__device__ __forceinline__ float tree_score(const TreeArgs & a, float dot, float slope_log2, float away) {
    float z = dot * a.scale_log2;
    if (a.cap_log2 > 0.0f) z = a.cap_log2 * tanhf(dot * a.over_cap);
    return z - slope_log2 * fabsf(away);
}

// Four dims of a row from c, zeros past d.
template <typename T>
__device__ __forceinline__ void load_dims4(const T * row, int c, int d, bool vec, float (&out)[4]) {
    if (vec && c + 4 <= d) {
        T e[4];
        __builtin_memcpy(e, __builtin_assume_aligned(row + c, 4 * sizeof(T)), sizeof(e));
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = load_f32(e + i);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = c + i < d ? load_f32(row + c + i) : 0.0f;
}

__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// A row of an item again, a key after the other, tokens that it does not see left out altogether: for
// trees where a token's value is infinite or NaN, which times a weight of zero is NaN.  One wave;
// lane l holds dims l, l + 64, ...  Broken data alone comes here.
template <typename T, int NC>
__device__ __forceinline__ void tree_row_alone(const TreeArgs & a, const Item & w, int row, int lane, int64_t slot) {
    const int i = row / a.group;
    const int head = w.kv * a.group + row % a.group;
    const T * q = static_cast<const T *>(a.q) + (w.g.q0 + i) * a.ldq + static_cast<int64_t>(head) * a.d;
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    const int pos = a.slopes ? a.positions[w.g.q0 + i] : 0;
    float qv[NC], acc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        qv[c] = lane + 64 * c < a.d ? load_f32(q + lane + 64 * c) : 0.0f;
        acc[c] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    auto step = [&](const T * k, const T * v, int at) {
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < a.d) dot += qv[c] * load_f32(k + lane + 64 * c);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) dot += __shfl_xor(dot, off, 64);
        const float z = tree_score(a, dot, slope, static_cast<float>(pos - at));
        const float up = fmaxf(m, z);
        const float base = up == -INFINITY ? 0.0f : up;
        const float p = exp2f(z - base), keep = exp2f(m - base);
        l = l * keep + p;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < a.d) acc[c] = acc[c] * keep + p * load_f32(v + lane + 64 * c);
        m = up;
    };
    const int64_t col = static_cast<int64_t>(w.kv) * a.d;
    if (w.chunk == 0)
        for (int c = i; c >= 0; c = above(a, w.g.q0, c))
            step(static_cast<const T *>(a.k) + (w.g.q0 + c) * a.ldk + col, static_cast<const T *>(a.v) + (w.g.q0 + c) * a.ldv + col,
                 a.slopes ? a.positions[w.g.q0 + c] : 0);
    for (int j = w.key0; j < w.key1; ++j)
        step(static_cast<const T *>(a.kc) + (w.g.k0 + j) * a.ldkc + col, static_cast<const T *>(a.vc) + (w.g.k0 + j) * a.ldvc + col, j);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN sum stays NaN)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int dim = lane + 64 * c;
        if (dim >= a.d) continue;
        if (w.chunks > 1) a.part[slot * a.d + dim] = acc[c];
        else store_f32(static_cast<T *>(a.o) + (w.g.q0 + i) * a.ldo + static_cast<int64_t>(head) * a.d + dim, acc[c] * inv);
    }
    if (w.chunks > 1 && lane == 0) a.part_ml[slot] = make_float2(m, l);
}

// Any type, head size up to DP, stride and alignment, in fp32 on v_mfma_f32_32x32x2_f32.  The four
// waves of a workgroup have the same 32 rows and every fourth block of 32 keys each, straight from
// memory; S^T = K Q^T, so that a lane owns one row and half of its scores, and O^T += V^T P^T.
// Their results are joined through LDS.
template <typename T, int DP>
__global__ void __launch_bounds__(256) tree_attn_any_kernel(TreeArgs a) {
    constexpr int DT = DP / 32;
    extern __shared__ __align__(16) float tree_smem[];  // [4][32][DP] outputs, [4][32] maxima and sums
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;
    Item w;
    w.kv = static_cast<int>(blockIdx.x % a.kv_heads);
    if (!locate_item(a, static_cast<int>(blockIdx.x / a.kv_heads), lane, w)) return;

    const bool live = w.row0 + r < w.rows;
    const int row = live ? w.row0 + r : w.rows - 1;
    const int qi = row / a.group, head = w.kv * a.group + row % a.group;
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    const int pos = a.slopes ? a.positions[w.g.q0 + qi] : 0;
    const int64_t col = static_cast<int64_t>(w.kv) * a.d;
    const T * q = static_cast<const T *>(a.q) + (w.g.q0 + qi) * a.ldq + static_cast<int64_t>(head) * a.d;
    float qv[DP / 2];  // dims h DP/2 .. h DP/2 + DP/2 - 1
#pragma unroll
    for (int u = 0; u < DP / 8; ++u) {
        float f[4];
        load_dims4<T>(q, h * (DP / 2) + 4 * u, a.d, a.vec, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) qv[4 * u + e] = f[e];
    }
    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    bool odd = false;
    int walk = qi;  // the next of the row's tokens, from itself up

    const int tree_blocks = w.chunk == 0 ? (w.g.nq + 31) / 32 : 0;
    const int all = tree_blocks + (w.key1 - w.key0 + 31) / 32;
    for (int b = wave; b < all; b += 4) {
        const bool tree = b < tree_blocks;
        const int first = tree ? (tree_blocks - 1 - b) * 32 : w.key0 + (b - tree_blocks) * 32;
        const int limit = (tree ? w.g.nq : w.key1) - first;  // keys of the block, 32 or more: all
        const int64_t ldk = tree ? a.ldk : a.ldkc, ldv = tree ? a.ldv : a.ldvc;
        const int64_t at = (tree ? w.g.q0 : w.g.k0) + first;
        const T * k = static_cast<const T *>(tree ? a.k : a.kc) + at * ldk + col;
        const T * v = static_cast<const T *>(tree ? a.v : a.vc) + at * ldv + col;
        uint32_t seen = limit >= 32 ? ~0u : (1u << limit) - 1u;
        if (tree) {
            seen = 0;
            while (walk >= first + 32) walk = above(a, w.g.q0, walk);
            for (; walk >= first; walk = above(a, w.g.q0, walk)) seen |= 1u << (walk - first);
        }
        f32x16 s = {};
        const T * krow = k + min(r, limit - 1) * ldk;
#pragma unroll
        for (int u = 0; u < DP / 8; ++u) {
            float f[4];
            load_dims4<T>(krow, h * (DP / 2) + 4 * u, a.d, a.vec, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(f[e], qv[4 * u + e], s, 0, 0, 0);
        }
        // Register e holds key 8 (e / 4) + 4 h + e % 4 of the block.
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int key = 8 * (e >> 2) + 4 * h + (e & 3);
            float away = 0.0f;
            if (a.slopes) away = static_cast<float>(pos - (tree ? a.positions[w.g.q0 + first + min(key, limit - 1)] : first + key));
            const float z = tree_score(a, s[e], slope, away);
            s[e] = seen >> key & 1u ? z : -INFINITY;
            top = fmaxf(top, s[e]);
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = fmaxf(m, top);
        const float base = up == -INFINITY ? 0.0f : up;  // nothing seen yet: every weight is 0
        const float keep = exp2f(m - base);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = exp2f(s[e] - base);
            sum += s[e];
        }
        sum += __shfl_xor(sum, 32, 64);
        l = l * keep + sum;
        m = up;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[dt][e] *= keep;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int key = 8 * (e >> 2) + 4 * h + (e & 3);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const float x = key < limit && dt * 32 + r < a.d ? load_f32(v + key * ldv + dt * 32 + r) : 0.0f;
                odd |= tree && !finite(x);
                oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[e], oacc[dt], 0, 0, 0);
            }
        }
    }
    const int64_t slot0 = (static_cast<int64_t>(w.slot) * a.kv_heads + w.kv) * kTreeRows;
    if (__syncthreads_or(odd)) {
        for (int i = wave; i < kTreeRows; i += 4)
            if (w.row0 + i < w.rows) tree_row_alone<T, (DP + 63) / 64>(a, w, w.row0 + i, lane, slot0 + i);
        return;
    }
    float2 * ml = reinterpret_cast<float2 *>(tree_smem + 4 * 32 * DP);
    if (h == 0) ml[wave * 32 + r] = make_float2(m, l);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4 *>(tree_smem + (wave * 32 + r) * DP + dt * 32 + 8 * g + 4 * h) =
                make_float4(oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]);
    __syncthreads();
    const int jr = tid >> 3;  // 8 threads a row
    if (w.row0 + jr >= w.rows) return;
    float base = -INFINITY, total = 0.0f, f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) base = fmaxf(base, ml[i * 32 + jr].x);
    const float ref = base == -INFINITY ? 0.0f : base;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = exp2f(ml[i * 32 + jr].x - ref);
        total += ml[i * 32 + jr].y * f[i];
    }
    const int to = (w.row0 + jr) / a.group, to_head = w.kv * a.group + (w.row0 + jr) % a.group;
    T * o = static_cast<T *>(a.o) + (w.g.q0 + to) * a.ldo + static_cast<int64_t>(to_head) * a.d;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (w.chunks > 1 && (tid & 7) == 0) a.part_ml[slot0 + jr] = make_float2(base, total);
    for (int c = tid & 7; c < a.d; c += 8) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) x += tree_smem[(i * 32 + jr) * DP + c] * f[i];
        if (w.chunks > 1) a.part[(slot0 + jr) * a.d + c] = x;
        else store_f32(o + c, x * inv);
    }
}

// Joins the chunks of a (query, head): eight groups of 32 lanes, each every eighth chunk, then
// their results in order.
template <typename T>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a) {
    constexpr int kGroups = 8, kMost = 8;  // head sizes up to 32 kMost
    __shared__ float2 ml[kGroups];
    __shared__ float acc_of[kGroups][32 * kMost];
    const int lane = threadIdx.x & 63, l32 = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int qi = static_cast<int>(blockIdx.x / a.heads);
    const int head = static_cast<int>(blockIdx.x % a.heads);
    Item w;
    w.kv = head / a.group;
    if (!locate_query(a, qi, lane, w) || w.chunks <= 1) return;
    const int tiles = row_tiles_of(a, w.g), row = (qi - w.g.q0) * a.group + head % a.group;
    if (w.slot + static_cast<int64_t>(tiles) * w.chunks > a.slots) return;  // (of bounds that fall: no such items)
    const int64_t at = ((w.slot + row / kTreeRows) * static_cast<int64_t>(a.kv_heads) + w.kv) * kTreeRows + row % kTreeRows;
    const int64_t step = static_cast<int64_t>(tiles) * a.kv_heads * kTreeRows;
    float m = -INFINITY, l = 0.0f, acc[kMost];
#pragma unroll
    for (int c = 0; c < kMost; ++c) acc[c] = 0.0f;
    for (int i = grp; i < w.chunks; i += kGroups) {
        const float2 p = a.part_ml[at + i * step];
        const float up = fmaxf(m, p.x), ref = up == -INFINITY ? 0.0f : up;
        const float keep = exp2f(m - ref), f = exp2f(p.x - ref);
        l = l * keep + p.y * f;
#pragma unroll
        for (int c = 0; c < kMost; ++c) {
            const float o = l32 + 32 * c < a.d ? a.part[(at + i * step) * a.d + l32 + 32 * c] : 0.0f;
            acc[c] = acc[c] * keep + o * f;
        }
        m = up;
    }
    if (l32 == 0) ml[grp] = make_float2(m, l);
#pragma unroll
    for (int c = 0; c < kMost; ++c) acc_of[grp][l32 + 32 * c] = acc[c];
    __syncthreads();
    const int dim = threadIdx.x;
    if (dim >= a.d) return;
    float base = -INFINITY, total = 0.0f, v = 0.0f;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) base = fmaxf(base, ml[i].x);
    const float ref = base == -INFINITY ? 0.0f : base;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const float f = exp2f(ml[i].x - ref);
        total += ml[i].y * f;
        v += acc_of[i][dim] * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    store_f32(static_cast<T *>(a.o) + qi * a.ldo + static_cast<int64_t>(head) * a.d + dim, v * inv);
}

// For more segments than a wave's lanes: items before each segment [nseg], all of them, the chunk,
// and items with partial results before each segment [nseg].
__global__ void __launch_bounds__(1024) tree_table_kernel(TreeArgs a, int64_t * __restrict__ table) {
    __shared__ double works[16];
    __shared__ int64_t waves[2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double work = 0.0;
    for (int s = tid; s < a.nseg; s += 1024) {
        const Tree g = load_tree(a, s);
        work += static_cast<double>(row_tiles_of(a, g)) * g.nk;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) work += __shfl_xor(work, d, 64);
    if (lane == 0) works[wave] = work;
    __syncthreads();
    work = 0.0;
    for (int i = 0; i < 16; ++i) work += works[i];
    const int chunk = chunk_of(a, work);
    int64_t before[2] = {0, 0};
    for (int s0 = 0; s0 < a.nseg; s0 += 1024) {
        const int s = s0 + tid;
        int64_t count[2] = {0, 0}, sum[2], ahead[2];
        if (s < a.nseg) {
            const Tree g = load_tree(a, s);
            const int64_t tiles = row_tiles_of(a, g);
            count[0] = tiles * chunks_of(g, chunk);
            count[1] = count[0] > tiles ? count[0] : 0;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            sum[c] = count[c];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int64_t below = __shfl_up(sum[c], d, 64);
                if (lane >= d) sum[c] += below;
            }
            if (lane == 63) waves[c][wave] = sum[c];
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            ahead[c] = before[c] + sum[c] - count[c];
            for (int i = 0; i < 16; ++i) {
                if (i < wave) ahead[c] += waves[c][i];
                before[c] += waves[c][i];
            }
        }
        if (s < a.nseg) {
            table[s] = ahead[0];
            table[a.nseg + 2 + s] = min(ahead[1], a.slots);
        }
        __syncthreads();
    }
    if (tid == 0) {
        table[a.nseg] = min(before[0], static_cast<int64_t>(INT32_MAX));
        table[a.nseg + 1] = chunk;
    }
}

// ---- host -----------------------------------------------------------------------

constexpr int kTreeMaxDim = 256;
constexpr int64_t kTreeMaxRows = INT32_MAX - 1023;  // rows and keys are counted in 32 bits, a tile past their end
constexpr int kWaveSegments = 64;
constexpr int64_t kTreeItems = 1024;  // workgroups that chunks past the first add at most

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int64_t tree_target(int kv_heads) { return std::max<int64_t>(1, kTreeItems / kv_heads); }
// Items a key/value head has at most: its row tiles, and the target of chunks past their first.
int64_t tree_items(int nseg, int64_t total_q, int kv_heads, int group) {
    return total_q * group / kTreeRows + nseg + tree_target(kv_heads);
}
// Those with partial results: a segment of len keys in more chunks than one has at most 2 len / chunk.
int64_t tree_slots(int kv_heads) { return 2 * tree_target(kv_heads); }
size_t tree_table_bytes(int nseg) { return round256((2 * static_cast<size_t>(nseg) + 2) * sizeof(int64_t)); }
size_t tree_part_rows(int kv_heads) { return static_cast<size_t>(tree_slots(kv_heads)) * kv_heads * kTreeRows; }

template <typename T, int DP>
int launch_tree_any(const TreeArgs & a, hipStream_t s) {
    constexpr int smem = 4 * 32 * DP * 4 + 4 * 32 * 8;
    auto kernel = &tree_attn_any_kernel<T, DP>;
    if constexpr (smem > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), smem, done, "hipFuncSetAttribute(tree_attn)")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.items * a.kv_heads)), dim3(256), smem, s, a);
    return check_launch("tree attention");
}

template <typename T>
int run_tree(const TreeArgs & a, hipStream_t s) {
    int rc = a.d <= 64 ? launch_tree_any<T, 64>(a, s) : a.d <= 128 ? launch_tree_any<T, 128>(a, s) : launch_tree_any<T, 256>(a, s);
    if (rc || a.cache_rows <= kTreeUnit) return rc;  // (no chunk is shorter than a unit)
    hipLaunchKernelGGL(tree_join_kernel<T>, dim3(static_cast<unsigned>(a.total_q * a.heads)), dim3(256), 0, s, a);
    return check_launch("tree attention join");
}

bool whole_pieces(const void * p, int64_t ld, int d, int elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * elem % 16 == 0 && d * elem % 16 == 0;
}

} // namespace
} // namespace pxs

using namespace pxs;

extern "C" {

size_t pxs_tree_attention_workspace_bytes(int nseg, int64_t total_q, int heads, int kv_heads, int head_dim) {
    if (nseg <= 0 || total_q <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 256;
    const size_t rows = tree_part_rows(kv_heads);
    return tree_table_bytes(nseg) + round256(rows * sizeof(float2)) + round256(rows * head_dim * sizeof(float));
}

int pxs_tree_attention(int dtype, const void * q, int64_t ld_q, const void * k, int64_t ld_k, const void * v, int64_t ld_v,
                       const int64_t * cu_q, const int32_t * parents, const void * k_cache, int64_t ld_k_cache,
                       const void * v_cache, int64_t ld_v_cache, const int64_t * cache_start, const int64_t * cache_len,
                       int nseg, int64_t total_q, int64_t cache_rows, int heads, int kv_heads, int head_dim, float scale,
                       float cap, const float * slopes, const int32_t * positions, void * o, int64_t ld_o, void * workspace,
                       void * stream) {
    PXS_CHECK_WORKSPACE(workspace, "pxs_tree_attention");
    PXS_CHECK(dtype == PXS_F32 || dtype == PXS_BF16, PXS_ERR_ARG, "pxs_tree_attention: bad dtype");
    PXS_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 65535, PXS_ERR_ARG,
              "pxs_tree_attention: heads must be a multiple of kv_heads, up to 65535");
    PXS_CHECK(head_dim > 0 && head_dim <= kTreeMaxDim, PXS_ERR_ARG, "pxs_tree_attention: head_dim must be in 1..256");
    PXS_CHECK(scale > 0.0f && std::isfinite(scale), PXS_ERR_ARG, "pxs_tree_attention: scale must be finite and positive");
    PXS_CHECK(cap >= 0.0f && std::isfinite(cap), PXS_ERR_ARG, "pxs_tree_attention: cap must be finite, and 0 for none");
    PXS_CHECK(std::isfinite(scale * kLog2e) && (cap == 0.0f || std::isfinite(scale / cap)), PXS_ERR_ARG,
              "pxs_tree_attention: scale and cap out of range");
    PXS_CHECK(!slopes || positions, PXS_ERR_ARG, "pxs_tree_attention: slopes need the tokens' positions");
    PXS_CHECK(nseg >= 0 && total_q >= 0 && cache_rows >= 0 && total_q <= kTreeMaxRows / (heads / kv_heads) &&
                  cache_rows <= kTreeMaxRows,
              PXS_ERR_ARG, "pxs_tree_attention: row counts must be in 0..2^31 - 1024, as total_q * heads / kv_heads");
    const int64_t wq = static_cast<int64_t>(heads) * head_dim, wk = static_cast<int64_t>(kv_heads) * head_dim;
    PXS_CHECK(ld_q >= wq && ld_k >= wk && ld_v >= wk && ld_o >= wq && (cache_rows == 0 || (ld_k_cache >= wk && ld_v_cache >= wk)),
              PXS_ERR_ARG, "pxs_tree_attention: row stride smaller than heads * head_dim");
    if (nseg == 0 || total_q == 0) return PXS_OK;
    PXS_CHECK(q && k && v && o && cu_q && parents && cache_start && cache_len && workspace &&
                  (cache_rows == 0 || (k_cache && v_cache)),
              PXS_ERR_ARG, "pxs_tree_attention: null pointer");
    hipStream_t s = as_stream(stream);
    TreeArgs a{};
    a.q = q; a.k = k; a.v = v; a.ldq = ld_q; a.ldk = ld_k; a.ldv = ld_v;
    a.kc = k_cache; a.vc = v_cache; a.ldkc = ld_k_cache; a.ldvc = ld_v_cache;
    a.cu_q = cu_q; a.parents = parents; a.start = cache_start; a.len = cache_len; a.positions = positions;
    a.nseg = nseg; a.total_q = total_q; a.cache_rows = cache_rows;
    a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.d = head_dim;
    // (Caps that cap nothing fp32 holds are taken lower, so that scale / cap stays a normal number.)
    cap = std::min({cap, std::numeric_limits<float>::max() / 4, scale * 0x1p126f});
    a.scale_log2 = scale * kLog2e;
    a.cap_log2 = cap * kLog2e;
    a.over_cap = cap > 0.0f ? scale / cap : 0.0f;
    a.slopes = slopes; a.o = o; a.ldo = ld_o;
    const int elem = dtype == PXS_BF16 ? 2 : 4;
    a.vec = whole_pieces(q, ld_q, head_dim, elem) && whole_pieces(k, ld_k, head_dim, elem) &&
            whole_pieces(v, ld_v, head_dim, elem) &&
            (cache_rows == 0 || (whole_pieces(k_cache, ld_k_cache, head_dim, elem) && whole_pieces(v_cache, ld_v_cache, head_dim, elem)));
    a.items = tree_items(nseg, total_q, kv_heads, a.group);
    a.slots = tree_slots(kv_heads);
    a.per_target = 1.0 / static_cast<double>(tree_target(kv_heads));
    PXS_CHECK(a.items * kv_heads <= UINT32_MAX / 256 && total_q * heads <= UINT32_MAX / 256, PXS_ERR_ARG,
              "pxs_tree_attention: grid too large");
    char * ws = static_cast<char *>(workspace);
    if (nseg > kWaveSegments) {
        a.table = reinterpret_cast<int64_t *>(ws);
        hipLaunchKernelGGL(tree_table_kernel, dim3(1), dim3(1024), 0, s, a, reinterpret_cast<int64_t *>(ws));
        if (int rc = check_launch("tree attention table")) return rc;
    }
    ws += tree_table_bytes(nseg);
    const size_t rows = tree_part_rows(kv_heads);
    a.part_ml = reinterpret_cast<float2 *>(ws);
    a.part = reinterpret_cast<float *>(ws + round256(rows * sizeof(float2)));
    return dtype == PXS_F32 ? run_tree<float>(a, s) : run_tree<uint16_t>(a, s);
}

} // extern "C"
