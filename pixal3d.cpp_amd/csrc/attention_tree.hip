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
// A row is a (query, head) of a key/value head's group, 32 or 128 rows a tile.  A tile's work is cut
// into chunks of the cached keys, an item each, the tree's keys with the first.  How long the
// caches are only the device knows: every workgroup takes the chunk's size from the lengths
// (segment_plan), so that a call has about `target` items, whatever the lengths, and a captured
// call follows the cache as it grows.  Chunks write maximum, sum and unnormalised output in fp32,
// which a second launch joins in order.
//
// Who is above a token is walked once per row, from the token up, while the tree's keys are
// taken from the last to the first: no mask is stored, whatever the tree's size.  A parent that
// is no earlier token of the tree ends the walk.

#include "attn_scores.h"

#include <algorithm>
#include <cmath>
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
    float scale_log2, cap_log2, over_cap, exp_mul;
    const float * slopes;      // [heads] or null
    void * o;
    int64_t ldo;
    int vec;                   // rows of q, k and v in whole 16-byte pieces
    int64_t items;             // launched (bound)
    int64_t slots;             // items with partial results (bound)
    float per_target;          // 1 / (items that the chunks add at most * 2 kTreeUnit)
    int row_shift;             // log2 of a tile's rows
    int slot_rows;             // those that one of the call's can have
    float * part;              // [slots * kv_heads * slot_rows][d] unnormalised outputs
    float2 * part_ml;          // [..] maxima (log2 units) and sums
};

constexpr int kTreeUnit = 64;  // keys that a chunk starts at a multiple of, a tile's

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

__host__ __device__ __forceinline__ int row_tiles_of(const TreeArgs & a, const Tree & g) {
    return static_cast<int>((static_cast<int64_t>(g.nq) * a.group + (1 << a.row_shift) - 1) >> a.row_shift);
}
// Keys of a chunk, from the sum of row tiles times cached keys: `work` of them over the target's items, and
// so much more that the chunks past a tile's first are at most the target: to the next multiple of two units (of
// one: eight caches of 0 to 40,001 keys 126 us, 92 so), or one unit where that is enough (12 tokens over 1,501
// keys 13.7 us, with two 14.3; one over 300 12.0 and 13.1).
// (Rounded sums of it: they are the same in every wave, and off by so little that the target, at most 512, holds.)
__host__ __device__ __forceinline__ int chunk_of(const TreeArgs & a, float work) {
    const float pairs = floorf(work * a.per_target) + 1.0f, most = static_cast<float>(a.cache_rows / (2 * kTreeUnit) + 1);
    return work * a.per_target <= 0.5f ? kTreeUnit : static_cast<int>(fminf(pairs, most)) * (2 * kTreeUnit);
}
__host__ __device__ __forceinline__ int chunks_of(const Tree & g, int chunk) { return g.nk > chunk ? (g.nk - 1) / chunk + 1 : 1; }
// First key of chunk i of a segment's: as even as whole units make them, where the first chunk has the tree's too.
__host__ __device__ __forceinline__ int chunk_start(const Tree & g, int i, int chunks) {
    if (i == 0) return 0;
    const int cached = static_cast<int>((static_cast<int64_t>(g.nk) + kTreeUnit - 1) / kTreeUnit);
    const int tree = min((g.nq - 1) / kTreeUnit + 1, cached / chunks);  // (no chunk but the first is left without keys)
    const int units = cached + tree, each = units / chunks, more = units - each * chunks;  // (the first `more` have one more)
    return static_cast<int>(min(static_cast<int64_t>(i * each + min(i, more) - tree) * kTreeUnit, static_cast<int64_t>(g.nk)));
}

// The fast kernel's steps for an item, a tile of `keys` keys each: the tree's tiles (with the first chunk), all of
// them, and those that take a maximum: the tree's, the cache's last where it ends inside, and one whole tile.
struct TreeSteps {
    int tree, all, exact;
};
__host__ __device__ __forceinline__ TreeSteps tree_steps(int nq, int chunk, int key0, int key1, int keys) {
    const int tree = chunk == 0 ? (nq + keys - 1) / keys : 0, all = tree + (key1 + keys - 1) / keys - key0 / keys;
    return {tree, all, std::min(all, tree + (key1 % keys != 0 ? 1 : 0) + 1)};
}

// An item: a row tile and the chunk's keys.
struct Item {
    Tree g;
    int kv;
    int row0, rows;       // first row of the tile; rows of the segment
    int key0, key1;       // cached keys
    int chunk, chunks;
    int slot;             // of the item's partial results, where there are more chunks than one
};

// v summed over the lanes up to each, through the lanes' own paths (a shuffle through LDS takes ten times as long).
template <typename V> __device__ __forceinline__ V tree_sums(V v) {
    auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value,
                                                               0xF, false));
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});  // from 1, 2, 4, 8 lanes below in a row of 16
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // the last of row 0 to row 1, of 2 to 3
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // lane 31 to rows 2 and 3
    return v;
}

// Of up to 64 segments, one a lane: its bounds, its items and those up to it, the same of
// items with partial results, and the chunk.  The attention's kernels and the joins' each make it and need the
// same: a product and an addition of the sum are two roundings, and no compiler's choice of one fused.
struct Plan {
    Tree g;
    int items, end, slots, slots_end, chunk;
};
__device__ __forceinline__ Plan segment_plan(const TreeArgs & a, int lane) {
#pragma clang fp contract(off)
    Plan p{};
    if (lane < a.nseg) p.g = load_tree(a, lane);
    const int tiles = row_tiles_of(a, p.g);
    const float work = tree_sums(static_cast<float>(tiles) * static_cast<float>(p.g.nk));
    p.chunk = chunk_of(a, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, work), 63)));
    p.items = tiles * chunks_of(p.g, p.chunk);
    p.end = tree_sums(p.items);
    p.slots = p.items > tiles ? p.items : 0;
    p.slots_end = tree_sums(p.slots);
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
    w.row0 = i % tiles << a.row_shift;
    w.key0 = chunk_start(g, w.chunk, w.chunks);
    w.key1 = chunk_start(g, w.chunk + 1, w.chunks);
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

// The item's rows of partial results.
__device__ __forceinline__ int64_t item_rows(const TreeArgs & a, const Item & w) {
    return (static_cast<int64_t>(w.slot) * a.kv_heads + w.kv) * a.slot_rows;
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

// Outputs are sums of weights up to 1 times values until the last division, and a mean of values below the largest
// number may be a sum above it.  So sums past kTreeOutLimit (512 chunks' of those below it are joined inside fp32)
// are taken again with weights that are lower by this power of two: all keys' together are then at most 1/2.
constexpr float kTreeOutLimit = 0x1p117f;
__device__ __forceinline__ float tree_lift(const Tree & g) {
    return static_cast<float>(33 - __clz(static_cast<int>(static_cast<uint32_t>(g.nk) + static_cast<uint32_t>(g.nq))));
}

// A row of an item again, a key after the other, tokens that it does not see left out altogether: for
// trees where a token's value is infinite or NaN, which times a weight of zero is NaN, and for sums past
// kTreeOutLimit.  One wave; lane l holds dims l, l + 64, ...  Broken or enormous data alone comes here.
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
    const float lift = tree_lift(w.g);
    float m = -INFINITY, l = 0.0f;
    auto step = [&](const T * k, const T * v, int at) {
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < a.d) dot += qv[c] * load_f32(k + lane + 64 * c);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) dot += __shfl_xor(dot, off, 64);
        const float z = tree_score(a, dot, slope, static_cast<float>(pos - at));
        const float up = fmaxf(m, z + lift);
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

// A row's walk up the tree, a tile of tokens at a time from the last: `at` is the next token that the lane's row
// sees, `done` the first token of the tile before.  A tile's parents are loaded by its lanes together, and the
// steps of the walk go through them and not to memory.
struct TreeWalk {
    int at, done;
};
// The tokens first .. first + KEYS - 1 that the row sees, as bits; tiles between `done` and those are passed.
template <int KEYS>
__device__ __forceinline__ uint64_t tree_bits(const TreeArgs & a, const Tree & g, TreeWalk & walk, int first, int lane) {
    static_assert(KEYS <= 64, "a lane a token");
    uint64_t bits = 0;
    while (walk.done > first) {
        walk.done -= KEYS;
        const int from = walk.done;
        const int up = a.parents[g.q0 + min(from + (lane & (KEYS - 1)), g.nq - 1)];
        while (__ballot(walk.at >= from)) {
            const bool here = walk.at >= from;
            const int k = here ? walk.at - from : 0;
            if (here) bits |= uint64_t(1) << k;
            const int next = __shfl(up, k, 64);
            if (here) walk.at = next >= 0 && next < walk.at ? next : -1;
        }
        if (from > first) bits = 0;
    }
    return bits;
}
// The first `seen` keys of a tile, as bits.
__device__ __forceinline__ uint64_t first_bits(int seen) { return seen >= 64 ? ~uint64_t(0) : (uint64_t(1) << seen) - 1; }

// How heads lie in memory: anywhere, in whole 16-byte pieces, or as such of DP values.
enum { kAnyRows, kPieceRows, kWholeRows };
// A row's floats in LDS: four more than its values, which spreads 32 rows' pieces over the banks.
constexpr int tree_any_pitch(int dp) { return dp + 4; }

// Any type, head size up to DP, stride and alignment, in fp32 on v_mfma_f32_32x32x2_f32.  The four
// waves of a workgroup have the same 32 rows and every fourth block of 32 keys each, straight from
// memory; S^T = K Q^T, so that a lane owns one row and half of its scores, and O^T += V^T P^T.
// Their results are joined through LDS.  The products bound it where rows are many (32,000 keys for 128 tokens of 16
// heads of 64 in 42 us, 3.1 TB/s; a block of 32 keys is 1.75 us of a wave's products), the way from the
// lengths to the first loads, and the joins, where they are few (37 and 100 tokens over 2,370 and 517 keys 26 us).
// Where the registers hold them, a block's keys and values are loaded while the block before is multiplied;
// otherwise q is in LDS and keys and values come a piece ahead of the products.
template <typename T, int DP, int FORM>
__global__ void __launch_bounds__(256) tree_attn_any_kernel(TreeArgs a) {
    constexpr int DT = DP / 32;
    constexpr bool kAhead = DP <= (FORM == kAnyRows ? 64 : 128);
    constexpr int P = tree_any_pitch(DP);
    extern __shared__ __align__(16) float tree_smem[];  // [4][32][P] outputs, [4][32] maxima and sums
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;
    Item w;
    w.kv = static_cast<int>(blockIdx.x % a.kv_heads);
    if (!locate_item(a, static_cast<int>(blockIdx.x / a.kv_heads), lane, w)) return;

    const bool live = w.row0 + r < w.rows;
    const int row = live ? w.row0 + r : w.rows - 1;
    const int qi = row / a.group, head = w.kv * a.group + row % a.group;
    const RowScore rs = row_score<kCap | kFar>(a, head);
    const bool capped = a.cap_log2 > 0.0f;
    const float slope = a.slopes ? -kLog2e * a.slopes[head] : 0.0f;
    const int pos = a.slopes ? a.positions[w.g.q0 + qi] : 0;
    const int64_t col = static_cast<int64_t>(w.kv) * a.d;

    const int tree_blocks = w.chunk == 0 ? (w.g.nq + 31) / 32 : 0;
    const int all = tree_blocks + (w.key1 - w.key0 + 31) / 32;
    struct Block {
        bool tree;
        int first, limit;  // its first key, and the keys there are from it on (32 or more: all of it)
    };
    auto block = [&](int b) {
        Block o;
        o.tree = b < tree_blocks;
        o.first = o.tree ? (tree_blocks - 1 - b) * 32 : w.key0 + (b - tree_blocks) * 32;
        o.limit = (o.tree ? w.g.nq : w.key1) - o.first;
        return o;
    };
    // Dims h DP/2 + at .. of a row, N of them; zeros past d
    auto load_part = [&](const T * p, int at, auto & out) __attribute__((always_inline)) {
        constexpr int N = sizeof(out) / sizeof(float);
        if constexpr (FORM != kAnyRows) {
            constexpr int V = 16 / static_cast<int>(sizeof(T));
#pragma unroll
            for (int u = 0; u < N / V; ++u) {
                const int dim = h * (DP / 2) + at + V * u;
                T e[V];
                __builtin_memcpy(e, __builtin_assume_aligned(p + (FORM == kWholeRows ? dim : min(dim, a.d - V)), 16), 16);
#pragma unroll
                for (int i = 0; i < V; ++i) out[V * u + i] = FORM == kWholeRows || dim < a.d ? load_f32(e + i) : 0.0f;
            }
        } else {
            int d = a.d;
            asm volatile("" : "+s"(d));  // (the comparisons stay here: kept over the loop they cost more registers than there are)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int dim = h * (DP / 2) + at + i;
                const float x = load_f32(p + min(dim, d - 1));
                out[i] = dim < d ? x : 0.0f;
            }
        }
    };
    auto load_k = [&](const Block & o, int at, auto & kk) __attribute__((always_inline)) {
        const int key = o.first + min(r, o.limit - 1);
        load_part(o.tree ? static_cast<const T *>(a.k) + static_cast<int64_t>(w.g.q0 + key) * a.ldk + col
                         : static_cast<const T *>(a.kc) + (w.g.k0 + key) * a.ldkc + col, at, kk);
    };
    // Register e of dims dt: key 8 (e / 4) + 4 h + e % 4 of the block, dim 32 dt + r.  (Those of dims past d
    // make outputs that are not stored.)
    auto load_v = [&](const Block & o, int from, auto & vv) __attribute__((always_inline)) {
        constexpr int N = sizeof(vv) / sizeof(vv[0]);
        const int64_t ldv = o.tree ? a.ldv : a.ldvc;
        const T * v = (o.tree ? static_cast<const T *>(a.v) + static_cast<int64_t>(w.g.q0 + o.first) * ldv
                              : static_cast<const T *>(a.vc) + (w.g.k0 + o.first) * ldv) + col;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int key = 8 * ((from + e) >> 2) + 4 * h + (e & 3);
            const T * p = v + min(key, o.limit - 1) * ldv;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) vv[e][dt] = load_f32(p + (FORM == kWholeRows ? dt * 32 + r : min(dt * 32 + r, a.d - 1)));
        }
    };
    constexpr int KN = kAhead ? DP / 2 : 32, KP = DP / 2 / KN, VN = kAhead ? 16 : 16 / static_cast<int>(sizeof(T)), VP = 16 / VN;
    float kk[2][KN], vv[2][VN][DT];
    const T * qrow = static_cast<const T *>(a.q) + (w.g.q0 + qi) * a.ldq + static_cast<int64_t>(head) * a.d;
    if (wave < all) {
        load_k(block(wave), 0, kk[0]);
        if (kAhead) load_v(block(wave), 0, vv[0]);
    }
    float qv[KN];
    float * qs = tree_smem + r * P + h * (DP / 2);
    if (kAhead) {
        load_part(qrow, 0, qv);
    } else {
        for (int u = wave; u < KP; u += 4) {
            load_part(qrow, KN * u, qv);
#pragma unroll
            for (int i = 0; i < KN; i += 4) *reinterpret_cast<float4 *>(qs + KN * u + i) = make_float4(qv[i], qv[i + 1], qv[i + 2], qv[i + 3]);
        }
        __syncthreads();
    }
    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    bool odd = false;
    TreeWalk walk{qi, tree_blocks * 32};
    for (int b = wave; b < all; b += 4) {
        const Block o = block(b);
        const uint32_t seen = o.tree ? static_cast<uint32_t>(tree_bits<32>(a, w.g, walk, o.first, lane))
                                     : static_cast<uint32_t>(first_bits(min(o.limit, 32)));
        f32x16 s = {};
#pragma unroll
        for (int u = 0; u < KP; ++u) {
            if (!kAhead) {
                if (u + 1 < KP) load_k(o, KN * (u + 1), kk[(u + 1) & 1]);
                else load_v(o, 0, vv[0]);
#pragma unroll
                for (int i = 0; i < KN; i += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(qs + KN * u + i);
                    qv[i] = x.x, qv[i + 1] = x.y, qv[i + 2] = x.z, qv[i + 3] = x.w;
                }
                asm volatile("" ::: "memory");  // (keeps the pieces' loads from being moved to one place)
            }
#pragma unroll
            for (int i = 0; i < KN; ++i) s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk[u & 1][i], qv[i], s, 0, 0, 0);
        }
        if (b + 4 < all) load_k(block(b + 4), 0, kk[0]);
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int key = 8 * (e >> 2) + 4 * h + (e & 3);
            float z = capped ? score_of<kCap | kFar>(rs, s[e], 0.0f, 0.0f) : s[e] * a.scale_log2;
            if (a.slopes) {
                const int at = o.tree ? a.positions[w.g.q0 + o.first + min(key, o.limit - 1)] : o.first + key;
                z = __builtin_fmaf(slope, fabsf(static_cast<float>(pos - at)), z);
            }
            s[e] = seen >> key & 1u ? z : -INFINITY;
            top = fmaxf(top, s[e]);
        }
        const float up = fmaxf(m, lane_pair_max(top));
        const float base = up == -INFINITY ? 0.0f : up;  // nothing seen yet: every weight is 0
        const float keep = __builtin_amdgcn_exp2f(m - base);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e] - base);
            sum += s[e];
        }
        l = l * keep + lane_pair_sum(sum);
        m = up;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[dt][e] *= keep;
#pragma unroll
        for (int u = 0; u < VP; ++u) {
            if (u + 1 < VP) {
                load_v(o, VN * (u + 1), vv[(u + 1) & 1]);
                asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int e = VN * u; e < VN * (u + 1); ++e) {
                const bool in = 8 * (e >> 2) + 4 * h + (e & 3) < o.limit;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const float x = in ? vv[u & 1][e - VN * u][dt] : 0.0f;
                    odd |= o.tree && !is_finite_bits(x);
                    oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[e], oacc[dt], 0, 0, 0);
                }
            }
        }
        if (kAhead && b + 4 < all) load_v(block(b + 4), 0, vv[0]);
    }
    const int64_t slot0 = item_rows(a, w);
    if (!kAhead) __syncthreads();  // (q's place is the outputs')
    float2 * ml = reinterpret_cast<float2 *>(tree_smem + 4 * 32 * P);
    int again = lane;
    asm volatile("" : "+v"(again));  // (h and r taken anew: kept over the loop they cost more registers than there are)
    const int to_h = again >> 5, to_r = again & 31;
    if (to_h == 0) ml[wave * 32 + to_r] = make_float2(m, l);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4 *>(tree_smem + (wave * 32 + to_r) * P + dt * 32 + 8 * g + 4 * to_h) =
                make_float4(oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]);
    __syncthreads();
    const int jr = tid >> 3;  // 8 threads a row
    float base = -INFINITY, total = 0.0f, f[4], x[DP / 8];
#pragma unroll
    for (int i = 0; i < 4; ++i) base = fmaxf(base, ml[i * 32 + jr].x);
    const float ref = base == -INFINITY ? 0.0f : base;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = exp2f(ml[i * 32 + jr].x - ref);
        total += ml[i * 32 + jr].y * f[i];
    }
    bool past = false;
#pragma unroll
    for (int u = 0; u < DP / 8; ++u) {
        x[u] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u] += tree_smem[(i * 32 + jr) * P + u * 8 + (tid & 7)] * f[i];
        past |= !(fabsf(x[u]) < kTreeOutLimit);  // (a row of no query repeats the last, dims past d its last one's)
    }
    if (__builtin_expect(__syncthreads_or(odd || (past && is_finite_bits(total))), 0)) {
        for (int i = wave; i < 32; i += 4)
            if (w.row0 + i < w.rows) tree_row_alone<T, (DP + 63) / 64>(a, w, w.row0 + i, lane, slot0 + i);
        return;
    }
    if (w.row0 + jr >= w.rows) return;
    const int to = (w.row0 + jr) / a.group, to_head = w.kv * a.group + (w.row0 + jr) % a.group;
    T * o = static_cast<T *>(a.o) + (w.g.q0 + to) * a.ldo + static_cast<int64_t>(to_head) * a.d;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (w.chunks > 1 && (tid & 7) == 0) a.part_ml[slot0 + jr] = make_float2(base, total);
#pragma unroll
    for (int u = 0; u < DP / 8; ++u) {
        const int c = u * 8 + (tid & 7);
        if (c >= a.d) continue;
        if (w.chunks > 1) a.part[(slot0 + jr) * a.d + c] = x[u];
        else store_f32(o + c, x[u] * inv);
    }
}

// ---- bf16, head sizes of whole 16-byte pieces up to 128 -----------------------------------------------------
// The tiles, products and weights of the scored attention's kernels (attn_scores.h).  An item's tiles are walked as
// the tree's from the last to the first, each with the keys that a row sees as bits, then the cache's.

// One row's place: its query, head, constants and first fragments.
template <int DH, int MODE> struct TreeRow {
    RowScore rs;
    bf16x8 qf[Fast<DH>::NST];
    int row, qi, head, pos;
    bool live;
};
template <int DH, int MODE>
__device__ __forceinline__ void load_row(const TreeArgs & a, const Item & w, int row, int h, TreeRow<DH, MODE> & o) {
    o.live = row < w.rows;
    o.row = o.live ? row : w.rows - 1;
    o.qi = o.row / a.group;
    o.head = w.kv * a.group + o.row % a.group;
    o.rs = row_score<MODE>(a, o.head);
    o.pos = MODE & kBias ? a.positions[w.g.q0 + o.qi] : 0;
    load_q_row<DH>(static_cast<const uint16_t *>(a.q) + (w.g.q0 + o.qi) * a.ldq + static_cast<int64_t>(o.head) * a.d, a.d, o.live, h,
                   o.qf);
}

template <int DH> struct TreeSources {
    TileSource<DH> tree, cache;
};
template <int DH>
__device__ __forceinline__ TreeSources<DH> tree_sources(const TreeArgs & a, const Item & w) {
    const int64_t col = static_cast<int64_t>(w.kv) * a.d;
    const int64_t q0 = w.g.q0;
    return {tile_source_of<DH>(static_cast<const uint16_t *>(a.k) + q0 * a.ldk + col,
                               static_cast<const uint16_t *>(a.v) + q0 * a.ldv + col, a.ldk, a.ldv, w.g.nq),
            tile_source_of<DH>(static_cast<const uint16_t *>(a.kc) + w.g.k0 * a.ldkc + col,
                               static_cast<const uint16_t *>(a.vc) + w.g.k0 * a.ldvc + col, a.ldkc, a.ldvc, w.key1)};
}

// The exact step of a tile of the tree (its first token) or of the cache (its first key), whose keys the row
// sees as bits.
template <int DH, int MODE>
__device__ __forceinline__ void tree_exact(const TreeArgs & a, const Item & w, const TreeRow<DH, MODE> & o, bool tree, int first,
                                           uint64_t bits, int h, typename Fast<DH>::Scores & s, typename Fast<DH>::Weights & p,
                                           typename Fast<DH>::Out & oacc, RowState & st, float lift) {
    const uint32_t lo = static_cast<uint32_t>(bits) >> (4 * h), hi = static_cast<uint32_t>(bits >> 32) >> (4 * h);
    auto seen = [&](int kt, int e) __attribute__((always_inline)) {  // (key_of is a constant)
        return ((kt == 0 ? lo : hi) >> (key_of(0, e)) & 1u) != 0;
    };
    const float behind = static_cast<float>(o.pos - first - 4 * h);
    if ((MODE & kBias) && tree) {
        float at[Fast<DH>::KT][16];
#pragma unroll
        for (int kt = 0; kt < Fast<DH>::KT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                at[kt][e] = static_cast<float>(o.pos - a.positions[w.g.q0 + min(first + key_of(kt, e) + 4 * h, w.g.nq - 1)]);
        tile_exact_of<DH, MODE>(o.rs, a.cap_log2, s, p, oacc, st,
                                [&](int kt, int e) __attribute__((always_inline)) { return at[kt][e]; }, seen, lift);
    } else {
        tile_exact_of<DH, MODE>(o.rs, a.cap_log2, s, p, oacc, st,
                                [&](int kt, int e) __attribute__((always_inline)) { return behind - static_cast<float>(key_of(kt, e)); },
                                seen, lift);
    }
}

// Four waves of 32 rows share the key tiles, a ring of four slots of K and V, as the scored attention's kernel of many
// rows does.  The tree's tiles and the cache's last, which may end inside, are exact steps
// (maximum, weights, product), and one whole tile after them, so that every row has a base that one of its own
// scores set.  From there on a step issues the products that do not depend on its weights, O += V P of the tile before
// and S of the next, and takes its weights while they run, without a maximum: a row's are redone with one
// where their sum passes 2^40, and an item whose outputs pass kTreeOutLimit is walked again with exact steps alone.
// Waves past the segment's rows only help to load: with one row or 32 the cache's bytes bound it (eight caches of
// 32,768 keys, one token each, 5.2 TB/s; two waves a workgroup with a ring of their own were 2 to 9% slower from
// one row to 64), with 256 a segment the products and the weights' exponentials (620 TFLOP/s, 515 with a cap).
template <int DH, int MODE, bool WHOLE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) tree_attn_rows_kernel(TreeArgs a) {
    using F = Fast<DH>;
    constexpr int kMine = 2 * F::kUnits / 4;  // DMA instructions of a wave and tile
    __shared__ __align__(16) char lds[kSlots * 2 * F::kTileBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;
    Item w;
    w.kv = static_cast<int>(blockIdx.x % a.kv_heads);
    if (!locate_item(a, static_cast<int>(blockIdx.x / a.kv_heads), lane, w)) return;
    const TreeSteps steps = tree_steps(w.g.nq, w.chunk, w.key0, w.key1, F::kKeys);
    const int tree_tiles = steps.tree, cache1 = (w.key1 + F::kKeys - 1) / F::kKeys;
    // Steps 0 .. n - 1: the tree's tiles from the last, then the cache's from the last.
    const int n = __builtin_amdgcn_readfirstlane(steps.all);
    const int exact = __builtin_amdgcn_readfirstlane(steps.exact);
    const int wave_row0 = w.row0 + wave * 32;
    const bool wave_live = wave_row0 < w.rows;

    TreeSources<DH> src = tree_sources<DH>(a, w);
    uint32_t off_tree[kMine], off_cache[kMine];
    tile_offsets<DH>(src.tree, a.d, wave * kMine, lane, off_tree);
    tile_offsets<DH>(src.cache, a.d, wave * kMine, lane, off_cache);
    const uint32_t lds0 = lds_offset(&lds[0]);
    auto slot = [](int i) { return (i % kSlots) * 2 * F::kTileBytes; };
    auto cache_tile = [&](int i) { return cache1 - 1 - (i - tree_tiles); };
    auto issue = [&](int i) __attribute__((always_inline)) {
        if (i < tree_tiles) tile_issue<DH, WHOLE>(src.tree, tree_tiles - 1 - i, wave * kMine, off_tree, lds0 + slot(i), lane);
        else tile_issue<DH, WHOLE>(src.cache, cache_tile(i), wave * kMine, off_cache, lds0 + slot(i), lane);
    };
    auto issue_cache = [&](int i) __attribute__((always_inline)) {
        tile_issue<DH, WHOLE>(src.cache, cache_tile(i), wave * kMine, off_cache, lds0 + slot(i), lane);
    };
    auto k_of = [&](int i) { return lds + slot(i); };
    auto v_of = [&](int i) { return lds + slot(i) + F::kTileBytes; };
    issue(0);  // (an item has a tile: its segment's tokens, or keys)
    if (n > 1) issue(1);
    // (The steps' order of waits, barriers and loads is the same for all waves.)
    auto await = [&](int i, bool more) __attribute__((always_inline)) {
        if (more && i + 1 < n) wait_vmcnt(kMine);
        else wait_vmcnt(0);
        barrier_no_fence();
    };
    TreeRow<DH, MODE> o;
    load_row<DH, MODE>(a, w, wave_row0 + r, h, o);
    const float cap_log2 = a.cap_log2;
    auto behind = [&](int i) { return static_cast<float>(o.pos - 4 * h - cache_tile(i) * F::kKeys); };
    typename F::Out oacc;
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt) oacc[dt] = f32x16{};
    RowState st{-INFINITY, 0.0f};
    bool odd = false, past = false;
    typename F::Scores s_a, s_b;
    typename F::Weights p;
    int i = 0;
    TreeWalk walk{o.qi, tree_tiles * F::kKeys};
    auto exact_step = [&](float lift) __attribute__((always_inline)) {
        const bool tree = i < tree_tiles;
        const int first = (tree ? tree_tiles - 1 - i : cache_tile(i)) * F::kKeys;
        const uint64_t bits = tree ? tree_bits<F::kKeys>(a, w.g, walk, first, lane) : first_bits(w.key1 - first);
        await(i, true);
        if (i + 2 < n) issue(i + 2);
        if (tree) odd |= tile_odd<DH>(v_of(i), tid, 256);
        if (wave_live) {
            tile_qk<DH>(k_of(i), o.qf, s_a, h, r);
            tree_exact<DH, MODE>(a, w, o, tree, first, bits, h, s_a, p, oacc, st, lift);
            tile_pv<DH>(v_of(i), p, oacc, lane);
        }
    };
    for (; i < exact; ++i) exact_step(-0.0f);
    i = __builtin_amdgcn_readfirstlane(i);
    if (!wave_live) {
        for (; i < n; ++i) {
            await(i, i == exact);
            if (i > exact && i + 1 < n) issue_cache(i + 1);
        }
    } else if (i < n) {
        auto weights = [&](int i, typename F::Scores & s) __attribute__((always_inline)) {
            float sum = tile_weights<DH, MODE>(o.rs, cap_log2, s, p, st.base, behind(i));
            if (__builtin_expect(__ballot(!(sum <= kSumLimit)) != 0, 0)) {
                const float top = fmaxf(st.base, tile_max<DH, MODE>(o.rs, cap_log2, s, behind(i)));
                const float up = top == -INFINITY ? 0.0f : top;  // scores of minus infinity, or NaN, only
                const float keep = __builtin_amdgcn_exp2f(st.base - up);
                st.base = up;
                st.sum *= keep;
#pragma unroll
                for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[dt][e] *= keep;
                sum = tile_weights<DH, MODE>(o.rs, cap_log2, s, p, st.base, behind(i));
            }
            st.sum += sum;
        };
        await(i, true);
        tile_qk<DH>(k_of(i), o.qf, s_a, h, r);
        // The first: no product before it.
        if (i + 1 < n) {
            await(i + 1, false);
            if (i + 2 < n) issue_cache(i + 2);
            tile_qk<DH>(k_of(i + 1), o.qf, s_b, h, r);
        }
        weights(i, s_a);
        ++i;
        auto step = [&](typename F::Scores & now, typename F::Scores & next) __attribute__((always_inline)) {
            await(i + 1, false);
            if (i + 2 < n) issue_cache(i + 2);
            tile_pv<DH>(v_of(i - 1), p, oacc, lane);
            tile_qk<DH>(k_of(i + 1), o.qf, next, h, r);
            weights(i, now);
            ++i;
        };
        while (i + 2 < n) {
            step(s_b, s_a);
            step(s_a, s_b);
        }
        if (i + 1 < n) {
            step(s_b, s_a);
#pragma unroll
            for (int kt = 0; kt < F::KT; ++kt) s_b[kt] = s_a[kt];
        }
        tile_pv<DH>(v_of(i - 1), p, oacc, lane);
        if (i < n) {
            weights(i, s_b);
            tile_pv<DH>(v_of(i), p, oacc, lane);
        }
    }
    // (A sum of magnitudes: infinities and NaN stay in it.)
    float size[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) size[e & 3] += fabsf(oacc[dt][e]);
    past = o.live && !((size[0] + size[1]) + (size[2] + size[3]) < kTreeOutLimit) && is_finite_bits(st.sum);
    const int64_t part = item_rows(a, w) + wave * 32;
    if (__builtin_expect(__syncthreads_or(odd || past), 0)) {
        if (__syncthreads_or(odd)) {
            for (int j = 0; j < 32; ++j)
                if (wave_row0 + j < w.rows) tree_row_alone<uint16_t, DH / 64>(a, w, wave_row0 + j, lane, part + j);
            return;
        }
        issue(0);  // (every wave is done with the slots)
        if (n > 1) issue(1);
#pragma unroll
        for (int dt = 0; dt < F::NDT; ++dt) oacc[dt] = f32x16{};
        st = {-INFINITY, 0.0f};
        walk = {o.qi, tree_tiles * F::kKeys};
        const float lift = tree_lift(w.g);
        for (i = 0; i < n; ++i) exact_step(lift);
    }
    const float sum = lane_pair_sum(st.sum);
    if (!o.live) return;
    if (w.chunks > 1) {
        if (h == 0) a.part_ml[part + r] = make_float2(st.base, sum);
        float * to = a.part + (part + r) * a.d;
#pragma unroll
        for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (WHOLE || dt * 32 + 8 * g + 4 * h < a.d)
                    *reinterpret_cast<float4 *>(to + dt * 32 + 8 * g + 4 * h) =
                        make_float4(oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]);
        return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t * to = static_cast<uint16_t *>(a.o) + (w.g.q0 + o.qi) * a.ldo + static_cast<int64_t>(o.head) * a.d;
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (WHOLE || dt * 32 + 8 * g + 4 * h < a.d)
                *reinterpret_cast<uint2 *>(to + dt * 32 + 8 * g + 4 * h) =
                    make_uint2(pack_bf16x2(oacc[dt][4 * g] * inv, oacc[dt][4 * g + 1] * inv),
                               pack_bf16x2(oacc[dt][4 * g + 2] * inv, oacc[dt][4 * g + 3] * inv));
}

// Joins the chunks of (query, head) rows, in their order; 32 lanes a row and chunk, four dims a lane.
// kRowsEach: a workgroup's eight groups of lanes have a row each, of eight heads of a query; otherwise they share one
// row, each every eighth chunk, and their results are joined through LDS.  The first for calls of kJoinRows rows
// and more, whose chunks are few.
template <typename T, bool kRowsEach>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a) {
    constexpr int kGroups = 8, kParts = 2;  // head sizes up to 128 kParts
    __shared__ float2 ml[kGroups];
    __shared__ __align__(16) float acc_of[kRowsEach ? 1 : kGroups][128 * kParts];
    const int lane = threadIdx.x & 63, l32 = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int per = kRowsEach ? (a.heads + kGroups - 1) / kGroups : a.heads;
    const int qi = static_cast<int>(blockIdx.x / per);
    int head = static_cast<int>(blockIdx.x % per);
    Item w;
    w.kv = 0;
    if (!locate_query(a, qi, lane, w) || w.chunks <= 1) return;
    if (kRowsEach) {
        head = head * kGroups + grp;
        if (head >= a.heads) return;
    }
    w.kv = head / a.group;
    const int tiles = row_tiles_of(a, w.g), row = (qi - w.g.q0) * a.group + head % a.group;
    if (w.slot + static_cast<int64_t>(tiles) * w.chunks > a.slots) return;  // (of bounds that fall: no such items)
    w.slot += row >> a.row_shift;
    const int64_t at = item_rows(a, w) + (row & ((1 << a.row_shift) - 1));
    const int64_t step = static_cast<int64_t>(tiles) * a.kv_heads * a.slot_rows;
    const bool whole = (a.d & 3) == 0;
    float m = -INFINITY, l = 0.0f, acc[kParts][4] = {};
#pragma unroll 4
    for (int i = kRowsEach ? 0 : grp; i < w.chunks; i += kRowsEach ? 1 : kGroups) {
        const float2 p = a.part_ml[at + i * step];
        float o[kParts][4];
#pragma unroll
        for (int c = 0; c < kParts; ++c) load_dims4<float>(a.part + (at + i * step) * a.d, 128 * c + 4 * l32, a.d, whole, o[c]);
        const float up = fmaxf(m, p.x), ref = up == -INFINITY ? 0.0f : up;
        const float keep = __builtin_amdgcn_exp2f(m - ref), f = __builtin_amdgcn_exp2f(p.x - ref);
        l = l * keep + p.y * f;
#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][e] = acc[c][e] * keep + o[c][e] * f;
        m = up;
    }
    T * to = static_cast<T *>(a.o) + qi * a.ldo + static_cast<int64_t>(head) * a.d;
    if constexpr (kRowsEach) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < kParts; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (128 * c + 4 * l32 + e < a.d) store_f32(to + 128 * c + 4 * l32 + e, acc[c][e] * inv);
        return;
    }
    if (l32 == 0) ml[grp] = make_float2(m, l);
#pragma unroll
    for (int c = 0; c < kParts; ++c)
        *reinterpret_cast<float4 *>(&acc_of[kRowsEach ? 0 : grp][128 * c + 4 * l32]) = make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]);
    __syncthreads();
    const int dim = threadIdx.x;
    if (dim >= a.d) return;
    float base = -INFINITY, total = 0.0f, v = 0.0f;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) base = fmaxf(base, ml[i].x);
    const float ref = base == -INFINITY ? 0.0f : base;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const float f = __builtin_amdgcn_exp2f(ml[i].x - ref);
        total += ml[i].y * f;
        v += acc_of[kRowsEach ? 0 : i][dim] * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    store_f32(to + dim, v * inv);
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
    const int chunk = chunk_of(a, static_cast<float>(work));
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
// (query, head) rows from which a group of lanes joins one alone: many rows have few chunks each.  16,384 rows of 4
// chunks 110 us with the attention, a workgroup a row 125; 4,096 of 8 68 and 71; 192 of 12 17.7 and 15.0; 1,024 of
// 64 55 and 49.
constexpr int64_t kJoinRows = 4096;
bool joins_rows_each(int64_t total_q, int heads) { return total_q * heads >= kJoinRows; }
// Workgroups of the join; none where no chunk is shorter than the cache.
int64_t join_groups(const TreeArgs & a) {
    if (a.cache_rows <= kTreeUnit) return 0;
    return a.total_q * (joins_rows_each(a.total_q, a.heads) ? (a.heads + 7) / 8 : a.heads);
}
// Workgroups that chunks past the first add at most: one round of the kernels' two a CU (eight trees of 64 over
// 8,192 keys 112 us, with 384 119, with 768 133, with 1,024 126; eight trees over caches of 0 to 40,001 keys 93, 97,
// 106 and 100; 64 of 8 over 4,096 198, 198, 220 and 221; in fp32 eight of 16 over 4,000 51, 57, 63 and 58).
constexpr int64_t kTreeItems = 512;

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int64_t tree_target(int kv_heads) { return std::max<int64_t>(1, kTreeItems / kv_heads); }
// Items a key/value head has at most: its row tiles, and the target of chunks past their first.
int64_t tree_items(int nseg, int64_t total_q, int kv_heads, int group, int row_shift) {
    return (total_q * group >> row_shift) + nseg + tree_target(kv_heads);
}
// Those with partial results: a segment of len keys in more chunks than one has at most 2 len / chunk.
int64_t tree_slots(int kv_heads) { return 2 * tree_target(kv_heads); }
size_t tree_table_bytes(int nseg) { return round256((2 * static_cast<size_t>(nseg) + 2) * sizeof(int64_t)); }
int tree_slot_rows(int64_t rows, int row_shift) { return static_cast<int>(std::min<int64_t>(rows, int64_t(1) << row_shift)); }
size_t tree_part_rows(int kv_heads, int slot_rows) { return static_cast<size_t>(tree_slots(kv_heads)) * kv_heads * slot_rows; }

void set_tree_cuts(TreeArgs & a, bool fast) {
    a.row_shift = fast ? 7 : 5;
    a.per_target = 1.0f / static_cast<float>(tree_target(a.kv_heads) * 2 * kTreeUnit);
}

template <typename T, int DP, int FORM>
int launch_tree_any(const TreeArgs & a, hipStream_t s) {
    constexpr int smem = 4 * 32 * tree_any_pitch(DP) * 4 + 4 * 32 * 8;
    auto kernel = &tree_attn_any_kernel<T, DP, FORM>;
    if constexpr (smem > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), smem, done, "hipFuncSetAttribute(tree_attn)")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.items * a.kv_heads)), dim3(256), smem, s, a);
    return check_launch("tree attention");
}

template <typename T, int FORM>
int launch_tree_any(const TreeArgs & a, hipStream_t s) {
    return a.d <= 64    ? launch_tree_any<T, 64, FORM>(a, s)
           : a.d <= 128 ? launch_tree_any<T, 128, FORM>(a, s)
                        : launch_tree_any<T, 256, FORM>(a, s);
}

// kernel<mode of the call>
template <typename F> int with_tree_mode(const TreeArgs & a, F && launch) {
    auto capped = [&](auto rest) {
        constexpr int kRest = decltype(rest)::value;
        if (a.cap_log2 == 0.0f) return launch(rest);
        if (a.cap_log2 <= kNearCap * kLog2e) return launch(std::integral_constant<int, kCap | kRest>{});
        return launch(std::integral_constant<int, kCap | kFar | kRest>{});
    };
    if (a.slopes) return capped(std::integral_constant<int, kBias>{});
    return capped(std::integral_constant<int, 0>{});
}

template <int DH, bool WHOLE>
int launch_tree_fast(const TreeArgs & a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.items * a.kv_heads));
    return with_tree_mode(a, [&](auto mode) {
        constexpr int kMode = decltype(mode)::value;
        hipLaunchKernelGGL((tree_attn_rows_kernel<DH, kMode, WHOLE>), grid, dim3(256), 0, s, a);
        return check_launch("tree attention");
    });
}

template <typename T>
int run_tree(const TreeArgs & a, bool fast, hipStream_t s) {
    int rc;
    if (fast && a.d == 64) rc = launch_tree_fast<64, true>(a, s);
    else if (fast && a.d == 128) rc = launch_tree_fast<128, true>(a, s);
    else if (fast) rc = a.d < 64 ? launch_tree_fast<64, false>(a, s) : launch_tree_fast<128, false>(a, s);
    else if (a.vec && (a.d == 64 || a.d == 128 || a.d == 256)) rc = launch_tree_any<T, kWholeRows>(a, s);
    else rc = a.vec ? launch_tree_any<T, kPieceRows>(a, s) : launch_tree_any<T, kAnyRows>(a, s);
    const dim3 groups(static_cast<unsigned>(join_groups(a)));
    if (rc || groups.x == 0) return rc;
    if (joins_rows_each(a.total_q, a.heads)) hipLaunchKernelGGL((tree_join_kernel<T, true>), groups, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((tree_join_kernel<T, false>), groups, dim3(256), 0, s, a);
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
    const int64_t group = (heads - 1) / kv_heads + 1;
    const size_t rows = tree_part_rows(kv_heads, tree_slot_rows(std::min<int64_t>(total_q, 128) * group, 7));  // (fp32's are fewer)
    return tree_table_bytes(nseg) + round256(rows * sizeof(float2)) + round256(rows * head_dim * sizeof(float));
}

int pxs_tree_attention_plan(int dtype, const int64_t * q_len, const int64_t * cache_len, int nseg, int64_t cache_rows,
                            int heads, int kv_heads, int head_dim, int * plan) {
    PXS_CHECK(dtype == PXS_F32 || dtype == PXS_BF16, PXS_ERR_ARG, "pxs_tree_attention_plan: bad dtype");
    PXS_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 65535 && head_dim > 0 && head_dim <= kTreeMaxDim,
              PXS_ERR_ARG, "pxs_tree_attention_plan: bad heads");
    PXS_CHECK(nseg > 0 && q_len && cache_len && plan, PXS_ERR_ARG, "pxs_tree_attention_plan: null pointer");
    PXS_CHECK(cache_rows >= 0 && cache_rows <= kTreeMaxRows, PXS_ERR_ARG, "pxs_tree_attention_plan: bad cache");
    TreeArgs a{};
    a.cache_rows = cache_rows; a.kv_heads = kv_heads; a.group = heads / kv_heads;
    const bool fast = dtype == PXS_BF16 && head_dim <= 128 && head_dim % 8 == 0;
    set_tree_cuts(a, fast);
    const int keys = !fast || head_dim > 64 ? 32 : 64;
    double work = 0.0;
    int64_t total_q = 0;
    for (int s = 0; s < nseg; ++s) {
        PXS_CHECK(q_len[s] >= 0 && q_len[s] <= kTreeMaxRows / a.group - total_q && cache_len[s] >= 0 && cache_len[s] <= cache_rows,
                  PXS_ERR_ARG, "pxs_tree_attention_plan: bad length");
        total_q += q_len[s];
        work += static_cast<double>(row_tiles_of(a, {0, static_cast<int>(q_len[s]), 0, 0})) * static_cast<double>(cache_len[s]);
    }
    const int chunk = chunk_of(a, static_cast<float>(work));
    int most[2] = {0, 0}, joined = 0;  // (of an even and of an odd number)
    for (int s = 0; s < nseg; ++s) {
        const Tree g{0, static_cast<int>(q_len[s]), static_cast<int>(cache_len[s]), 0};
        const int chunks = chunks_of(g, chunk);
        for (int i = 0; g.nq > 0 && i < chunks; ++i) {
            const TreeSteps t = tree_steps(g.nq, i, chunk_start(g, i, chunks), chunk_start(g, i + 1, chunks), keys);
            int & of = most[(t.all - t.exact) % 2];
            if (fast) of = std::max(of, t.all - t.exact);
        }
        if (g.nq > 0 && chunks > 1) joined = joins_rows_each(total_q, heads) ? 2 : 1;
    }
    plan[0] = 1 << a.row_shift;
    plan[1] = keys;
    plan[2] = chunk;
    plan[3] = most[0];
    plan[4] = most[1];
    plan[5] = joined;
    return PXS_OK;
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
    score_constants(a, scale, cap);
    a.slopes = slopes; a.o = o; a.ldo = ld_o;
    const int elem = dtype == PXS_BF16 ? 2 : 4;
    a.vec = whole_pieces(q, ld_q, head_dim, elem) && whole_pieces(k, ld_k, head_dim, elem) &&
            whole_pieces(v, ld_v, head_dim, elem) &&
            (cache_rows == 0 || (whole_pieces(k_cache, ld_k_cache, head_dim, elem) && whole_pieces(v_cache, ld_v_cache, head_dim, elem)));
    // The fast kernels' 32-bit offsets within a key tile hold row strides below 2^24.
    const bool fast = dtype == PXS_BF16 && head_dim <= 128 && a.vec && ld_k < (1 << 24) && ld_v < (1 << 24) &&
                      (cache_rows == 0 || (ld_k_cache < (1 << 24) && ld_v_cache < (1 << 24))) &&
                      reinterpret_cast<uintptr_t>(o) % 8 == 0 && ld_o % 4 == 0;
    set_tree_cuts(a, fast);
    a.items = tree_items(nseg, total_q, kv_heads, a.group, a.row_shift);
    a.slot_rows = tree_slot_rows(total_q * a.group, a.row_shift);
    a.slots = tree_slots(kv_heads);
    PXS_CHECK(a.items * kv_heads <= UINT32_MAX / 256 && join_groups(a) <= UINT32_MAX / 256, PXS_ERR_ARG,
              "pxs_tree_attention: grid too large");
    char * ws = static_cast<char *>(workspace);
    if (nseg > kWaveSegments) {
        a.table = reinterpret_cast<int64_t *>(ws);
        hipLaunchKernelGGL(tree_table_kernel, dim3(1), dim3(1024), 0, s, a, reinterpret_cast<int64_t *>(ws));
        if (int rc = check_launch("tree attention table")) return rc;
    }
    ws += tree_table_bytes(nseg);
    const size_t rows = tree_part_rows(kv_heads, a.slot_rows);
    a.part_ml = reinterpret_cast<float2 *>(ws);
    a.part = reinterpret_cast<float *>(ws + round256(rows * sizeof(float2)));
    return dtype == PXS_F32 ? run_tree<float>(a, false, s) : run_tree<uint16_t>(a, fast, s);
}

} // extern "C"
