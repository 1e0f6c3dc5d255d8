// Varlen attention whose scores are capped, biased by distance and masked
// (pxs_varlen_attention in attention.hip has plain scores and no mask).
//
//   s(i, j) = scale * q_i . k_j
//   s = cap * tanh(s / cap)                     with a cap
//   s = s - slope[head] * |p_i - j|             with slopes
//   seen(i, j): not causal, or j <= p_i, or j < prefix[segment]
//   o_i = sum_seen exp(s) v_j / sum_seen exp(s), zeros where nothing is seen
//
// p_i = i + (keys - queries) of the segment: its queries are the last positions of
// its keys, as new tokens over a cache are.  The segments are the documents of a
// packed batch: nothing is seen across them.
//
// `group` query heads share a key/value head.  They are rows of one tile, row
// r of a (segment, key/value head) being query r / group of its head r % group: a
// key tile is read once for the group, and a single token fills group rows.
//
// Scores are kept in units of log2: z = s * log2(e).  One pass over the keys with
// the running maximum and sum in fp32.  Where a call's row tiles leave CUs idle the
// keys are split; every split writes its maximum, sum and unnormalised output in
// fp32, and a second launch joins them in order.

#include "attn_common.h"
#include "split3.h"
#include "tiles.h"

#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

namespace pxs {
namespace {

struct ScoreArgs {
    const void * q;
    const void * k;
    const void * v;
    int64_t ldq, ldk, ldv;
    const int64_t * cu_q;
    const int64_t * cu_k;
    int nseg;
    int64_t total_q, total_k;
    const int64_t * tile_start;  // [nseg + 1] items before each segment; null: at most 64 segments
    int chunk;                   // keys of an item of a segment with one row tile; 0: not cut
    int heads, kv_heads, group, d;
    float scale_log2;            // scale * log2(e)
    float cap_log2;              // cap * log2(e); 0: no cap
    float over_cap;              // scale / cap
    float exp_mul;               // 2 log2(e) scale / cap
    const float * slopes;        // [heads] or null
    int causal;
    const int64_t * prefix;      // [nseg] or null
    void * o;
    int64_t ldo;
    int vec;                     // rows of q, k and v in whole 16-byte pieces
    int64_t tiles;               // row tiles launched (bound)
    int splits;
    float * part;                // [partial rows][d] unnormalised outputs
    float2 * part_ml;            // [partial rows] maxima (log2 units) and sums
};

// A workgroup's rows: a tile of a segment and key/value head, and the keys that its rows see.
struct Rows {
    int kv;
    int q0, k0;           // the segment's first query and key
    int nk;
    int row0;             // first row of the tile
    int rows;             // of the segment: queries * group
    int shift;            // position of query i: i + shift
    int prefix;           // keys that every row sees, 0..nk
    int chunk, chunks;    // of the segment's keys; 0 of 1 where they are not cut
    int splits;           // of its keys where all of a call's are split alike: up to a.splits
};

constexpr int kSplitKeys = 256;  // keys that a split has at least

// Splits that a segment of nk keys has of a call's.
__device__ __forceinline__ int segment_splits(const ScoreArgs & a, int nk) {
    return max(1, min(a.splits, (nk + kSplitKeys - 1) / kSplitKeys));
}

// Items of a segment: its row tiles, or where it has one and a.chunk is set the chunks of its keys.
__device__ __forceinline__ int64_t segment_items(int64_t nq, int64_t nk, int group, int rows_per_tile, int chunk) {
    const int64_t rows = nq * group;
    if (rows <= 0) return 0;
    if (chunk > 0 && rows <= rows_per_tile) return max((nk + chunk - 1) / chunk, int64_t(1));
    return (rows + rows_per_tile - 1) / rows_per_tile;
}

// A segment's first query and key, its queries, keys and prefix (0..keys).
struct Segment {
    int q0, k0, nq, nk, prefix;
};
// (Bounds are kept within the call's rows, whatever cu_q and cu_k hold.)
__device__ __forceinline__ Segment load_segment(const ScoreArgs & a, int s) {
    auto within = [](int64_t v, int64_t lo, int64_t hi) { return static_cast<int>(max(min(v, hi), lo)); };
    const int q0 = within(a.cu_q[s], 0, a.total_q), q1 = within(a.cu_q[s + 1], q0, a.total_q);
    const int k0 = within(a.cu_k[s], 0, a.total_k), k1 = within(a.cu_k[s + 1], k0, a.total_k);
    return {q0, k0, q1 - q0, k1 - k0, a.causal && a.prefix ? within(a.prefix[s], 0, k1 - k0) : 0};
}
// The segment that lane `from` (the same in all lanes) holds.
__device__ __forceinline__ Segment segment_of(const Segment & g, int from) {
    return {__builtin_amdgcn_readlane(g.q0, from), __builtin_amdgcn_readlane(g.k0, from),
            __builtin_amdgcn_readlane(g.nq, from), __builtin_amdgcn_readlane(g.nk, from),
            __builtin_amdgcn_readlane(g.prefix, from)};
}
// Up to 64 segments, one a lane, read together (a segment's bounds are then no second wait).
__device__ __forceinline__ Segment lane_segment(const ScoreArgs & a, int lane) {
    Segment g{};
    if (lane < a.nseg) g = load_segment(a, lane);
    return g;
}

// Item i of a segment; false where it has no such rows.
__device__ __forceinline__ bool segment_rows(const ScoreArgs & a, const Segment & g, int i, int rows_per_tile, Rows & w) {
    w.q0 = g.q0;
    w.k0 = g.k0;
    w.nk = g.nk;
    w.rows = g.nq * a.group;
    w.shift = g.nk - g.nq;
    w.prefix = g.prefix;
    const bool cut = a.chunk > 0 && w.rows <= rows_per_tile;
    w.row0 = cut ? 0 : i * rows_per_tile;
    w.chunk = cut ? i : 0;
    w.chunks = !cut ? 1 : g.nk > 0 ? (g.nk - 1) / a.chunk + 1 : 0;
    w.splits = segment_splits(a, g.nk);
    return w.row0 < w.rows;
}

// v summed over the lanes up to each.
__device__ __forceinline__ int lane_sums(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int below = __shfl_up(v, d, 64);
        if (lane >= d) v += below;
    }
    return v;
}

// Item t; false past the last.
__device__ __forceinline__ bool locate_rows(const ScoreArgs & a, int t, int rows_per_tile, int lane, Rows & w) {
    if (a.tile_start) {
        if (t >= a.tile_start[a.nseg]) return false;
        const int seg = __builtin_amdgcn_readfirstlane(find_segment(a.tile_start, a.nseg, t, lane));
        return segment_rows(a, load_segment(a, seg), __builtin_amdgcn_readfirstlane(static_cast<int>(t - a.tile_start[seg])),
                            rows_per_tile, w);
    }
    const Segment g = lane_segment(a, lane);
    const int items = static_cast<int>(segment_items(g.nq, g.nk, a.group, rows_per_tile, a.chunk));
    const int end = lane_sums(items, lane);
    const int seg = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < a.nseg && end <= t)));  // those that end at or before t
    if (seg >= a.nseg) return false;
    return segment_rows(a, segment_of(g, seg), t - __builtin_amdgcn_readlane(end - items, seg), rows_per_tile, w);
}

// Row tiles of a segment with `tiles` of them whose rows see fewer than x keys (they come first:
// later rows see no fewer).
__device__ __forceinline__ int tiles_below(int x, int nq, int nk, int prefix, int group, int tiles, int shift) {
    if (x <= prefix || x <= 0) return 0;  // (keys seen are at least the prefix, up to nk)
    if (x > nk) return tiles;
    // the first tile with a row of query x - 1 - (nk - nq) or later
    const int64_t query = static_cast<int64_t>(x) - 1 - (nk - nq);
    return query <= 0 ? 0 : static_cast<int>(min(query * group >> shift, static_cast<int64_t>(tiles)));
}

// The t-th row tile of a call with a causal mask and 2 to 64 segments, those that see most keys
// first: 64 classes of keys seen, counted by a lane each, then the tile within its class.  (In
// the segments' order, reversed, the last of a call's tiles may be long ones: 16 heads of 128 over 4, eight prompts
// of 2,048 tokens 172 us against 187; ten of 100 to 5,000, 295 against 306; five of 8,000 to 500, 365 against
// 376; 8192, 2903 and 4739 with a cap, 483 against 495.  Two prompts whose first 1370 tokens all see lose 3%.)
__device__ __forceinline__ bool locate_sorted(const ScoreArgs & a, int t, int rows_per_tile, int lane, Rows & w) {
    const int shift = 31 - __clz(rows_per_tile);
    const Segment g = lane_segment(a, lane);
    const int nq = g.nq, nk = g.nk, prefix = g.prefix;
    const int tiles = static_cast<int>((static_cast<int64_t>(nq) * a.group + rows_per_tile - 1) >> shift);
    int most = nk;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) most = max(most, __shfl_xor(most, d, 64));
    const int unit = most / 64 + 1;  // most < 64 unit
    int count = 0;                   // tiles that see at least lane * unit keys
    for (int s = 0; s < a.nseg; ++s) {
        const int of = __builtin_amdgcn_readlane(tiles, s);
        count += of - tiles_below(lane * unit, __builtin_amdgcn_readlane(nq, s), __builtin_amdgcn_readlane(nk, s),
                                  __builtin_amdgcn_readlane(prefix, s), a.group, of, shift);
    }
    const int cls = __popcll(__ballot(count > t)) - 1;
    if (cls < 0) return false;
    const int ahead = cls == 63 ? 0 : __builtin_amdgcn_readlane(count, cls + 1);
    const int lo = tiles_below(cls * unit, nq, nk, prefix, a.group, tiles, shift);
    const int hi = cls == 63 ? tiles : tiles_below((cls + 1) * unit, nq, nk, prefix, a.group, tiles, shift);
    const int end = lane_sums(hi - lo, lane);  // the class's tiles of the segments up to this lane's
    const int at = t - ahead;
    const int seg = __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < a.nseg && end <= at)));
    const int within = at - __builtin_amdgcn_readlane(end - (hi - lo), seg);
    return segment_rows(a, segment_of(g, seg), __builtin_amdgcn_readlane(hi, seg) - 1 - within, rows_per_tile, w);
}

// A workgroup's row tile and split: key/value heads next to one another, so that an XCD, which
// takes every eighth workgroup, reads few of them; the longest tiles first.
__device__ __forceinline__ bool locate_work(const ScoreArgs & a, int rows_per_tile, int lane, Rows & w, int & split) {
    const int per = a.kv_heads * a.splits, rest = static_cast<int>(blockIdx.x % per);
    const int t = static_cast<int>(blockIdx.x / per);
    w.kv = rest % a.kv_heads;
    split = rest / a.kv_heads;
    const bool found = a.causal && !a.tile_start && a.nseg > 1
                           ? locate_sorted(a, t, rows_per_tile, lane, w)
                           : locate_rows(a, static_cast<int>(a.tiles) - 1 - t, rows_per_tile, lane, w);
    return found && split < w.splits;
}

// Query qi of the call: its segment, and the first of the segment's items; false for a row of no segment.
__device__ __forceinline__ bool locate_query(const ScoreArgs & a, int qi, int rows_per_tile, int lane, Rows & w, int & item) {
    if (a.tile_start) {
        if (qi < a.cu_q[0] || qi >= a.cu_q[a.nseg]) return false;
        const int seg = find_segment(a.cu_q, a.nseg, qi, lane);
        const Segment g = load_segment(a, seg);
        if (qi < g.q0 || qi >= g.q0 + g.nq) return false;  // (bounds that fall)
        item = static_cast<int>(min(a.tile_start[seg], a.tiles));
        return segment_rows(a, g, 0, rows_per_tile, w);
    }
    const Segment g = lane_segment(a, lane);
    const int items = static_cast<int>(segment_items(g.nq, g.nk, a.group, rows_per_tile, a.chunk));
    const int end = lane_sums(items, lane);
    const uint64_t mine = __ballot(lane < a.nseg && qi >= g.q0 && qi < g.q0 + g.nq);
    if (mine == 0) return false;
    const int seg = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(mine)) - 1);
    item = __builtin_amdgcn_readlane(end - items, seg);
    return segment_rows(a, segment_of(g, seg), 0, rows_per_tile, w);
}

// One past the last key that any of the rows up to `row` (inclusive) sees.
__device__ __forceinline__ int keys_end(const ScoreArgs & a, const Rows & w, int row) {
    if (!a.causal) return w.nk;
    return min(w.nk, max(min(row, w.rows - 1) / a.group + w.shift + 1, w.prefix));
}
// The keys that every row from `row` on sees: all below.
__device__ __forceinline__ int keys_all(const ScoreArgs & a, const Rows & w, int row) {
    if (!a.causal) return w.nk;
    return min(w.nk, max(row / a.group + w.shift + 1, w.prefix));
}

// A score in log2 units, from a product q . k and the key's distance behind the query.
__device__ __forceinline__ float score_log2(const ScoreArgs & a, float dot, float slope_log2, float away) {
    float z = dot * a.scale_log2;
    if (a.cap_log2 > 0.0f) z = a.cap_log2 * tanhf(dot * a.over_cap);
    return z - slope_log2 * fabsf(away);
}

template <typename T>
__device__ __forceinline__ void load_dims(const T * row, int c, int d, bool vec, T (&out)[16 / sizeof(T)]) {
    constexpr int kVec = 16 / sizeof(T);
    if (vec && c + kVec <= d) {
        *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(row + c);
        return;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = c + e < d ? row[c + e] : T(0);
}

__device__ __forceinline__ bool is_finite_bits(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// A row again, one key after the other, keys that it does not see left out
// altogether: for tiles where an unseen key's value is infinite or NaN, which
// times a weight of zero is NaN.  One wave per row; lane l holds dims l, l + 64, ...
// Slow, a key a step: where a causal prompt's last value is NaN, 16 heads of 128, 1,024 tokens take 7.4 ms
// (87 us without), 8,192 take 327 (0.33); 8 tokens over 8,192 keys 0.42 (0.09).  The last row sees such a value
// and is NaN itself, so it is met in broken data alone.
// (Inlined: a call would take the arguments in memory, and with them every kernel's scalars.)
template <typename T, int NC>
__device__ __forceinline__ void row_alone(const ScoreArgs & a, const Rows & w, int row, int key0, int key1, int lane, bool partial,
                          int64_t slot) {
    const int i = row / a.group;
    const int head = w.kv * a.group + row % a.group;
    const T * q = static_cast<const T *>(a.q) + (w.q0 + i) * a.ldq + static_cast<int64_t>(head) * a.d;
    const T * k = static_cast<const T *>(a.k) + w.k0 * a.ldk + static_cast<int64_t>(w.kv) * a.d;
    const T * v = static_cast<const T *>(a.v) + w.k0 * a.ldv + static_cast<int64_t>(w.kv) * a.d;
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    float qv[NC], acc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        qv[c] = lane + 64 * c < a.d ? load_f32(q + lane + 64 * c) : 0.0f;
        acc[c] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int end = min(key1, keys_end(a, w, row));
    for (int64_t j = key0; j < end; ++j) {
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < a.d) dot += qv[c] * load_f32(k + j * a.ldk + lane + 64 * c);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) dot += __shfl_xor(dot, off, 64);
        const float z = score_log2(a, dot, slope, static_cast<float>(i + w.shift - j));
        const float up = fmaxf(m, z);
        const float base = up == -INFINITY ? 0.0f : up;
        const float p = exp2f(z - base), keep = exp2f(m - base);
        l = l * keep + p;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < a.d) acc[c] = acc[c] * keep + p * load_f32(v + j * a.ldv + lane + 64 * c);
        m = up;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN sum stays NaN)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int dim = lane + 64 * c;
        if (dim >= a.d) continue;
        if (partial) a.part[slot * a.d + dim] = acc[c];
        else store_f32(static_cast<T *>(a.o) + (w.q0 + i) * a.ldo + static_cast<int64_t>(head) * a.d + dim, acc[c] * inv);
    }
    if (partial && lane == 0) a.part_ml[slot] = make_float2(m, l);
}

// Partial row of a (query, head) in split `split` of a call whose keys are split alike for all rows.
__device__ __forceinline__ int64_t split_slot(const ScoreArgs & a, const Rows & w, int split, int row) {
    return (split * a.total_q + w.q0 + row / a.group) * a.heads + w.kv * a.group + row % a.group;
}

// Any dtype, head size up to DP, stride and alignment.  Four waves of 32 rows
// share tiles of kKeys keys, staged through registers into LDS.  As in
// attention.hip a wave computes S^T = K Q^T, so that a lane owns one row and half of
// its scores, and O^T += V^T P^T with P straight from those registers.  Waves past the segment's
// rows only help to stage: a new token's tile costs one wave's products.
//
// bf16: V is staged transposed, four keys of a dim a read.
// fp32, SPLIT (heads up to 128): operands and weights split in three bf16 terms, six of their
//   products (split3.h), 192 cycles where v_mfma_f32_32x32x2_f32 takes 512; K and V in three planes,
//   laid out as the bf16 kernels' tiles are.  Bound by the vector instructions that split beside the
//   matrix cores.  A workgroup that meets values the terms may not hold (above 2^50, not finite, or in V
//   below 2^-110 and not zero) writes nothing and takes the next form.  (The scores' losses stay under
//   128 x 2^50 x 2^-134 of the scale, at most 2^41.)  4,000 tokens, 16 heads of 64: 400 us against 587.
// fp32 otherwise: v_mfma_f32_32x32x2_f32, V read as it lies, 32 dims of a key side by side.
template <typename T, int DP, bool SPLIT> struct AnyTile {
    static constexpr bool kTransposed = sizeof(T) == 2;
    static constexpr int kKeys = DP == 64 ? 64 : 32;
    static constexpr int kPlane = kKeys * DP * 2;  // SPLIT: one term of a K or V tile
    static constexpr int kKPitch = DP * static_cast<int>(sizeof(T)) + 16;
    static constexpr int kVPitch = kTransposed ? kKeys * 2 + 8 : kKPitch;
    static constexpr int kBytes = SPLIT ? 6 * kPlane : kKeys * kKPitch + (kTransposed ? DP : kKeys) * kVPitch;
};
constexpr uint32_t kSplitHighBits = 177u << 23, kSplitWholeBits = 17u << 23;  // 2^50, 2^-110

// One pass over the keys of a row tile's split; false where SPLIT does not hold its values.
template <typename T, int DP, bool SPLIT>
__device__ __forceinline__ bool any_pass(const ScoreArgs & a, const Rows & w, int split, char * smem) {
    static_assert(!SPLIT || (sizeof(T) == 4 && DP <= 128), "the split is of fp32");
    using Tile = AnyTile<T, DP, SPLIT>;
    constexpr int kVec = 16 / static_cast<int>(sizeof(T)), kKeys = Tile::kKeys, KT = kKeys / 32, DT = DP / 32;
    constexpr int kPieces = DP / kVec;  // 16-byte pieces of a padded row
    constexpr int NST = DP / 16, kHalf = kKeys * 128;
    char * k_lds = smem;
    char * v_lds = smem + (SPLIT ? 3 * Tile::kPlane : kKeys * Tile::kKPitch);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;

    const int end = keys_end(a, w, w.row0 + 127);
    const int key_tiles = (end + kKeys - 1) / kKeys;
    const int kt_first = static_cast<int>(static_cast<int64_t>(key_tiles) * split / w.splits);
    const int kt_last = static_cast<int>(static_cast<int64_t>(key_tiles) * (split + 1) / w.splits);

    const T * k = static_cast<const T *>(a.k) + w.k0 * a.ldk + static_cast<int64_t>(w.kv) * a.d;
    const T * v = static_cast<const T *>(a.v) + w.k0 * a.ldv + static_cast<int64_t>(w.kv) * a.d;

    // This lane's row and its Q fragment (dims h DP/2 .. h DP/2 + DP/2 - 1, or as the planes hold them).
    const int wave_row0 = w.row0 + wave * 32;
    const int row = wave_row0 + r;
    const bool live = row < w.rows;
    const int qi = (live ? row : 0) / a.group;
    const int head = w.kv * a.group + (live ? row : 0) % a.group;
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    const T * q = static_cast<const T *>(a.q) + (w.q0 + qi) * a.ldq + static_cast<int64_t>(head) * a.d;
    T qv[SPLIT ? 1 : DP / 2];
    bf16x8 qf[SPLIT ? 3 : 1][SPLIT ? NST : 1];
    uint32_t hi_bits = 0;  // the largest magnitude met
    bool wild = false;
    float unused = 0.0f;
    if constexpr (SPLIT) {
#pragma unroll
        for (int st = 0; st < NST; ++st) {
            float f[2][4] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (live) load_dims<float>(q, (st / 4) * 64 + 32 * h + 8 * (st % 4) + 4 * i, a.d, a.vec, f[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) hi_bits = max(hi_bits, __float_as_uint(f[i][e]) & 0x7FFFFFFFu);
            }
            uint2 lo4[3], hi4[3];
            split4(make_float4(f[0][0], f[0][1], f[0][2], f[0][3]), lo4, unused);
            split4(make_float4(f[1][0], f[1][1], f[1][2], f[1][3]), hi4, unused);
#pragma unroll
            for (int t = 0; t < 3; ++t)
                qf[t][st] = __builtin_bit_cast(bf16x8, make_uint4(lo4[t].x, lo4[t].y, hi4[t].x, hi4[t].y));
        }
    } else {
#pragma unroll
        for (int c = 0; c < DP / 2 / kVec; ++c) {
            T tmp[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) tmp[e] = T(0);
            if (live) load_dims<T>(q, h * (DP / 2) + c * kVec, a.d, a.vec, tmp);
#pragma unroll
            for (int e = 0; e < kVec; ++e) qv[c * kVec + e] = tmp[e];
        }
    }
    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    const int my_end = live ? keys_end(a, w, row) : 0;  // keys >= my_end are masked
    const int wave_all = keys_all(a, w, wave_row0);     // keys below are seen by all of the wave's rows
    const int tile_all = keys_all(a, w, w.row0);
    bool again = false;

    // This thread's pieces of a K and a V tile, the next tile's loaded while one is multiplied.
    constexpr int kMine = kKeys * kPieces / 256;
    T kk[kMine][kVec], vv[kMine][kVec];
    auto load = [&](int kt0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int key = (tid + 256 * j) / kPieces, piece = (tid + 256 * j) % kPieces;
#pragma unroll
            for (int e = 0; e < kVec; ++e) kk[j][e] = vv[j][e] = T(0);
            if (kt0 + key < w.nk) {
                load_dims<T>(k + static_cast<int64_t>(kt0 + key) * a.ldk, piece * kVec, a.d, a.vec, kk[j]);
                load_dims<T>(v + static_cast<int64_t>(kt0 + key) * a.ldv, piece * kVec, a.d, a.vec, vv[j]);
            }
        }
    };
    if (kt_first < kt_last) load(kt_first * kKeys);
    for (int kt0 = kt_first * kKeys; kt0 < kt_last * kKeys; kt0 += kKeys) {
        barrier_no_fence();  // every wave has read the tile before
        bool odd = false;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int key = (tid + 256 * j) / kPieces, piece = (tid + 256 * j) % kPieces;
            if constexpr (SPLIT) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t kb = __float_as_uint(kk[j][e]) & 0x7FFFFFFFu, vb = __float_as_uint(vv[j][e]) & 0x7FFFFFFFu;
                    hi_bits = max(hi_bits, max(kb, vb));
                    wild |= vb - 1u < kSplitWholeBits - 1u;
                }
                const int at = (piece >> 4) * kHalf + key * 128 + (piece & 1) * 8, p16 = (piece & 15) >> 1;
                uint2 t[3];
                split4(make_float4(kk[j][0], kk[j][1], kk[j][2], kk[j][3]), t, unused);
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<uint2 *>(k_lds + p * Tile::kPlane + at + ((p16 ^ kswz(key)) << 4)) = t[p];
                split4(make_float4(vv[j][0], vv[j][1], vv[j][2], vv[j][3]), t, unused);
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<uint2 *>(v_lds + p * Tile::kPlane + at + ((p16 ^ vswz(key)) << 4)) = t[p];
                continue;
            }
            *reinterpret_cast<uint4 *>(k_lds + key * Tile::kKPitch + piece * 16) = *reinterpret_cast<const uint4 *>(kk[j]);
            if constexpr (!Tile::kTransposed)
                *reinterpret_cast<uint4 *>(v_lds + key * Tile::kVPitch + piece * 16) = *reinterpret_cast<const uint4 *>(vv[j]);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                odd |= !is_finite_bits(load_f32(&vv[j][e]));
                if constexpr (Tile::kTransposed)
                    *reinterpret_cast<T *>(v_lds + (piece * kVec + e) * Tile::kVPitch + key * static_cast<int>(sizeof(T))) = vv[j][e];
            }
        }
        // A tile with keys that some row does not see, and values that are not finite.
        again |= odd && min(kt0 + kKeys, w.nk) > tile_all;
        if (kt0 + kKeys < kt_last * kKeys) load(kt0 + kKeys);
        barrier_no_fence();  // the tile is written
        if (wave_row0 >= w.rows) continue;

        f32x16 s[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = f32x16{};
        if constexpr (SPLIT) {
#pragma unroll
            for (int st = 0; st < NST; ++st) {
                bf16x8 kf[KT][3];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const int rw = kt * 32 + r;
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        kf[kt][p] = *reinterpret_cast<const bf16x8 *>(k_lds + p * Tile::kPlane + (st / 4) * kHalf + rw * 128 +
                                                                      (((4 * h + st % 4) ^ kswz(rw)) << 4));
                }
#pragma unroll
                for (int n = 0; n < 6; ++n)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
                        s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kt][kSplitTermA[n]], qf[kSplitTermB[n]][st],
                                                                        s[kt], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const char * krow = k_lds + (kt * 32 + r) * Tile::kKPitch;
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int st = 0; st < NST; ++st) {
                        const bf16x8 kf = *reinterpret_cast<const bf16x8 *>(krow + h * DP + st * 16);
                        bf16x8 qb;
#pragma unroll
                        for (int e = 0; e < 8; ++e) qb[e] = __builtin_bit_cast(__bf16, qv[st * 8 + e]);
                        s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qb, s[kt], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < DP / 8; ++u) {
                        const f32x4 kf = *reinterpret_cast<const f32x4 *>(krow + (h * (DP / 2) + 4 * u) * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[kt] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], __builtin_bit_cast(float, qv[4 * u + e]),
                                                                         s[kt], 0, 0, 0);
                    }
                }
            }
        }
        // Register e of sub-tile kt holds key kt * 32 + 8 (e / 4) + 4 h + e % 4.
        const bool masked = kt0 + kKeys > wave_all || kt0 + kKeys > w.nk;
        const int behind = qi + w.shift - kt0, seen = my_end - kt0;
        float top = -INFINITY;
        if (a.cap_log2 > 0.0f || a.slopes || masked) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = kt * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                    float z = score_log2(a, s[kt][e], slope, static_cast<float>(behind - key));
                    if (key >= seen) z = -INFINITY;
                    s[kt][e] = z;
                    top = fmaxf(top, z);
                }
        } else {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[kt][e] *= a.scale_log2;
                    top = fmaxf(top, s[kt][e]);
                }
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = fmaxf(m, top);
        const float base = up == -INFINITY ? 0.0f : up;  // nothing seen yet: every weight is 0
        const float keep = __builtin_amdgcn_exp2f(m - base);
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(s[kt][e] - base);  // (0 below 2^-126)
                s[kt][e] = p;
                sum += p;
            }
        sum += __shfl_xor(sum, 32, 64);
        l = l * keep + sum;
        m = up;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[dt][e] *= keep;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            if constexpr (SPLIT) {
                const int G = lane >> 4, jl = lane & 15;
                const int key_off = 4 * (G >> 1) + (jl >> 2), dim_off = 16 * (G & 1) + 4 * (jl & 3);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    bf16x8 pf[3];
                    uint2 lo4[3], hi4[3];
                    split4(make_float4(s[kt][8 * u], s[kt][8 * u + 1], s[kt][8 * u + 2], s[kt][8 * u + 3]), lo4, unused);
                    split4(make_float4(s[kt][8 * u + 4], s[kt][8 * u + 5], s[kt][8 * u + 6], s[kt][8 * u + 7]), hi4, unused);
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        pf[p] = __builtin_bit_cast(bf16x8, make_uint4(lo4[p].x, lo4[p].y, hi4[p].x, hi4[p].y));
                    const int ka = kt * 32 + 16 * u + key_off, kb = ka + 8;
#pragma unroll
                    for (int d2 = 0; d2 < DT; d2 += 2) {
                        bf16x8 vf[2][3];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int dbyte = (i * 32 + dim_off) * 2, p16 = dbyte >> 4, within = dbyte & 15;
#pragma unroll
                            for (int p = 0; p < 3; ++p) {
                                const char * vh = v_lds + p * Tile::kPlane + (d2 / 2) * kHalf;
                                const char * pa = vh + ka * 128 + ((p16 ^ vswz(ka)) << 4) + within;
                                const char * pb = vh + kb * 128 + ((p16 ^ vswz(kb)) << 4) + within;
                                const uint2 lo2 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                                                (v4i16 __attribute__((address_space(3))) *)(pa)));
                                const uint2 hi2 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                                                (v4i16 __attribute__((address_space(3))) *)(pb)));
                                vf[i][p] = __builtin_bit_cast(bf16x8, make_uint4(lo2.x, lo2.y, hi2.x, hi2.y));
                            }
                        }
#pragma unroll
                        for (int n = 0; n < 6; ++n)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                oacc[d2 + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i][kSplitTermA[n]], pf[kSplitTermB[n]],
                                                                                       oacc[d2 + i], 0, 0, 0);
                    }
                }
            } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    bf16x8 p;  // weights round to bf16, as the values they multiply are
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = static_cast<__bf16>(s[kt][8 * u + e]);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const char * vrow = v_lds + (dt * 32 + r) * Tile::kVPitch;
                        const int key = kt * 32 + 16 * u + 4 * h;
                        const uint2 lo = *reinterpret_cast<const uint2 *>(vrow + key * 2);
                        const uint2 hi = *reinterpret_cast<const uint2 *>(vrow + (key + 8) * 2);
                        oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            __builtin_bit_cast(bf16x8, make_uint4(lo.x, lo.y, hi.x, hi.y)), p, oacc[dt], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const char * vrow = v_lds + (kt * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * Tile::kVPitch + r * 4;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float *>(vrow + dt * 128),
                                                                        s[kt][e], oacc[dt], 0, 0, 0);
                }
            }
        }
    }
    if constexpr (SPLIT) {
        if (__syncthreads_or(wild || hi_bits > kSplitHighBits)) return false;
    } else if (__syncthreads_or(again)) {
        for (int i = 0; i < 32; ++i)
            if (wave_row0 + i < w.rows)
                row_alone<T, DP / 64>(a, w, wave_row0 + i, kt_first * kKeys, kt_last * kKeys, lane, w.splits > 1,
                                      split_slot(a, w, split, wave_row0 + i));
        return true;
    }
    if (!live) return true;
    const int64_t slot = split_slot(a, w, split, row);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T * o = static_cast<T *>(a.o) + (w.q0 + qi) * a.ldo + static_cast<int64_t>(head) * a.d;
    if (w.splits > 1 && h == 0) a.part_ml[slot] = make_float2(m, l);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int dim = dt * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (dim >= a.d) continue;
            if (w.splits > 1) a.part[slot * a.d + dim] = oacc[dt][e];
            else store_f32(o + dim, oacc[dt][e] * inv);
        }
    return true;
}

template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP == 64 || (DP == 128 && !SPLIT) ? 2 : 1)))
score_attn_any_kernel(ScoreArgs a) {
    extern __shared__ __align__(16) char smem[];
    Rows w;
    int split;
    if (!locate_work(a, 128, threadIdx.x & 63, w, split)) return;
    if constexpr (SPLIT) {
        if (any_pass<T, DP, true>(a, w, split, smem)) return;
    }
    any_pass<T, DP, false>(a, w, split, smem);
}

// ---- bf16, head sizes of whole 16-byte pieces up to 128 -----------------------------------------------------
// Tiles of kKeys keys, 8 KB of K and 8 KB of V, go from HBM to LDS by DMA, rows of
// DH / 64 halves of 128 bytes; V is read transposed from LDS (ds_read_b64_tr_b16).
// 16 matrix instructions a tile and wave, as many for S as for O.

__device__ __align__(16) uint4 g_score_zero[8];  // what keys past a segment's end are read as

// MODE bits: scores are capped, biased, of a biased call that its mask lets queries see only keys at
// or before them in the tiles taken without a maximum, and of a capped call that its cap is above kNearCap.
constexpr int kCap = 1, kBias = 2, kBehind = 4, kFar = 8;
constexpr float kNearCap = 256.0f;
constexpr bool near_cap(int mode) { return (mode & (kCap | kFar)) == kCap; }

// Head sizes that are multiples of 8 up to 128 run as the next of 64 and 128 (WHOLE false): the
// missing pieces of a row come from a line of zeros.
template <int DH> struct Fast {
    static constexpr int KT = DH == 64 ? 2 : 1;   // 32-key sub-tiles of a tile
    static constexpr int kKeys = 32 * KT;
    static constexpr int kHalves = DH / 64;
    static constexpr int kHalfBytes = kKeys * 128;
    static constexpr int kTileBytes = kHalves * kHalfBytes;  // 8 KB
    static constexpr int kUnits = kTileBytes / 1024;         // DMA instructions of a K or V tile (8 rows of a half)
    static constexpr int NST = DH / 16, NDT = DH / 32;
    typedef f32x16 Scores[KT];
    typedef bf16x8 Weights[KT][2];
    typedef f32x16 Out[NDT];
};

// One row's constants of the map from a product q . k to a weight's exponent:
//   z = raw * mul + add                              (no cap)
//   z = add + top / (1 + 2^(raw * mul))              (cap: cap tanh(x) = cap - 2 cap / (1 + e^2x))
//   with a bias, add - slope * |behind - key|.
// That form of the cap is off by up to 2^-23 of the cap, whatever the score: 3e-5 at kNearCap, about what
// the products' sums in fp32 are off by.  A larger cap (kFar) takes a form that is right relative to the
// score, x = raw * over:
//   z = add + raw * mul * (1 - x^2/3 + 2 x^4/15 - ...)        |x| < 1/4; the next term is 2^-26 there
//   z = add + top - 2 top / (1 + e^2x)                        above, where the cap is at most 4.1 scores
// Ten operations a score more than the near form: causal prompts of 8192, 2903 and 4739, 16 heads of 128 over
// 4, 690 us against 485, 8,192 tokens without a mask, 16 heads of 64, 708 against 420; eight tokens over 170,161
// keys 150 against 144.
struct RowScore {
    float mul, top, slope, over, part;
};

template <int MODE>
__device__ __forceinline__ RowScore row_score(const ScoreArgs & a, int head) {
    RowScore s;
    s.mul = near_cap(MODE) ? a.exp_mul : a.scale_log2;
    s.top = near_cap(MODE) ? -2.0f * a.cap_log2 : a.cap_log2;
    s.over = a.over_cap;
    s.part = -2.0f * a.cap_log2;
    s.slope = MODE & kBias ? -kLog2e * a.slopes[head] : 0.0f;
    return s;
}

// z - base of a product; key: behind - key is the distance.  add is cap_log2 - base with a near cap, -base otherwise.
template <int MODE>
__device__ __forceinline__ float score_of(const RowScore & s, float raw, float add, float away) {
    float b = add;
    if constexpr (MODE & kBias) b = __builtin_fmaf(s.slope, fabsf(away), add);
    if constexpr (MODE & kFar) {
        const float x = raw * s.over, y = x * x;
        const float series = __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 0x1.664f48p-6f, -0x1.ba1ba2p-5f),
                                                                                0x1.111112p-3f), -0x1.555556p-2f), 1.0f);
        const float rest = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * (2.0f * kLog2e)));
        // (Of the two forms' cheap parts one is taken: between their results the compiler branches.)
        const bool near = fabsf(x) < 0.25f;
        const float whole = near ? raw * s.mul * series : s.top, part = near ? 0.0f : s.part;
        return __builtin_fmaf(part, rest, whole) + b;
    }
    if constexpr (MODE & kCap)
        return __builtin_fmaf(s.top, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(raw * s.mul)), b);
    return __builtin_fmaf(raw, s.mul, b);
}

template <int DH>
__device__ __forceinline__ void tile_qk(const char * kl, const bf16x8 (&qf)[Fast<DH>::NST],
                                        typename Fast<DH>::Scores & s, int h, int r) {
    using F = Fast<DH>;
#pragma unroll
    for (int kt = 0; kt < F::KT; ++kt) {
        const int row = kt * 32 + r;
#pragma unroll
        for (int st = 0; st < F::NST; ++st) {
            const bf16x8 kf = *reinterpret_cast<const bf16x8 *>(
                kl + (st / 4) * F::kHalfBytes + row * 128 + (((4 * h + st % 4) ^ kswz(row)) << 4));
            if (st == 0) s[kt] = f32x16{};
            s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[st], s[kt], 0, 0, 0);
        }
    }
}

template <int DH>
__device__ __forceinline__ void tile_pv(const char * vl, const typename Fast<DH>::Weights & p,
                                        typename Fast<DH>::Out & oacc, int lane) {
    using F = Fast<DH>;
    const int G = lane >> 4, jl = lane & 15;
    const int key_off = 4 * (G >> 1) + (jl >> 2), dim_off = 16 * (G & 1) + 4 * (jl & 3);
#pragma unroll
    for (int kt = 0; kt < F::KT; ++kt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int ka = kt * 32 + 16 * u + key_off, kb = ka + 8;
#pragma unroll
            for (int dt = 0; dt < F::NDT; ++dt) {
                const int dbyte = ((dt % 2) * 32 + dim_off) * 2, piece = dbyte >> 4, within = dbyte & 15;
                const char * vh = vl + (dt / 2) * F::kHalfBytes;
                const char * pa = vh + ka * 128 + ((piece ^ vswz(ka)) << 4) + within;
                const char * pb = vh + kb * 128 + ((piece ^ vswz(kb)) << 4) + within;
                const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                               (v4i16 __attribute__((address_space(3))) *)(pa)));
                const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                               (v4i16 __attribute__((address_space(3))) *)(pb)));
                oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    __builtin_bit_cast(bf16x8, make_uint4(lo.x, lo.y, hi.x, hi.y)), p[kt][u], oacc[dt], 0, 0, 0);
            }
        }
}

// Key of register e of sub-tile kt, and its part beyond 4 h.
__device__ __forceinline__ constexpr int key_of(int kt, int e) { return kt * 32 + 8 * (e >> 2) + (e & 3); }

// The running state of a lane's row: base (the maximum that weights are relative
// to) and this lane's half of their sum.
struct RowState {
    float base, sum;
};

// Weights of a tile relative to state.base: p = 2^(z - base), and their sum over this lane.  They are rounded to
// bf16, as pxs_varlen_attention's are and as the values that they multiply are: the matrix cores take both operands
// in one type, and a second term of each weight would be half as many products again.  The sum is of the rounded
// weights, so their errors' mean cancels.  Relative L2 error against 64 bits 0.0017 to 0.0020, of which the
// output's own rounding is 0.0017.
// behind: the lane's query position minus the tile's first key and 4 h.
// With kBehind the bias is a line over the keys, one operation a score and not two.
template <int DH, int MODE>
__device__ __forceinline__ float tile_weights(const RowScore & rs, float cap_log2, const typename Fast<DH>::Scores & s,
                                              typename Fast<DH>::Weights & p, float base, float behind) {
    const bf16x2 ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
    const float add = near_cap(MODE) ? cap_log2 - base : -base;
    const float start = MODE & kBehind ? __builtin_fmaf(rs.slope, behind, add) : 0.0f;
    auto weight = [&](int kt, int e) __attribute__((always_inline)) {
        const float key = static_cast<float>(key_of(kt, e));
        const float z = MODE & kBehind ? score_of<MODE & (kCap | kFar)>(rs, s[kt][e], __builtin_fmaf(rs.slope, -key, start), 0.0f)
                                       : score_of<MODE>(rs, s[kt][e], add, behind - key);
        return static_cast<__bf16>(__builtin_amdgcn_exp2f(z));
    };
    float sum = 0.0f;
#pragma unroll
    for (int kt = 0; kt < Fast<DH>::KT; ++kt)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const int i = 8 * u + e;
                bf16x2 pp;
                pp[0] = weight(kt, i);
                pp[1] = weight(kt, i + 1);
                p[kt][u][e] = pp[0];
                p[kt][u][e + 1] = pp[1];
                sum = __builtin_amdgcn_fdot2_f32_bf16(pp, ones, sum, false);  // of the rounded weights
            }
    return sum;
}

// The largest z of a tile over the row's two lanes.
template <int DH, int MODE>
__device__ __forceinline__ float tile_max(const RowScore & rs, float cap_log2, const typename Fast<DH>::Scores & s,
                                          float behind) {
    const float add = near_cap(MODE) ? cap_log2 : 0.0f;
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < Fast<DH>::KT; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            top = fmaxf(top, score_of<MODE>(rs, s[kt][e], add, behind - static_cast<float>(key_of(kt, e))));
    return lane_pair_max(top);
}

// The exact step of a tile: hidden keys (at or past `seen` of the tile's keys, less 4 h)
// get weight 0, the base rises to the maximum and the output with it.
template <int DH, int MODE>
__device__ __forceinline__ void tile_exact(const RowScore & rs, float cap_log2, typename Fast<DH>::Scores & s,
                                           typename Fast<DH>::Weights & p, typename Fast<DH>::Out & oacc,
                                           RowState & st, float behind, int seen) {
    using F = Fast<DH>;
    const float add = near_cap(MODE) ? cap_log2 : 0.0f;
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < F::KT; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float z = score_of<MODE>(rs, s[kt][e], add, behind - static_cast<float>(key_of(kt, e)));
            s[kt][e] = key_of(kt, e) < seen ? z : -INFINITY;
            top = fmaxf(top, s[kt][e]);
        }
    const float up = fmaxf(st.base, lane_pair_max(top));
    const float base = up == -INFINITY ? 0.0f : up;  // nothing seen yet: every weight is 0
    const float keep = __builtin_amdgcn_exp2f(st.base - base);
    const bf16x2 ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
    float sum = st.sum * keep;
#pragma unroll
    for (int kt = 0; kt < F::KT; ++kt)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                bf16x2 pp;
                pp[0] = static_cast<__bf16>(__builtin_amdgcn_exp2f(s[kt][8 * u + e] - base));
                pp[1] = static_cast<__bf16>(__builtin_amdgcn_exp2f(s[kt][8 * u + e + 1] - base));
                p[kt][u][e] = pp[0];
                p[kt][u][e + 1] = pp[1];
                sum = __builtin_amdgcn_fdot2_f32_bf16(pp, ones, sum, false);
            }
    st.sum = sum;
    st.base = up;
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[dt][e] *= keep;
}

// A tile's 2 * kUnits DMA instructions, those of index first, first + step, ...: K then V units.
template <int DH>
struct TileSource {
    const char * k;      // the segment's first key, this head
    const char * v;
    int64_t ldk, ldv;    // bytes
    int nk;
    uint64_t zero;
    uint32_t lacks;      // bit j: instruction j's piece of this lane lies past the head
};

template <int DH, int COUNT>
__device__ __forceinline__ void tile_offsets(TileSource<DH> & src, int d, int first, int lane, uint32_t (&off)[COUNT]) {
    using F = Fast<DH>;
    src.lacks = 0;
    const int lrow = lane >> 3, lslot = lane & 7;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        const int unit = first + j;
        const bool is_v = unit >= F::kUnits;
        const int half = unit % F::kUnits / (F::kKeys / 8), row = unit % (F::kKeys / 8) * 8 + lrow;
        const int byte = half * 128 + (lslot ^ (is_v ? vswz(row) : kswz(row))) * 16;
        off[j] = static_cast<uint32_t>(row * (is_v ? src.ldv : src.ldk) + byte);
        src.lacks |= (byte >= 2 * d ? 1u : 0u) << j;
    }
}

// Units first .. first + COUNT - 1 of tile t into the slot at LDS offset `lds` (K, then V).
template <int DH, bool WHOLE, int COUNT>
__device__ __forceinline__ void tile_issue(const TileSource<DH> & src, int t, int first, const uint32_t (&off)[COUNT],
                                           uint32_t lds, int lane) {
    using F = Fast<DH>;
    const int kt0 = t * F::kKeys;
    const char * kb = src.k + static_cast<int64_t>(kt0) * src.ldk;
    const char * vb = src.v + static_cast<int64_t>(kt0) * src.ldv;
    const bool whole = kt0 + F::kKeys <= src.nk;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        const int unit = first + j;
        const bool is_v = unit >= F::kUnits;
        const uint32_t at = lds + unit * 1024;
        if (WHOLE && whole) {
            lds_dma16_sbase(is_v ? vb : kb, off[j], at);
        } else {
            const int row = unit % (F::kKeys / 8) * 8 + (lane >> 3);
            const bool in = kt0 + row < src.nk && (WHOLE || !(src.lacks >> j & 1u));
            lds_dma16(in ? (is_v ? vb : kb) + off[j] : reinterpret_cast<const char *>(src.zero), at);
        }
    }
}

// Whether this thread's share of a V tile (of `threads` threads) holds an infinity or a NaN.
template <int DH>
__device__ __forceinline__ bool tile_odd(const char * vl, int thread, int threads) {
    bool odd = false;
    for (int i = thread; i < Fast<DH>::kTileBytes / 16; i += threads) {
        const uint4 u = *reinterpret_cast<const uint4 *>(vl + i * 16);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            odd |= (x[e] & 0x7F800000u) == 0x7F800000u || (x[e] & 0x7F80u) == 0x7F80u;
    }
    return odd;
}

template <int DH>
__device__ __forceinline__ void load_q(const ScoreArgs & a, const Rows & w, int qi, int head, bool live, int h,
                                       bf16x8 (&qf)[Fast<DH>::NST]) {
    const uint16_t * q = static_cast<const uint16_t *>(a.q) + (w.q0 + qi) * a.ldq + static_cast<int64_t>(head) * a.d;
#pragma unroll
    for (int st = 0; st < Fast<DH>::NST; ++st) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (live && (st / 4) * 64 + 32 * h + 8 * (st % 4) < a.d) u = *reinterpret_cast<const uint4 *>(q + (st / 4) * 64 + 32 * h + 8 * (st % 4));
        qf[st] = __builtin_bit_cast(bf16x8, u);
    }
}

template <int DH>
__device__ __forceinline__ TileSource<DH> tile_source(const ScoreArgs & a, const Rows & w) {
    TileSource<DH> s;
    s.k = uniform_ptr(reinterpret_cast<const char *>(static_cast<const uint16_t *>(a.k) + w.k0 * a.ldk + static_cast<int64_t>(w.kv) * a.d));
    s.v = uniform_ptr(reinterpret_cast<const char *>(static_cast<const uint16_t *>(a.v) + w.k0 * a.ldv + static_cast<int64_t>(w.kv) * a.d));
    s.ldk = a.ldk * 2;
    s.ldv = a.ldv * 2;
    s.nk = w.nk;
    s.zero = reinterpret_cast<uint64_t>(&g_score_zero[0]);
    asm volatile("" : "+s"(s.zero));
    return s;
}

// Many rows a segment: four waves of 32 rows share the key tiles, a ring of four
// slots of K and V.  The keys are walked from the last that is seen to the first:
// the tiles with hidden keys come first, each an exact step (maximum, weights, product),
// then one exact step on whole keys, after which every row has a base that one of its
// own scores set.  From there on tile j's step issues the products that do not depend on
// its weights, O += V P of the tile before and S of the next, and takes its weights while
// they run, without a maximum: a row's weights are redone with one where their sum passes
// 2^40.  With a bias that falls with the distance the nearest keys come first, so that is rare.
// Weights past 1 may take large values past what fp32 holds: where outputs pass 2^118 (512 splits of
// them can be joined) the tile is walked again with exact steps alone, whose weights are at most 1, as those
// of the other kernels are.  Bound by the vector instructions of the weights beside the products,
// and by the waits between the two: 8,192 tokens, 16 heads of 128, 0.53 to 0.56 ms (980 to 1,040 TFLOP/s; the
// matrix cores busy in 55% of the cycles), of 64 0.30 to 0.32 ms, with a cap 0.41, with a bias of both sides 0.45.
constexpr int kSlots = 4;
constexpr float kSumLimit = 0x1p40f;
constexpr float kOutLimit = 0x1p118f;

template <int DH, int MODE, bool WHOLE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) score_attn_rows_kernel(ScoreArgs a) {
    using F = Fast<DH>;
    constexpr int kMine = 2 * F::kUnits / 4;  // DMA instructions of a wave and tile
    __shared__ __align__(16) char lds[kSlots * 2 * F::kTileBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;
    Rows w;
    int split;
    if (!locate_work(a, 128, lane, w, split)) return;
    const int end = keys_end(a, w, w.row0 + 127);
    const int all = (end + F::kKeys - 1) / F::kKeys;
    const int first = static_cast<int>(static_cast<int64_t>(all) * split / w.splits);
    const int last = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / w.splits) - 1;
    const int n = last - first + 1;  // tiles, walked from `last` down: step i is tile last - i

    const int wave_row0 = w.row0 + wave * 32;
    const bool live = wave_row0 + r < w.rows;
    const int row = live ? wave_row0 + r : w.rows - 1;
    const int qi = row / a.group;
    const int head = w.kv * a.group + row % a.group;
    const RowScore rs = row_score<MODE>(a, head);
    const float cap_log2 = a.cap_log2;
    bf16x8 qf[F::NST];
    load_q<DH>(a, w, qi, head, live, h, qf);
    const int seen = keys_end(a, w, row) - 4 * h;
    const int pos = qi + w.shift - 4 * h;
    // Tiles below hold seen keys only, and with kBehind none after a query.
    const int first_pos = w.row0 / a.group + w.shift;
    const int whole = max(MODE & kBehind ? min(keys_all(a, w, w.row0), first_pos + 1) : keys_all(a, w, w.row0), 0) / F::kKeys;
    const int wave_end = wave_row0 < w.rows ? keys_end(a, w, wave_row0 + 31) : 0;

    TileSource<DH> src = tile_source<DH>(a, w);
    uint32_t off[kMine];
    tile_offsets<DH>(src, a.d, wave * kMine, lane, off);
    const uint32_t lds0 = lds_offset(&lds[0]);
    auto slot = [](int i) { return (i % kSlots) * 2 * F::kTileBytes; };
    auto issue = [&](int i) __attribute__((always_inline)) {
        tile_issue<DH, WHOLE>(src, last - i, wave * kMine, off, lds0 + slot(i), lane);
    };
    auto k_of = [&](int i) { return lds + slot(i); };
    auto v_of = [&](int i) { return lds + slot(i) + F::kTileBytes; };
    auto behind = [&](int i) { return static_cast<float>(pos - (last - i) * F::kKeys); };

    typename F::Out oacc;
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt) oacc[dt] = f32x16{};
    RowState st{-INFINITY, 0.0f};
    bool odd = false, past = false;
    // Exact steps: tiles with hidden keys, and one of whole keys.
    const int exact = min(n, max(last + 1 - whole, 0) + 1);
    if (n > 0) issue(0);
    if (n > 1) issue(1);
    typename F::Scores s_a, s_b;
    typename F::Weights p;
    int i = 0;
    auto exact_step = [&]() __attribute__((always_inline)) {
        if (i + 1 < n) wait_vmcnt(kMine);
        else wait_vmcnt(0);
        barrier_no_fence();
        if (i + 2 < n) issue(i + 2);
        const int tile = last - i;
        if (tile >= whole) odd |= tile_odd<DH>(v_of(i), tid, 256);
        if (tile * F::kKeys < wave_end) {
            tile_qk<DH>(k_of(i), qf, s_a, h, r);
            tile_exact<DH, MODE>(rs, cap_log2, s_a, p, oacc, st, behind(i), seen - tile * F::kKeys);
            tile_pv<DH>(v_of(i), p, oacc, lane);
        }
    };
    for (; i < exact; ++i) exact_step();
    // (The step as a scalar: taken for a lane's, it kept a second copy of the output alive through the
    // loop, and the compiler, out of registers, waited for every read of LDS: 475 us against 529 for the
    // capped prompts above.)
    i = __builtin_amdgcn_readfirstlane(i);
    if (i < __builtin_amdgcn_readfirstlane(n)) {
        // Steps exact .. n - 1, one tile's products behind its weights.  Slot use: step i
        // reads V of i - 1 and K of i + 1 while i + 2 lands.
        auto weights = [&](int i, typename F::Scores & s) __attribute__((always_inline)) {
            float sum = tile_weights<DH, MODE>(rs, cap_log2, s, p, st.base, behind(i));
            if (__builtin_expect(__ballot(!(sum <= kSumLimit)) != 0, 0)) {
                const float top = fmaxf(st.base, tile_max<DH, MODE>(rs, cap_log2, s, behind(i)));
                const float up = top == -INFINITY ? 0.0f : top;  // scores of minus infinity, or NaN, only
                const float keep = __builtin_amdgcn_exp2f(st.base - up);
                st.base = up;
                st.sum *= keep;
#pragma unroll
                for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[dt][e] *= keep;
                sum = tile_weights<DH, MODE>(rs, cap_log2, s, p, st.base, behind(i));
            }
            st.sum += sum;
        };
        if (i + 1 < n) wait_vmcnt(kMine);
        else wait_vmcnt(0);
        barrier_no_fence();
        tile_qk<DH>(k_of(i), qf, s_a, h, r);
        // The first: no product before it.
        if (i + 1 < n) {
            wait_vmcnt(0);
            barrier_no_fence();
            if (i + 2 < n) issue(i + 2);
            tile_qk<DH>(k_of(i + 1), qf, s_b, h, r);
        }
        weights(i, s_a);
        ++i;
        auto step = [&](typename F::Scores & now, typename F::Scores & next) __attribute__((always_inline)) {
            wait_vmcnt(0);
            barrier_no_fence();
            if (i + 2 < n) issue(i + 2);
            tile_pv<DH>(v_of(i - 1), p, oacc, lane);
            tile_qk<DH>(k_of(i + 1), qf, next, h, r);
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
        // (A sum of magnitudes: infinities and NaN stay in it.)
        float size[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) size[e & 3] += fabsf(oacc[dt][e]);
        past = live && !((size[0] + size[1]) + (size[2] + size[3]) < kOutLimit) && is_finite_bits(st.sum);
    }
    if (__builtin_expect(__syncthreads_or(odd || past), 0)) {
        if (__syncthreads_or(odd)) {
            for (int j = 0; j < 32; ++j)
                if (wave_row0 + j < w.rows)
                    row_alone<uint16_t, DH / 64>(a, w, wave_row0 + j, first * F::kKeys, (last + 1) * F::kKeys, lane,
                                                 w.splits > 1, split_slot(a, w, split, wave_row0 + j));
            return;
        }
        issue(0);  // (every wave is done with the slots)
        if (n > 1) issue(1);
#pragma unroll
        for (int dt = 0; dt < F::NDT; ++dt) oacc[dt] = f32x16{};
        st = {-INFINITY, 0.0f};
        for (i = 0; i < n; ++i) exact_step();
    }
    const float sum = lane_pair_sum(st.sum);
    if (!live) return;
    const int64_t part = split_slot(a, w, split, row);
    if (w.splits > 1) {
        if (h == 0) a.part_ml[part] = make_float2(st.base, sum);
        float * o = a.part + part * a.d;
#pragma unroll
        for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (WHOLE || dt * 32 + 8 * g + 4 * h < a.d)
                    *reinterpret_cast<float4 *>(o + dt * 32 + 8 * g + 4 * h) =
                        make_float4(oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]);
        return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t * o = static_cast<uint16_t *>(a.o) + (w.q0 + qi) * a.ldo + static_cast<int64_t>(head) * a.d;
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (WHOLE || dt * 32 + 8 * g + 4 * h < a.d)
                *reinterpret_cast<uint2 *>(o + dt * 32 + 8 * g + 4 * h) =
                    make_uint2(pack_bf16x2(oacc[dt][4 * g] * inv, oacc[dt][4 * g + 1] * inv),
                               pack_bf16x2(oacc[dt][4 * g + 2] * inv, oacc[dt][4 * g + 3] * inv));
}

// Few rows a segment (new tokens over caches): a workgroup has one tile of 32 rows
// and a chunk of the segment's keys, its two waves every second key tile of it, each
// through a ring of its own in LDS, with no barrier before the end, where the waves'
// results are joined.  Bound by reading the keys and values once (4.9 TB/s, where a copy
// reaches 4.85).  Two waves and two workgroups a CU: with four waves and one, the start and end
// of a chunk were not hidden (158 us against 142 for eight tokens over 170,161 keys).
//
// Segments of up to 32 rows are cut into chunks of a.chunk keys, an item each; so long
// and short caches of one call load the CUs alike.  Others have an item per 32 rows.
constexpr int kFewRows = 32;

constexpr int kFewWaves = 2, kFewStages = 2;  // 64 KB of LDS: two workgroups a CU
template <int DH> constexpr int kFewWaveBytes = kFewStages * 2 * Fast<DH>::kTileBytes;
template <int DH> constexpr int kFewBytes = kFewWaves * kFewWaveBytes<DH> + kFewWaves * 32 * 2 * static_cast<int>(sizeof(float));

// A wave's own LDS reads are done, and none is moved over this.
__device__ __forceinline__ void wave_reads_done() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

template <int DH, int MODE, bool WHOLE>
__global__ void __launch_bounds__(kFewWaves * 64) score_attn_few_kernel(ScoreArgs a) {
    using F = Fast<DH>;
    constexpr int kInstr = 2 * F::kUnits;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;
    Rows w;
    w.kv = static_cast<int>(blockIdx.x % a.kv_heads);
    const int item = static_cast<int>(blockIdx.x / a.kv_heads);
    if (!locate_rows(a, item, kFewRows, lane, w)) return;
    const bool live = w.row0 + r < w.rows;
    const int row = live ? w.row0 + r : w.rows - 1;
    const int qi = row / a.group;
    const int head = w.kv * a.group + row % a.group;
    int first = 0, last = (keys_end(a, w, w.row0 + kFewRows - 1) + F::kKeys - 1) / F::kKeys;
    if (w.chunks > 1) {
        first = w.chunk * (a.chunk / F::kKeys);
        last = min(last, first + a.chunk / F::kKeys);
    }
    const RowScore rs = row_score<MODE>(a, head);
    const float cap_log2 = a.cap_log2;
    TileSource<DH> src = tile_source<DH>(a, w);
    char * ring = smem + wave * kFewWaveBytes<DH>;
    const uint32_t lds0 = lds_offset(ring);
    uint32_t off[kInstr];
    tile_offsets<DH>(src, a.d, 0, lane, off);
    const int n = last - first > wave ? (last - first - wave + kFewWaves - 1) / kFewWaves : 0;
    auto tile = [&](int i) { return first + wave + kFewWaves * i; };
    auto slot = [](int i) { return i % kFewStages * 2 * F::kTileBytes; };
    auto issue = [&](int i) __attribute__((always_inline)) {
        tile_issue<DH, WHOLE>(src, tile(i), 0, off, lds0 + slot(i), lane);
    };
    if (n > 0) issue(0);
    bf16x8 qf[F::NST];
    load_q<DH>(a, w, qi, head, live, h, qf);
    const int seen = keys_end(a, w, row) - 4 * h;
    const int pos = qi + w.shift - 4 * h;
    const int whole = keys_all(a, w, w.row0) / F::kKeys;
    typename F::Out oacc;
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt) oacc[dt] = f32x16{};
    RowState st{-INFINITY, 0.0f};
    bool odd = false;
#pragma unroll
    for (int i = 1; i < kFewStages; ++i)
        if (i < n) issue(i);
    for (int i = 0; i < n; ++i) {
        wait_stages<kFewStages - 1, kInstr>(n - 1 - i);
        asm volatile("" ::: "memory");
        const char * kl = ring + slot(i);
        const char * vl = kl + F::kTileBytes;
        if (tile(i) >= whole) odd |= tile_odd<DH>(vl, lane, 64);
        typename F::Scores s;
        typename F::Weights p;
        tile_qk<DH>(kl, qf, s, h, r);
        tile_exact<DH, MODE>(rs, cap_log2, s, p, oacc, st, static_cast<float>(pos - tile(i) * F::kKeys),
                             seen - tile(i) * F::kKeys);
        tile_pv<DH>(vl, p, oacc, lane);
        wave_reads_done();
        if (i + kFewStages < n) issue(i + kFewStages);
    }
    const int64_t part = (static_cast<int64_t>(item) * a.kv_heads + w.kv) * kFewRows;  // this item's rows of partial results
    if (__syncthreads_or(odd)) {
        for (int j = wave; j < kFewRows; j += kFewWaves)
            if (w.row0 + j < w.rows)
                row_alone<uint16_t, DH / 64>(a, w, w.row0 + j, first * F::kKeys, last * F::kKeys, lane, w.chunks > 1,
                                             part + j);
        return;
    }
    // The waves' results: outputs in their own rings, bases and sums behind the rings.
    float * mine = reinterpret_cast<float *>(ring);
    float2 * ml = reinterpret_cast<float2 *>(smem + kFewWaves * kFewWaveBytes<DH>);
    const float sum = lane_pair_sum(st.sum);
    if (h == 0) ml[wave * 32 + r] = make_float2(st.base, sum);
#pragma unroll
    for (int dt = 0; dt < F::NDT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4 *>(mine + r * DH + dt * 32 + 8 * g + 4 * h) =
                make_float4(oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]);
    __syncthreads();
    const int jc = tid & 7;  // 8 threads a row
#pragma unroll
    for (int jr = tid >> 3; jr < kFewRows; jr += kFewWaves * 8) {
        if (w.row0 + jr >= w.rows) return;
        float base = -INFINITY;
#pragma unroll
        for (int i = 0; i < kFewWaves; ++i) base = fmaxf(base, ml[i * 32 + jr].x);
        const float ref = base == -INFINITY ? 0.0f : base;
        float total = 0.0f, f[kFewWaves];
#pragma unroll
        for (int i = 0; i < kFewWaves; ++i) {
            const float2 v = ml[i * 32 + jr];
            f[i] = __builtin_amdgcn_exp2f(v.x - ref);
            total += v.y * f[i];
        }
        const int token = (w.row0 + jr) / a.group;
        const int to_head = w.kv * a.group + (w.row0 + jr) % a.group;
        uint16_t * o = static_cast<uint16_t *>(a.o) + (w.q0 + token) * a.ldo + static_cast<int64_t>(to_head) * a.d;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        if (w.chunks > 1 && jc == 0) a.part_ml[part + jr] = make_float2(base, total);
#pragma unroll
        for (int c = jc * 4; c < DH; c += 32) {
            if (!WHOLE && c >= a.d) break;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kFewWaves; ++i) {
                const float4 x = *reinterpret_cast<const float4 *>(
                    reinterpret_cast<const float *>(smem + i * kFewWaveBytes<DH>) + jr * DH + c);
                v[0] += x.x * f[i]; v[1] += x.y * f[i]; v[2] += x.z * f[i]; v[3] += x.w * f[i];
            }
            if (w.chunks > 1)
                *reinterpret_cast<float4 *>(a.part + (part + jr) * a.d + c) = make_float4(v[0], v[1], v[2], v[3]);
            else
                *reinterpret_cast<uint2 *>(o + c) =
                    make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
        }
    }
}

// Joins the chunks of a (query, head): eight groups of 32 lanes, each every eighth chunk, then
// their results in order.  Lane l of a group has dims DH / 32 l on.
template <int DH>
__global__ void __launch_bounds__(256) score_join_few_kernel(ScoreArgs a) {
    constexpr int V = DH / 32, kGroups = 8;
    typedef float vec __attribute__((ext_vector_type(V)));
    __shared__ float2 ml[kGroups];
    __shared__ float acc_of[kGroups][DH];
    const int lane = threadIdx.x & 63, l32 = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int qi = static_cast<int>(blockIdx.x / a.heads);
    const int head = static_cast<int>(blockIdx.x % a.heads);
    Rows w;
    w.kv = head / a.group;
    int item;
    if (!locate_query(a, qi, kFewRows, lane, w, item) || w.chunks <= 1) return;
    if (item + w.chunks > a.tiles) return;  // (of segments that overlap: no such items)
    const int row = (qi - w.q0) * a.group + head % a.group;
    const int64_t at = (static_cast<int64_t>(item) * a.kv_heads + w.kv) * kFewRows + row;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * kFewRows;
    const bool in = l32 * V < a.d;
    float m = -INFINITY, l = 0.0f;
    vec acc = {};
#pragma unroll 4
    for (int i = grp; i < w.chunks; i += kGroups) {
        const float2 p = a.part_ml[at + i * step];
        vec o = {};
        if (in) o = *reinterpret_cast<const vec *>(a.part + (at + i * step) * a.d + l32 * V);
        const float up = fmaxf(m, p.x), ref = up == -INFINITY ? 0.0f : up;
        const float keep = __builtin_amdgcn_exp2f(m - ref), f = __builtin_amdgcn_exp2f(p.x - ref);
        l = l * keep + p.y * f;
#pragma unroll
        for (int c = 0; c < V; ++c) acc[c] = acc[c] * keep + o[c] * f;
        m = up;
    }
    if (l32 == 0) ml[grp] = make_float2(m, l);
    *reinterpret_cast<vec *>(&acc_of[grp][l32 * V]) = acc;
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
        v += acc_of[i][dim] * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    static_cast<uint16_t *>(a.o)[qi * a.ldo + static_cast<int64_t>(head) * a.d + dim] = f32_to_bf16(v * inv);
}

// Joins the splits of a (query, head), in their order: a thread has four of its dims.
template <typename T>
__global__ void __launch_bounds__(256) score_join_kernel(ScoreArgs a) {
    const int quads = (a.d + 3) / 4;
    const int64_t rows = a.total_q * a.heads;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / quads, query = row / a.heads;
    const int dim = static_cast<int>(i % quads) * 4, dims = min(4, a.d - dim);
    if (row >= rows || query < a.cu_q[0] || query >= a.cu_q[a.nseg]) return;  // (rows of no segment)
    int seg = 0;  // the last that starts at or before the query
    for (int left = a.nseg; left > 1;) {
        const int half = left / 2;
        if (a.cu_q[seg + half] <= query) seg += half;
        left -= half;
    }
    const int splits = segment_splits(a, load_segment(a, seg).nk);
    if (splits == 1) return;  // written whole
    float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const int64_t at = s * rows + row;
        const float2 ml = a.part_ml[at];
        const float * o = a.part + at * a.d + dim;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (dims == 4) {
            __builtin_memcpy(v, o, 16);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c < dims) v[c] = o[c];
        }
        const float up = fmaxf(m, ml.x), ref = up == -INFINITY ? 0.0f : up;
        const float keep = exp2f(m - ref), f = exp2f(ml.x - ref);  // 0 for a split that saw nothing
        l = l * keep + ml.y * f;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = acc[c] * keep + v[c] * f;
        m = up;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T * o = static_cast<T *>(a.o) + row / a.heads * a.ldo + row % a.heads * a.d + dim;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c < dims) store_f32(o + c, acc[c] * inv);
}

// tile_start[s] = items of the segments before s, for more segments than a wave's lanes.
__global__ void __launch_bounds__(1024) score_tiles_kernel(ScoreArgs a, int rows_per_tile,
                                                           int64_t * __restrict__ tile_start) {
    __shared__ int64_t waves[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t before = 0;
    for (int s0 = 0; s0 < a.nseg; s0 += 1024) {
        const int s = s0 + tid;
        int64_t tiles = 0;
        if (s < a.nseg) {
            const Segment g = load_segment(a, s);
            tiles = segment_items(g.nq, g.nk, a.group, rows_per_tile, a.chunk);
        }
        int64_t sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t below = __shfl_up(sum, d, 64);
            if (lane >= d) sum += below;
        }
        if (lane == 63) waves[wave] = sum;
        __syncthreads();
        int64_t ahead = before, all = 0;
        for (int i = 0; i < 16; ++i) {
            if (i < wave) ahead += waves[i];
            all += waves[i];
        }
        if (s < a.nseg) tile_start[s] = ahead + sum - tiles;
        before += all;
        __syncthreads();
    }
    if (tid == 0) tile_start[a.nseg] = before;
}

// ---- host -----------------------------------------------------------------------

constexpr int kScoreMaxDim = 256;
constexpr int64_t kScoreMaxRows = INT32_MAX - 1023;  // rows and keys are counted in 32 bits, a tile past their end
constexpr int kWaveSegments = 64;   // segments that a wave's lanes hold; more take a table
constexpr int kRowTile = 128;
constexpr int64_t kSplitGrid = 512; // workgroups (two a CU) up to which a call's keys are split
// fp32: one and a half rounds of the two workgroups a CU (heads up to 64), or two of its one.  Twelve calls of
// 256 to 4,000 queries over 1,000 to 8,192 keys, 4 to 32 heads, geometric mean: heads of 64 the same with 512
// (single calls 20% faster to 24% slower) and 2% slower with 1024; heads of 128 23% slower with 256, 7% with 768.
constexpr int64_t kSplitGridF32 = 768, kSplitGridF32Wide = 512;

int64_t row_tiles(int64_t total_q, int nseg, int group) { return total_q * group / kRowTile + nseg; }

// Splits of the longest segment's keys at most: as many as keep row tiles * key/value heads * splits
// within `grid`.  (How long it is the host does not know: all the keys may be its.)
int score_splits(int64_t grid, int nseg, int64_t total_q, int64_t total_k, int kv_heads, int group) {
    const int64_t fit = grid / (row_tiles(total_q, nseg, group) * kv_heads);
    return static_cast<int>(std::max<int64_t>(1, std::min(fit, total_k / kSplitKeys)));
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Rows of partial results at most: a split call has at most the largest split grid's workgroups of
// kRowTile rows, whatever its other sizes; so the size never falls as a call grows.
int64_t split_rows(int64_t total_q, int64_t total_k, int heads) {
    constexpr int64_t kGrid = std::max({kSplitGrid, kSplitGridF32, kSplitGridF32Wide}), kMost = kGrid * kRowTile;
    const int64_t most = std::max<int64_t>(1, std::min(kGrid, total_k / kSplitKeys));
    if (most == 1) return 0;
    return std::min(kMost, total_q > kMost ? kMost : total_q * heads * most);
}

// Few rows a segment: keys of a chunk, so that a call has about kFewItems items, two rounds of two
// workgroups a CU.  Ragged caches want them: eight tokens over 170,161 keys in caches of 1 to 65,536, 8 key/value
// heads of 128: 138 us (5.05 TB/s), with 512 items 168, with 2,048 149.  Of twelve other calls (1 to 128
// tokens, caches alike or one) five take the same with 512 and seven 3 to 24% less; 2,048 costs 6% on average.
// At least 128 keys, a tile or two for each wave: one token over 1,501 keys, 16 heads of 64, 10.2 us against
// 11.5 with 256; of the others four are 5 to 23% slower with 256 and two 21 to 23% faster.
constexpr int64_t kFewItems = 1024;
constexpr int64_t kFewKeys = 128;  // at least, and a multiple of
int64_t few_chunk(int64_t total_k, int kv_heads) {
    const int64_t keys = (total_k * kv_heads + kFewItems - 1) / kFewItems;
    return std::min<int64_t>(std::max<int64_t>(1, (keys + kFewKeys - 1) / kFewKeys) * kFewKeys, 1 << 30);
}
bool few_rows(int64_t total_q, int nseg, int group) { return total_q * group <= static_cast<int64_t>(kFewRows) * nseg; }
int64_t few_items(int64_t total_q, int64_t total_k, int nseg, int kv_heads, int group) {
    return total_q * group / kFewRows + total_k / few_chunk(total_k, kv_heads) + nseg + 1;
}
// Rows of partial results of any such call of up to these sizes: its queries' rows fill at
// most nseg tiles, and total_k / chunk is at most both total_k / kFewKeys and kFewItems / kv_heads.
int64_t few_part_rows(int64_t total_k, int nseg, int kv_heads) {
    return ((2 * static_cast<int64_t>(nseg) + 3) * kv_heads + std::min(total_k / kFewKeys * kv_heads, kFewItems)) * kFewRows;
}

// Rows of partial results of any call of up to these sizes, and the workspace that holds them.
int64_t score_part_rows(int nseg, int64_t total_q, int64_t total_k, int heads, int kv_heads) {
    return std::max(split_rows(total_q, total_k, heads), few_part_rows(total_k, nseg, kv_heads));
}
size_t score_workspace(int nseg, int64_t part_rows, int head_dim) {
    const size_t rows = static_cast<size_t>(part_rows);
    return round256((static_cast<size_t>(nseg) + 1) * sizeof(int64_t)) + round256(rows * sizeof(float2)) +
           round256(rows * head_dim * sizeof(float));
}

template <typename T, int DP, bool SPLIT = false>
int launch_any(const ScoreArgs & a, int64_t blocks, hipStream_t s) {
    constexpr int plain = AnyTile<T, DP, false>::kBytes, smem = SPLIT ? std::max(plain, AnyTile<T, DP, true>::kBytes) : plain;
    auto kernel = &score_attn_any_kernel<T, DP, SPLIT>;
    if constexpr (smem > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), smem, done, "hipFuncSetAttribute(score_attn)")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), smem, s, a);
    return check_launch("scored attention");
}

template <typename T>
int run_any(const ScoreArgs & a, int64_t blocks, hipStream_t s) {
    if constexpr (sizeof(T) == 4) {
        if (a.d <= 128 && a.scale_log2 <= 0x1p41f) {
            if (a.d <= 64) return launch_any<T, 64, true>(a, blocks, s);
            return launch_any<T, 128, true>(a, blocks, s);
        }
    }
    if (a.d <= 64) return launch_any<T, 64>(a, blocks, s);
    if (a.d <= 128) return launch_any<T, 128>(a, blocks, s);
    return launch_any<T, 256>(a, blocks, s);
}

// kernel<mode of the call>
template <bool BEHIND, typename F> int with_mode(const ScoreArgs & a, F && launch) {
    auto capped = [&](auto rest) {
        constexpr int kRest = decltype(rest)::value;
        if (a.cap_log2 == 0.0f) return launch(rest);
        if (a.cap_log2 <= kNearCap * kLog2e) return launch(std::integral_constant<int, kCap | kRest>{});
        return launch(std::integral_constant<int, kCap | kFar | kRest>{});
    };
    if constexpr (BEHIND)
        if (a.slopes && a.causal) return capped(std::integral_constant<int, kBias | kBehind>{});
    if (a.slopes) return capped(std::integral_constant<int, kBias>{});
    return capped(std::integral_constant<int, 0>{});
}

template <int DH, bool WHOLE>
int run_rows(const ScoreArgs & a, int64_t blocks, hipStream_t s) {
    return with_mode<true>(a, [&](auto mode) {
        hipLaunchKernelGGL((score_attn_rows_kernel<DH, decltype(mode)::value, WHOLE>), dim3(static_cast<unsigned>(blocks)),
                           dim3(256), 0, s, a);
        return check_launch("scored attention");
    });
}

template <int DH, bool WHOLE>
int run_few(const ScoreArgs & a, int64_t blocks, bool join, hipStream_t s) {
    const int rc = with_mode<false>(a, [&](auto mode) {
        auto kernel = &score_attn_few_kernel<DH, decltype(mode)::value, WHOLE>;
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), kFewBytes<DH>, done, "hipFuncSetAttribute(score_attn_few)")) return rc;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kFewWaves * 64), kFewBytes<DH>, s, a);
        return check_launch("scored attention of few rows");
    });
    if (rc || !join) return rc;
    hipLaunchKernelGGL(score_join_few_kernel<DH>, dim3(static_cast<unsigned>(a.total_q * a.heads)), dim3(256), 0, s, a);
    return check_launch("scored attention join");
}

bool rows_of_pieces(const void * p, int64_t ld, int d, int elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * elem % 16 == 0 && d * elem % 16 == 0;
}

} // namespace
} // namespace pxs

using namespace pxs;

extern "C" {

size_t pxs_attention_scores_workspace_bytes(int nseg, int64_t total_q, int64_t total_k, int heads, int kv_heads,
                                            int head_dim) {
    if (nseg <= 0 || total_q <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 256;
    return score_workspace(nseg, score_part_rows(nseg, total_q, std::max<int64_t>(total_k, 0), heads, kv_heads), head_dim);
}

int pxs_varlen_attention_scores(int dtype, const void * q, int64_t ld_q, const void * k, int64_t ld_k, const void * v,
                                int64_t ld_v, const int64_t * cu_q, const int64_t * cu_k, int nseg, int64_t total_q,
                                int64_t total_k, int heads, int kv_heads, int head_dim, float scale, float cap,
                                const float * slopes, int causal, const int64_t * prefix, void * o, int64_t ld_o,
                                void * workspace, void * stream) {
    PXS_CHECK_WORKSPACE(workspace, "pxs_varlen_attention_scores");
    PXS_CHECK(dtype == PXS_F32 || dtype == PXS_BF16, PXS_ERR_ARG, "pxs_varlen_attention_scores: bad dtype");
    PXS_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 65535, PXS_ERR_ARG,
              "pxs_varlen_attention_scores: heads must be a multiple of kv_heads, up to 65535");
    PXS_CHECK(head_dim > 0 && head_dim <= kScoreMaxDim, PXS_ERR_ARG,
              "pxs_varlen_attention_scores: head_dim must be in 1..256");
    PXS_CHECK(scale > 0.0f && std::isfinite(scale), PXS_ERR_ARG,
              "pxs_varlen_attention_scores: scale must be finite and positive");
    PXS_CHECK(cap >= 0.0f && std::isfinite(cap), PXS_ERR_ARG,
              "pxs_varlen_attention_scores: cap must be finite, and 0 for none");
    PXS_CHECK(causal == 0 || causal == 1, PXS_ERR_ARG, "pxs_varlen_attention_scores: causal must be 0 or 1");
    PXS_CHECK(causal || !prefix, PXS_ERR_ARG, "pxs_varlen_attention_scores: a prefix needs the causal mask");
    PXS_CHECK(std::isfinite(scale * kLog2e) && (cap == 0.0f || std::isfinite(scale / cap)),
              PXS_ERR_ARG, "pxs_varlen_attention_scores: scale and cap out of range");
    PXS_CHECK(nseg >= 0 && total_q >= 0 && total_k >= 0 && total_q <= kScoreMaxRows / (heads / kv_heads) &&
                  total_k <= kScoreMaxRows,
              PXS_ERR_ARG, "pxs_varlen_attention_scores: row counts must be in 0..2^31 - 1024, as total_q * heads / kv_heads");
    const int64_t wq = static_cast<int64_t>(heads) * head_dim, wk = static_cast<int64_t>(kv_heads) * head_dim;
    PXS_CHECK(ld_q >= wq && ld_k >= wk && ld_v >= wk && ld_o >= wq, PXS_ERR_ARG,
              "pxs_varlen_attention_scores: row stride smaller than heads * head_dim");
    if (nseg == 0 || total_q == 0) return PXS_OK;
    PXS_CHECK(q && o && cu_q && cu_k && workspace && (total_k == 0 || (k && v)), PXS_ERR_ARG,
              "pxs_varlen_attention_scores: null pointer");
    hipStream_t s = as_stream(stream);
    ScoreArgs a{};
    a.q = q; a.k = k; a.v = v; a.ldq = ld_q; a.ldk = ld_k; a.ldv = ld_v;
    a.cu_q = cu_q; a.cu_k = cu_k; a.nseg = nseg; a.total_q = total_q; a.total_k = total_k;
    a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.d = head_dim;
    // (Caps near the largest number, or that products of 2^113 at least are small against, cap nothing that
    // fp32 holds: taken lower, so that scale / cap stays a normal number.  A multiplier past the largest
    // number is cut, so that a product of zero stays zero under it.)
    constexpr float kLargest = std::numeric_limits<float>::max();
    cap = std::min({cap, kLargest / 4, scale * 0x1p126f});
    a.scale_log2 = scale * kLog2e;
    a.cap_log2 = cap * kLog2e;
    a.over_cap = cap > 0.0f ? scale / cap : 0.0f;
    a.exp_mul = std::min(2.0f * kLog2e * a.over_cap, kLargest);
    a.slopes = slopes; a.causal = causal; a.prefix = prefix; a.o = o; a.ldo = ld_o;
    const int elem = dtype == PXS_BF16 ? 2 : 4;
    a.vec = rows_of_pieces(q, ld_q, head_dim, elem) && rows_of_pieces(k, ld_k, head_dim, elem) &&
            rows_of_pieces(v, ld_v, head_dim, elem);
    // The fast kernels' 32-bit offsets within a key tile hold row strides below 2^24.
    const bool fast = dtype == PXS_BF16 && head_dim <= 128 && a.vec && ld_k < (1 << 24) &&
                      ld_v < (1 << 24) && reinterpret_cast<uintptr_t>(o) % 8 == 0 && ld_o % 4 == 0;
    const bool few = fast && few_rows(total_q, nseg, a.group);
    a.splits = 1;
    int64_t blocks, part_rows = 0;
    if (few) {
        a.chunk = static_cast<int>(few_chunk(total_k, kv_heads));
        a.tiles = few_items(total_q, total_k, nseg, kv_heads, a.group);
        blocks = a.tiles * kv_heads;
        part_rows = blocks * kFewRows;
    } else {
        a.tiles = row_tiles(total_q, nseg, a.group);
        const int64_t grid = dtype == PXS_BF16 ? kSplitGrid : head_dim <= 64 ? kSplitGridF32 : kSplitGridF32Wide;
        a.splits = score_splits(grid, nseg, total_q, total_k, kv_heads, a.group);
        blocks = a.tiles * kv_heads * a.splits;
        if (a.splits > 1) part_rows = a.splits * total_q * heads;
    }
    PXS_CHECK(blocks <= UINT32_MAX / 256 && (!few || total_q * heads <= UINT32_MAX / 256), PXS_ERR_ARG,
              "attention grid too large");
    // (The bounds that the workspace's size is made of hold for every rule above.)
    PXS_CHECK(part_rows <= score_part_rows(nseg, total_q, total_k, heads, kv_heads), PXS_ERR_ARG,
              "pxs_varlen_attention_scores: partial results past the workspace");
    char * ws = static_cast<char *>(workspace);
    if (nseg > kWaveSegments) {
        a.tile_start = reinterpret_cast<int64_t *>(ws);
        hipLaunchKernelGGL(score_tiles_kernel, dim3(1), dim3(1024), 0, s, a, few ? kFewRows : kRowTile,
                           reinterpret_cast<int64_t *>(ws));
        if (int rc = check_launch("scored attention tiles")) return rc;
    }
    ws += round256((static_cast<size_t>(nseg) + 1) * sizeof(int64_t));
    a.part_ml = reinterpret_cast<float2 *>(ws);
    a.part = reinterpret_cast<float *>(ws + round256(static_cast<size_t>(part_rows) * sizeof(float2)));
    if (few) {
        const bool join = total_k > a.chunk;  // otherwise no segment is cut
        if (head_dim == 64) return run_few<64, true>(a, blocks, join, s);
        if (head_dim == 128) return run_few<128, true>(a, blocks, join, s);
        return head_dim < 64 ? run_few<64, false>(a, blocks, join, s) : run_few<128, false>(a, blocks, join, s);
    }
    int rc;
    if (fast && head_dim == 64) rc = run_rows<64, true>(a, blocks, s);
    else if (fast && head_dim == 128) rc = run_rows<128, true>(a, blocks, s);
    else if (fast) rc = head_dim < 64 ? run_rows<64, false>(a, blocks, s) : run_rows<128, false>(a, blocks, s);
    else rc = dtype == PXS_F32 ? run_any<float>(a, blocks, s) : run_any<uint16_t>(a, blocks, s);
    if (rc || a.splits == 1) return rc;
    const dim3 grid(grid_for(total_q * heads * ((head_dim + 3) / 4), 256));
    if (dtype == PXS_F32) hipLaunchKernelGGL(score_join_kernel<float>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(score_join_kernel<uint16_t>, grid, dim3(256), 0, s, a);
    return check_launch("scored attention join");
}

} // extern "C"
