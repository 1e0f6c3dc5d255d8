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

#include <algorithm>
#include <atomic>
#include <cmath>

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
    int64_t total_q;
    const int64_t * tile_start;  // [nseg + 1] row tiles before each segment; null: at most 64 segments
    int heads, kv_heads, group, d;
    float scale_log2;            // scale * log2(e), or with a cap scale / cap
    float cap_log2;              // cap * log2(e); 0: no cap
    const float * slopes;        // [heads] or null
    int causal;
    const int64_t * prefix;      // [nseg] or null
    void * o;
    int64_t ldo;
    int vec;                     // rows of q, k and v in whole 16-byte pieces
    int64_t tiles;               // row tiles launched (bound)
    int splits;
    float * part;                // [splits][total_q][heads][d] unnormalised outputs
    float2 * part_ml;            // [splits][total_q][heads] maxima (log2 units) and sums
};

// A workgroup's rows: a tile of a segment and key/value head, and the keys that its rows see.
struct Rows {
    int seg;
    int kv;
    int64_t q0, k0;       // the segment's first query and key
    int64_t nq, nk;
    int64_t row0;         // first row of the tile
    int64_t rows;         // of the segment: nq * group
    int64_t shift;        // position of query i: i + shift
    int64_t prefix;
};

// Row tile t of `rows_per_tile` rows (a power of two); false past the last.
__device__ __forceinline__ bool locate_rows(const ScoreArgs & a, int64_t t, int rows_per_tile, int lane, Rows & w) {
    const int shift = 31 - __clz(rows_per_tile);
    int64_t first;
    if (a.tile_start) {
        if (t >= a.tile_start[a.nseg]) return false;
        w.seg = find_segment(a.tile_start, a.nseg, t, lane);
        first = a.tile_start[w.seg];
    } else {
        int64_t tiles = 0;
        if (lane < a.nseg)
            tiles = ((a.cu_q[lane + 1] - a.cu_q[lane]) * a.group + rows_per_tile - 1) >> shift;
        int64_t end = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t below = __shfl_up(end, d, 64);
            if (lane >= d) end += below;
        }
        const uint64_t before = __ballot(lane < a.nseg && end <= t);  // segments that end at or before t
        w.seg = __popcll(before);
        if (w.seg >= a.nseg) return false;
        first = __shfl(end - tiles, w.seg, 64);
    }
    w.seg = __builtin_amdgcn_readfirstlane(w.seg);
    w.q0 = a.cu_q[w.seg];
    w.k0 = a.cu_k[w.seg];
    w.nq = a.cu_q[w.seg + 1] - w.q0;
    w.nk = a.cu_k[w.seg + 1] - w.k0;
    w.rows = w.nq * a.group;
    w.row0 = (t - first) * rows_per_tile;
    w.shift = w.nk - w.nq;
    w.prefix = a.causal && a.prefix ? a.prefix[w.seg] : 0;
    return true;
}

// One past the last key that any of the rows up to `row` (inclusive) sees.
__device__ __forceinline__ int64_t keys_end(const ScoreArgs & a, const Rows & w, int64_t row) {
    if (!a.causal) return w.nk;
    const int64_t last = min(row, w.rows - 1) / a.group;
    return min(w.nk, max(last + w.shift + 1, max(w.prefix, int64_t(0))));
}
// The keys that every row from `row` on sees: all below.
__device__ __forceinline__ int64_t keys_all(const ScoreArgs & a, const Rows & w, int64_t row) {
    if (!a.causal) return w.nk;
    return min(w.nk, max(row / a.group + w.shift + 1, max(w.prefix, int64_t(0))));
}

// A score in log2 units, from a product q . k and the key's distance behind the query.
__device__ __forceinline__ float score_log2(const ScoreArgs & a, float dot, float slope_log2, float away) {
    float z = dot * a.scale_log2;
    if (a.cap_log2 > 0.0f) z = a.cap_log2 * tanhf(z);
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
template <typename T, int NC>
__device__ void row_alone(const ScoreArgs & a, const Rows & w, int64_t row, int64_t key0, int64_t key1, int lane,
                          int64_t slot_split) {
    const int64_t i = row / a.group;
    const int head = w.kv * a.group + static_cast<int>(row % a.group);
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
    const int64_t end = min(key1, keys_end(a, w, row));
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
    const int64_t slot = (slot_split * a.total_q + w.q0 + i) * a.heads + head;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN sum stays NaN)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int dim = lane + 64 * c;
        if (dim >= a.d) continue;
        if (a.splits > 1) a.part[slot * a.d + dim] = acc[c];
        else store_f32(static_cast<T *>(a.o) + (w.q0 + i) * a.ldo + static_cast<int64_t>(head) * a.d + dim, acc[c] * inv);
    }
    if (a.splits > 1 && lane == 0) a.part_ml[slot] = make_float2(m, l);
}

// Any dtype, head size up to DP, stride and alignment.  Four waves of 32 rows
// share tiles of kKeys keys, staged through registers into LDS (V transposed).  As in
// attention.hip a wave computes S^T = K Q^T, so that a lane owns one row and half of
// its scores, and O^T += V^T P^T with P straight from those registers.
template <typename T, int DP> struct AnyTile {
    static constexpr int kKeys = DP == 64 ? 64 : 32;
    static constexpr int kKPitch = DP * static_cast<int>(sizeof(T)) + 16;
    static constexpr int kVPitch = kKeys * static_cast<int>(sizeof(T)) + (sizeof(T) == 2 ? 8 : 16);
    static constexpr int kBytes = kKeys * kKPitch + DP * kVPitch;
};

template <typename T, int DP>
__global__ void __launch_bounds__(256) score_attn_any_kernel(ScoreArgs a) {
    using Tile = AnyTile<T, DP>;
    constexpr int kVec = 16 / static_cast<int>(sizeof(T)), kKeys = Tile::kKeys, KT = kKeys / 32, DT = DP / 32;
    constexpr int kPieces = DP / kVec;  // 16-byte pieces of a padded row
    extern __shared__ __align__(16) char smem[];
    char * k_lds = smem;
    char * vt_lds = smem + kKeys * Tile::kKPitch;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, r = lane & 31;

    // The row tiles of a key/value head and split from the last, which sees most, to the first.
    const int64_t t = a.tiles - 1 - blockIdx.x % a.tiles;
    const int rest = static_cast<int>(blockIdx.x / a.tiles);
    const int split = rest % a.splits;
    Rows w;
    w.kv = rest / a.splits;
    if (!locate_rows(a, t, 128, lane, w)) return;
    const int64_t end = keys_end(a, w, w.row0 + 127);
    const int64_t key_tiles = (end + kKeys - 1) / kKeys;
    const int64_t kt_first = key_tiles * split / a.splits, kt_last = key_tiles * (split + 1) / a.splits;

    const T * k = static_cast<const T *>(a.k) + w.k0 * a.ldk + static_cast<int64_t>(w.kv) * a.d;
    const T * v = static_cast<const T *>(a.v) + w.k0 * a.ldv + static_cast<int64_t>(w.kv) * a.d;

    // This lane's row and its Q fragment (dims h DP/2 .. h DP/2 + DP/2 - 1).
    const int64_t wave_row0 = w.row0 + wave * 32;
    const int64_t row = wave_row0 + r;
    const bool live = row < w.rows;
    const int64_t qi = (live ? row : 0) / a.group;
    const int head = w.kv * a.group + static_cast<int>((live ? row : 0) % a.group);
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    T qv[DP / 2];
#pragma unroll
    for (int c = 0; c < DP / 2 / kVec; ++c) {
        T tmp[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) tmp[e] = T(0);
        if (live)
            load_dims<T>(static_cast<const T *>(a.q) + (w.q0 + qi) * a.ldq + static_cast<int64_t>(head) * a.d,
                         h * (DP / 2) + c * kVec, a.d, a.vec, tmp);
#pragma unroll
        for (int e = 0; e < kVec; ++e) qv[c * kVec + e] = tmp[e];
    }
    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    const int64_t my_end = live ? keys_end(a, w, row) : 0;  // keys >= my_end are masked
    const int64_t wave_all = keys_all(a, w, wave_row0);     // keys below are seen by all of the wave's rows
    const int64_t tile_all = keys_all(a, w, w.row0);
    bool again = false;

    for (int64_t kt0 = kt_first * kKeys; kt0 < kt_last * kKeys; kt0 += kKeys) {
        __syncthreads();
        bool odd = false;
        for (int c = tid; c < kKeys * kPieces; c += 256) {
            const int key = c / kPieces, piece = c % kPieces;
            T kk[kVec], vv[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) kk[e] = vv[e] = T(0);
            if (kt0 + key < w.nk) {
                load_dims<T>(k + (kt0 + key) * a.ldk, piece * kVec, a.d, a.vec, kk);
                load_dims<T>(v + (kt0 + key) * a.ldv, piece * kVec, a.d, a.vec, vv);
            }
            *reinterpret_cast<uint4 *>(k_lds + key * Tile::kKPitch + piece * 16) = *reinterpret_cast<const uint4 *>(kk);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                odd |= !is_finite_bits(load_f32(&vv[e]));
                *reinterpret_cast<T *>(vt_lds + (piece * kVec + e) * Tile::kVPitch + key * static_cast<int>(sizeof(T))) = vv[e];
            }
        }
        // A tile with keys that some row does not see, and values that are not finite.
        again |= __syncthreads_or(odd && min(kt0 + kKeys, w.nk) > tile_all);

        f32x16 s[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            s[kt] = f32x16{};
            const char * krow = k_lds + (kt * 32 + r) * Tile::kKPitch;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int st = 0; st < DP / 16; ++st) {
                    const bf16x8 kf = *reinterpret_cast<const bf16x8 *>(krow + h * DP + st * 16);
                    bf16x8 qf;
#pragma unroll
                    for (int e = 0; e < 8; ++e) qf[e] = __builtin_bit_cast(__bf16, qv[st * 8 + e]);
                    s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf, s[kt], 0, 0, 0);
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
        // Register e of sub-tile kt holds key kt * 32 + 8 (e / 4) + 4 h + e % 4.
        const bool masked = kt0 + kKeys > wave_all || kt0 + kKeys > w.nk;
        const int behind = static_cast<int>(qi + w.shift - kt0), seen = static_cast<int>(my_end - kt0);
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int key = kt * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                float z = score_log2(a, s[kt][e], slope, static_cast<float>(behind - key));
                if (masked && key >= seen) z = -INFINITY;
                s[kt][e] = z;
                top = fmaxf(top, z);
            }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = fmaxf(m, top);
        const float base = up == -INFINITY ? 0.0f : up;  // nothing seen yet: every weight is 0
        const float keep = exp2f(m - base);
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = exp2f(s[kt][e] - base);
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
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    bf16x8 p;  // weights round to bf16, as the values they multiply are
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = static_cast<__bf16>(s[kt][8 * u + e]);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const char * vrow = vt_lds + (dt * 32 + r) * Tile::kVPitch;
                        const int key = kt * 32 + 16 * u + 4 * h;
                        const uint2 lo = *reinterpret_cast<const uint2 *>(vrow + key * 2);
                        const uint2 hi = *reinterpret_cast<const uint2 *>(vrow + (key + 8) * 2);
                        oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            __builtin_bit_cast(bf16x8, make_uint4(lo.x, lo.y, hi.x, hi.y)), p, oacc[dt], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const f32x4 vf = *reinterpret_cast<const f32x4 *>(vt_lds + (dt * 32 + r) * Tile::kVPitch +
                                                                          (kt * 32 + 8 * i + 4 * h) * 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[j], s[kt][4 * i + j], oacc[dt], 0, 0, 0);
                    }
            }
        }
    }
    if (again) {
        for (int i = 0; i < 32; ++i)
            if (wave_row0 + i < w.rows)
                row_alone<T, DP / 64>(a, w, wave_row0 + i, kt_first * kKeys, kt_last * kKeys, lane, split);
        return;
    }
    if (!live) return;
    const int64_t slot = (static_cast<int64_t>(split) * a.total_q + w.q0 + qi) * a.heads + head;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T * o = static_cast<T *>(a.o) + (w.q0 + qi) * a.ldo + static_cast<int64_t>(head) * a.d;
    if (a.splits > 1 && h == 0) a.part_ml[slot] = make_float2(m, l);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int dim = dt * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (dim >= a.d) continue;
            if (a.splits > 1) a.part[slot * a.d + dim] = oacc[dt][e];
            else store_f32(o + dim, oacc[dt][e] * inv);
        }
}

// Joins the splits of a row: one wave per (query, head), in the splits' order.
template <typename T>
__global__ void __launch_bounds__(256) score_join_kernel(ScoreArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t rows = a.total_q * a.heads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= rows || row < a.cu_q[0] * a.heads || row >= a.cu_q[a.nseg] * a.heads) return;  // (rows of no segment)
    float m = -INFINITY;
    for (int i = 0; i < a.splits; ++i) m = fmaxf(m, a.part_ml[i * rows + row].x);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < a.splits; ++i) {
        const float2 ml = a.part_ml[i * rows + row];
        if (ml.y == 0.0f) continue;  // saw nothing
        const float f = exp2f(ml.x - base);
        l += ml.y * f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < a.d) acc[c] += a.part[(i * rows + row) * a.d + lane + 64 * c] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T * o = static_cast<T *>(a.o) + row / a.heads * a.ldo + row % a.heads * a.d;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < a.d) store_f32(o + lane + 64 * c, acc[c] * inv);
}

// tile_start[s] = row tiles of the segments before s, for more segments than a wave's lanes.
__global__ void __launch_bounds__(1024) score_tiles_kernel(const int64_t * __restrict__ cu_q, int nseg, int group,
                                                           int rows_per_tile, int64_t * __restrict__ tile_start) {
    __shared__ int64_t waves[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int64_t before = 0;
    for (int s0 = 0; s0 < nseg; s0 += 1024) {
        const int s = s0 + tid;
        const int64_t tiles = s < nseg ? ((cu_q[s + 1] - cu_q[s]) * group + rows_per_tile - 1) / rows_per_tile : 0;
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
        if (s < nseg) tile_start[s] = ahead + sum - tiles;
        before += all;
        __syncthreads();
    }
    if (tid == 0) tile_start[nseg] = before;
}

// ---- host -----------------------------------------------------------------------

constexpr int kScoreMaxDim = 256;
constexpr int kWaveSegments = 64;   // segments that a wave's lanes hold; more take a table
constexpr int kRowTile = 128;
constexpr int64_t kSplitGrid = 512; // workgroups (two a CU) up to which a call's keys are split
constexpr int64_t kSplitKeys = 256; // keys that a split has at least, of the segments' mean

int64_t row_tiles(int64_t total_q, int nseg, int group) { return total_q * group / kRowTile + nseg; }

// Splits of the keys: as many as keep row tiles * key/value heads * splits within
// kSplitGrid, and kSplitKeys keys each.
int score_splits(int nseg, int64_t total_q, int64_t total_k, int kv_heads, int group) {
    const int64_t fit = kSplitGrid / (row_tiles(total_q, nseg, group) * kv_heads);
    return static_cast<int>(std::max<int64_t>(1, std::min(fit, total_k / nseg / kSplitKeys)));
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Rows of partial results at most: a split call has at most kSplitGrid workgroups of
// kRowTile rows, whatever its other sizes; so the size never falls as a call grows.
int64_t split_rows(int64_t total_q, int64_t total_k, int heads) {
    const int64_t most = std::max<int64_t>(1, std::min(kSplitGrid, total_k / kSplitKeys));
    if (most == 1) return 0;
    return std::min(kSplitGrid * kRowTile, total_q > kSplitGrid * kRowTile ? kSplitGrid * kRowTile : total_q * heads * most);
}

template <typename T, int DP>
int launch_any(const ScoreArgs & a, int64_t blocks, hipStream_t s) {
    constexpr int smem = AnyTile<T, DP>::kBytes;
    auto kernel = &score_attn_any_kernel<T, DP>;
    if constexpr (smem > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != hipSuccess) return check_hip(e, "hipFuncSetAttribute(score_attn)");
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), smem, s, a);
    return check_launch("scored attention");
}

template <typename T>
int run_scores(ScoreArgs a, int64_t blocks, hipStream_t s) {
    int rc;
    if (a.d <= 64) rc = launch_any<T, 64>(a, blocks, s);
    else if (a.d <= 128) rc = launch_any<T, 128>(a, blocks, s);
    else rc = launch_any<T, 256>(a, blocks, s);
    if (rc || a.splits == 1) return rc;
    hipLaunchKernelGGL(score_join_kernel<T>, dim3(grid_for(a.total_q * a.heads, 4)), dim3(256), 0, s, a);
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
    (void)kv_heads;
    if (nseg <= 0 || total_q <= 0 || heads <= 0 || head_dim <= 0) return 256;
    const size_t rows = static_cast<size_t>(split_rows(total_q, std::max<int64_t>(total_k, 0), heads));
    return round256((static_cast<size_t>(nseg) + 1) * sizeof(int64_t)) + round256(rows * sizeof(float2)) +
           round256(rows * head_dim * sizeof(float));
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
    PXS_CHECK(std::isfinite(scale * kLog2e) && (cap == 0.0f || (std::isfinite(scale / cap) && std::isfinite(cap * kLog2e))),
              PXS_ERR_ARG, "pxs_varlen_attention_scores: scale and cap out of range");
    PXS_CHECK(nseg >= 0 && total_q >= 0 && total_k >= 0 && total_q <= INT32_MAX && total_k <= INT32_MAX, PXS_ERR_ARG,
              "pxs_varlen_attention_scores: row counts must be in 0..2^31 - 1");
    const int64_t wq = static_cast<int64_t>(heads) * head_dim, wk = static_cast<int64_t>(kv_heads) * head_dim;
    PXS_CHECK(ld_q >= wq && ld_k >= wk && ld_v >= wk && ld_o >= wq, PXS_ERR_ARG,
              "pxs_varlen_attention_scores: row stride smaller than heads * head_dim");
    if (nseg == 0 || total_q == 0) return PXS_OK;
    PXS_CHECK(q && o && cu_q && cu_k && workspace && (total_k == 0 || (k && v)), PXS_ERR_ARG,
              "pxs_varlen_attention_scores: null pointer");
    hipStream_t s = as_stream(stream);
    ScoreArgs a{};
    a.q = q; a.k = k; a.v = v; a.ldq = ld_q; a.ldk = ld_k; a.ldv = ld_v;
    a.cu_q = cu_q; a.cu_k = cu_k; a.nseg = nseg; a.total_q = total_q;
    a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.d = head_dim;
    a.scale_log2 = cap > 0.0f ? scale / cap : scale * kLog2e;
    a.cap_log2 = cap * kLog2e;
    a.slopes = slopes; a.causal = causal; a.prefix = prefix; a.o = o; a.ldo = ld_o;
    const int elem = dtype == PXS_BF16 ? 2 : 4;
    a.vec = rows_of_pieces(q, ld_q, head_dim, elem) && rows_of_pieces(k, ld_k, head_dim, elem) &&
            rows_of_pieces(v, ld_v, head_dim, elem);
    a.tiles = row_tiles(total_q, nseg, a.group);
    a.splits = score_splits(nseg, total_q, total_k, kv_heads, a.group);
    const int64_t blocks = a.tiles * kv_heads * a.splits;
    PXS_CHECK(blocks <= UINT32_MAX / 256, PXS_ERR_ARG, "attention grid too large");
    char * ws = static_cast<char *>(workspace);
    if (nseg > kWaveSegments) {
        a.tile_start = reinterpret_cast<int64_t *>(ws);
        hipLaunchKernelGGL(score_tiles_kernel, dim3(1), dim3(1024), 0, s, cu_q, nseg, a.group, kRowTile,
                           reinterpret_cast<int64_t *>(ws));
        if (int rc = check_launch("scored attention tiles")) return rc;
    }
    if (a.splits > 1) {
        const size_t rows = static_cast<size_t>(a.splits) * total_q * heads;
        ws += round256((static_cast<size_t>(nseg) + 1) * sizeof(int64_t));
        a.part_ml = reinterpret_cast<float2 *>(ws);
        a.part = reinterpret_cast<float *>(ws + round256(rows * sizeof(float2)));
    }
    return dtype == PXS_F32 ? run_scores<float>(a, blocks, s) : run_scores<uint16_t>(a, blocks, s);
}

} // extern "C"
