// Shared by the attention kernels whose scores are capped and biased (attention_scores.hip,
// attention_tree.hip), bf16, head sizes of whole 16-byte pieces up to 128: a score's map to a weight's
// exponent, the products and weights of a tile of keys, and its DMA.
#pragma once

#include "attn_common.h"
#include "tiles.h"

#include <algorithm>
#include <limits>

namespace pxs {

// The constants of a call's scores, from its scale (finite, positive) and cap (finite, 0 for none).
// (Caps near the largest number, or that products of 2^113 at least are small against, cap nothing that
// fp32 holds: taken lower, so that scale / cap stays a normal number.  A multiplier past the largest
// number is cut, so that a product of zero stays zero under it.)
template <typename Args>
inline void score_constants(Args & a, float scale, float cap) {
    constexpr float kLargest = std::numeric_limits<float>::max();
    cap = std::min({cap, kLargest / 4, scale * 0x1p126f});
    a.scale_log2 = scale * kLog2e;
    a.cap_log2 = cap * kLog2e;
    a.over_cap = cap > 0.0f ? scale / cap : 0.0f;
    a.exp_mul = std::min(2.0f * kLog2e * a.over_cap, kLargest);
}

__device__ __forceinline__ bool is_finite_bits(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// Tiles of kKeys keys, 8 KB of K and 8 KB of V, go from HBM to LDS by DMA, rows of
// DH / 64 halves of 128 bytes; V is read transposed from LDS (ds_read_b64_tr_b16).
// 16 matrix instructions a tile and wave, as many for S as for O.

static __device__ __align__(16) uint4 g_score_zero[8];  // what keys past a segment's end are read as

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

// (Args: scale_log2, cap_log2, over_cap and exp_mul as score_constants makes them, and slopes.)
template <int MODE, typename Args>
__device__ __forceinline__ RowScore row_score(const Args & a, int head) {
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

// The exact step of a tile: hidden keys get weight 0, the base rises to the maximum and the output
// with it.  away(kt, e) and seen(kt, e) of the lane's keys.  lift: how far above the maximum the base is kept, so
// that weights are at most 2^-lift (-0, which adds nothing to any number).
template <int DH, int MODE, typename Away, typename Seen>
__device__ __forceinline__ void tile_exact_of(const RowScore & rs, float cap_log2, typename Fast<DH>::Scores & s,
                                              typename Fast<DH>::Weights & p, typename Fast<DH>::Out & oacc,
                                              RowState & st, Away away, Seen seen, float lift = -0.0f) {
    using F = Fast<DH>;
    const float add = near_cap(MODE) ? cap_log2 : 0.0f;
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < F::KT; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float z = score_of<MODE>(rs, s[kt][e], add, away(kt, e));
            s[kt][e] = seen(kt, e) ? z : -INFINITY;
            top = fmaxf(top, s[kt][e]);
        }
    const float up = fmaxf(st.base, lane_pair_max(top) + lift);
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

// Keys at or past `seen` of the tile's (less 4 h) hidden, distances counted from `behind`.
template <int DH, int MODE>
__device__ __forceinline__ void tile_exact(const RowScore & rs, float cap_log2, typename Fast<DH>::Scores & s,
                                           typename Fast<DH>::Weights & p, typename Fast<DH>::Out & oacc,
                                           RowState & st, float behind, int seen) {
    tile_exact_of<DH, MODE>(
        rs, cap_log2, s, p, oacc, st,
        [&](int kt, int e) __attribute__((always_inline)) { return behind - static_cast<float>(key_of(kt, e)); },
        [&](int kt, int e) __attribute__((always_inline)) { return key_of(kt, e) < seen; });
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
__device__ __forceinline__ void load_q_row(const uint16_t * q, int d, bool live, int h, bf16x8 (&qf)[Fast<DH>::NST]) {
#pragma unroll
    for (int st = 0; st < Fast<DH>::NST; ++st) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (live && (st / 4) * 64 + 32 * h + 8 * (st % 4) < d) u = *reinterpret_cast<const uint4 *>(q + (st / 4) * 64 + 32 * h + 8 * (st % 4));
        qf[st] = __builtin_bit_cast(bf16x8, u);
    }
}

template <int DH>
__device__ __forceinline__ TileSource<DH> tile_source_of(const uint16_t * k, const uint16_t * v, int64_t ldk, int64_t ldv, int nk) {
    TileSource<DH> s;
    s.k = uniform_ptr(reinterpret_cast<const char *>(k));
    s.v = uniform_ptr(reinterpret_cast<const char *>(v));
    s.ldk = ldk * 2;
    s.ldv = ldv * 2;
    s.nk = nk;
    s.zero = reinterpret_cast<uint64_t>(&g_score_zero[0]);
    asm volatile("" : "+s"(s.zero));
    return s;
}

// The steps without a maximum: sums past this are redone with one, and outputs past that walked again.
constexpr int kSlots = 4;
constexpr float kSumLimit = 0x1p40f;
constexpr float kOutLimit = 0x1p118f;

// A wave's own LDS reads are done, and none is moved over this.
__device__ __forceinline__ void wave_reads_done() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

} // namespace pxs
