// 8-bit linears: rows quantized to 8-bit integers with a scale each, and their
// products with weights quantized the same way, row by output channel.
//
//   scale[r] = max_c |x[r, c]| / 127         q[r, c] = rint(x[r, c] * (127 / max))
//   Y[m, n]  = (sum_k q[m, k] w[n, k]) * x_scale[m] * w_scale[n] + bias[n]
//
// then one of the epilogues of the linears in 16 and 32 bits (dense.hip): store
// with an activation, add to an fp32 residual, add to it through the adaLN gate.
// The sum is an int32 and exact (cin is bounded so that it cannot overflow), so
// no order of it, and no tile, changes an output's bits.

#include "pxs_common.h"
#include "tiles.h"

#include <algorithm>
#include <iterator>
#include <type_traits>

namespace pxs {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- rows to 8 bits -----------------------------------------------------------
// One pass: a row stays in registers between its maximum and its rounding, so
// the bytes are those of x, q and the scales.  The maximum is taken of the bit
// patterns of |x| as integers, which puts NaN above infinity above all numbers.
// The product and the rounding are two roundings, as the formula says, never one
// fused: adding 1.5 * 2^23 rounds the product to an integer, ties to even, and
// leaves it in the sum's low byte.
constexpr uint32_t kQuantFinite = 0x7F800000u;   // infinity's bits
constexpr float kQuantLeast = 0x1p-100f;         // rows below count as zero: 127 / max stays finite
constexpr float kRoundMagic = 12582912.0f;       // 1.5 * 2^23

struct QuantArgs {
    const void * x;
    int64_t ldx;
    int64_t rows;
    int channels;
    int8_t * q;
    float * scales;
};

// The 8 elements from column c of a row of 8 or more, or its last 8 (which a neighbour then holds
// too, and stores alike); of fewer, those there are.  Rows start at any element.
template <typename T, bool VEC>
__device__ __forceinline__ void load_elems8(const T * row, int c, int channels, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (c >= channels) return;
    if constexpr (VEC) {
        T e[8];
        __builtin_memcpy(e, row + min(c, channels - 8), sizeof(e));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = load_f32(e + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < channels) v[i] = load_f32(row + c + i);
    }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The scale of a row with this largest magnitude, and what its values are multiplied with.
__device__ __forceinline__ void row_scale(uint32_t top_bits, float & scale, float & per) {
    const float top = __uint_as_float(top_bits);
    scale = 0.0f;
    per = 0.0f;
    if (top_bits >= kQuantFinite) {
        scale = __uint_as_float(0x7FC00000u);  // NaN: the row's products are NaN
    } else if (top >= kQuantLeast) {
        scale = top / 127.0f;
        per = 127.0f / top;
    }
}

template <bool VEC>
__device__ __forceinline__ void store_q8(int8_t * row, int c, int channels, const float (&v)[8], float per,
                                         bool finite) {
#pragma clang fp contract(off)
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(v[i] * per + kRoundMagic);
    uint2 u;
    u.x = (b[0] & 255u) | (b[1] & 255u) << 8 | (b[2] & 255u) << 16 | b[3] << 24;
    u.y = (b[4] & 255u) | (b[5] & 255u) << 8 | (b[6] & 255u) << 16 | b[7] << 24;
    if (!finite) u = make_uint2(0u, 0u);
    if constexpr (VEC) {
        if (c < channels) __builtin_memcpy(row + min(c, channels - 8), &u, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < channels) row[c + i] = static_cast<int8_t>((i < 4 ? u.x >> (8 * i) : u.y >> (8 * (i - 4))) & 255u);
    }
}

// WPR waves share a row of up to WPR * 64 * 8 * NV channels; rows of any number
// (HELD false) are read a second time for the rounding.
template <typename T, int WPR, int NV, bool VEC, bool HELD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantArgs a) {
    constexpr int kLanes = WPR * 64;
    __shared__ uint32_t tops[4];
    const int wave = threadIdx.x >> 6;
    const int l = threadIdx.x % kLanes;
    float v[NV][8];
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / WPR) + wave / WPR; row < a.rows;
         row += static_cast<int64_t>(gridDim.x) * (4 / WPR)) {
        const T * x = static_cast<const T *>(a.x) + row * a.ldx;
        uint32_t top = 0;
        if constexpr (HELD) {
#pragma unroll
            for (int j = 0; j < NV; ++j) load_elems8<T, VEC>(x, (j * kLanes + l) * 8, a.channels, v[j]);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[j][i]));
        } else {
            for (int c = l * 8; c < a.channels; c += kLanes * 8) {
                load_elems8<T, VEC>(x, c, a.channels, v[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[0][i]));
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64)));
        if constexpr (WPR > 1) {
            if ((threadIdx.x & 63) == 0) tops[wave] = top;
            __syncthreads();
            top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
            __syncthreads();  // (every wave has the same rows)
        }
        float scale, per;
        row_scale(top, scale, per);
        if (l == 0) a.scales[row] = scale;
        int8_t * q = a.q + row * a.channels;
        const bool finite = top < kQuantFinite;
        if constexpr (HELD) {
#pragma unroll
            for (int j = 0; j < NV; ++j) store_q8<VEC>(q, (j * kLanes + l) * 8, a.channels, v[j], per, finite);
        } else {
            for (int c = l * 8; c < a.channels; c += kLanes * 8) {
                load_elems8<T, VEC>(x, c, a.channels, v[0]);
                store_q8<VEC>(q, c, a.channels, v[0], per, finite);
            }
        }
    }
}

template <typename T>
int launch_quantize(const QuantArgs & a, hipStream_t s) {
    const int64_t one = (a.rows + 3) / 4;
    auto launch = [&](auto kernel, int64_t blocks) {  // a workgroup takes more rows past 2^20 of them
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20))), dim3(256), 0, s, a);
    };
    if (a.channels < 8) launch(quantize_rows_kernel<T, 1, 1, false, true>, one);
    else if (a.channels <= 512) launch(quantize_rows_kernel<T, 1, 1, true, true>, one);
    else if (a.channels <= 1024) launch(quantize_rows_kernel<T, 1, 2, true, true>, one);
    else if (a.channels <= 2048) launch(quantize_rows_kernel<T, 4, 1, true, true>, a.rows);
    else if (a.channels <= 4096) launch(quantize_rows_kernel<T, 4, 2, true, true>, a.rows);
    else if (a.channels <= 8192) launch(quantize_rows_kernel<T, 4, 4, true, true>, a.rows);
    else launch(quantize_rows_kernel<T, 4, 1, true, false>, a.rows);
    return check_launch("quantize rows");
}

// ---- products -------------------------------------------------------------------

enum I8Epi { kI8Store = 0, kI8AddResidual = 1, kI8Gate = 2 };

struct I8Args {
    const int8_t * x;        // [m, k]
    const float * x_scales;  // [m]
    const int8_t * w;        // [n, k]
    const float * w_scales;  // [n]
    const float * bias;      // [n] or null
    int64_t m;
    int k;
    int n;
    int act;
    void * y;                // [m, n], store epilogue
    float * residual;        // [m, n] fp32, residual epilogues
    const int32_t * coords;  // [m, 4], gate epilogue: batch of each row
    const float * block_mod; // gate = block_mod[gate_offset + c] + time_mod[b, gate_offset + c]
    const float * time_mod;  // [batch, 6 n]
    int gate_offset;
    int vec_out;             // 1: 4-channel vector accesses of all that the epilogue touches; 2: y in whole 16-byte pieces
    int group_m;             // tile order (tile_of)
};

// The activations of pxs_linear through one exponential and one reciprocal: 0.5 v (1 + tanh u)
// is v / (1 + e^-2u).  Within a few steps of the library's forms, which took a third of a
// short product's time.
__device__ __forceinline__ float i8_gelu(float v) {
    const float e = v * __builtin_fmaf(v * v, -0.10294324f, -2.3022082f);  // -2 log2(e) u
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e));
}
__device__ __forceinline__ float i8_silu(float v) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

// The scales and biases of four channels from c (c < n; past n, the last channel's).
struct I8Channels {
    float ws[4], bias[4];
};
__device__ __forceinline__ I8Channels i8_channels(const I8Args & a, int c, bool vec) {
    I8Channels o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.bias[e] = 0.0f;
    if (vec) {
        const float4 w4 = *reinterpret_cast<const float4 *>(a.w_scales + c);
        o.ws[0] = w4.x; o.ws[1] = w4.y; o.ws[2] = w4.z; o.ws[3] = w4.w;
        if (a.bias) {
            const float4 b4 = *reinterpret_cast<const float4 *>(a.bias + c);
            o.bias[0] = b4.x; o.bias[1] = b4.y; o.bias[2] = b4.z; o.bias[3] = b4.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int ce = min(c + e, a.n - 1);
            o.ws[e] = a.w_scales[ce];
            if (a.bias) o.bias[e] = a.bias[ce];
        }
    }
    return o;
}

// Four values of a row: (sum * x_scale) * w_scale + bias, then the activation.  (The sum, up
// to 2^31, rounds to fp32 once, each product and the bias once.)
__device__ __forceinline__ void i8_values4(const I8Args & a, const I8Channels & ch, const int (&sum)[4], float xs,
                                           float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (static_cast<float>(sum[e]) * xs) * ch.ws[e] + ch.bias[e];
    if (a.act == PXS_ACT_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i8_gelu(v[e]);
    } else if (a.act == PXS_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i8_silu(v[e]);
    }
}

template <typename T> __device__ __forceinline__ void i8_put4(T * p, const float (&v)[4]) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

template <typename T, int EPI>
__device__ __forceinline__ void i8_epilogue4(const I8Args & a, const I8Channels & ch, int64_t row, int batch, int c,
                                             const int (&sum)[4], float xs) {
    const bool vec = a.vec_out && c + 3 < a.n;
    float v[4];
    i8_values4(a, ch, sum, xs, v);
    if constexpr (EPI == kI8Store) {
        T * p = static_cast<T *>(a.y) + row * a.n + c;
        if (vec) {
            i8_put4(p, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.n) store_f32(p + e, v[e]);
        }
    } else {
        float * p = a.residual + row * a.n + c;
        float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (EPI == kI8Gate) {
            const float * bm = a.block_mod + a.gate_offset;
            const float * tm = a.time_mod + static_cast<int64_t>(batch) * 6 * a.n + a.gate_offset;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int ce = min(c + e, a.n - 1);
                g[e] = bm[ce] + tm[ce];
            }
        }
        if (vec) {
            float4 o = *reinterpret_cast<const float4 *>(p);
            o.x += v[0] * g[0]; o.y += v[1] * g[1]; o.z += v[2] * g[2]; o.w += v[3] * g[3];
            *reinterpret_cast<float4 *>(p) = o;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.n) p[e] += v[e] * g[e];
        }
    }
}

// Row pitch in LDS of 32 rows of a wave's block, and 16 bytes against bank conflicts.
template <typename T, int WN> constexpr int i8_pitch() { return WN * static_cast<int>(sizeof(T)) + 16; }

// One wave's block of outputs: acc[i][j] holds 32 rows by 32 channels, lane (h, r) row r and
// channels 8 g + 4 h + e.  Stores go through the wave's region of LDS (which no other wave uses
// any more), 32 rows at a time, so that an instruction covers row segments of 64 to 128 bytes: whole
// 16-byte pieces (vec_out 2), or elements (4,739 x 1370 -> 1021 in fp32 25 us, 34 without).
// HOIST: every channel's scale and bias loaded ahead of the first value, one wait for all, where
// the registers are there (8 waves a workgroup: 1,370 x 1024 -> 4096 14.0 -> 12.9 us; 16 waves: 42,017 x
// 4096 -> 1024 179 -> 203).
template <typename T, int TI, int TJ, int EPI, bool HOIST>
__device__ __forceinline__ void i8_tile_out(const I8Args & a, const i32x16 (&acc)[TI][TJ], char * region, int64_t row0,
                                            int col0, int h, int r, int lane) {
    constexpr int WN = TJ * 32, kPitch = i8_pitch<T, WN>(), kElems = 16 / static_cast<int>(sizeof(T));
    constexpr int kLanesPerRow = WN / kElems, kRowsPerPass = 64 / kLanesPerRow;
    constexpr bool staged = EPI == kI8Store;
    auto channels = [&](int j, int g) __attribute__((always_inline)) {
        const int c = min(col0 + j * 32 + 8 * g + 4 * h, a.n - 1);
        return i8_channels(a, c, a.vec_out && c + 3 < a.n);
    };
    I8Channels held[HOIST ? TJ : 1][4];
    float scale[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) scale[i] = a.x_scales[min(row0 + i * 32 + r, a.m - 1)];
    if constexpr (HOIST) {
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) held[j][g] = channels(j, g);
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int64_t row = row0 + i * 32 + r;
        const float xs = scale[i];
        const int batch = EPI == kI8Gate && row < a.m ? a.coords[row * 4] : 0;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int cl = j * 32 + 8 * g + 4 * h, c = col0 + cl;
                const int sum[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                const I8Channels ch = HOIST ? held[HOIST ? j : 0][g] : channels(j, g);
                if constexpr (staged) {
                    float v[4];
                    i8_values4(a, ch, sum, xs, v);  // (past n: not stored)
                    i8_put4(reinterpret_cast<T *>(region + r * kPitch + cl * static_cast<int>(sizeof(T))), v);
                } else if (row < a.m && c < a.n) {
                    i8_epilogue4<T, EPI>(a, ch, row, batch, c, sum, xs);
                }
            }
        if constexpr (staged) {
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own writes
            if (a.vec_out != 2) {  // an element a lane, in the order of their addresses
#pragma unroll 2
                for (int pass = 0; pass < 32 * WN / 64; ++pass) {
                    const int rl = (pass * 64 + lane) / WN, cl = (pass * 64 + lane) % WN;
                    const T v = *reinterpret_cast<const T *>(region + rl * kPitch + cl * static_cast<int>(sizeof(T)));
                    const int64_t to = row0 + i * 32 + rl;
                    if (to < a.m && col0 + cl < a.n) static_cast<T *>(a.y)[to * a.n + col0 + cl] = v;
                }
                continue;
            }
            const int lr = lane / kLanesPerRow, lc = lane % kLanesPerRow;
#pragma unroll
            for (int pass = 0; pass < 32 / kRowsPerPass; ++pass) {
                const int rl = pass * kRowsPerPass + lr;
                const uint4 v = *reinterpret_cast<const uint4 *>(region + rl * kPitch + lc * 16);
                const int64_t to = row0 + i * 32 + rl;
                const int c = col0 + lc * kElems;
                if (to < a.m && c < a.n) *reinterpret_cast<uint4 *>(static_cast<T *>(a.y) + to * a.n + c) = v;
            }
        }
    }
}

// 16 bytes of a row at K offset k0 for a product over k: a whole piece as it lies,
// or the row's last 16 bytes with those before k0 zeroed (ZERO; the other operand
// may keep them, its products are zero), nothing read outside the row.
template <bool ZERO>
__device__ __forceinline__ uint4 load_piece(const int8_t * row, int k0, int k) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (k0 >= k) return v;
    if (k < 16) {  // k0 is 0
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < k) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[i])) << (8 * (i & 3));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const int at = min(k0, k - 16), skip = k0 - at;
    __builtin_memcpy(&v, row + at, 16);
    if (ZERO && skip > 0) {
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = skip - 4 * i;  // bytes of this word to zero
            w[i] = s >= 4 ? 0u : (s > 0 ? w[i] & (0xFFFFFFFFu << (8 * s)) : w[i]);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}

// BM x BN outputs, NW waves in a WAVES_M x (NW / WAVES_M) grid, rows of any length and
// alignment.  128 bytes of K a stage, two stages in LDS, and every thread's 16-byte pieces of
// the next in registers, loaded while the ones before are multiplied (a further stage in
// registers changed nothing, and pieces put together from aligned words cost more: 1,000 x 1370 -> 1021
// 14.5 us, 14.3 and 17.5).  What bounds it: the loads, whose rows lie across the cache's lines; 1,000 x
// 1376 -> 1024 on the kernel below takes 7.8 us.
template <typename T, int BM, int BN, int NW, int WAVES_M, int EPI>
__global__ void __launch_bounds__(NW * 64) linear_i8_any_kernel(I8Args a) {
    constexpr int KB = 128, P = 8, NT = NW * 64, RS = NT / P;
    constexpr int WAVES_N = NW / WAVES_M, WM = BM / WAVES_M, WN = BN / WAVES_N, TI = WM / 32, TJ = WN / 32;
    constexpr int XI = BM / RS, WI = BN / RS, kStage = (BM + BN) * KB, kOut = NW * 32 * i8_pitch<T, WN>();
    static_assert(2 * kStage >= kOut, "the store regions lie in the stages");
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int h = lane >> 5, r = lane & 31;
    const int tiles_n = (a.n + BN - 1) / BN, tiles_m = static_cast<int>((a.m + BM - 1) / BM);
    int tm, tn;
    tile_of(remap_xcd(blockIdx.x, gridDim.x), tiles_m, tiles_n, a.group_m, tm, tn);
    const int64_t p0 = static_cast<int64_t>(tm) * BM;
    const int n0 = tn * BN;
    const int piece = tid & (P - 1), row0 = tid / P;
    const int8_t * xr[XI];
    const int8_t * wr[WI];
#pragma unroll
    for (int i = 0; i < XI; ++i) xr[i] = a.x + min(p0 + row0 + RS * i, a.m - 1) * a.k;
#pragma unroll
    for (int i = 0; i < WI; ++i) wr[i] = a.w + static_cast<int64_t>(min(n0 + row0 + RS * i, a.n - 1)) * a.k;
    auto load = [&](int s, uint4 (&vx)[XI], uint4 (&vw)[WI]) __attribute__((always_inline)) {
        const int k0 = s * KB + piece * 16;
        if (s * KB + KB <= a.k) {
#pragma unroll
            for (int i = 0; i < XI; ++i) __builtin_memcpy(&vx[i], xr[i] + k0, 16);
#pragma unroll
            for (int i = 0; i < WI; ++i) __builtin_memcpy(&vw[i], wr[i] + k0, 16);
        } else {
#pragma unroll
            for (int i = 0; i < XI; ++i) vx[i] = load_piece<true>(xr[i], k0, a.k);
#pragma unroll
            for (int i = 0; i < WI; ++i) vw[i] = load_piece<false>(wr[i], k0, a.k);
        }
    };
    auto put = [&](int s, const uint4 (&vx)[XI], const uint4 (&vw)[WI]) __attribute__((always_inline)) {
        char * stage = smem + (s & 1) * kStage;
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const int row = row0 + RS * i;
            *reinterpret_cast<uint4 *>(stage + row * KB + ((piece ^ piece_swz<KB>(row)) << 4)) = vx[i];
        }
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int row = row0 + RS * i;
            *reinterpret_cast<uint4 *>(stage + (BM + row) * KB + ((piece ^ piece_swz<KB>(row)) << 4)) = vw[i];
        }
    };
    i32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = i32x16{};
    const int stages = (a.k + KB - 1) / KB;
    uint4 vx[XI], vw[WI];
    load(0, vx, vw);
    put(0, vx, vw);
    if (stages > 1) load(1, vx, vw);
    for (int s = 0; s < stages; ++s) {
        barrier_no_fence();  // stage s is written, and stage s - 1 read, by every wave
        if (s + 1 < stages) put(s + 1, vx, vw);
        if (s + 2 < stages) load(s + 2, vx, vw);
        const char * stage = smem + (s & 1) * kStage;
#pragma unroll
        for (int u = 0; u < P / 2; ++u) {
            const int pc = (P / 2) * h + u;
            i32x4 xf[TI], wf[TJ];
#pragma unroll
            for (int i = 0; i < TI; ++i) {
                const int row = wm * WM + i * 32 + r;
                xf[i] = *reinterpret_cast<const i32x4 *>(stage + row * KB + ((pc ^ piece_swz<KB>(row)) << 4));
            }
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                const int row = wn * WN + j * 32 + r;
                wf[j] = *reinterpret_cast<const i32x4 *>(stage + (BM + row) * KB + ((pc ^ piece_swz<KB>(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
        }
    }
    barrier_no_fence();
    i8_tile_out<T, TI, TJ, EPI, NW <= 8>(a, acc, smem + wave * 32 * i8_pitch<T, WN>(), p0 + wm * WM, n0 + wn * WN, h, r, lane);
}

// Up to 16 RB rows (single tokens): bound by reading the weights once.  A workgroup has 16
// output channels; its eight waves take every eighth 128 bytes of K, straight from memory to
// the operands of 16 x 16 x 64 products (a lane holds 32 contiguous bytes of a channel's and
// of a row's 128), and their sums are joined through LDS.
constexpr int kFewWaves = 8;
template <typename T, int RB, int EPI>
__global__ void __launch_bounds__(kFewWaves * 64) linear_i8_few_kernel(I8Args a) {
    __shared__ __align__(16) int part[kFewWaves][RB * 16][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * RB);
    const int8_t * w = a.w + static_cast<int64_t>(min(n0 + l16, a.n - 1)) * a.k;
    const int8_t * x[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) x[b] = a.x + min(static_cast<int64_t>(m0 + b * 16 + l16), a.m - 1) * a.k;
    i32x4 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = i32x4{};
    const int whole = a.k / 128;
    // U chunks of the wave from c: all their loads before the first product.
    auto chunks = [&](int c, auto count) __attribute__((always_inline)) {
        constexpr int U = decltype(count)::value;
        i32x4 wf[U][2], xf[U][RB][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (c + u * kFewWaves) * 128 + kq * 32;
            __builtin_memcpy(wf[u], w + k0, 32);
#pragma unroll
            for (int b = 0; b < RB; ++b) __builtin_memcpy(xf[u][b], x[b] + k0, 32);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][e], xf[u][b][e], acc[b], 0, 0, 0);
    };
    int c = wave;
    for (; c + 3 * kFewWaves < whole; c += 4 * kFewWaves) chunks(c, std::integral_constant<int, 4>{});
    for (; c < whole; c += kFewWaves) chunks(c, std::integral_constant<int, 1>{});
    if (a.k % 128 != 0 && wave == whole % kFewWaves) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int k0 = whole * 128 + kq * 32 + e * 16;
            const i32x4 wf = __builtin_bit_cast(i32x4, load_piece<false>(w, k0, a.k));
#pragma unroll
            for (int b = 0; b < RB; ++b)
                acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                    wf, __builtin_bit_cast(i32x4, load_piece<true>(x[b], k0, a.k)), acc[b], 0, 0, 0);
        }
    }
    // Lane (kq, l16) holds row l16's channels 4 kq .. 4 kq + 3.
#pragma unroll
    for (int b = 0; b < RB; ++b) *reinterpret_cast<i32x4 *>(&part[wave][b * 16 + l16][4 * kq]) = acc[b];
    __syncthreads();
    if (tid >= RB * 64) return;
    const int rl = tid >> 2, cl = (tid & 3) * 4;
    const int64_t row = m0 + rl;
    const int col = n0 + cl;
    if (row >= a.m || col >= a.n) return;
    int sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) {
        const i32x4 p = *reinterpret_cast<const i32x4 *>(&part[i][rl][cl]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += p[e];
    }
    i8_epilogue4<T, EPI>(a, i8_channels(a, col, a.vec_out && col + 3 < a.n), row,
                         EPI == kI8Gate ? a.coords[row * 4] : 0, col, sum, a.x_scales[row]);
}

// Rows of whole 16-byte pieces (cin a multiple of 16).  As the 16-bit products
// (dense.hip): BM rows of X and BN rows of W go 128 bytes of K at a time from L2 to LDS by
// DMA, NSTAGE stages in flight, and a lane reads 16 contiguous bytes per fragment, the K
// order inside a stage being permuted alike for both operands.  A 32 x 32 x 32 product
// takes the cycles of a 16-bit one of half its depth, so bytes, stages and LDS traffic
// are those of the 16-bit kernel and the rate is twice its.
//
// KG groups of NW waves share a tile and take every KG-th stage each, in stages of their
// own; the groups' sums are added through LDS.  For calls of few tiles, whose time is
// the chain of stages.
__device__ __align__(16) uint4 g_i8_zero[8];  // K pieces past the end

template <typename T, int BM, int BN, int NW, int WAVES_M, int NSTAGE, int KG, int EPI>
__global__ void __launch_bounds__(NW * KG * 64) linear_i8_kernel(I8Args a) {
    constexpr int KB = 128, P = 8, RPI = 8;  // bytes, pieces per row of a stage; rows per DMA instruction
    constexpr int WAVES_N = NW / WAVES_M, WM = BM / WAVES_M, WN = BN / WAVES_N, TI = WM / 32, TJ = WN / 32;
    constexpr int kStage = (BM + BN) * KB;
    constexpr int AI = BM / (RPI * NW), BI = BN / (RPI * NW), kPerStage = AI + BI;
    static_assert(AI * RPI * NW == BM && BI * RPI * NW == BN, "tile rows must split over the waves");
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int group = KG > 1 ? __builtin_amdgcn_readfirstlane(tid / (NW * 64)) : 0;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) - group * NW;  // in its group
    char * ring = smem + group * NSTAGE * kStage;
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int h = lane >> 5, r = lane & 31;
    const int tiles_n = (a.n + BN - 1) / BN, tiles_m = static_cast<int>((a.m + BM - 1) / BM);
    int tm, tn;
    tile_of(remap_xcd(blockIdx.x, gridDim.x), tiles_m, tiles_n, a.group_m, tm, tn);
    const int64_t p0 = static_cast<int64_t>(tm) * BM;
    const int n0 = tn * BN;
    const int8_t * xs = a.x + p0 * a.k;
    const int8_t * wsb = a.w + static_cast<int64_t>(n0) * a.k;
    const int all_stages = (a.k + KB - 1) / KB;
    const int stages = (all_stages - group + KG - 1) / KG;       // of this group
    const int steps = KG > 1 ? (all_stages + KG - 1) / KG : stages;  // of every group
    const bool ragged = a.k % KB != 0;  // the last stage holds pieces past k
    const int lrow = lane / P, lslot = lane % P;
    const int64_t last_x = a.m - 1 - p0;
    const int last_w = a.n - 1 - n0;
    uint32_t off[kPerStage];  // rows past the end are clamped; their outputs are not stored
#pragma unroll
    for (int j = 0; j < kPerStage; ++j) {
        const bool is_x = j < AI;
        const int row = (wave * (is_x ? AI : BI) + (is_x ? j : j - AI)) * RPI + lrow;
        const int64_t at = is_x ? min(static_cast<int64_t>(row), last_x) : static_cast<int64_t>(min(row, last_w));
        off[j] = static_cast<uint32_t>(at * a.k + (lslot ^ piece_swz<KB>(row)) * 16);
    }
    auto issue_one = [&](int s, int q) __attribute__((always_inline)) {
        const bool is_x = q < AI;
        const int row0 = (wave * (is_x ? AI : BI) + (is_x ? q : q - AI)) * RPI;
        const uint32_t lds = lds_offset(ring + (s % NSTAGE) * kStage + ((is_x ? 0 : BM) + row0) * KB);
        const int at = s * KG + group;
        const int8_t * src = (is_x ? xs : wsb) + static_cast<int64_t>(at) * KB;
        if (ragged && at == all_stages - 1) {
            const bool in = at * KB + (lslot ^ piece_swz<KB>(row0 + lrow)) * 16 < a.k;
            lds_dma16(in ? static_cast<const void *>(src + off[q]) : static_cast<const void *>(g_i8_zero), lds);
        } else {
            lds_dma16_sbase(src, off[q], lds);
        }
    };
    i32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = i32x16{};
#pragma unroll
    for (int s = 0; s < NSTAGE - 1; ++s)
        if (s < stages) {
#pragma unroll
            for (int q = 0; q < kPerStage; ++q) issue_one(s, q);
        }
    for (int s = 0; s < steps; ++s) {
        if (KG == 1 || s < stages) wait_stages<NSTAGE - 2, kPerStage>(stages - 1 - s);
        barrier_no_fence();
        if (KG > 1 && s >= stages) continue;
        const bool more = s + NSTAGE - 1 < stages;
        const char * sx = ring + (s % NSTAGE) * kStage;
        const char * sw = sx + BM * KB;
        i32x4 xf[2][TI], wf[2][TJ];
        auto read_frags = [&](int u, i32x4 (&xo)[TI], i32x4 (&wo)[TJ]) __attribute__((always_inline)) {
            const int piece = (P / 2) * h + u;
#pragma unroll
            for (int i = 0; i < TI; ++i) {
                const int row = wm * WM + i * 32 + r;
                xo[i] = *reinterpret_cast<const i32x4 *>(sx + row * KB + ((piece ^ piece_swz<KB>(row)) << 4));
            }
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                const int row = wn * WN + j * 32 + r;
                wo[j] = *reinterpret_cast<const i32x4 *>(sw + row * KB + ((piece ^ piece_swz<KB>(row)) << 4));
            }
        };
        read_frags(0, xf[0], wf[0]);
#pragma unroll
        for (int u = 0; u < P / 2; ++u) {
            // The next stage's DMA in four parts, one per K step.
#pragma unroll
            for (int q = 0; q < kPerStage; ++q)
                if (more && q * (P / 2) / kPerStage == u) issue_one(s + NSTAGE - 1, q);
            if (u + 1 < P / 2) read_frags(u + 1, xf[(u + 1) & 1], wf[(u + 1) & 1]);
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[u & 1][j], xf[u & 1][i], acc[i][j], 0, 0, 0);
        }
    }
    barrier_no_fence();  // every wave is done with the stages
    constexpr int kOut = NW * 32 * i8_pitch<T, WN>();
    if constexpr (KG > 1) {
        // [group - 1][wave][register][lane], behind the first group's store regions
        int * sums = reinterpret_cast<int *>(smem + kOut) + wave * TI * TJ * 16 * 64 + lane;
        constexpr int kGroup = NW * TI * TJ * 16 * 64;
        if (group > 0) {
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sums[(group - 1) * kGroup + ((i * TJ + j) * 16 + e) * 64] = acc[i][j][e];
        }
        barrier_no_fence();
        if (group > 0) return;
#pragma unroll
        for (int g = 0; g < KG - 1; ++g)
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][j][e] += sums[g * kGroup + ((i * TJ + j) * 16 + e) * 64];
    }
    i8_tile_out<T, TI, TJ, EPI, NW <= 8>(a, acc, smem + wave * 32 * i8_pitch<T, WN>(), p0 + wm * WM, n0 + wn * WN, h, r, lane);
}

bool aligned_to(const void * p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_i8_grid(int64_t blocks, int threads) {
    PXS_CHECK(blocks <= UINT32_MAX / threads, PXS_ERR_ARG, "8-bit linear grid too large");
    return PXS_OK;
}

template <typename T, int BM, int BN, int NW, int WAVES_M, int NSTAGE, int KG, int EPI>
int launch_i8_tiles(I8Args a, hipStream_t s) {
    constexpr int WN = BN / (NW / WAVES_M), kOut = NW * 32 * i8_pitch<T, WN>();
    constexpr int kStages = KG * NSTAGE * (BM + BN) * 128, kEnd = kOut + (KG - 1) * BM * BN * 4;
    constexpr int smem = kStages > kEnd ? kStages : kEnd;
    static_assert(smem <= 160 * 1024, "LDS");
    const int64_t blocks = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    if (int rc = check_i8_grid(blocks, NW * KG * 64)) return rc;
    auto kernel = &linear_i8_kernel<T, BM, BN, NW, WAVES_M, NSTAGE, KG, EPI>;
    if constexpr (smem > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), smem, done, "hipFuncSetAttribute(linear_i8)")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(NW * KG * 64), smem, s, a);
    return check_launch("8-bit linear");
}

template <typename T, int BM, int BN, int NW, int WAVES_M, int EPI>
int launch_i8_any(const I8Args & a, hipStream_t s) {
    constexpr int smem = 2 * (BM + BN) * 128;
    const int64_t blocks = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    if (int rc = check_i8_grid(blocks, NW * 64)) return rc;
    auto kernel = &linear_i8_any_kernel<T, BM, BN, NW, WAVES_M, EPI>;
    if constexpr (smem > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), smem, done, "hipFuncSetAttribute(linear_i8_any)")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(NW * 64), smem, s, a);
    return check_launch("8-bit linear");
}

template <typename T, int RB, int EPI>
int launch_i8_few(const I8Args & a, hipStream_t s) {
    const dim3 grid(grid_for(a.n, 16), grid_for(a.m, 16 * RB));
    if (int rc = check_i8_grid(grid.x, kFewWaves * 64)) return rc;
    hipLaunchKernelGGL((linear_i8_few_kernel<T, RB, EPI>), grid, dim3(kFewWaves * 64), 0, s, a);
    return check_launch("8-bit linear of few rows");
}

// Tile shapes, their time alone on a CU and their share of a full CU's time, in us for
// 1024 bytes of K more and without any: fitted to each shape's times at 68 sizes (65 to 206,980
// rows, 256 to 8192 deep), where the shape picked takes 0.5% more than the best on average (at the larger
// sizes the whole card runs slower than one tile alone):
//   256 x 256, 16 waves of 64 x 64, one workgroup a CU:  8,192 x 8192 -> 4096 242 us (2,270 TOP/s)
//   192 x 128 and 128 x 128, 8 waves, two workgroups:    287 and 289; 1,370 x 1024 -> 4096 13.1 and 13.6
//   128 x 64, 8 waves, two:                              1,370 x 4096 -> 1024 17.8 against 20.3
//   64 x 64, 4 waves, two:                               150 x 4096 -> 4096 15.1 against 17.0
//   32 x 64, four groups of two waves over K, one:       300 x 4096 -> 1024 8.4 against 14.8
struct I8Shape {
    int bm, bn, stages;
    double alone0, alone1, each0, each1;
};
constexpr I8Shape kI8Shapes[] = {
    {256, 256, 2, 7.3, 8.9, 10.8, 13.4}, {192, 128, 2, 4.9, 4.8, 4.2, 5.9}, {128, 128, 2, 3.9, 4.0, 2.7, 4.4},
    {128, 64, 3, 3.6, 3.3, 2.0, 2.8},    {64, 64, 4, 3.1, 2.9, 1.4, 2.0},   {32, 64, 3, 3.7, 1.1, 2.7, 1.2},
};

int i8_shape(int64_t m, int n, int k) {
    int best = 0;
    double least = 0.0;
    for (int i = 0; i < static_cast<int>(std::size(kI8Shapes)); ++i) {
        const I8Shape & c = kI8Shapes[i];
        const double deep = k / 1024.0, alone = c.alone0 + c.alone1 * deep, each = c.each0 + c.each1 * deep;
        const int64_t tiles = ((m + c.bm - 1) / c.bm) * ((n + c.bn - 1) / c.bn);
        const double time = tiles <= 256 ? alone + std::max(0.0, each - alone) * (tiles / 256.0)
                                         : std::max(alone, ((tiles + 255) / 256) * each);
        if (i == 0 || time < least) {
            least = time;
            best = i;
        }
    }
    return best;
}

constexpr int kI8DeepK = 1024;  // a longer K is worth a third stage (i8_plan)

// Up to kI8FewRows rows: 16 output channels a workgroup, and as few of its 16-row blocks as
// keep the workgroups near one a CU.
constexpr int64_t kI8FewRows = 64;

// What a call runs on: its tile of rows by output channels, and its stages of K in LDS by DMA; 1 through
// registers (linear_i8_any_kernel), 0 straight from memory (linear_i8_few_kernel).
struct I8Plan {
    int bm, bn, stages;
};

// pieces: cin and the operands' addresses are multiples of 16.
I8Plan i8_plan(int64_t m, int n, int k, bool pieces) {
    if (m <= kI8FewRows) {
        const int64_t blocks = (n + 15) / 16 * ((m + 15) / 16);
        if (blocks <= 256 || m <= 16) return {16, 16, 0};
        if (blocks <= 512 || m <= 32) return {32, 16, 0};
        return {64, 16, 0};
    }
    auto tiles = [&](int bm, int bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
    if (!pieces) {
        // Rounds of tiles over the 256 CUs, 12.6 us each of 128 rows and 21.7 of 192 (4,739 x 1370 ->
        // 1021: 23.7 us in two rounds, 20.5 in one; 20,000 rows 58 and 61).  At 43 of 55 sizes, 500 to 42,000 rows
        // and 130 to 4090 deep, the pick is the faster form or within 5%; where 128 rows take three rounds
        // or more it is up to 20% slower (42,000 x 1370 -> 1021 122 us, 108 with 192 rows).
        auto rounds = [&](int bm) { return (tiles(bm, 128) + 255) / 256; };
        return {21.7 * rounds(192) < 12.6 * rounds(128) ? 192 : 128, 128, 1};
    }
    const I8Shape & c = kI8Shapes[i8_shape(m, n, k)];
    // Three stages where a CU has one tile at most, so that no second tile's stages need fit, and K is
    // longer than their start (1,500 x 4096 -> 2048 22 us against 27, 1,370 x 2048 -> 4096 19.6 against 20.4,
    // but 1,000 x 1024 -> 4096 9.8 against 9.5; four stages the same as three).
    const bool deep = k > kI8DeepK && tiles(c.bm, c.bn) <= 256;
    return {c.bm, c.bn, c.stages + (c.bn == 128 && deep ? 1 : 0)};
}

template <typename T, int EPI>
int launch_i8(I8Args a, hipStream_t s) {
    a.group_m = 8;
    const I8Plan p = i8_plan(a.m, a.n, a.k, a.k % 16 == 0 && aligned_to(a.x, 16) && aligned_to(a.w, 16));
    if (p.stages == 0) {
        if (p.bm == 16) return launch_i8_few<T, 1, EPI>(a, s);
        return p.bm == 32 ? launch_i8_few<T, 2, EPI>(a, s) : launch_i8_few<T, 4, EPI>(a, s);
    }
    if (p.stages == 1)
        return p.bm == 192 ? launch_i8_any<T, 192, 128, 8, 2, EPI>(a, s) : launch_i8_any<T, 128, 128, 8, 2, EPI>(a, s);
    switch (p.bm) {
    case 256: return launch_i8_tiles<T, 256, 256, 16, 4, 2, 1, EPI>(a, s);
    case 192:
        if (p.stages == 3) return launch_i8_tiles<T, 192, 128, 8, 2, 3, 1, EPI>(a, s);
        return launch_i8_tiles<T, 192, 128, 8, 2, 2, 1, EPI>(a, s);
    case 128:
        if (p.bn == 64) return launch_i8_tiles<T, 128, 64, 8, 4, 3, 1, EPI>(a, s);
        if (p.stages == 3) return launch_i8_tiles<T, 128, 128, 8, 2, 3, 1, EPI>(a, s);
        return launch_i8_tiles<T, 128, 128, 8, 2, 2, 1, EPI>(a, s);
    case 64: return launch_i8_tiles<T, 64, 64, 4, 2, 4, 1, EPI>(a, s);
    default: return launch_i8_tiles<T, 32, 64, 2, 1, 3, 4, EPI>(a, s);
    }
}

constexpr int kI8MaxInputs = 131071;  // 131,071 products of -128 by -128 stay below 2^31
constexpr int kI8MaxColumns = 1 << 30;  // columns are counted in 32 bits, a tile past their end

// The checks that the 8-bit linears share; *run is false where there is nothing to do.
int check_i8(const char * what, const int8_t * x, const float * x_scales, int64_t rows, int cin,
             const int8_t * weight, const float * w_scales, int cout, const void * out, bool * run) {
    *run = false;
    if (rows < 0 || cin <= 0 || cout <= 0) return fail_call(what, "bad shape");
    if (cin > kI8MaxInputs) return fail_call(what, "more than 131071 inputs (their sum may not fit 32 bits)");
    if (cout > kI8MaxColumns) return fail_call(what, "more than 2^30 outputs");
    if (rows == 0) return PXS_OK;
    if (!x || !x_scales || !weight || !w_scales || !out) return fail_call(what, "null pointer");
    *run = true;
    return PXS_OK;
}

} // namespace
} // namespace pxs

using namespace pxs;

extern "C" {

int pxs_quantize_rows_i8(int dtype, const void * x, int64_t ld_x, int64_t rows, int channels, int8_t * q,
                         float * scales, void * stream) {
    PXS_CHECK(dtype == PXS_F32 || dtype == PXS_BF16, PXS_ERR_ARG, "pxs_quantize_rows_i8: bad dtype");
    PXS_CHECK(rows >= 0 && channels > 0 && ld_x >= channels, PXS_ERR_ARG, "pxs_quantize_rows_i8: bad shape");
    PXS_CHECK(channels <= kI8MaxColumns, PXS_ERR_ARG, "pxs_quantize_rows_i8: more than 2^30 channels");
    if (rows == 0) return PXS_OK;
    PXS_CHECK(x && q && scales, PXS_ERR_ARG, "pxs_quantize_rows_i8: null pointer");
    QuantArgs a{x, ld_x, rows, channels, q, scales};
    return dtype == PXS_F32 ? launch_quantize<float>(a, as_stream(stream))
                            : launch_quantize<uint16_t>(a, as_stream(stream));
}

int pxs_linear_i8(const int8_t * x, const float * x_scales, int64_t rows, int cin, const int8_t * weight,
                  const float * w_scales, const float * bias, int cout, int act, int y_dtype, void * y,
                  void * stream) {
    PXS_CHECK(y_dtype == PXS_F32 || y_dtype == PXS_BF16, PXS_ERR_ARG, "pxs_linear_i8: bad dtype");
    PXS_CHECK(act == PXS_ACT_NONE || act == PXS_ACT_GELU_TANH || act == PXS_ACT_SILU, PXS_ERR_ARG,
              "pxs_linear_i8: bad activation");
    bool run;
    if (int rc = check_i8("pxs_linear_i8", x, x_scales, rows, cin, weight, w_scales, cout, y, &run)) return rc;
    if (!run) return PXS_OK;
    I8Args a{};
    a.x = x; a.x_scales = x_scales; a.w = weight; a.w_scales = w_scales; a.bias = bias;
    a.m = rows; a.k = cin; a.n = cout; a.act = act; a.y = y;
    a.vec_out = cout % 4 == 0 && aligned_to(y, y_dtype == PXS_BF16 ? 8 : 16) && aligned_to(w_scales, 16) &&
                (!bias || aligned_to(bias, 16));
    if (a.vec_out && cout % (y_dtype == PXS_BF16 ? 8 : 4) == 0 && aligned_to(y, 16)) a.vec_out = 2;
    return y_dtype == PXS_F32 ? launch_i8<float, kI8Store>(a, as_stream(stream))
                              : launch_i8<uint16_t, kI8Store>(a, as_stream(stream));
}

int pxs_linear_i8_tile(int64_t rows, int cin, int cout, int whole_pieces, int * tile) {
    bool run;
    const int8_t some = 0;
    const float one = 1.0f;
    if (int rc = check_i8("pxs_linear_i8_tile", &some, &one, rows, cin, &some, &one, cout, tile, &run)) return rc;
    PXS_CHECK(tile, PXS_ERR_ARG, "pxs_linear_i8_tile: null pointer");
    const I8Plan p = run ? i8_plan(rows, cout, cin, whole_pieces && cin % 16 == 0) : I8Plan{};
    tile[0] = p.bm;
    tile[1] = p.bn;
    tile[2] = p.stages;
    return PXS_OK;
}

int pxs_linear_i8_residual(const int8_t * x, const float * x_scales, int64_t rows, int cin, const int8_t * weight,
                           const float * w_scales, const float * bias, int cout, float * residual, void * stream) {
    bool run;
    if (int rc = check_i8("pxs_linear_i8_residual", x, x_scales, rows, cin, weight, w_scales, cout, residual, &run))
        return rc;
    if (!run) return PXS_OK;
    I8Args a{};
    a.x = x; a.x_scales = x_scales; a.w = weight; a.w_scales = w_scales; a.bias = bias;
    a.m = rows; a.k = cin; a.n = cout; a.residual = residual;
    a.vec_out = cout % 4 == 0 && aligned_to(residual, 16) && aligned_to(w_scales, 16) &&
                (!bias || aligned_to(bias, 16));
    return launch_i8<float, kI8AddResidual>(a, as_stream(stream));
}

int pxs_linear_i8_gate_residual(const int8_t * x, const float * x_scales, int64_t rows, int cin,
                                const int8_t * weight, const float * w_scales, const float * bias, int cout,
                                const int32_t * coords, const float * block_mod, const float * time_mod,
                                int gate_offset, float * residual, void * stream) {
    PXS_CHECK(gate_offset >= 0 && gate_offset <= 5 * static_cast<int64_t>(cout), PXS_ERR_ARG,
              "pxs_linear_i8_gate_residual: bad gate offset");
    bool run;
    if (int rc = check_i8("pxs_linear_i8_gate_residual", x, x_scales, rows, cin, weight, w_scales, cout, residual,
                          &run))
        return rc;
    if (!run) return PXS_OK;
    PXS_CHECK(coords && block_mod && time_mod, PXS_ERR_ARG, "pxs_linear_i8_gate_residual: null pointer");
    I8Args a{};
    a.x = x; a.x_scales = x_scales; a.w = weight; a.w_scales = w_scales; a.bias = bias;
    a.m = rows; a.k = cin; a.n = cout; a.residual = residual;
    a.coords = coords; a.block_mod = block_mod; a.time_mod = time_mod; a.gate_offset = gate_offset;
    a.vec_out = cout % 4 == 0 && aligned_to(residual, 16) && aligned_to(w_scales, 16) &&
                (!bias || aligned_to(bias, 16));
    return launch_i8<float, kI8Gate>(a, as_stream(stream));
}

} // extern "C"
