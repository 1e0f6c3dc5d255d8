// Microscaled 4-bit linears: blocks of 32 values of a row share a power of two, and a
// value is a sign, two bits of exponent and one of mantissa (e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6).
//
//   e = floor(log2 max|x|) - 2 of the block, -127 at least    scale byte = e + 127
//   code = the nearest of the eight magnitudes to |x| 2^-e, ties to the even code, past 6 6
//   Y[m, n] = sum_k x[m, k] w[n, k] + bias[n]      of the values that the codes stand for
//
// then an epilogue of the linears in 8 bits (linear_i8.hip): store with an activation, add to
// an fp32 residual, add to it through the adaLN gate.  A product of two values is exact, and
// the matrix cores take both operands' scales (v_mfma_scale_f32_*_f8f6f4); sums are fp32.
//
// Layout.  A row of codes is a whole number of blocks of 16 bytes, the earlier value of a byte in
// its low half, codes past the row's end zero.  A row of scale bytes is a whole number of 16
// bytes; what those past the last block hold does not matter.

#include "pxs_common.h"
#include "tiles.h"

#include <algorithm>
#include <iterator>
#include <limits>
#include <type_traits>

namespace pxs {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ constexpr int mx_blocks(int channels) { return channels / 32 + (channels % 32 != 0); }
__host__ __device__ constexpr int mx_scale_pitch(int channels) { return (mx_blocks(channels) + 15) / 16 * 16; }

// Units of a call from which a thread quantizes two: 42,017 x 4096 bf16 84 us (5.2 TB/s) with two, 90 with one;
// 1,370 x 1024 3.6 and 3.2, 4,739 x 1370 fp32 9.1 and 8.1.
constexpr int64_t kMxTwoUnits = 1 << 22;

constexpr uint32_t kMxNan = 255;  // the scale byte of a block that holds an infinity or a NaN

// ---- values to 4 bits and back ---------------------------------------------------

struct MxRows {
    const void * x;
    int64_t ldx;
    int64_t rows;
    int channels;
    uint8_t * codes;
    uint8_t * scales;
    void * y;
    int64_t ldy;
};

// The scale byte of a block with this largest magnitude (bits).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    return top >= 0x7F800000u ? kMxNan : static_cast<uint32_t>(max(static_cast<int>(top >> 23) - 2, 0));
}
// 2^-e of a scale byte below 253 (as any that mx_scale_byte gives).
__device__ __forceinline__ float mx_unscale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^e (2^-127 is no normal number).
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
    return __uint_as_float(byte == kMxNan ? 0x7FC00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// Rows and units of eight values of a range of (row, unit): i / per_row and i % per_row through a
// reciprocal, right for i below 2^51 (a 64-bit division took a third of a short call).
struct MxUnit {
    int64_t row;
    int unit;
};
__device__ __forceinline__ MxUnit mx_unit(int64_t i, int per_row, double inv) {
    int64_t row = static_cast<int64_t>(static_cast<double>(i) * inv);
    int64_t unit = i - row * per_row;
    if (unit < 0) {
        --row;
        unit += per_row;
    } else if (unit >= per_row) {
        ++row;
        unit -= per_row;
    }
    return {row, static_cast<int>(unit)};
}

// Four lanes a block, eight values each (16 bytes of bf16 or 32 of fp32 from any element, 4 bytes of codes);
// U of them a thread, 256 apart, all loaded ahead of the first's maximum.
template <typename T, int U>
__global__ void __launch_bounds__(256) quantize_mxfp4_kernel(MxRows a) {
    const int blocks = mx_blocks(a.channels), pitch = mx_scale_pitch(a.channels), per_row = blocks * 4;
    const double inv = 1.0 / per_row;
    const int64_t lanes = a.rows * per_row;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * (256 * U); i0 < lanes;
         i0 += static_cast<int64_t>(gridDim.x) * (256 * U)) {
        MxUnit at[U];
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + u * 256 + threadIdx.x;
            at[u] = mx_unit(min(i, lanes - 1), per_row, inv);
            const int c = at[u].unit * 8;
            const T * x = static_cast<const T *>(a.x) + at[u].row * a.ldx;
            if (i >= lanes) at[u].unit = -1;
            if (c + 8 <= a.channels) {
                T e[8];
                __builtin_memcpy(e, x + c, sizeof(e));
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = load_f32(e + j);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = c + j < a.channels ? load_f32(x + c + j) : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[u][j]) & 0x7FFFFFFFu);
            // (A block's four lanes are inside the range together: it is a multiple of four.)
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1, 64)));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2, 64)));
            const uint32_t byte = mx_scale_byte(top);
            const float per = mx_unscale(min(byte, 252u));  // exact, as is the product
            uint32_t code = 0;
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[u][0] * per, v[u][1] * per, 1.0f, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[u][2] * per, v[u][3] * per, 1.0f, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[u][4] * per, v[u][5] * per, 1.0f, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[u][6] * per, v[u][7] * per, 1.0f, 3);
            if (byte == kMxNan) code = 0;
            const int unit = at[u].unit, block = unit >> 2;
            if (unit < 0) continue;
            *reinterpret_cast<uint32_t *>(a.codes + (at[u].row * blocks + block) * 16 + (unit & 3) * 4) = code;
            uint8_t * scales = a.scales + at[u].row * pitch;
            if ((unit & 3) == 0) scales[block] = static_cast<uint8_t>(byte);
            if (block == blocks - 1)  // the row's padding
                for (int b = blocks + (unit & 3); b < pitch; b += 4) scales[b] = 127;
        }
    }
}

// 16 bytes of values a lane (eight of bf16, four of fp32), so that a wave's stores are one piece.  The stores
// pass the caches by: 42,017 x 4096 in bf16 87 us (5.0 TB/s) against 115, 8,192 x 8192 29 against 49.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_mxfp4_kernel(MxRows a) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const int blocks = mx_blocks(a.channels), pitch = mx_scale_pitch(a.channels), per_row = blocks * (32 / V);
    const double inv = 1.0 / per_row;
    const int64_t lanes = a.rows * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < lanes; i += static_cast<int64_t>(gridDim.x) * 256) {
        const MxUnit at = mx_unit(i, per_row, inv);
        const uint8_t * codes = a.codes + (at.row * per_row + at.unit) * (V / 2);
        uint32_t code;
        if constexpr (V == 8) code = *reinterpret_cast<const uint32_t *>(codes);
        else code = *reinterpret_cast<const uint16_t *>(codes);
        const float scale = mx_scale_value(a.scales[at.row * pitch + at.unit / (32 / V)]);
        T e[V];
        auto put = [&](int j, auto pair) __attribute__((always_inline)) {
            store_f32(e + j, pair[0] * scale);
            store_f32(e + j + 1, pair[1] * scale);
        };
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1));
        if constexpr (V == 8) {
            put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2));
            put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3));
        }
        const int c = at.unit * V;
        T * y = static_cast<T *>(a.y) + at.row * a.ldy + c;
        if (c + V <= a.channels) {
            store16_past(y, e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < a.channels) y[j] = e[j];
        }
    }
}

// ---- products -------------------------------------------------------------------

enum MxEpi { kMxStore = 0, kMxAddResidual = 1, kMxGate = 2 };

struct MxArgs {
    const uint8_t * x;         // [m, 16 blocks] codes
    const uint8_t * x_scales;  // [m, pitch]
    const uint8_t * w;         // [n, 16 blocks]
    const uint8_t * w_scales;  // [n, pitch]
    const float * bias;        // [n] or null
    int64_t m;
    int n;
    int blocks, pitch;         // of a row
    int act;
    void * y;                  // [m, n], store epilogue
    float * residual;          // [m, n] fp32, residual epilogues
    const int32_t * coords;    // [m, 4], gate epilogue: batch of each row
    const float * block_mod;   // gate = block_mod[gate_offset + c] + time_mod[b, gate_offset + c]
    const float * time_mod;    // [batch, 6 n]
    int gate_offset;
    int vec_out;               // 1: 4-channel vector accesses of all that the epilogue touches; 2: y in whole 16-byte pieces
    int group_m;               // tile order (tile_of)
};

// The activations through one exponential and one reciprocal, as the 8-bit linears'.
__device__ __forceinline__ float mx_gelu(float v) {
    const float e = v * __builtin_fmaf(v * v, -0.10294324f, -2.3022082f);  // -2 log2(e) u
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e));
}
__device__ __forceinline__ float mx_silu(float v) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

// The biases of four channels from c (past n, the last channel's).
struct MxBias {
    float v[4];
};
__device__ __forceinline__ MxBias mx_bias(const MxArgs & a, int c, bool vec) {
    MxBias o = {};
    if (!a.bias) return o;
    if (vec) {
        const float4 b4 = *reinterpret_cast<const float4 *>(a.bias + c);
        o.v[0] = b4.x; o.v[1] = b4.y; o.v[2] = b4.z; o.v[3] = b4.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = a.bias[min(c + e, a.n - 1)];
    }
    return o;
}

__device__ __forceinline__ void mx_values4(const MxArgs & a, const MxBias & b, const float (&sum)[4], float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sum[e] + b.v[e];
    if (a.act == PXS_ACT_GELU_TANH) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = mx_gelu(v[e]);
    } else if (a.act == PXS_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = mx_silu(v[e]);
    }
}

template <typename T> __device__ __forceinline__ void mx_put4(T * p, const float (&v)[4]) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

template <typename T, int EPI>
__device__ __forceinline__ void mx_epilogue4(const MxArgs & a, const MxBias & b, int64_t row, int batch, int c,
                                             const float (&sum)[4]) {
    const bool vec = a.vec_out && c + 3 < a.n;
    float v[4];
    mx_values4(a, b, sum, v);
    if constexpr (EPI == kMxStore) {
        T * p = static_cast<T *>(a.y) + row * a.n + c;
        if (vec) {
            mx_put4(p, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.n) store_f32(p + e, v[e]);
        }
    } else {
        float * p = a.residual + row * a.n + c;
        float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (EPI == kMxGate) {
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

// 16 bytes of codes as an operand (the instruction reads four registers of a 4-bit operand's eight).
__device__ __forceinline__ i32x8 mx_operand(const uint4 & v) {
    return i32x8{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
}

constexpr int kMxFp4 = 4;  // the operands' format: e2m1

// Up to 16 RB rows (single tokens): bound by reading the weights once.  A workgroup has 16
// output channels; its eight waves take every eighth group of 8 blocks of K, straight from memory to
// the operands of 16 x 16 x 128 products, and their sums are joined through LDS.  Of a group, lane
// (kq, l16) holds blocks 2 kq and 2 kq + 1 of channel l16 and of row l16.
constexpr int kFewWaves = 8;
template <typename T, int RB, int EPI>
__global__ void __launch_bounds__(kFewWaves * 64) linear_mxfp4_few_kernel(MxArgs a) {
    __shared__ __align__(16) float part[kFewWaves][RB * 16][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * RB);
    const int64_t wrow = min(n0 + l16, a.n - 1);
    const uint8_t * w = a.w + wrow * a.blocks * 16;
    const uint8_t * ws = a.w_scales + wrow * a.pitch;
    const uint8_t * x[RB];
    const uint8_t * xs[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int64_t row = min(m0 + b * 16 + l16, a.m - 1);
        x[b] = a.x + row * a.blocks * 16;
        xs[b] = a.x_scales + row * a.pitch;
    }
    f32x4 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = f32x4{};
    for (int g = wave; g * 8 < a.blocks; g += kFewWaves) {
        const int k0 = g * 8 + 2 * kq;
        const bool in[2] = {k0 < a.blocks, k0 + 1 < a.blocks};
        auto codes = [&](const uint8_t * row, int e) __attribute__((always_inline)) {
            return in[e] ? *reinterpret_cast<const uint4 *>(row + (k0 + e) * 16) : make_uint4(0u, 0u, 0u, 0u);
        };
        // Two scale bytes; past the last block 1, which the zero codes are multiplied with.
        auto scales = [&](const uint8_t * row) __attribute__((always_inline)) {
            const uint32_t s = *reinterpret_cast<const uint16_t *>(row + k0);
            return static_cast<int>((in[0] ? s & 255u : 127u) | (in[1] ? s & 0xFF00u : 127u << 8));
        };
        uint4 wf[2], xf[RB][2];
        int wsc = scales(ws), xsc[RB];
#pragma unroll
        for (int e = 0; e < 2; ++e) wf[e] = codes(w, e);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            xsc[b] = scales(xs[b]);
#pragma unroll
            for (int e = 0; e < 2; ++e) xf[b][e] = codes(x[b], e);
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(wf[0]), mx_operand(xf[b][0]), acc[b], kMxFp4,
                                                                      kMxFp4, 0, wsc, 0, xsc[b]);
            acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(wf[1]), mx_operand(xf[b][1]), acc[b], kMxFp4,
                                                                      kMxFp4, 1, wsc, 1, xsc[b]);
        }
    }
    // Lane (kq, l16) holds row l16's channels 4 kq .. 4 kq + 3.
#pragma unroll
    for (int b = 0; b < RB; ++b) *reinterpret_cast<f32x4 *>(&part[wave][b * 16 + l16][4 * kq]) = acc[b];
    __syncthreads();
    if (tid >= RB * 64) return;
    const int rl = tid >> 2, cl = (tid & 3) * 4;
    const int64_t row = m0 + rl;
    const int col = n0 + cl;
    if (row >= a.m || col >= a.n) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) {
        const f32x4 p = *reinterpret_cast<const f32x4 *>(&part[i][rl][cl]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += p[e];
    }
    mx_epilogue4<T, EPI>(a, mx_bias(a, col, a.vec_out && col + 3 < a.n), row, EPI == kMxGate ? a.coords[row * 4] : 0, col, sum);
}

// Row pitch in LDS of 32 rows of a wave's block, and 16 bytes against bank conflicts.
template <typename T, int WN> constexpr int mx_pitch() { return WN * static_cast<int>(sizeof(T)) + 16; }

// The gates of K channels from c, kept from a row to the next of its batch item.
template <int K> struct MxGates {
    int batch = -1;
    float g[K];
    __device__ __forceinline__ void to(const MxArgs & a, int item, int c) {
        if (item == batch) return;
        batch = item;
        const float * bm = a.block_mod + a.gate_offset;
        const float * tm = a.time_mod + static_cast<int64_t>(item) * 6 * a.n + a.gate_offset;
#pragma unroll
        for (int e = 0; e < K; ++e) {
            const int ce = min(c + e, a.n - 1);
            g[e] = bm[ce] + tm[ce];
        }
    }
};

// One wave's block of outputs: acc[i][j] holds 32 rows by 32 channels, lane (h, r) row r and
// channels 8 g + 4 h + e.  Values go through the wave's region of LDS (which no other wave uses
// any more), 32 rows at a time, so that an instruction covers row segments of 64 bytes and more.  Stores
// pass the caches by: what reads y next runs on other XCDs (8,192 x 8192 -> 4096 155 -> 148 us, 1,370 x 1024 -> 4096
// 12.6 -> 11.5).  A residual's values are loaded ahead of the block's (into one, 42,017 x 4096 -> 1024 214 -> 166 us).
template <typename T, int TI, int TJ, int EPI>
__device__ __forceinline__ void mx_tile_out(const MxArgs & a, const f32x16 (&acc)[TI][TJ], char * region, int64_t row0,
                                            int col0, int h, int r, int lane) {
    constexpr int WN = TJ * 32, kPitch = mx_pitch<T, WN>(), kElems = 16 / static_cast<int>(sizeof(T));
    constexpr int kLanesPerRow = WN / kElems, kRowsPerPass = 64 / kLanesPerRow, kPasses = 32 / kRowsPerPass;
    constexpr bool kAdds = EPI != kMxStore;
    static_assert(!kAdds || sizeof(T) == 4, "residuals are fp32");
    auto bias = [&](int j, int g) __attribute__((always_inline)) {
        const int c = min(col0 + j * 32 + 8 * g + 4 * h, a.n - 1);
        return mx_bias(a, c, a.vec_out && c + 3 < a.n);
    };
    MxBias held[TJ][4];  // every channel's, ahead of the first value
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) held[j][g] = bias(j, g);
    const int lr = lane / kLanesPerRow, lc = lane % kLanesPerRow, c16 = col0 + lc * kElems;
    static_assert(64 % WN == 0, "a lane's elements are of one channel");
    MxGates<4> gates;
    MxGates<1> gate;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int64_t block = row0 + i * 32;
        float4 old[kAdds ? kPasses : 1];
        int batch[EPI == kMxGate ? kPasses : 1];
        if (kAdds && a.vec_out == 2) {
#pragma unroll
            for (int pass = 0; pass < kPasses; ++pass) {
                const int64_t to = min(block + pass * kRowsPerPass + lr, a.m - 1);
                old[kAdds ? pass : 0] = *reinterpret_cast<const float4 *>(a.residual + to * a.n + min(c16, a.n - 4));
                if (EPI == kMxGate) batch[EPI == kMxGate ? pass : 0] = a.coords[to * 4];
            }
        }
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float sum[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                float v[4];
                mx_values4(a, held[j][g], sum, v);  // (past n: not stored)
                mx_put4(reinterpret_cast<T *>(region + r * kPitch + (j * 32 + 8 * g + 4 * h) * static_cast<int>(sizeof(T))), v);
            }
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own writes
        if (a.vec_out != 2) {  // an element a lane, in the order of their addresses
            constexpr int kStep = 64 / WN;  // rows of a pass
            const int rl = lane / WN, cl = lane % WN, c = col0 + cl;
            const int64_t left = c < a.n ? a.m - block - rl : 0;
            const char * from = region + rl * kPitch + cl * static_cast<int>(sizeof(T));
            T * to = static_cast<T *>(kAdds ? static_cast<void *>(a.residual) : a.y) + (block + rl) * a.n + c;
            const int64_t step = static_cast<int64_t>(kStep) * a.n;
#pragma unroll
            for (int first = 0; first < 32; first += 8 * kStep) {
                T v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const T *>(from + (first + u * kStep) * kPitch);
                if constexpr (kAdds) {
                    float o[8];
                    int item[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (first + u * kStep < left) {
                            o[u] = to[u * step];
                            item[u] = EPI == kMxGate ? a.coords[(block + rl + first + u * kStep) * 4] : 0;
                        }
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (first + u * kStep < left) {
                            if constexpr (EPI == kMxGate) gate.to(a, item[u], c);
                            to[u * step] = o[u] + (EPI == kMxGate ? v[u] * gate.g[0] : v[u]);
                        }
                } else {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (first + u * kStep < left) to[u * step] = v[u];
                }
                to += 8 * step;
            }
            continue;
        }
#pragma unroll
        for (int pass = 0; pass < kPasses; ++pass) {
            const int rl = pass * kRowsPerPass + lr;
            uint4 v = *reinterpret_cast<const uint4 *>(region + rl * kPitch + lc * 16);
            const int64_t to = block + rl;
            if (to < a.m && c16 < a.n) {
                if constexpr (kAdds) {
                    float4 f = __builtin_bit_cast(float4, v), & o = old[pass];
                    if constexpr (EPI == kMxGate) {
                        gates.to(a, batch[pass], c16);
                        f.x *= gates.g[0]; f.y *= gates.g[1]; f.z *= gates.g[2]; f.w *= gates.g[3];
                    }
                    o.x += f.x; o.y += f.y; o.z += f.z; o.w += f.w;
                    *reinterpret_cast<float4 *>(a.residual + to * a.n + c16) = o;
                } else {
                    store16_past(static_cast<T *>(a.y) + to * a.n + c16, &v);
                }
            }
        }
    }
}

// As the 8-bit products (linear_i8.hip): BM rows of X and BN rows of W go 128 bytes of codes (8 blocks)
// at a time from L2 to LDS by DMA, NSTAGE stages in flight, and a lane reads 16 contiguous bytes per
// fragment, one block; the K order inside a stage is permuted alike for both operands, lane (h, r) of
// step u taking block 4 h + u.  So the four steps' scales of a lane are one 32-bit word of the row's
// scale bytes, and the instruction picks its byte.  Scale bytes come by DMA as well, 32 of a row (four
// stages) at a time, ahead of the codes of the first of the four.
// A 32 x 32 x 64 product takes the cycles of an 8-bit one of half its depth: bytes, stages and LDS
// traffic are those of the 8-bit kernel and the rate is twice its.  Bound by no single unit: at 8,192 x 8192
// -> 4096 (144 us, 3,830 TFLOP/s, 3.6 times the 16-bit library product's rate) the matrix cores are busy 48%
// of the cycles, the return path of the DMA 56% and LDS 56% (17 of them bank conflicts), in step with one
// another.  (Beside 148 us on another card, 64 x 64 a wave and 16 waves 162, 128 x 128 and four waves 184.)
//
// KG groups of NW waves share a tile and take every KG-th stage each, in stages of their own (KG 4:
// a group's stages are one of each four, and each loads its own scales); the groups' sums are added
// through LDS in their order.  For calls of few tiles, whose time is the chain of stages.
__device__ __align__(16) uint4 g_mx_zero[8];  // K pieces past the end

constexpr int kMxKB = 128;           // bytes of codes of a row and stage
constexpr int kMxScaleStages = 4;    // stages that a slot of scale bytes serves
constexpr int kMxScaleRow = 32;      // its bytes of a row
// (Those of stage s + nstage are loaded as stage s begins.)
constexpr int mx_scale_slots(int nstage) { return (nstage + kMxScaleStages - 1) / kMxScaleStages + 1; }

template <int U>
__device__ __forceinline__ f32x16 mx_mfma(const uint4 & w, const uint4 & x, const f32x16 & acc, uint32_t ws, uint32_t xs) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(w), mx_operand(x), acc, kMxFp4, kMxFp4, U,
                                                           static_cast<int>(ws), U, static_cast<int>(xs));
}

template <typename T, int BM, int BN, int NW, int WAVES_M, int NSTAGE, int KG, int EPI>
__global__ void __launch_bounds__(NW * KG * 64) linear_mxfp4_kernel(MxArgs a) {
    constexpr int KB = kMxKB, P = 8, RPI = 8;  // bytes, pieces per row of a stage; rows per DMA instruction
    constexpr int WAVES_N = NW / WAVES_M, WM = BM / WAVES_M, WN = BN / WAVES_N, TI = WM / 32, TJ = WN / 32;
    constexpr int kStage = (BM + BN) * KB;
    constexpr int AI = BM / (RPI * NW), BI = BN / (RPI * NW), kPerStage = AI + BI;
    static_assert(AI * RPI * NW == BM && BI * RPI * NW == BN, "tile rows must split over the waves");
    // Scales: a DMA instruction takes 32 rows; slots of all rows behind the stages.
    constexpr int kSlots = mx_scale_slots(KG > 1 ? 4 * NSTAGE : NSTAGE), kSlot = (BM + BN) * kMxScaleRow, kScaleInstr = (BM + BN) / 32;
    constexpr int kScalePerWave = (kScaleInstr + NW - 1) / NW;
    constexpr int kRing = NSTAGE * kStage + kSlots * kSlot;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int group = KG > 1 ? __builtin_amdgcn_readfirstlane(tid / (NW * 64)) : 0;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) - group * NW;  // in its group
    char * ring = smem + group * kRing;
    char * scale_ring = ring + NSTAGE * kStage;
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int h = lane >> 5, r = lane & 31;
    const int tiles_n = (a.n + BN - 1) / BN, tiles_m = static_cast<int>((a.m + BM - 1) / BM);
    int tm, tn;
    tile_of(remap_xcd(blockIdx.x, gridDim.x), tiles_m, tiles_n, a.group_m, tm, tn);
    const int64_t p0 = static_cast<int64_t>(tm) * BM;
    const int n0 = tn * BN;
    const int64_t row_bytes = static_cast<int64_t>(a.blocks) * 16;
    const uint8_t * xs = a.x + p0 * row_bytes;
    const uint8_t * wsb = a.w + static_cast<int64_t>(n0) * row_bytes;
    const int all_stages = (a.blocks + P - 1) / P;
    const int stages = (all_stages - group + KG - 1) / KG;       // of this group
    const int steps = KG > 1 ? (all_stages + KG - 1) / KG : stages;  // of every group
    const int lrow = lane / P, lslot = lane % P;
    const int64_t last_x = a.m - 1 - p0;
    const int last_w = a.n - 1 - n0;
    uint32_t off[kPerStage];  // rows past the end are clamped; their outputs are not stored
#pragma unroll
    for (int j = 0; j < kPerStage; ++j) {
        const bool is_x = j < AI;
        const int row = (wave * (is_x ? AI : BI) + (is_x ? j : j - AI)) * RPI + lrow;
        const int64_t at = is_x ? min(static_cast<int64_t>(row), last_x) : static_cast<int64_t>(min(row, last_w));
        off[j] = static_cast<uint32_t>(at * row_bytes + (lslot ^ piece_swz<KB>(row)) * 16);
    }
    // This lane's row of each of the wave's scale instructions, two lanes a row.
    const uint8_t * scale_row[kScalePerWave];
#pragma unroll
    for (int j = 0; j < kScalePerWave; ++j) {
        const int row = (wave + j * NW) * 32 + (lane >> 1);
        const bool is_x = row < BM;
        const int64_t at = is_x ? p0 + min(static_cast<int64_t>(row), last_x) : n0 + static_cast<int64_t>(min(row - BM, last_w));
        scale_row[j] = (is_x ? a.x_scales : a.w_scales) + at * a.pitch + (lane & 1) * 16;
    }
    // Stage s of this group is stage s * KG + group of the row; its scales lie in the 32 bytes of its four.
    auto issue_scales = [&](int s) __attribute__((always_inline)) {
        if (s % kMxScaleStages != 0 && KG == 1) return;
        const int at = (s * KG + group) / kMxScaleStages;
        const int slot = (KG == 1 ? s / kMxScaleStages : s) % kSlots;
#pragma unroll
        for (int j = 0; j < kScalePerWave; ++j) {
            const int instr = wave + j * NW;
            if (instr >= kScaleInstr) break;
            const bool in = at * kMxScaleRow + (lane & 1) * 16 < a.pitch;
            lds_dma16(in ? static_cast<const void *>(scale_row[j] + at * kMxScaleRow) : static_cast<const void *>(g_mx_zero),
                      lds_offset(scale_ring + slot * kSlot + instr * 1024));
        }
    };
    auto issue_one = [&](int s, int q, bool last) __attribute__((always_inline)) {
        const bool is_x = q < AI;
        const int row0 = (wave * (is_x ? AI : BI) + (is_x ? q : q - AI)) * RPI;
        const uint32_t lds = lds_offset(ring + (s % NSTAGE) * kStage + ((is_x ? 0 : BM) + row0) * KB);
        const int at = s * KG + group;
        const uint8_t * src = (is_x ? xs : wsb) + static_cast<int64_t>(at) * KB;
        if (last) {
            const bool in = at * P + (lslot ^ piece_swz<KB>(row0 + lrow)) < a.blocks;  // (a last stage may hold pieces past the row)
            lds_dma16(in ? static_cast<const void *>(src + off[q]) : static_cast<const void *>(g_mx_zero), lds);
        } else {
            lds_dma16_sbase(src, off[q], lds);
        }
    };
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = f32x16{};
#pragma unroll
    for (int s = 0; s < NSTAGE; ++s)
        if (s < stages) {
            issue_scales(s);
#pragma unroll
            for (int q = 0; q < kPerStage; ++q) issue_one(s, q, true);
        }
    // A step's fragments are read while the step before multiplies, those of a stage's first step beside the last
    // products of the stage before: the wait for its DMA and the barrier lie ahead of those, when every wave holds
    // the last fragments of its stage, whose slot is filled anew at once.
    uint4 xf[2][TI], wf[2][TJ];
    uint32_t xsc[TI], wsc[TJ], xnext[TI], wnext[TJ];
    auto read_frags = [&](int s, int u, uint4 (&xo)[TI], uint4 (&wo)[TJ]) __attribute__((always_inline)) {
        const char * sx = ring + (s % NSTAGE) * kStage;
        const char * sw = sx + BM * KB;
        const int piece = (P / 2) * h + u;
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            const int row = wm * WM + i * 32 + r;
            xo[i] = *reinterpret_cast<const uint4 *>(sx + row * KB + ((piece ^ piece_swz<KB>(row)) << 4));
        }
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            const int row = wn * WN + j * 32 + r;
            wo[j] = *reinterpret_cast<const uint4 *>(sw + row * KB + ((piece ^ piece_swz<KB>(row)) << 4));
        }
    };
    // The lanes' scale words.
    auto read_scales = [&](int s, uint32_t (&xo)[TI], uint32_t (&wo)[TJ]) __attribute__((always_inline)) {
        const int at = s * KG + group;
        const char * sc = scale_ring + (KG == 1 ? s / kMxScaleStages : s) % kSlots * kSlot + at % kMxScaleStages * 8 + 4 * h;
#pragma unroll
        for (int i = 0; i < TI; ++i) xo[i] = *reinterpret_cast<const uint32_t *>(sc + (wm * WM + i * 32 + r) * kMxScaleRow);
#pragma unroll
        for (int j = 0; j < TJ; ++j) wo[j] = *reinterpret_cast<const uint32_t *>(sc + (BM + wn * WN + j * 32 + r) * kMxScaleRow);
    };
    // Stage s's, taken into use: those of blocks past the row's end, in its last stage, count as 1, whatever the
    // bytes hold.
    auto use_scales = [&](int s, bool ends) __attribute__((always_inline)) {
        const int valid = a.blocks - ((s * KG + group) * P + 4 * h);
        const uint32_t keep = !ends || valid >= 4 ? ~0u : valid <= 0 ? 0u : (1u << (8 * valid)) - 1u;
#pragma unroll
        for (int i = 0; i < TI; ++i) xsc[i] = (xnext[i] & keep) | (~keep & 0x7F7F7F7Fu);
#pragma unroll
        for (int j = 0; j < TJ; ++j) wsc[j] = (wnext[j] & keep) | (~keep & 0x7F7F7F7Fu);
    };
    // Stage s, whose first fragments and scales are read.  MORE: what is loaded beside its last products, 1 a stage
    // that is not the group's last, 2 the last, 0 none; 3: there is no next stage.  (Bodies without branches
    // between their products: the compiler moves the products past any to the stage's end, with all its
    // fragments alive until there, and the large tiles spill.)
    auto stage = [&](int s, auto what) __attribute__((always_inline)) {
        constexpr int MORE = decltype(what)::value;
        auto products = [&](auto which) __attribute__((always_inline)) {
            constexpr int u = decltype(which)::value;
            if constexpr (u + 1 < P / 2) read_frags(s, u + 1, xf[(u + 1) & 1], wf[(u + 1) & 1]);
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j) {
                    acc[i][j] = mx_mfma<u>(wf[u & 1][j], xf[u & 1][i], acc[i][j], wsc[j], xsc[i]);
                    if constexpr (u == P / 2 - 1 && (MORE == 1 || MORE == 2)) {
#pragma unroll
                        for (int q = 0; q < kPerStage; ++q)
                            if (q * (TI * TJ) / kPerStage == i * TJ + j) issue_one(s + NSTAGE, q, MORE == 2);
                    }
                }
        };
        if constexpr (MORE == 1 || MORE == 2) issue_scales(s + NSTAGE);
        products(std::integral_constant<int, 0>{});
        products(std::integral_constant<int, 1>{});
        products(std::integral_constant<int, 2>{});
        if constexpr (MORE != 3) {
            // (Counts codes alone: with scales of a later stage in flight it waits for some of that stage too.)
            wait_stages<NSTAGE - 2, kPerStage>(MORE > 0 ? NSTAGE : stages - 2 - s);
            barrier_no_fence();
            read_scales(s + 1, xnext, wnext);
            read_frags(s + 1, 0, xf[0], wf[0]);
        }
        products(std::integral_constant<int, 3>{});
        if constexpr (MORE != 3) use_scales(s + 1, MORE == 0);
    };
    if (KG == 1 || stages > 0) {
        wait_stages<NSTAGE - 1, kPerStage>(stages - 1);
        barrier_no_fence();
        read_scales(0, xnext, wnext);
        read_frags(0, 0, xf[0], wf[0]);
        use_scales(0, true);
        int s = 0;
        for (; s + NSTAGE + 1 < stages; ++s) stage(s, std::integral_constant<int, 1>{});
        if (s + NSTAGE + 1 == stages) stage(s++, std::integral_constant<int, 2>{});
        for (; s + 1 < stages; ++s) stage(s, std::integral_constant<int, 0>{});
        stage(s, std::integral_constant<int, 3>{});
    }
    // (Or the compiler moves the last products into the epilogue's branches, and spills.)
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) asm volatile("" : "+v"(acc[i][j]));
    if constexpr (KG > 1)
        for (int s = stages; s < steps; ++s) barrier_no_fence();  // (of groups with a stage more)
    barrier_no_fence();  // every wave is done with the stages
    constexpr int kOut = NW * 32 * mx_pitch<T, WN>();
    if constexpr (KG > 1) {
        // [group - 1][wave][register][lane], behind the first group's store regions
        float * sums = reinterpret_cast<float *>(smem + kOut) + wave * TI * TJ * 16 * 64 + lane;
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
    mx_tile_out<T, TI, TJ, EPI>(a, acc, smem + wave * 32 * mx_pitch<T, WN>(), p0 + wm * WM, n0 + wn * WN, h, r, lane);
}

bool aligned_to(const void * p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A launch counts its threads in 32 bits.
bool mx_grid_fits(int64_t workgroups, int threads) { return workgroups <= UINT32_MAX / threads; }
int check_mx_grid(int64_t workgroups, int threads) {
    PXS_CHECK(mx_grid_fits(workgroups, threads), PXS_ERR_ARG, "4-bit linear grid too large");
    return PXS_OK;
}

template <typename T, int RB, int EPI>
int launch_mx_few(const MxArgs & a, hipStream_t s) {
    const int64_t rows = (a.m + 16 * RB - 1) / (16 * RB);
    PXS_CHECK(rows <= 65535, PXS_ERR_ARG, "4-bit linear grid too large");
    const dim3 grid(grid_for(a.n, 16), static_cast<unsigned>(rows));
    if (int rc = check_mx_grid(grid.x * rows, kFewWaves * 64)) return rc;
    hipLaunchKernelGGL((linear_mxfp4_few_kernel<T, RB, EPI>), grid, dim3(kFewWaves * 64), 0, s, a);
    return check_launch("4-bit linear of few rows");
}

template <typename T, int BM, int BN, int NW, int WAVES_M, int NSTAGE, int KG, int EPI>
int launch_mx_tiles(const MxArgs & a, hipStream_t s) {
    constexpr int WN = BN / (NW / WAVES_M), kOut = NW * 32 * mx_pitch<T, WN>();
    constexpr int kStages = KG * (NSTAGE * (BM + BN) * kMxKB + mx_scale_slots(KG > 1 ? 4 * NSTAGE : NSTAGE) * (BM + BN) * kMxScaleRow);
    constexpr int kEnd = kOut + (KG - 1) * BM * BN * 4, smem = kStages > kEnd ? kStages : kEnd;
    static_assert(smem <= 160 * 1024, "LDS");
    const int64_t blocks = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    if (int rc = check_mx_grid(blocks, NW * KG * 64)) return rc;
    auto kernel = &linear_mxfp4_kernel<T, BM, BN, NW, WAVES_M, NSTAGE, KG, EPI>;
    if constexpr (smem > 64 * 1024) {
        static std::atomic<uint64_t> done{0};
        if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), smem, done, "hipFuncSetAttribute(linear_mxfp4)")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(NW * KG * 64), smem, s, a);
    return check_launch("4-bit linear");
}

// Tile shapes, their time alone on a CU and their share of a full CU's time, in us for
// 1024 bytes of codes a row more and without any: fitted to each shape's times at 64 sizes (66 to 42,017
// rows, 256 to 8192 deep), where the shape picked takes 0.6% more than the best on average, 17% at most (2,873 x
// 256 -> 1024):
//   256 x 256, 8 waves of 128 x 64, one workgroup a CU:  8,192 x 8192 -> 4096 144 us (3,830 TFLOP/s), next best 192
//   128 x 128, 8 waves, two stages and two workgroups:   1,370 x 1024 -> 4096 11.6 against 14.6
//   the same, three stages and one workgroup:            2,000 x 4096 -> 2048 17.9 against 19.5
//   64 x 64, 4 waves, two:                               150 x 4096 -> 4096 10.6 against 15.5
//   32 x 64, four groups of two waves over K, one:       87 x 8192 -> 1024 11.3 against 14.2
// (bf16 outputs; another output's bytes, or a residual's, change no choice.)
struct MxShape {
    int bm, bn, stages, threads;
    double alone0, alone1, each0, each1;
};
constexpr MxShape kMxShapes[] = {
    {256, 256, 2, 512, 11.4, 10.3, 8.5, 16.5}, {128, 128, 2, 512, 6.1, 4.9, 3.3, 4.5}, {128, 128, 3, 512, 6.5, 4.2, 4.3, 5.2},
    {64, 64, 4, 256, 6.0, 2.2, 1.9, 2.0},      {32, 64, 2, 512, 6.1, 1.5, 3.0, 1.9},
};

// Of the shapes whose grid can be launched, the one of the least time (the largest, if there is none: refused).
int mx_shape(int64_t m, int n, int blocks, double & least) {
    int best = 0;
    least = std::numeric_limits<double>::infinity();
    for (int i = 0; i < static_cast<int>(std::size(kMxShapes)); ++i) {
        const MxShape & c = kMxShapes[i];
        const double deep = blocks / 64.0, alone = c.alone0 + c.alone1 * deep, each = c.each0 + c.each1 * deep;
        const int64_t tiles = ((m + c.bm - 1) / c.bm) * ((n + c.bn - 1) / c.bn);
        const double time = tiles <= 256 ? alone + std::max(0.0, each - alone) * (tiles / 256.0)
                                         : std::max(alone, ((tiles + 255) / 256) * each);
        if (time < least && mx_grid_fits(tiles, c.threads)) {
            least = time;
            best = i;
        }
    }
    return best;
}

// Up to kMxFewRows rows a workgroup may have 16 output channels and as few of the rows' 16-row blocks as keep the
// workgroups near one a CU, straight from memory.  Its time is its launch's and that of the codes that a CU
// loads, 24 KB a us (within 10% of the measured at 32 sizes of 1 to 64 rows), and it is taken where that is
// less than the tiles': 1 x 1024 -> 4096 4.8 us against 6.2, 16 x 4096 -> 4096 7.0 and 9.1, 16 x 4096 -> 14336 15.2
// and 10.9, 64 x 8192 -> 1024 9.5 and 12.1, 64 x 4096 -> 4096 11.5 and 9.4.
constexpr int64_t kMxFewRows = 64;

// What a call runs on: its tile of rows by output channels, and its stages of K in LDS by DMA; 0
// straight from memory (linear_mxfp4_few_kernel).
struct MxPlan {
    int bm, bn, stages;
};
MxPlan mx_plan(int64_t m, int n, int blocks) {
    double tiles;
    const MxShape & c = kMxShapes[mx_shape(m, n, blocks, tiles)];
    if (m <= kMxFewRows) {
        const int64_t columns = (n + 15) / 16, row_blocks = (m + 15) / 16;
        const int rb = columns * row_blocks <= 256 || m <= 16 ? 1 : columns * row_blocks <= 512 || m <= 32 ? 2 : 4;
        const int64_t workgroups = columns * ((row_blocks + rb - 1) / rb);
        const int64_t rows = 16 + std::min<int64_t>(16 * rb, m);  // of codes that one loads, its channels' and its rows'
        const double few = 4.3 + 0.042 * static_cast<double>((workgroups + 255) / 256 * rows) * blocks / 64.0;
        if (few < tiles && mx_grid_fits(workgroups, kFewWaves * 64)) return {16 * rb, 16, 0};
    }
    return {c.bm, c.bn, c.stages};
}

template <typename T, int EPI>
int launch_mx(MxArgs a, hipStream_t s) {
    a.group_m = 8;
    const MxPlan p = mx_plan(a.m, a.n, a.blocks);
    if (p.stages == 0) {
        if (p.bm == 16) return launch_mx_few<T, 1, EPI>(a, s);
        return p.bm == 32 ? launch_mx_few<T, 2, EPI>(a, s) : launch_mx_few<T, 4, EPI>(a, s);
    }
    switch (p.bm) {
    case 256: return launch_mx_tiles<T, 256, 256, 8, 2, 2, 1, EPI>(a, s);
    case 128:
        if (p.stages == 3) return launch_mx_tiles<T, 128, 128, 8, 2, 3, 1, EPI>(a, s);
        return launch_mx_tiles<T, 128, 128, 8, 2, 2, 1, EPI>(a, s);
    case 64: return launch_mx_tiles<T, 64, 64, 4, 2, 4, 1, EPI>(a, s);
    default: return launch_mx_tiles<T, 32, 64, 2, 1, 2, 4, EPI>(a, s);
    }
}

constexpr int kMxMaxColumns = 1 << 30;  // columns are counted in 32 bits, a tile past their end
constexpr int kMxMaxInputs = 1 << 24;   // a tile's 256 rows of codes are reached with 32-bit offsets

// The checks that the 4-bit linears share; *run is false where there is nothing to do.
int check_mx(const char * what, const uint8_t * x, const uint8_t * x_scales, int64_t rows, int cin, const uint8_t * weight,
             const uint8_t * w_scales, int cout, const void * out, bool * run) {
    *run = false;
    if (rows < 0 || cin <= 0 || cout <= 0) return fail_call(what, "bad shape");
    if (cin > kMxMaxInputs) return fail_call(what, "more than 2^24 inputs");
    if (cout > kMxMaxColumns) return fail_call(what, "more than 2^30 outputs");
    if (rows == 0) return PXS_OK;
    if (!x || !x_scales || !weight || !w_scales || !out) return fail_call(what, "null pointer");
    if (!aligned_to(x, 16) || !aligned_to(x_scales, 16) || !aligned_to(weight, 16) || !aligned_to(w_scales, 16))
        return fail_call(what, "codes and scales must be 16-byte aligned");
    *run = true;
    return PXS_OK;
}

MxArgs mx_args(const uint8_t * x, const uint8_t * x_scales, int64_t rows, int cin, const uint8_t * weight,
               const uint8_t * w_scales, const float * bias, int cout, const void * out, int out_bytes) {
    MxArgs a{};
    a.x = x; a.x_scales = x_scales; a.w = weight; a.w_scales = w_scales; a.bias = bias;
    a.m = rows; a.n = cout; a.blocks = mx_blocks(cin); a.pitch = mx_scale_pitch(cin);
    a.vec_out = cout % 4 == 0 && aligned_to(out, 4 * out_bytes) && (!bias || aligned_to(bias, 16));
    if (a.vec_out && cout % (16 / out_bytes) == 0 && aligned_to(out, 16)) a.vec_out = 2;
    return a;
}

// The checks and arguments of the two conversions.
int check_mx_rows(const char * what, int dtype, const void * values, int64_t ld, int64_t rows, int channels,
                  const uint8_t * codes, const uint8_t * scales) {
    if (dtype != PXS_F32 && dtype != PXS_BF16) return fail_call(what, "bad dtype");
    if (rows < 0 || channels <= 0 || ld < channels) return fail_call(what, "bad shape");
    if (channels > kMxMaxColumns) return fail_call(what, "more than 2^30 channels");
    if (rows == 0) return PXS_OK;
    if (!values || !codes || !scales) return fail_call(what, "null pointer");
    if (!aligned_to(codes, 16) || !aligned_to(scales, 16)) return fail_call(what, "codes and scales must be 16-byte aligned");
    return PXS_OK;
}
unsigned mx_grid(int64_t lanes, int each) {
    return static_cast<unsigned>(std::min<int64_t>((lanes + 256 * each - 1) / (256 * each), 1 << 20));
}

template <typename T>
int launch_quantize(const MxRows & a, hipStream_t s) {
    const int64_t lanes = a.rows * mx_blocks(a.channels) * 4;  // (eight values each)
    if (lanes >= kMxTwoUnits) hipLaunchKernelGGL((quantize_mxfp4_kernel<T, 2>), dim3(mx_grid(lanes, 2)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((quantize_mxfp4_kernel<T, 1>), dim3(mx_grid(lanes, 1)), dim3(256), 0, s, a);
    return check_launch("quantize to 4 bits");
}

template <typename T>
int launch_dequantize(const MxRows & a, hipStream_t s) {
    hipLaunchKernelGGL(dequantize_mxfp4_kernel<T>, dim3(mx_grid(a.rows * mx_blocks(a.channels) * (sizeof(T) == 2 ? 4 : 8), 1)), dim3(256), 0, s, a);
    return check_launch("values of 4 bits");
}

} // namespace
} // namespace pxs

using namespace pxs;

extern "C" {

size_t pxs_mxfp4_code_bytes(int channels) { return channels > 0 ? static_cast<size_t>(mx_blocks(channels)) * 16 : 0; }
size_t pxs_mxfp4_scale_bytes(int channels) { return channels > 0 ? static_cast<size_t>(mx_scale_pitch(channels)) : 0; }

int pxs_quantize_mxfp4(int dtype, const void * x, int64_t ld_x, int64_t rows, int channels, uint8_t * codes,
                       uint8_t * scales, void * stream) {
    if (int rc = check_mx_rows("pxs_quantize_mxfp4", dtype, x, ld_x, rows, channels, codes, scales)) return rc;
    if (rows == 0) return PXS_OK;
    MxRows a{x, ld_x, rows, channels, codes, scales, nullptr, 0};
    return dtype == PXS_F32 ? launch_quantize<float>(a, as_stream(stream)) : launch_quantize<uint16_t>(a, as_stream(stream));
}

int pxs_dequantize_mxfp4(const uint8_t * codes, const uint8_t * scales, int64_t rows, int channels, int dtype, void * y,
                         int64_t ld_y, void * stream) {
    if (int rc = check_mx_rows("pxs_dequantize_mxfp4", dtype, y, ld_y, rows, channels, codes, scales)) return rc;
    if (rows == 0) return PXS_OK;
    MxRows a{nullptr, 0, rows, channels, const_cast<uint8_t *>(codes), const_cast<uint8_t *>(scales), y, ld_y};
    return dtype == PXS_F32 ? launch_dequantize<float>(a, as_stream(stream)) : launch_dequantize<uint16_t>(a, as_stream(stream));
}

int pxs_linear_mxfp4(const uint8_t * x, const uint8_t * x_scales, int64_t rows, int cin, const uint8_t * weight,
                     const uint8_t * w_scales, const float * bias, int cout, int act, int y_dtype, void * y, void * stream) {
    PXS_CHECK(y_dtype == PXS_F32 || y_dtype == PXS_BF16, PXS_ERR_ARG, "pxs_linear_mxfp4: bad dtype");
    PXS_CHECK(act == PXS_ACT_NONE || act == PXS_ACT_GELU_TANH || act == PXS_ACT_SILU, PXS_ERR_ARG,
              "pxs_linear_mxfp4: bad activation");
    bool run;
    if (int rc = check_mx("pxs_linear_mxfp4", x, x_scales, rows, cin, weight, w_scales, cout, y, &run)) return rc;
    if (!run) return PXS_OK;
    MxArgs a = mx_args(x, x_scales, rows, cin, weight, w_scales, bias, cout, y, y_dtype == PXS_BF16 ? 2 : 4);
    a.act = act; a.y = y;
    return y_dtype == PXS_F32 ? launch_mx<float, kMxStore>(a, as_stream(stream))
                              : launch_mx<uint16_t, kMxStore>(a, as_stream(stream));
}

int pxs_linear_mxfp4_tile(int64_t rows, int cin, int cout, int * tile) {
    PXS_CHECK(rows >= 0 && cin > 0 && cout > 0 && cin <= kMxMaxInputs && cout <= kMxMaxColumns, PXS_ERR_ARG,
              "pxs_linear_mxfp4_tile: bad shape");
    PXS_CHECK(tile, PXS_ERR_ARG, "pxs_linear_mxfp4_tile: null pointer");
    const MxPlan p = rows > 0 ? mx_plan(rows, cout, mx_blocks(cin)) : MxPlan{};
    tile[0] = p.bm;
    tile[1] = p.bn;
    tile[2] = p.stages;
    return PXS_OK;
}

int pxs_linear_mxfp4_residual(const uint8_t * x, const uint8_t * x_scales, int64_t rows, int cin, const uint8_t * weight,
                              const uint8_t * w_scales, const float * bias, int cout, float * residual, void * stream) {
    bool run;
    if (int rc = check_mx("pxs_linear_mxfp4_residual", x, x_scales, rows, cin, weight, w_scales, cout, residual, &run))
        return rc;
    if (!run) return PXS_OK;
    MxArgs a = mx_args(x, x_scales, rows, cin, weight, w_scales, bias, cout, residual, 4);
    a.residual = residual;
    return launch_mx<float, kMxAddResidual>(a, as_stream(stream));
}

int pxs_linear_mxfp4_gate_residual(const uint8_t * x, const uint8_t * x_scales, int64_t rows, int cin,
                                   const uint8_t * weight, const uint8_t * w_scales, const float * bias, int cout,
                                   const int32_t * coords, const float * block_mod, const float * time_mod,
                                   int gate_offset, float * residual, void * stream) {
    PXS_CHECK(gate_offset >= 0 && gate_offset <= 5 * static_cast<int64_t>(cout), PXS_ERR_ARG,
              "pxs_linear_mxfp4_gate_residual: bad gate offset");
    bool run;
    if (int rc = check_mx("pxs_linear_mxfp4_gate_residual", x, x_scales, rows, cin, weight, w_scales, cout, residual, &run))
        return rc;
    if (!run) return PXS_OK;
    PXS_CHECK(coords && block_mod && time_mod, PXS_ERR_ARG, "pxs_linear_mxfp4_gate_residual: null pointer");
    MxArgs a = mx_args(x, x_scales, rows, cin, weight, w_scales, bias, cout, residual, 4);
    a.residual = residual;
    a.coords = coords; a.block_mod = block_mod; a.time_mod = time_mod; a.gate_offset = gate_offset;
    return launch_mx<float, kMxGate>(a, as_stream(stream));
}

} // extern "C"
