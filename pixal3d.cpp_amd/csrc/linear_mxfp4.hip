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

bool aligned_to(const void * p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_mx_grid(int64_t blocks, int threads) {
    PXS_CHECK(blocks <= UINT32_MAX / threads, PXS_ERR_ARG, "4-bit linear grid too large");
    return PXS_OK;
}

template <typename T, int RB, int EPI>
int launch_mx_few(const MxArgs & a, hipStream_t s) {
    const int64_t rows = (a.m + 16 * RB - 1) / (16 * RB);
    PXS_CHECK(rows <= 65535, PXS_ERR_ARG, "4-bit linear grid too large");
    const dim3 grid(grid_for(a.n, 16), static_cast<unsigned>(rows));
    if (int rc = check_mx_grid(grid.x, kFewWaves * 64)) return rc;
    hipLaunchKernelGGL((linear_mxfp4_few_kernel<T, RB, EPI>), grid, dim3(kFewWaves * 64), 0, s, a);
    return check_launch("4-bit linear of few rows");
}

template <typename T, int EPI>
int launch_mx(const MxArgs & a, hipStream_t s) {
    if (a.m <= 16) return launch_mx_few<T, 1, EPI>(a, s);
    return launch_mx_few<T, 4, EPI>(a, s);
}

constexpr int kMxMaxColumns = 1 << 30;  // columns are counted in 32 bits, a tile past their end

// The checks that the 4-bit linears share; *run is false where there is nothing to do.
int check_mx(const char * what, const uint8_t * x, const uint8_t * x_scales, int64_t rows, int cin, const uint8_t * weight,
             const uint8_t * w_scales, int cout, const void * out, bool * run) {
    *run = false;
    if (rows < 0 || cin <= 0 || cout <= 0) return fail_call(what, "bad shape");
    if (cin > kMxMaxColumns) return fail_call(what, "more than 2^30 inputs");
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
