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

// The 8 elements from column c of a row; those past the end are 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load_elems8(const T * row, int c, int channels, float (&v)[8]) {
    if constexpr (VEC) {
        if (c < channels) {
            if constexpr (sizeof(T) == 2) {
                const uint4 u = *reinterpret_cast<const uint4 *>(row + c);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
            } else {
                const float4 a = *reinterpret_cast<const float4 *>(row + c);
                const float4 b = *reinterpret_cast<const float4 *>(row + c + 4);
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < channels ? load_f32(row + c + i) : 0.0f;
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
        if (c < channels) *reinterpret_cast<uint2 *>(row + c) = u;
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
    const bool vec = a.channels % 8 == 0 && a.ldx % (16 / sizeof(T)) == 0 &&
                     reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.q) % 8 == 0;
    const int64_t one = (a.rows + 3) / 4;
    auto launch = [&](auto kernel, int64_t blocks) {  // a workgroup takes more rows past 2^20 of them
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20))), dim3(256), 0, s, a);
    };
    auto pick = [&](auto v) {
        constexpr bool VEC = decltype(v)::value;
        if (a.channels <= 512) launch(quantize_rows_kernel<T, 1, 1, VEC, true>, one);
        else if (a.channels <= 1024) launch(quantize_rows_kernel<T, 1, 2, VEC, true>, one);
        else if (a.channels <= 2048) launch(quantize_rows_kernel<T, 4, 1, VEC, true>, a.rows);
        else if (a.channels <= 4096) launch(quantize_rows_kernel<T, 4, 2, VEC, true>, a.rows);
        else if (a.channels <= 8192) launch(quantize_rows_kernel<T, 4, 4, VEC, true>, a.rows);
        else launch(quantize_rows_kernel<T, 4, 1, VEC, false>, a.rows);
    };
    if (vec) pick(std::true_type{});
    else pick(std::false_type{});
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
    int vec_out;             // 4-channel vector accesses of all that the epilogue touches
    int group_m;             // tile order (tile_of)
};

// Four outputs of a row, from column c (c < n): value = (sum * x_scale) * w_scale + bias.
// (The sum of up to 2^31 rounds to fp32 once, each product and the bias once.)
template <typename T, int EPI>
__device__ __forceinline__ void i8_epilogue4(const I8Args & a, int64_t row, int batch, int c, const int (&sum)[4],
                                             float xs) {
    const bool vec = a.vec_out && c + 3 < a.n;
    float ws[4], b[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4];
    if (vec) {
        const float4 w4 = *reinterpret_cast<const float4 *>(a.w_scales + c);
        ws[0] = w4.x; ws[1] = w4.y; ws[2] = w4.z; ws[3] = w4.w;
        if (a.bias) {
            const float4 b4 = *reinterpret_cast<const float4 *>(a.bias + c);
            b[0] = b4.x; b[1] = b4.y; b[2] = b4.z; b[3] = b4.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int ce = min(c + e, a.n - 1);
            ws[e] = a.w_scales[ce];
            if (a.bias) b[e] = a.bias[ce];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (static_cast<float>(sum[e]) * xs) * ws[e] + b[e];
    if constexpr (EPI == kI8Store) {
        if (a.act == PXS_ACT_GELU_TANH) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_f(v[e]);
        } else if (a.act == PXS_ACT_SILU) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = silu_f(v[e]);
        }
        T * p = static_cast<T *>(a.y) + row * a.n + c;
        if (vec) {
            if constexpr (sizeof(T) == 2)
                *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            else
                *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
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

// BM x BN outputs, NW waves in a WAVES_M x (NW / WAVES_M) grid.  128 bytes of K a
// stage: every thread loads its 16-byte pieces of the next stage's rows into
// registers while the stage in LDS is multiplied.  Rows of any length and alignment.
template <typename T, int BM, int BN, int NW, int WAVES_M, int EPI>
__global__ void __launch_bounds__(NW * 64) linear_i8_any_kernel(I8Args a) {
    constexpr int KB = 128, P = 8, NT = NW * 64, RS = NT / P;
    constexpr int WAVES_N = NW / WAVES_M, WM = BM / WAVES_M, WN = BN / WAVES_N, TI = WM / 32, TJ = WN / 32;
    constexpr int XI = BM / RS, WI = BN / RS;
    __shared__ __align__(16) char smem[(BM + BN) * KB];
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
    uint4 vx[XI], vw[WI];
    auto load = [&](int s) __attribute__((always_inline)) {
        const int k0 = s * KB + piece * 16;
#pragma unroll
        for (int i = 0; i < XI; ++i) vx[i] = load_piece<true>(xr[i], k0, a.k);
#pragma unroll
        for (int i = 0; i < WI; ++i) vw[i] = load_piece<false>(wr[i], k0, a.k);
    };
    i32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = i32x16{};
    const int stages = (a.k + KB - 1) / KB;
    load(0);
    for (int s = 0; s < stages; ++s) {
        __syncthreads();  // every wave has read the stage before
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const int row = row0 + RS * i;
            *reinterpret_cast<uint4 *>(smem + row * KB + ((piece ^ piece_swz<KB>(row)) << 4)) = vx[i];
        }
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int row = row0 + RS * i;
            *reinterpret_cast<uint4 *>(smem + (BM + row) * KB + ((piece ^ piece_swz<KB>(row)) << 4)) = vw[i];
        }
        __syncthreads();
        if (s + 1 < stages) load(s + 1);
#pragma unroll
        for (int u = 0; u < P / 2; ++u) {
            const int pc = (P / 2) * h + u;
            i32x4 xf[TI], wf[TJ];
#pragma unroll
            for (int i = 0; i < TI; ++i) {
                const int row = wm * WM + i * 32 + r;
                xf[i] = *reinterpret_cast<const i32x4 *>(smem + row * KB + ((pc ^ piece_swz<KB>(row)) << 4));
            }
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                const int row = wn * WN + j * 32 + r;
                wf[j] = *reinterpret_cast<const i32x4 *>(smem + (BM + row) * KB + ((pc ^ piece_swz<KB>(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int64_t row = p0 + wm * WM + i * 32 + r;
        if (row >= a.m) continue;
        const float xs = a.x_scales[row];
        const int batch = EPI == kI8Gate ? a.coords[row * 4] : 0;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = n0 + wn * WN + j * 32 + 8 * g + 4 * h;
                if (c >= a.n) continue;
                const int sum[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                i8_epilogue4<T, EPI>(a, row, batch, c, sum, xs);
            }
    }
}

template <typename T, int EPI>
int launch_i8(I8Args a, hipStream_t s) {
    constexpr int BM = 128, BN = 128;
    const int64_t blocks = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    PXS_CHECK(blocks <= UINT32_MAX / 512, PXS_ERR_ARG, "8-bit linear grid too large");
    a.group_m = 8;
    hipLaunchKernelGGL((linear_i8_any_kernel<T, BM, BN, 8, 2, EPI>), dim3(static_cast<unsigned>(blocks)), dim3(512), 0,
                       s, a);
    return check_launch("8-bit linear");
}

bool aligned_to(const void * p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

constexpr int kI8MaxInputs = 131071;  // 131,071 products of -128 by -128 stay below 2^31

// The checks that the 8-bit linears share; *run is false where there is nothing to do.
int check_i8(const char * what, const int8_t * x, const float * x_scales, int64_t rows, int cin,
             const int8_t * weight, const float * w_scales, int cout, const void * out, bool * run) {
    *run = false;
    if (rows < 0 || cin <= 0 || cout <= 0) return fail_call(what, "bad shape");
    if (cin > kI8MaxInputs) return fail_call(what, "more than 131071 inputs (their sum may not fit 32 bits)");
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
    return y_dtype == PXS_F32 ? launch_i8<float, kI8Store>(a, as_stream(stream))
                              : launch_i8<uint16_t, kI8Store>(a, as_stream(stream));
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
