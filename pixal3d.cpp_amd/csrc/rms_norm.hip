// The residual's addition and the root-mean-square norm of its rows, for token
// models (layer norms and the per-head RMS norm are in pointwise.hip):
//
//   h    = residual + x          one rounding in fp32, then that of the residual's type; stored
//   inv  = 1 / sqrt(sum h^2 / channels + eps)                         of the stored h
//   y    = h * inv * gamma       rows in fp32 or bf16, or
//   t    = h * gamma;  q = rint(t * (127 / max|t|));  scale = max|t| / 127 * inv
//
// inv is one positive factor of a row, so the bytes do not depend on it: they are those that
// the row quantizer makes of t (rows_i8.h), whatever order the squares are summed in.  The
// squares are summed in 64 bits, which hold the square of every fp32 value.

#include "pxs_common.h"
#include "rows_i8.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace pxs {
namespace {

struct NormArgs {
    const void * x;
    int64_t ldx;
    const void * residual;  // [rows, channels] or null
    void * residual_out;    // the same; may be residual
    int64_t rows;
    int channels;
    double eps;
    const float * gamma;    // [channels] or null: ones
    int y_dtype;
    void * y;               // [rows, channels], or
    int8_t * q;             // [rows, channels]
    float * scales;         // [rows]
    int past;               // y is stored past the caches
};

struct None {};

// A row's h from its x and residual (RT None: h is x).
template <typename XT, typename RT>
__device__ __forceinline__ float norm_sum(const XT * x, const RT * res, RT * out, int c) {
    if constexpr (std::is_same<RT, None>::value) {
        return load_f32(x + c);
    } else {
        store_f32(out + c, load_f32(res + c) + load_f32(x + c));
        return load_f32(out + c);
    }
}

__device__ __forceinline__ void norm_store(const NormArgs & a, int64_t at, float v) {
    if (a.y_dtype == PXS_BF16) static_cast<uint16_t *>(a.y)[at] = f32_to_bf16(v);
    else static_cast<float *>(a.y)[at] = v;
}

// Workgroups launched at most: each then takes several rows, with the gains loaded once.  Of three rules the one
// that is nowhere more than 2.5% behind the best: 42,017 x 1024 bf16 on an fp32 residual into 8-bit rows 90 us with
// 4,096, 94 with 2,048, 89 with one for every four rows; 8,192 x 4096 of the same 49.9, 48.7 and 49.0; 4,739 x 1370
// in bf16 throughout 14.5, 14.3 and 15.8.
constexpr int64_t kNormGrid = 4096;

// A workgroup a row, a value at a time, the row read again for its output: rows of more than 16,384 channels.
template <typename XT, typename RT, bool Q>
__global__ void __launch_bounds__(256) rms_norm_any_kernel(NormArgs a) {
    __shared__ double sums[4];
    __shared__ uint32_t tops[4];
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const XT * x = static_cast<const XT *>(a.x) + row * a.ldx;
        const RT * res = static_cast<const RT *>(a.residual) + row * a.channels;  // (None: not read)
        RT * out = static_cast<RT *>(a.residual_out) + row * a.channels;
        double sum = 0.0;
        uint32_t top = 0;
        for (int c = tid; c < a.channels; c += 256) {
            const float h = norm_sum<XT, RT>(x, res, out, c);
            sum += static_cast<double>(h) * h;
            top = max(top, abs_bits(a.gamma ? h * a.gamma[c] : h));
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            sum += __shfl_xor(sum, d, 64);
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64)));
        }
        if ((tid & 63) == 0) {
            sums[wave] = sum;
            tops[wave] = top;
        }
        __syncthreads();
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        __syncthreads();
        const float inv = static_cast<float>(rsqrt(sum / a.channels + a.eps));
        float scale, per;
        row_scale(top, scale, per);
        if (Q && tid == 0) a.scales[row] = scale == 0.0f ? 0.0f : scale * inv;
        for (int c = tid; c < a.channels; c += 256) {
            float h;
            if constexpr (std::is_same<RT, None>::value) h = load_f32(x + c);
            else h = load_f32(out + c);  // (this thread's own)
            const float g = a.gamma ? a.gamma[c] : 1.0f;
            if constexpr (Q) {
                const float v[8] = {h * g, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                a.q[row * a.channels + c] = top < kQuantFinite ? static_cast<int8_t>(q8_bytes(v, per).x & 255u) : int8_t(0);
            } else {
                norm_store(a, row * a.channels + c, h * inv * g);
            }
        }
    }
}

// Eight values of a row from column c, those past its end zero.
template <typename T>
__device__ __forceinline__ void norm_load8(const T * row, int c, int channels, float (&v)[8]) {
    if (c + 8 <= channels) {
        T e[8];
        __builtin_memcpy(e, row + c, sizeof(e));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = load_f32(e + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < channels ? load_f32(row + c + i) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void norm_store8(T * row, int c, int channels, const float (&v)[8], bool past = false) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) store_f32(e + i, v[i]);
    if (c + 8 <= channels) {
        if (past) {
            asm volatile("");  // (here and behind, or the compiler makes one store of both branches', through the caches)
#pragma unroll
            for (int k = 0; k < static_cast<int>(sizeof(e) / 16); ++k)
                store16_past(reinterpret_cast<char *>(row + c) + 16 * k, reinterpret_cast<const char *>(e) + 16 * k);
            asm volatile("");
        } else {
            __builtin_memcpy(row + c, e, sizeof(e));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < channels) row[c + i] = e[i];
    }
}

constexpr int norm_threads(int wpr) { return wpr > 4 ? wpr * 64 : 256; }

// WPR waves share a row of up to WPR * 64 * 8 * NV channels, which they hold in registers between
// the sums and the rounding: every value is read and written once.  Rows start at any element.  The
// gains are loaded once for all the rows that a wave takes.  Bound by HBM: 42,017 x 1024, bf16 on an fp32
// residual, 90 us, 5.2 TB/s (the kernel above, a value at a time, 175); one row of 1024 3.4 us, its launch, loads and
// two reductions.
template <typename XT, typename RT, bool Q, int WPR, int NV>
__global__ void __launch_bounds__(norm_threads(WPR)) rms_norm_rows_kernel(NormArgs a) {
    constexpr int kLanes = WPR * 64, kRows = norm_threads(WPR) / kLanes;
    __shared__ double sums[WPR];
    __shared__ uint32_t tops[WPR];
    const int wave = threadIdx.x >> 6, l = threadIdx.x % kLanes;
    float gain[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (a.gamma) norm_load8(a.gamma, (j * kLanes + l) * 8, a.channels, gain[j]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) gain[j][i] = 1.0f;
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + wave / WPR; row < a.rows;
         row += static_cast<int64_t>(gridDim.x) * kRows) {
        const XT * x = static_cast<const XT *>(a.x) + row * a.ldx;
        float h[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j) norm_load8(x, (j * kLanes + l) * 8, a.channels, h[j]);
        if constexpr (!std::is_same<RT, None>::value) {
            const RT * res = static_cast<const RT *>(a.residual) + row * a.channels;
            RT * out = static_cast<RT *>(a.residual_out) + row * a.channels;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * kLanes + l) * 8;
                float r[8];
                norm_load8(res, c, a.channels, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    RT e;
                    store_f32(&e, r[i] + h[j][i]);
                    h[j][i] = load_f32(&e);
                }
                norm_store8(out, c, a.channels, h[j]);
            }
        }
        double sum = 0.0;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum += static_cast<double>(h[j][i]) * h[j][i];
                if constexpr (Q) {
                    h[j][i] *= gain[j][i];
                    top = max(top, abs_bits(h[j][i]));
                }
            }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            sum += __shfl_xor(sum, d, 64);
            if constexpr (Q) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64)));
        }
        if constexpr (WPR > 1) {
            if ((threadIdx.x & 63) == 0) {
                sums[wave] = sum;
                if constexpr (Q) tops[wave] = top;
            }
            __syncthreads();
            sum = sums[0];
#pragma unroll
            for (int i = 1; i < WPR; ++i) sum += sums[i];
            if constexpr (Q) {
                top = tops[0];
#pragma unroll
                for (int i = 1; i < WPR; ++i) top = max(top, tops[i]);
            }
            __syncthreads();  // (every wave has the same rows)
        }
        const float inv = static_cast<float>(rsqrt(sum / a.channels + a.eps));
        if constexpr (Q) {
            float scale, per;
            row_scale(top, scale, per);
            if (l == 0) a.scales[row] = scale == 0.0f ? 0.0f : scale * inv;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * kLanes + l) * 8;
                uint2 u = q8_bytes(h[j], per);
                if (top >= kQuantFinite) u = make_uint2(0u, 0u);
                int8_t * q = a.q + row * a.channels + c;
                if (c + 8 <= a.channels) {
                    __builtin_memcpy(q, &u, 8);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + i < a.channels) q[i] = static_cast<int8_t>((i < 4 ? u.x >> (8 * i) : u.y >> (8 * (i - 4))) & 255u);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * kLanes + l) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) h[j][i] = h[j][i] * inv * gain[j][i];
                if (a.y_dtype == PXS_BF16) norm_store8(static_cast<uint16_t *>(a.y) + row * a.channels, c, a.channels, h[j], a.past);
                else norm_store8(static_cast<float *>(a.y) + row * a.channels, c, a.channels, h[j], a.past);
            }
        }
    }
}

// Waves a row: as few as hold it in 16 values a lane or less, one up to 1024 channels (42,017 x 512 47 us, with four
// 61; at 1024 channels they meet: 42,017 rows 90 and 88 to 92, 2,000 7.1 and 7.1, one 3.4 and 3.3), four to 2048
// (4,739 x 1370 14.5, with one 16.1), eight to 8192 (10,000 x 4096 84, with four 87, with sixteen 123; 15,000 x 2600 85, 92
// and 179; 5,000 x 8192 88, 90 and 89), sixteen to 16,384 (2,500 x 16,384 101, a value at a time 197).
// (4,739 x 1370 in bf16 throughout, the others bf16 on an fp32 residual into 8-bit rows.)
template <typename XT, typename RT, bool Q>
int launch_norm(const NormArgs & a, hipStream_t s) {
    const int64_t one = (a.rows + 3) / 4;
    auto launch = [&](auto kernel, int64_t blocks, int threads = 256) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, kNormGrid))), dim3(threads), 0, s, a);
    };
    if (a.channels <= 512) launch(rms_norm_rows_kernel<XT, RT, Q, 1, 1>, one);
    else if (a.channels <= 1024) launch(rms_norm_rows_kernel<XT, RT, Q, 1, 2>, one);
    else if (a.channels <= 2048) launch(rms_norm_rows_kernel<XT, RT, Q, 4, 1>, a.rows);
    else if (a.channels <= 4096) launch(rms_norm_rows_kernel<XT, RT, Q, 8, 1>, a.rows, norm_threads(8));
    else if (a.channels <= 8192) launch(rms_norm_rows_kernel<XT, RT, Q, 8, 2>, a.rows, norm_threads(8));
    else if (a.channels <= 16384) launch(rms_norm_rows_kernel<XT, RT, Q, 16, 2>, a.rows, norm_threads(16));
    else launch(rms_norm_any_kernel<XT, RT, Q>, a.rows);
    return check_launch("RMS norm");
}

template <typename XT, bool Q>
int norm_residual(const NormArgs & a, int residual_dtype, hipStream_t s) {
    if (!a.residual) return launch_norm<XT, None, Q>(a, s);
    return residual_dtype == PXS_F32 ? launch_norm<XT, float, Q>(a, s) : launch_norm<XT, uint16_t, Q>(a, s);
}

template <bool Q>
int run_norm(const NormArgs & a, int x_dtype, int residual_dtype, hipStream_t s) {
    return x_dtype == PXS_F32 ? norm_residual<float, Q>(a, residual_dtype, s)
                              : norm_residual<uint16_t, Q>(a, residual_dtype, s);
}

constexpr int kNormMaxChannels = 1 << 30;
constexpr int64_t kNormPast = 32 << 20;  // bytes of y that the L2s do not hold

// The checks that both calls share.
int check_norm(const char * what, int x_dtype, const void * x, int64_t ld_x, int residual_dtype, const void * residual,
               const void * residual_out, int64_t rows, int channels, float eps, const void * out) {
    if (x_dtype != PXS_F32 && x_dtype != PXS_BF16) return fail_call(what, "bad dtype");
    if (residual && residual_dtype != PXS_F32 && residual_dtype != PXS_BF16) return fail_call(what, "bad residual dtype");
    if (rows < 0 || channels <= 0 || ld_x < channels) return fail_call(what, "bad shape");
    if (channels > kNormMaxChannels) return fail_call(what, "more than 2^30 channels");
    if (!(eps > 0.0f) || !std::isfinite(eps)) return fail_call(what, "eps must be finite and positive");
    if (!residual != !residual_out) return fail_call(what, "residual and residual_out must both be given, or neither");
    if (rows > 0 && (!x || !out)) return fail_call(what, "null pointer");
    return PXS_OK;
}

} // namespace
} // namespace pxs

using namespace pxs;

extern "C" {

int pxs_rms_norm(int x_dtype, const void * x, int64_t ld_x, int residual_dtype, const void * residual,
                 void * residual_out, int64_t rows, int channels, float eps, const float * gamma, int y_dtype, void * y,
                 void * stream) {
    PXS_CHECK(y_dtype == PXS_F32 || y_dtype == PXS_BF16, PXS_ERR_ARG, "pxs_rms_norm: bad dtype");
    if (int rc = check_norm("pxs_rms_norm", x_dtype, x, ld_x, residual_dtype, residual, residual_out, rows, channels, eps, y))
        return rc;
    if (rows == 0) return PXS_OK;
    // (8,192 x 4096 in bf16, no residual: 24 us past the caches, 29 through them.)
    const int past = rows * channels * (y_dtype == PXS_BF16 ? 2 : 4) > kNormPast;
    NormArgs a{x, ld_x, residual, residual_out, rows, channels, eps, gamma, y_dtype, y, nullptr, nullptr, past};
    return run_norm<false>(a, x_dtype, residual_dtype, as_stream(stream));
}

int pxs_rms_norm_i8(int x_dtype, const void * x, int64_t ld_x, int residual_dtype, const void * residual,
                    void * residual_out, int64_t rows, int channels, float eps, const float * gamma, int8_t * q,
                    float * scales, void * stream) {
    if (int rc = check_norm("pxs_rms_norm_i8", x_dtype, x, ld_x, residual_dtype, residual, residual_out, rows, channels,
                            eps, q))
        return rc;
    PXS_CHECK(rows == 0 || scales, PXS_ERR_ARG, "pxs_rms_norm_i8: null pointer");
    if (rows == 0) return PXS_OK;
    NormArgs a{x, ld_x, residual, residual_out, rows, channels, eps, gamma, PXS_F32, nullptr, q, scales, 0};
    return run_norm<true>(a, x_dtype, residual_dtype, as_stream(stream));
}

} // extern "C"
