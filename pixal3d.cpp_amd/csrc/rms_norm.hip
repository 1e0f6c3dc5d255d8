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

// A workgroup a row, a value at a time, the row read again for its output: any width.
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
        const float inv = static_cast<float>(1.0 / sqrt(sum / a.channels + a.eps));
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

template <typename XT, typename RT, bool Q>
int launch_norm(const NormArgs & a, hipStream_t s) {
    hipLaunchKernelGGL((rms_norm_any_kernel<XT, RT, Q>), dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, 1 << 20))),
                       dim3(256), 0, s, a);
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
    NormArgs a{x, ld_x, residual, residual_out, rows, channels, eps, gamma, y_dtype, y, nullptr, nullptr};
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
    NormArgs a{x, ld_x, residual, residual_out, rows, channels, eps, gamma, PXS_F32, nullptr, q, scales};
    return run_norm<true>(a, x_dtype, residual_dtype, as_stream(stream));
}

} // extern "C"
