// Rotary positions of token sequences: each row's heads are turned by angles
// that grow with the row's position (pxs_rope in pointwise.hip turns by voxel
// coordinates).
//
//   angle_i = position * freq_i, i = 0 .. rotary / 2 - 1
//   (a, b) -> (a cos - b sin, a sin + b cos) * magnitude
//
// for the pairs (2 i, 2 i + 1) or (i, i + rotary / 2) of a head's first `rotary`
// values; the rest of the head is copied.
//
// The angle is taken in 64 bits: position 100,000 at frequency 1 in 32 bits is
// already off by up to 0.004.  It is reduced to a whole number of quarter turns
// and the rest, at most an eighth of a turn, which goes through the 32-bit sine and
// cosine; so those are within a few 2^-24 at any position.

#include "pxs_common.h"

#include <algorithm>
#include <cmath>

namespace pxs {
namespace {

struct RopeArgs {
    const void * x;
    int64_t ldx;
    void * y;
    int64_t ldy;
    const int32_t * positions;  // [rows]
    const double * freq;        // [rotary / 2], radians per position
    int64_t rows;
    int heads, head_dim, rotary;
    float magnitude;
    int rows_per_block;
};

// cos and sin of the angle, times the magnitude.
__device__ __forceinline__ float2 turn(int32_t position, double freq, float magnitude) {
    const double quarters = static_cast<double>(position) * freq * 0.63661977236758134308;  // 2 / pi
    const double whole = rint(quarters);
    const float rest = static_cast<float>(quarters - whole);  // of a quarter turn, in [-1/2, 1/2]
    float s, c;
    sincospif(0.5f * rest, &s, &c);
    // whole modulo 4 in 64 bits: a position times a frequency may be any number
    const int q = static_cast<int>(whole - 4.0 * floor(whole * 0.25));
    const float cs = (q & 1) ? s : c, sn = (q & 1) ? c : s;
    return make_float2(((q + 1) & 2) ? -cs * magnitude : cs * magnitude, (q & 2) ? -sn * magnitude : sn * magnitude);
}

// Every 256th (row, head, unit of a head) from the thread's own, without a division a step.
struct UnitWalk {
    int row, head, unit, heads, units, step_row, step_head, step_unit;
    __device__ __forceinline__ UnitWalk(int h, int u) : heads(h), units(u) {
        const int per_row = h * u, t = threadIdx.x;
        row = t / per_row;
        head = t % per_row / u;
        unit = t % u;
        step_row = 256 / per_row;
        step_head = 256 % per_row / u;
        step_unit = 256 % u;
    }
    __device__ __forceinline__ void next() {
        unit += step_unit;
        head += step_head;
        row += step_row;
        if (unit >= units) {
            unit -= units;
            ++head;
        }
        if (head >= heads) {
            head -= heads;
            ++row;
        }
    }
};

// One value pair or one value of the rest per thread: heads, widths, strides and
// alignments of any kind.
template <typename T, bool HALF>
__global__ void __launch_bounds__(256) rope_any_kernel(RopeArgs a) {
    extern __shared__ float2 turns[];  // [rows of the block][rotary / 2]
    const int pairs = a.rotary / 2, rest = a.head_dim - a.rotary;
    const int units = pairs + rest;  // of a head
    const T * x = static_cast<const T *>(a.x);
    T * y = static_cast<T *>(a.y);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.rows_per_block; row0 < a.rows;
         row0 += static_cast<int64_t>(gridDim.x) * a.rows_per_block) {
        const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows_per_block), a.rows - row0));
        __syncthreads();  // the turns of the rows before have been read
        for (int i = threadIdx.x; i < rows * pairs; i += 256)
            turns[i] = turn(a.positions[row0 + i / pairs], a.freq[i % pairs], a.magnitude);
        __syncthreads();
        for (UnitWalk at(a.heads, units); at.row < rows; at.next()) {
            const int r = at.row, u = at.unit;
            const T * xs = x + (row0 + r) * a.ldx + static_cast<int64_t>(at.head) * a.head_dim;
            T * ys = y + (row0 + r) * a.ldy + static_cast<int64_t>(at.head) * a.head_dim;
            if (u < pairs) {
                const int ia = HALF ? u : 2 * u, ib = HALF ? u + pairs : 2 * u + 1;
                const float va = load_f32(xs + ia), vb = load_f32(xs + ib);
                const float2 t = turns[r * pairs + u];
                store_f32(ys + ia, va * t.x - vb * t.y);
                store_f32(ys + ib, va * t.y + vb * t.x);
            } else {
                ys[pairs + u] = xs[pairs + u];
            }
        }
    }
}

// Heads, halves and rests of whole vectors: V values (16 bytes) a lane and load.  The same
// steps as above with a vector of pairs per unit; interleaved pairs lie inside a vector, those
// of the half layout in two vectors rotary / 2 apart.  Bound by reading and writing the heads once:
// 32,768 x 32 heads of 64 in bf16 44 us, 6.1 TB/s (92 us a value at a time).
template <typename T, int V> struct RopeVec {
    T v[V];
};

template <typename T, bool HALF>
__global__ void __launch_bounds__(256) rope_vec_kernel(RopeArgs a) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    using Vec = RopeVec<T, V>;
    extern __shared__ float2 turns[];  // [rows of the block][rotary / 2]
    const int pairs = a.rotary / 2;
    const int turned = HALF ? pairs / V : a.rotary / V;  // units of a head that are turned
    const int units = turned + (a.head_dim - a.rotary) / V;
    const T * x = static_cast<const T *>(a.x);
    T * y = static_cast<T *>(a.y);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.rows_per_block; row0 < a.rows;
         row0 += static_cast<int64_t>(gridDim.x) * a.rows_per_block) {
        const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows_per_block), a.rows - row0));
        __syncthreads();  // the turns of the rows before have been read
        for (int i = threadIdx.x; i < rows * pairs; i += 256)
            turns[i] = turn(a.positions[row0 + i / pairs], a.freq[i % pairs], a.magnitude);
        __syncthreads();
        for (UnitWalk walk(a.heads, units); walk.row < rows; walk.next()) {
            const int r = walk.row, u = walk.unit;
            const int64_t col = static_cast<int64_t>(walk.head) * a.head_dim;
            const T * xs = x + (row0 + r) * a.ldx + col;
            T * ys = y + (row0 + r) * a.ldy + col;
            const float2 * t = turns + r * pairs;
            if (u >= turned) {
                const int at = a.rotary + (u - turned) * V;
                *reinterpret_cast<uint4 *>(ys + at) = *reinterpret_cast<const uint4 *>(xs + at);
            } else if constexpr (HALF) {
                const int at = u * V;
                Vec va = *reinterpret_cast<const Vec *>(__builtin_assume_aligned(xs + at, 16));
                Vec vb = *reinterpret_cast<const Vec *>(__builtin_assume_aligned(xs + at + pairs, 16));
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float p = load_f32(&va.v[e]), q = load_f32(&vb.v[e]);
                    const float2 c = t[at + e];
                    store_f32(&va.v[e], p * c.x - q * c.y);
                    store_f32(&vb.v[e], p * c.y + q * c.x);
                }
                *reinterpret_cast<uint4 *>(ys + at) = __builtin_bit_cast(uint4, va);
                *reinterpret_cast<uint4 *>(ys + at + pairs) = __builtin_bit_cast(uint4, vb);
            } else {
                const int at = u * V;
                Vec va = *reinterpret_cast<const Vec *>(__builtin_assume_aligned(xs + at, 16));
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float p = load_f32(&va.v[2 * e]), q = load_f32(&va.v[2 * e + 1]);
                    const float2 c = t[at / 2 + e];
                    store_f32(&va.v[2 * e], p * c.x - q * c.y);
                    store_f32(&va.v[2 * e + 1], p * c.y + q * c.x);
                }
                *reinterpret_cast<uint4 *>(ys + at) = __builtin_bit_cast(uint4, va);
            }
        }
    }
}

constexpr int kRopeMaxDim = 1024;

template <typename T>
int launch_rope(RopeArgs a, bool half, hipStream_t s) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const bool vec = a.head_dim % V == 0 && a.rotary % (half ? 2 * V : V) == 0 && a.ldx % V == 0 && a.ldy % V == 0 &&
                     reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
    // Rows of a workgroup: about 4096 values (32,768 x 32 heads of 64, half layout: 44 us, with 2048
    // 47, with 16,384 51), if that leaves two workgroups a CU.
    const int64_t row = static_cast<int64_t>(a.heads) * a.head_dim;
    a.rows_per_block = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, 4096 / row),
                                                          std::max<int64_t>(1, a.rows / 512)));
    a.rows_per_block = std::min(a.rows_per_block, 32);
    const int smem = a.rows_per_block * (a.rotary / 2) * static_cast<int>(sizeof(float2));
    const int64_t blocks = std::min<int64_t>((a.rows + a.rows_per_block - 1) / a.rows_per_block, 1 << 20);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), smem, s, a);
    };
    if (vec && half) launch(rope_vec_kernel<T, true>);
    else if (vec) launch(rope_vec_kernel<T, false>);
    else if (half) launch(rope_any_kernel<T, true>);
    else launch(rope_any_kernel<T, false>);
    return check_launch("rotary positions");
}

} // namespace
} // namespace pxs

using namespace pxs;

extern "C" {

int pxs_rope_frequencies(int rotary_dim, double base, double factor, double original_length, double low_turns,
                         double high_turns, double * freq) {
    PXS_CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= kRopeMaxDim, PXS_ERR_ARG,
              "pxs_rope_frequencies: rotary_dim must be even and in 2..1024");
    PXS_CHECK(base > 0.0 && std::isfinite(base) && factor > 0.0 && std::isfinite(factor), PXS_ERR_ARG,
              "pxs_rope_frequencies: base and factor must be finite and positive");
    PXS_CHECK(original_length >= 0.0 && std::isfinite(original_length), PXS_ERR_ARG,
              "pxs_rope_frequencies: the original length must be finite and not negative");
    PXS_CHECK(original_length == 0.0 || (std::isfinite(low_turns) && std::isfinite(high_turns) && low_turns < high_turns),
              PXS_ERR_ARG, "pxs_rope_frequencies: low_turns must be below high_turns");
    PXS_CHECK(freq, PXS_ERR_ARG, "pxs_rope_frequencies: null pointer");
    for (int i = 0; i < rotary_dim / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / rotary_dim);
        double keep = 0.0;  // of the frequency; the rest of it is divided by the factor
        if (original_length > 0.0) {
            const double turns = original_length * f / 6.283185307179586477;
            keep = std::min(1.0, std::max(0.0, (turns - low_turns) / (high_turns - low_turns)));
        }
        freq[i] = f * (keep + (1.0 - keep) / factor);
    }
    return PXS_OK;
}

int pxs_rope_positions(int dtype, const int32_t * positions, const double * freq, const void * x, int64_t ld_x,
                       int64_t rows, int heads, int head_dim, int rotary_dim, int layout, float magnitude, void * y,
                       int64_t ld_y, void * stream) {
    PXS_CHECK(dtype == PXS_F32 || dtype == PXS_BF16, PXS_ERR_ARG, "pxs_rope_positions: bad dtype");
    PXS_CHECK(layout == PXS_ROPE_INTERLEAVED || layout == PXS_ROPE_HALF, PXS_ERR_ARG,
              "pxs_rope_positions: bad layout");
    PXS_CHECK(rows >= 0 && heads > 0 && head_dim > 0 && head_dim <= kRopeMaxDim && heads <= 65535, PXS_ERR_ARG,
              "pxs_rope_positions: head_dim must be in 1..1024, heads in 1..65535");
    PXS_CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, PXS_ERR_ARG,
              "pxs_rope_positions: rotary_dim must be even and in 2..head_dim");
    PXS_CHECK(ld_x >= static_cast<int64_t>(heads) * head_dim && ld_y >= static_cast<int64_t>(heads) * head_dim,
              PXS_ERR_ARG, "pxs_rope_positions: row stride smaller than heads * head_dim");
    PXS_CHECK(std::isfinite(magnitude), PXS_ERR_ARG, "pxs_rope_positions: magnitude must be finite");
    if (rows == 0) return PXS_OK;
    PXS_CHECK(positions && freq && x && y, PXS_ERR_ARG, "pxs_rope_positions: null pointer");
    PXS_CHECK(x != y || ld_x == ld_y, PXS_ERR_ARG, "pxs_rope_positions: in place, ld_x must be ld_y");
    RopeArgs a{x, ld_x, y, ld_y, positions, freq, rows, heads, head_dim, rotary_dim, magnitude, 1};
    const bool half = layout == PXS_ROPE_HALF;
    return dtype == PXS_F32 ? launch_rope<float>(a, half, as_stream(stream))
                            : launch_rope<uint16_t>(a, half, as_stream(stream));
}

} // extern "C"
