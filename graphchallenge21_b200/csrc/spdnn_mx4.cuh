// Microscaled 4-bit floats: a row of a matrix in blocks of 32 elements, each block one power of two (E8M0) and 32 values of E2M1.
//
//   e = clamp(floor(log2 max|v|) - 2, -127, 127)      code = v 2^-e rounded to E2M1, half to even, magnitudes above 6 to 6
//
// A block of zeros has the scale 2^-127 and zero codes.  A block that holds a NaN or an infinity has the scale byte 255: all its
// values are NaN.  Storage: codes [rows][blocks][16] (element 2i of a block in the low half of byte i), scales [rows][blocks]; the
// elements behind the last column of a row are zero.
#pragma once

#include "spdnn_ffn.cuh"

namespace spdnn_impl {
namespace ffn {

constexpr int kMx4Threads = 256;

// Eight values as a word of E2M1, the first in the lowest half-byte.
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{ .reg .b8 b0, b1, b2, b3; cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1; cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;"
        " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5; cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7; mov.b32 %0, {b0, b1, b2, b3}; }"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Where group `i` of a matrix with `per_row` groups a row is, and then those a block of threads further on: one division for a thread's whole
// batch (a division takes longer than the rest of a group's work).
struct Walk {
    int64_t row;
    uint32_t at;
    __device__ __forceinline__ Walk(int64_t i, uint32_t per_row) {
        row = i >> 32 ? i / per_row : (int64_t)((uint32_t)i / per_row);
        at = (uint32_t)(i - row * per_row);
    }
    __device__ __forceinline__ void step(uint32_t by, uint32_t per_row) {
        at += by;
        if (at < per_row) return;
        const uint32_t rows = per_row >= by ? 1u : at / per_row;
        row += rows;
        at -= rows * per_row;
    }
};

constexpr int kMx4Batch = 4;      // groups of a thread whose loads are in flight together

// Four lanes share a block, eight elements each.  BYTES: what the base and the row stride are multiples of, 16 at most.
template <class E, int BYTES, int BATCH>
__global__ void __launch_bounds__(kMx4Threads) mx4_quantize_kernel(const E *__restrict__ x, int64_t stride, int64_t rows, int cols, int blocks,
                                                                   uint32_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    const int64_t groups = rows * blocks * 4;
    const int64_t step = (int64_t)gridDim.x * kMx4Threads * BATCH;
    // whole warps stay together for the shuffles
    for (int64_t first = (int64_t)blockIdx.x * kMx4Threads * BATCH + (threadIdx.x & ~31); first < groups; first += step) {
        constexpr int PER = BYTES / (int)sizeof(E);
        Raw<E, PER> part[BATCH][8 / PER];
        Walk walk(first + (threadIdx.x & 31), (uint32_t)blocks * 4);
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int64_t i = first + m * kMx4Threads + (threadIdx.x & 31);
            if (m) walk.step(kMx4Threads, (uint32_t)blocks * 4);
#pragma unroll
            for (int h = 0; h < 8 / PER; ++h) part[m][h].clear();
            if (i >= groups) continue;
            const int col = (int)walk.at * 8;
            const E *from = x + walk.row * stride + col;
            if (col + 8 <= cols) {
#pragma unroll
                for (int h = 0; h < 8 / PER; ++h) part[m][h].load(from + h * PER);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (col + k < cols) part[m][k / PER].set(k % PER, from[k]);
            }
        }
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int64_t i = first + m * kMx4Threads + (threadIdx.x & 31);
            float v[8], most = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = bits_to_float<E>(part[m][k / PER].bits(k % PER));
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(v[k])));
            }
            // as bits: they are ordered as the magnitudes are, and NaN and infinity are the largest
            uint32_t top = __float_as_uint(most);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (i >= groups) continue;
            const bool finite = top < 0x7f800000u;
            // biased exponent of the scale; below 2^-125 (subnormals among them) it stays at the smallest
            const int e = max((int)(top >> 23) - 2, 0);
            // 2^-(e - 127), between 2^-125 and 2^127: a normal number, and the product is exact
            const float inverse = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= inverse;
            codes[i] = finite ? to_e2m1x8(v) : 0u;
            if ((i & 3) == 0) scales[i >> 2] = finite ? (uint8_t)e : (uint8_t)255;
        }
    }
}

// Groups of four values (16 bytes of float32, 8 of the 16-bit types): neighbouring lanes fill whole sectors, which eight values a lane did not
// (8191 x 4100 to float32: 29.9 and 34.6 us).  VECTOR: base and row stride are multiples of a group.
template <class E, bool VECTOR, int BATCH>
__global__ void __launch_bounds__(kMx4Threads) mx4_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t rows,
                                                                     int cols, int blocks, E *__restrict__ y, int64_t stride) {
    const uint32_t per_row = (uint32_t)(cols + 3) / 4;
    const int64_t groups = rows * per_row;
    const int64_t step = (int64_t)gridDim.x * kMx4Threads * BATCH;
    for (int64_t first = (int64_t)blockIdx.x * kMx4Threads * BATCH + threadIdx.x; first < groups; first += step) {
        uint32_t word[BATCH], scale[BATCH];
        int64_t to_at[BATCH];
        int left[BATCH];
        Walk walk(first, per_row);
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            if (m) walk.step(kMx4Threads, per_row);
            word[m] = scale[m] = 0;
            const int col = (int)walk.at * 4;
            to_at[m] = walk.row * stride + col;
            left[m] = cols - col;
            if (first + m * kMx4Threads >= groups) continue;
            const int64_t block = walk.row * blocks + (col >> 5);
            word[m] = __ldg((const uint16_t *)(codes + block * 16 + ((col & 31) >> 1)));
            scale[m] = __ldg(scales + block);
        }
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            if (first + m * kMx4Threads >= groups) break;
            float v[4];
            e2m1_values(word[m], v);
            const float factor = e8m0_value(scale[m]);
            __align__(16) E e[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = from_float<E>(v[k] * factor);
            E *to = y + to_at[m];
            if (VECTOR && left[m] >= 4) {
                if constexpr (sizeof(E) == 4) *(uint4 *)to = *(const uint4 *)e;
                else *(uint2 *)to = *(const uint2 *)e;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < left[m]) to[k] = e[k];
            }
        }
    }
}

}  // namespace ffn
}  // namespace spdnn_impl
