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

// Two values as one byte of E2M1, `lo` in the low half.
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{ .reg .b8 b, z; mov.b16 {b, z}, 0; cvt.rn.satfinite.e2m1x2.f32 b, %1, %2; mov.b32 %0, {b, z, z, z}; }" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Four lanes share a block, eight elements each.  VECTOR: base and row stride are multiples of 16 bytes.
template <class E, bool VECTOR>
__global__ void __launch_bounds__(kMx4Threads) mx4_quantize_kernel(const E *__restrict__ x, int64_t stride, int64_t rows, int cols, int blocks,
                                                                   uint32_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    const int64_t groups = rows * blocks * 4;
    const int64_t step = (int64_t)gridDim.x * kMx4Threads;
    // whole warps stay together for the shuffles
    for (int64_t first = (int64_t)blockIdx.x * kMx4Threads + (threadIdx.x & ~31); first < groups; first += step) {
        const int64_t i = first + (threadIdx.x & 31);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
        if (i < groups) {
            const int64_t row = i / (blocks * 4);
            const int col = (int)(i - row * (blocks * 4)) * 8;
            const E *from = x + row * stride + col;
            if (VECTOR && col + 8 <= cols) {
                Values<E, 16 / sizeof(E)> part[8 * sizeof(E) / 16];
#pragma unroll
                for (int h = 0; h < (int)(8 * sizeof(E) / 16); ++h) part[h].load(from + h * (16 / sizeof(E)));
#pragma unroll
                for (int k = 0; k < 4; ++k) unpack2(part[k / (8 / sizeof(E))].v[k % (8 / sizeof(E))], v[2 * k], v[2 * k + 1]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (col + k < cols) v[k] = to_float(from[k]);
            }
        }
        // the largest magnitude as bits: they are ordered as the values are, and NaN and infinity are the largest
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (i >= groups) continue;
        const bool finite = top < 0x7f800000u;
        // biased exponent of the scale; below 2^-125 (subnormals among them) it stays at the smallest
        const int e = max((int)(top >> 23) - 2, 0);
        // 2^-(e - 127), between 2^-125 and 2^127: a normal number, and the product is exact
        const float inverse = __uint_as_float((uint32_t)(254 - e) << 23);
        uint32_t word = 0;
        if (finite) {
#pragma unroll
            for (int k = 0; k < 4; ++k) word |= to_e2m1x2(v[2 * k] * inverse, v[2 * k + 1] * inverse) << (8 * k);
        }
        codes[i] = word;
        if ((i & 3) == 0) scales[i >> 2] = finite ? (uint8_t)e : (uint8_t)255;
    }
}

// Eight elements per thread.
template <class E>
__global__ void __launch_bounds__(kMx4Threads) mx4_dequantize_kernel(const uint32_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t rows,
                                                                     int cols, int blocks, E *__restrict__ y, int64_t stride) {
    const int64_t groups = rows * blocks * 4;
    const int64_t step = (int64_t)gridDim.x * kMx4Threads;
    for (int64_t i = (int64_t)blockIdx.x * kMx4Threads + threadIdx.x; i < groups; i += step) {
        const int64_t row = i / (blocks * 4);
        const int col = (int)(i - row * (blocks * 4)) * 8;
        const uint32_t word = __ldg(codes + i);
        const float scale = e8m0_value(__ldg(scales + (i >> 2)));
        E *to = y + row * stride + col;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (col + k < cols) to[k] = from_float<E>(e2m1_value(word >> (4 * k)) * scale);
    }
}

}  // namespace ffn
}  // namespace spdnn_impl
