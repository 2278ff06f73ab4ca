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

// i / n, in 32 bits where both fit (a division of 64 bits takes longer than the rest of the loop).
__device__ __forceinline__ int64_t quotient(int64_t i, uint32_t n) {
    return i >> 32 ? i / n : (int64_t)((uint32_t)i / n);
}

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
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int64_t i = first + m * kMx4Threads + (threadIdx.x & 31);
#pragma unroll
            for (int h = 0; h < 8 / PER; ++h) part[m][h].clear();
            if (i >= groups) continue;
            const int64_t row = quotient(i, (uint32_t)blocks * 4);
            const int col = (int)(i - row * (blocks * 4)) * 8;
            const E *from = x + row * stride + col;
#pragma unroll
            for (int h = 0; h < 8 / PER; ++h) {
                if (col + (h + 1) * PER <= cols) {
                    part[m][h].load(from + h * PER);
                } else {
#pragma unroll
                    for (int k = 0; k < PER; ++k)
                        if (col + h * PER + k < cols) part[m][h].set(k, from[h * PER + k]);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int64_t i = first + m * kMx4Threads + (threadIdx.x & 31);
            float v[8];
            // the largest magnitude as bits: they are ordered as the values are, and NaN and infinity are the largest
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = bits_to_float<E>(part[m][k / PER].bits(k % PER));
                top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
            }
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
}

// Groups of four values (16 bytes of float32, 8 of the 16-bit types).  VECTOR: base and row stride are multiples of that.
template <class E, bool VECTOR, int BATCH>
__global__ void __launch_bounds__(kMx4Threads) mx4_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t rows,
                                                                     int cols, int blocks, E *__restrict__ y, int64_t stride) {
    const uint32_t per_row = (uint32_t)(cols + 3) / 4;
    const int64_t groups = rows * per_row;
    const int64_t step = (int64_t)gridDim.x * kMx4Threads * BATCH;
    for (int64_t first = (int64_t)blockIdx.x * kMx4Threads * BATCH + threadIdx.x; first < groups; first += step) {
        uint32_t word[BATCH], scale[BATCH];
        int64_t row[BATCH];
        int col[BATCH];
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int64_t i = min(first + m * kMx4Threads, groups - 1);
            row[m] = quotient(i, per_row);
            col[m] = (int)(i - row[m] * per_row) * 4;
            const int64_t block = row[m] * blocks + (col[m] >> 5);
            word[m] = __ldg((const uint16_t *)(codes + block * 16 + ((col[m] & 31) >> 1)));
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
            E *to = y + row[m] * stride + col[m];
            if (VECTOR && col[m] + 4 <= cols) {
                if constexpr (sizeof(E) == 4) *(uint4 *)to = *(const uint4 *)e;
                else *(uint2 *)to = *(const uint2 *)e;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (col[m] + k < cols) to[k] = e[k];
            }
        }
    }
}

}  // namespace ffn
}  // namespace spdnn_impl
