// sm_100a kernels of the feed-forward operators: sparse layers on row-major activations [tokens][neurons], plain or gated,
// forward and backward.
//
//   forward    z_s[t,c] = b_s[c] + sum_j w_s[c,j] x[t,r(c,j)]         s = 0 .. G-1 sets of weights over one topology
//              y[t,c]   = act(z_0)            (G = 1)      act(z_0) z_1            (G = 2)
//   backward   d_0 = dy act'(z_0)             (G = 1)      d_0 = dy z_1 act'(z_0), d_1 = dy act(z_0)     (G = 2)
//              dx[t,i]  = sum over connections (c,j) with r(c,j) = i of  sum_s w_s[c,j] d_s[t,c]
//              dw_s[c,j] = sum_t d_s[t,c] x[t,r(c,j)],   db_s[c] = sum_t d_s[t,c]
//
// Of a pattern in general there is no dense contraction in this: what a multiply-add costs is fetching its activation.  So activations are gathered
// in vectors over TOKENS: an IMAGE holds the values of T tokens of every neuron side by side, one load brings a connection's
// activation for up to eight tokens, and its index and weights are fetched once for all of them.  prepare_kernel writes the
// images (and takes in whatever is irregular: strides, types, 4-bit blocks, the last tokens), gather_kernel brings one into
// shared memory and runs a range of neurons on it.  Where neurons share their connections, 16 of them over the same rows are a small dense
// contraction, and block_kernel and dw_block_kernel take it to the tensor cores.
//
// Roundings.  Sums and the pre-activations kept for the backward pass are float32.  Inside a tensor-core instruction products are added without
// rounding and cut off to float32 (16 products at a time in block_kernel, 32 tokens in dw_block_kernel).  The d that the weights' gradients are made of
// are float32 too; dw_block_kernel multiplies with their upper 22 bits.  The
// d that dx gathers is rounded to the activations' type: a gathered value costs what it is wide, in shared memory and in tokens per
// image, and the error is half a step of every term.  fp16 does not hold d's range (a product of two or three factors of the operands' order), so a
// token's d are gathered at a power of two of their own (token_scale_kernel), which the sums are divided by again.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace spdnn_impl {
namespace ffn {

typedef __nv_bfloat16 bf16;

enum Type { F32 = 0, F16 = 1, BF16 = 2, MX4 = 3 };
enum Act { NONE = 0, RELU = 1, CLIP = 2, SILU = 3, GELU = 4, GELU_TANH = 5 };

// ---- numbers ---------------------------------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
template <class E> __device__ __forceinline__ E from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float load_as_float(const void *p, int type, int64_t at) {
    if (type == F32) return __ldg((const float *)p + at);
    if (type == F16) return __half2float(__ushort_as_half(__ldg((const unsigned short *)p + at)));
    return __uint_as_float((uint32_t)__ldg((const unsigned short *)p + at) << 16);
}

__device__ __forceinline__ void store_from_float(void *p, int type, int64_t at, float v) {
    if (type == F32) ((float *)p)[at] = v;
    else if (type == F16) ((__half *)p)[at] = __float2half_rn(v);
    else ((bf16 *)p)[at] = __float2bfloat16_rn(v);
}

// E2M1 (sign, two bits of exponent, one of mantissa) shifted into the place of a float's exponent and mantissa is its value times
// 2^-126, the subnormal code among them.
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    return __uint_as_float((code & 7u) << 22 | (code & 8u) << 28) * 0x1p126f;
}

// E8M0: 2^(byte - 127), 255 is NaN; 2^-127 is a subnormal float
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// The values of a word of codes, lowest half-byte first.
template <int COUNT> __device__ __forceinline__ void e2m1_values(uint32_t word, float (&v)[COUNT]) {
#pragma unroll
    for (int k = 0; k < COUNT; ++k) v[k] = e2m1_value(word >> (4 * k));
}

// Element `col` of row `row` of a microscaled matrix: codes [rows][blocks][16], scales [rows][blocks].  The product with the
// power of two is exact (below 2^128; beyond that it is infinite, as a float32 product is).
__device__ __forceinline__ float mx4_value(const uint8_t *codes, const uint8_t *scales, int64_t blocks, int64_t row, int col) {
    const int64_t b = row * blocks + (col >> 5);
    const uint32_t byte = __ldg(codes + b * 16 + ((col & 31) >> 1));
    return e2m1_value((col & 1) ? byte >> 4 : byte & 15u) * e8m0_value(__ldg(scales + b));
}

// ---- activations ------------------------------------------------------------------------------

constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluA = 0.79788456080286536f, kGeluB = 0.044715f;

// v / (1 + e^-w), the shape of SILU (w = v) and of GELU_TANH (w = 2 a (v + b v^3): (1 + tanh(w / 2)) / 2 = 1 / (1 + e^-w)).  FAST:
// the hardware's exponential and reciprocal, for operands of 16 bits: off by (8 + 2 |w|) 2^-24 of the result, the part that grows with w being of the
// size of what the rounding of w itself does to the exponential.
template <bool FAST> __device__ __forceinline__ float sigmoid_times(float v, float w) {
    if (!FAST) return v / (1.0f + expf(-w));
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(w * -1.44269504088896341f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return v * r;
}

// The normal distribution at v and its density.  What is computed is the tail (below zero), not its distance from one, which has lost all digits
// at v = -6: e^(-v^2 / 2), the density's, times a function of v that changes slowly: t Q(t) with t = 1 / (1 + 0.305 |v|), Q of degree 7 fitted to it
// for the least relative error (2^-23.3 for |v| up to 13.5); with the roundings 1.6 (4 + v^2) 2^-24 of the tail.  FAST: and those of the hardware's
// exponential and reciprocal (2^-22).
template <bool FAST> __device__ __forceinline__ void normal(float v, float &phi, float &density) {
    float e, t;
    if (FAST) {
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * v * (-0.5f * 1.44269504088896341f)));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(fabsf(v), 0.305f, 1.0f)));
    } else {
        e = expf(-0.5f * v * v);
        t = 1.0f / fmaf(fabsf(v), 0.305f, 1.0f);
    }
    float q = fmaf(t, 0.036699183285236f, -0.152988344430923f);
    q = fmaf(t, q, 0.185717046260834f);
    q = fmaf(t, q, -0.037977069616318f);
    q = fmaf(t, q, 0.121021859347820f);
    q = fmaf(t, q, 0.103420801460743f);
    q = fmaf(t, q, 0.122466832399368f);
    q = fmaf(t, q, 0.121639735996723f);
    const float tail = t * q * e;
    phi = v >= 0.0f ? 1.0f - tail : tail;
    density = kInvSqrt2Pi * e;
}

// A NaN stays one (v < 0 is false for it).
template <bool FAST> __device__ __forceinline__ float activate(float v, int act, float clip) {
    switch (act) {
        case RELU: return v < 0.0f ? 0.0f : v;
        case CLIP: return v < 0.0f ? 0.0f : v > clip ? clip : v;
        case SILU: return sigmoid_times<FAST>(v, v);
        case GELU: {
            float phi, density;
            normal<FAST>(v, phi, density);
            return v * phi;
        }
        case GELU_TANH: return sigmoid_times<FAST>(v, 2.0f * kGeluA * (v + kGeluB * v * v * v));
        default: return v;
    }
}

// 1 / (1 + e^-w)
template <bool FAST> __device__ __forceinline__ float sigmoid(float w) { return sigmoid_times<FAST>(1.0f, w); }

// act(v) and act'(v) for the backward pass
template <bool FAST> __device__ __forceinline__ void activate_both(float v, int act, float clip, float &value, float &slope) {
    switch (act) {
        case RELU: value = v < 0.0f ? 0.0f : v; slope = v > 0.0f ? 1.0f : v != v ? v : 0.0f; return;
        case CLIP:
            value = v < 0.0f ? 0.0f : v > clip ? clip : v;
            slope = v > 0.0f && v < clip ? 1.0f : v != v ? v : 0.0f;
            return;
        case SILU: {
            const float s = sigmoid<FAST>(v);
            value = v * s; slope = s * (1.0f + v * (1.0f - s));
            return;
        }
        case GELU: {
            float phi, density;
            normal<FAST>(v, phi, density);
            value = v * phi; slope = phi + v * density;
            return;
        }
        case GELU_TANH: {
            const float s = sigmoid<FAST>(2.0f * kGeluA * (v + kGeluB * v * v * v));
            // where v^2 is infinite the factor before it is zero
            value = v * s; slope = s + v * s * (1.0f - s) * 2.0f * kGeluA * (1.0f + 3.0f * kGeluB * fminf(v * v, 1e30f));
            return;
        }
        default: value = v; slope = 1.0f;
    }
}

// Calls f with the activation as a constant; not at all for NONE.
template <class F> __device__ __forceinline__ void with_activation(int act, const F &f) {
    switch (act) {
        case RELU: f(std::integral_constant<int, RELU>()); return;
        case CLIP: f(std::integral_constant<int, CLIP>()); return;
        case SILU: f(std::integral_constant<int, SILU>()); return;
        case GELU: f(std::integral_constant<int, GELU>()); return;
        case GELU_TANH: f(std::integral_constant<int, GELU_TANH>()); return;
        default: return;
    }
}

// ---- packed arithmetic -------------------------------------------------------------------------

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Two values of a 32-bit word of a 16-bit type as a pair of floats (exact).
template <class E> __device__ __forceinline__ f32x2 widen(uint32_t w);        // 16-bit types only
template <> __device__ __forceinline__ f32x2 widen<bf16>(uint32_t w) {
    return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ f32x2 widen<__half>(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return pack2(f.x, f.y);
}

template <class E> __device__ __forceinline__ f32x2 widen_word(uint32_t w) {
    if constexpr (sizeof(E) == 4) return 0;
    else return widen<E>(w);
}

// V consecutive 16- or 32-bit values as they are in memory.
template <class E, int V> struct Raw {
    static constexpr int kBytes = V * (int)sizeof(E);
    uint32_t w[(kBytes + 3) / 4];
    __device__ __forceinline__ void load(const void *p) {
        if constexpr (kBytes == 16) { const uint4 r = *(const uint4 *)p; w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w; }
        else if constexpr (kBytes == 8) { const uint2 r = *(const uint2 *)p; w[0] = r.x; w[1] = r.y; }
        else if constexpr (kBytes == 4) w[0] = *(const uint32_t *)p;
        else w[0] = *(const uint16_t *)p;
    }
    __device__ __forceinline__ uint32_t bits(int i) const {
        if constexpr (sizeof(E) == 4) return w[i];
        else return i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (kBytes + 3) / 4; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void set(int i, E v) {        // of a cleared one
        if constexpr (sizeof(E) == 4) w[i] = __float_as_uint(v);
        else w[i >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t *>(&v) << (16 * (i & 1));
    }
};

template <class E> __device__ __forceinline__ float bits_to_float(uint32_t b) {
    if constexpr (sizeof(E) == 4) return __uint_as_float(b);
    else if constexpr (std::is_same<E, bf16>::value) return __uint_as_float(b << 16);
    else return __half2float(__ushort_as_half((uint16_t)b));
}

// c + a b in float32, from the bits of a and b.  Two operands of one 16-bit type go into the mixed-precision fma as they are: exact
// product, one rounding, and none of the conversions (two per pair of values) that took a third of the inner loop.
template <class E, class W> __device__ __forceinline__ float fma_bits(uint32_t a, uint32_t b, float c) {
    if constexpr (sizeof(E) == 4) {
        return fmaf(__uint_as_float(a), __uint_as_float(b), c);
    } else {
        const uint16_t x = (uint16_t)a, y = (uint16_t)b;
        float d;
        if constexpr (std::is_same<E, bf16>::value && std::is_same<W, bf16>::value)
            asm("fma.rn.f32.bf16 %0, %1, %2, %3;" : "=f"(d) : "h"(x), "h"(y), "f"(c));
        else if constexpr (std::is_same<E, __half>::value && std::is_same<W, __half>::value)
            asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(x), "h"(y), "f"(c));
        else
            d = fmaf(__half2float(__ushort_as_half(x)), __uint_as_float(b << 16), c);
        return d;
    }
}

// ---- images -------------------------------------------------------------------------------------

// An image: rows + 1 neurons (the last one zeros) x SETS values x T = V P tokens, in UNITS of V tokens (16 bytes, or less where a
// neuron's tokens are fewer).  A neuron has R = SETS P units in a row; unit u = s P + p of neuron n lies at n R + (u ^ x(n)).  x
// turns the units of neighbouring neurons against each other, so that the bank group of unit 0 (16 bytes, 8 of them) is made of the three
// low bits of n whatever R is: of bits 0 and 1 and 2 for its highest and middle and lowest bit (R = 2: 1, 0, 2).  Eight lanes are served
// at a time (16 of 8 bytes).  So where L = 4, 2 or 1 lanes read a neuron together, the 2, 4 or 8 neurons of eight lanes do not meet if
// they differ modulo 2, 4 or 8, and sixteen neurons of 8 bytes if they do modulo 16: what topology.h orders connections by.
__host__ __device__ __forceinline__ uint32_t image_units(int rows, int per_row) { return ((uint32_t)(rows + 1) * per_row + 7u) & ~7u; }
__host__ __device__ __forceinline__ uint32_t unit_place(uint32_t n, uint32_t per_row) {
    const uint32_t reversed = (n & 1u) << 2 | (n & 2u) | (n >> 2 & 1u);
    return n * per_row + (reversed & ((per_row < 8u ? per_row : 8u) - 1u));
}

struct Matrix {            // a caller's operand
    const void *data;
    const uint8_t *scales; // MX4 only
    int64_t stride;        // elements of a row; MX4: blocks of a row
    int type;
};

struct PackArgs {
    Matrix x;              // values, or (backward) dy
    const float *z0, *z1;  // backward: pre-activations saved by the forward call (z1 used for two sets)
    int64_t z_stride;
    void *image;           // tiles of image_bytes each, or nullptr
    int64_t image_bytes;
    void *columns;         // [rows][sets][token_stride], or nullptr: what dw_kernel reads (gradients as float; x followed by 16 bytes of zeros)
    int64_t token_stride;
    const float *scale;    // [token_stride] what a token's values in the image are multiplied by, or nullptr: see token_scale_kernel
    int rows, tokens;
    int v, p;              // the image's unit and units per neuron (powers of two)
    int vector;            // every row of every operand begins on 16 bytes
    int same;              // x has the image's type, its rows begin on 16 bytes
    int act;
    float clip;
};

constexpr int kPackThreads = 256;

// The tile of a block: a row of 64 tokens and 16 bytes for every set and neuron; of gradients in float32.
template <class E, int SETS, bool GRADIENT> __host__ __device__ constexpr int pack_tile_bytes() {
    using Tile = typename std::conditional<GRADIENT, float, E>::type;
    return SETS * 64 * (64 + 16 / (int)sizeof(Tile)) * (int)sizeof(Tile) + (sizeof(E) == 2 && !GRADIENT ? 64 * 128 : 0);
}

// `COUNT` neighbours of a row as floats, from column `col` on; zeros behind `cols`.
template <int COUNT>
__device__ __forceinline__ void load_row_part(const Matrix &x, bool vector, int64_t row, int col, int cols, float (&v)[COUNT]) {
    if (x.type == MX4) {
        const int64_t b = row * x.stride + (col >> 5);
        const float scale = e8m0_value(__ldg(x.scales + b));
        const uint8_t *from = (const uint8_t *)x.data + b * 16 + ((col & 31) >> 1);
        float e[COUNT];
        e2m1_values(COUNT == 8 ? __ldg((const uint32_t *)from) : __ldg((const uint16_t *)from), e);
#pragma unroll
        for (int k = 0; k < COUNT; ++k) v[k] = col + k < cols ? e[k] * scale : 0.0f;
        return;
    }
    if (vector && col + COUNT <= cols) {
        if (x.type == F32) {
#pragma unroll
            for (int k = 0; k < COUNT; k += 4) {
                const float4 r = __ldg((const float4 *)((const float *)x.data + row * x.stride + col + k));
                v[k] = r.x; v[k + 1] = r.y; v[k + 2] = r.z; v[k + 3] = r.w;
            }
            return;
        }
        Raw<bf16, COUNT> r;
        r.load((const uint16_t *)x.data + row * x.stride + col);
#pragma unroll
        for (int k = 0; k < COUNT / 2; ++k) {
            const f32x2 two = x.type == F16 ? widen<__half>(r.w[k]) : widen<bf16>(r.w[k]);
            unpack2(two, v[2 * k], v[2 * k + 1]);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < COUNT; ++k) v[k] = col + k < cols ? load_as_float(x.data, x.type, row * x.stride + col + k) : 0.0f;
}

template <class E> __device__ __forceinline__ uint32_t pair_bits(float lo, float hi) {
    if constexpr (std::is_same<E, bf16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&p);
    } else {
        const __half2 p = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&p);
    }
}

// COUNT neighbours of the tile (on their natural alignment) as values of type E, in words; one 16-bit value: in the low half.  scale: of these
// tokens, or nullptr (a tile of gradients in fp16 only).
template <class E, int COUNT, class Tile> __device__ __forceinline__ void tile_words(const Tile *p, uint32_t *w, const float *scale) {
    if constexpr (sizeof(Tile) == sizeof(E)) {
        Raw<E, COUNT> r;
        r.load(p);
#pragma unroll
        for (int i = 0; i < (COUNT * (int)sizeof(E) + 3) / 4; ++i) w[i] = r.w[i];
    } else if constexpr (COUNT == 1) {
        w[0] = pair_bits<E>(std::is_same<E, __half>::value && scale ? *p * __ldg(scale) : *p, 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; i += 2) {
            float2 v = *(const float2 *)(p + i);
            if (std::is_same<E, __half>::value && scale) {
                const float2 f = __ldg((const float2 *)(scale + i));
                v.x *= f.x; v.y *= f.y;
            }
            w[i / 2] = pair_bits<E>(v.x, v.y);
        }
    }
}

// The units of fewer than 16 bytes of a block's neurons: 16 bytes at a time.  (An image is whole groups of 16 bytes, and so is what the
// 64 neurons before n0 take.)
template <class E, int SETS, int V, class Tile, class At>
__device__ __forceinline__ void small_units(char *image, int64_t image_bytes, int parts, const Tile &tile, const At &at, int n0, int n_end,
                                            uint32_t units, int rows, const float *scale) {
    constexpr int N = 16 / (int)sizeof(E), PIECES = N / V;
    const int first = (int)((uint32_t)n0 * SETS * V / N);
    const int here = (int)(min((uint32_t)(n0 + n_end) * SETS, units) * V / N) - first;
    const int log_here = n_end == 64 ? 31 - __clz(here) : 0;              // 64 neurons: a power of two
    for (int i = threadIdx.x; i < parts * here; i += kPackThreads) {
        const int part = log_here ? i >> log_here : i / here, g = i - part * here;
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int q = g * PIECES + k, n = q / SETS, s = q % SETS;
            uint32_t v[2] = {0, 0};
            if (n < 64 && n0 + n < rows) tile_words<E, V>(&tile[s][n][at(n, part * V)], v, scale ? scale + part * V : nullptr);
            constexpr int WORDS = V * (int)sizeof(E) / 4;
            if constexpr (WORDS == 0) w[k / 2] |= v[0] << (16 * (k & 1)) & (k & 1 ? 0xffff0000u : 0xffffu);
            else
#pragma unroll
                for (int j = 0; j < WORDS; ++j) w[k * WORDS + j] = v[j];
        }
        ((uint4 *)(image + part * image_bytes))[first + g] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// dL/dz of N neurons of a token, from neuron `col` on; zeros behind the last.
template <class E, int SETS, int N>
__device__ __forceinline__ void gradient_part(const PackArgs &a, int64_t row, int col, float (&d0)[N], float (&d1)[N]) {
    float g[N], u[N], dy[N];
    load_row_part<N>(a.x, a.vector, row, col, a.rows, d0);
#pragma unroll
    for (int k = 0; k < N; ++k) dy[k] = d0[k];
    const bool saved = SETS == 2 || a.act != NONE;
    if (saved) load_row_part<N>(Matrix{a.z0, nullptr, a.z_stride, F32}, a.vector, row, col, a.rows, g);
    if (SETS == 2) load_row_part<N>(Matrix{a.z1, nullptr, a.z_stride, F32}, a.vector, row, col, a.rows, u);
    if (SETS == 2) {
#pragma unroll
        for (int k = 0; k < N; ++k) { d1[k] = d0[k] * g[k]; u[k] *= d0[k]; d0[k] = u[k]; }       // NONE
    }
    with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float value, slope;
            activate_both<sizeof(E) == 2>(g[k], act.value, a.clip, value, slope);
            if (SETS == 2) d1[k] = dy[k] * value;
            d0[k] *= slope;
        }
    });
}

// One block: 64 neurons x 64 tokens, through shared memory so that reads run along neurons and writes along tokens.  The tokens of a
// neuron are permuted in groups of N (16 bytes of the tile), for the writers of neighbouring neurons to hit different banks.
template <class E, int SETS, bool GRADIENT>
__device__ __forceinline__ void pack_block(const PackArgs &a, unsigned block, unsigned char *shared) {
    using Tile = typename std::conditional<GRADIENT, float, E>::type;
    constexpr int N = 16 / (int)sizeof(E);            // neurons a thread loads at a time
    constexpr int G = 16 / (int)sizeof(Tile);         // tokens of a permuted group
    constexpr int ROW = 64 + G;
    static_assert(sizeof(Tile[SETS][64][ROW]) <= pack_tile_bytes<E, SETS, GRADIENT>(), "the tile");
    Tile (&tile)[SETS][64][ROW] = *reinterpret_cast<Tile (*)[SETS][64][ROW]>(shared);
    const auto at = [](int n, int t) { return t ^ (((n / N) & (64 / G - 1)) * G); };
    const int blocks_n = (a.rows + 63) / 64;
    const int n0 = (int)(block % blocks_n) * 64;
    const int t0 = (int)(block / blocks_n) * 64;
    bool loaded = false;
    if constexpr (sizeof(E) == 2 && !GRADIENT) {
        // 16-bit values that stay as they are: rows come in with cp.async (behind the tile) and are turned by ldmatrix.trans, eight
        // tokens x eight neurons at a time, without a value passing through the ALU
        if (a.same && n0 + 64 <= a.rows) {
            loaded = true;
            const uint32_t rows = (uint32_t)__cvta_generic_to_shared(shared + sizeof(Tile[SETS][64][ROW]));
            const uint16_t *x = (const uint16_t *)a.x.data;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = i * 32 + threadIdx.x / 8, q = threadIdx.x & 7;
                const int64_t row = min(t0 + t, a.tokens - 1);
                const int bytes = t0 + t < a.tokens ? 16 : 0;         // zeros behind the last token
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(rows + t * 128 + ((q ^ (t & 7)) * 16)),
                             "l"(x + row * a.x.stride + n0 + q * 8), "r"(bytes) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
            const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;      // of eight tokens
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t w[4];
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(rows + (group * 8 + (lane & 7)) * 128 + (((i * 4 + lane / 8) ^ (lane & 7)) * 16)) : "memory");
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int n = (i * 4 + k) * 8 + lane / 4;
                    *(uint32_t *)&tile[0][n][at(n, group * 8) + (lane & 3) * 2] = w[k];
                }
            }
        }
    }
    for (int i = loaded ? 64 * 64 : threadIdx.x; i < 64 * 64 / N; i += kPackThreads) {
        const int t = i / (64 / N), n = i % (64 / N) * N;
        float d0[N], d1[N];
#pragma unroll
        for (int k = 0; k < N; ++k) d0[k] = d1[k] = 0.0f;
        if (t0 + t < a.tokens && n0 + n < a.rows) {
            if constexpr (GRADIENT) gradient_part<E, SETS, N>(a, t0 + t, n0 + n, d0, d1);
            else load_row_part<N>(a.x, a.vector, t0 + t, n0 + n, a.rows, d0);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            tile[0][n + k][at(n, t)] = from_float<Tile>(d0[k]);
            if (SETS == 2) tile[SETS - 1][n + k][at(n, t)] = from_float<Tile>(d1[k]);
        }
    }
    __syncthreads();
    if (a.image) {
        const float *scale = GRADIENT && a.scale ? a.scale + t0 : nullptr;
        const int log_p = 31 - __clz(a.p), T = a.v * a.p, per_row = a.p * SETS;
        const uint32_t units = image_units(a.rows, per_row);
        const int64_t tiles = ((int64_t)a.tokens + T - 1) / T;
        // the last block along n also writes the row of zeros and the units behind it
        const int n_end = n0 + 64 >= a.rows ? (int)((units + per_row - 1) / per_row) - n0 : 64;
        const int64_t tile0 = t0 / T;
        const int parts = (int)min((int64_t)(64 / T), tiles - tile0);
        if (a.v == N) {
            const int units_here = min(n_end * per_row, (int)(units - (uint32_t)n0 * per_row));
            const int log_units = n_end == 64 ? 31 - __clz(units_here) : 0;        // 64 neurons: a power of two
            for (int i = threadIdx.x; i < parts * units_here; i += kPackThreads) {
                const int part = log_units ? i >> log_units : i / units_here, u = i - part * units_here;
                const int p = u & (a.p - 1), s = (u >> log_p) & (SETS - 1), n = (u >> log_p) / SETS;
                const int t = part * T + p * N;
                uint32_t w[4] = {0, 0, 0, 0};
                if (n < 64 && n0 + n < a.rows) {
                    if constexpr (sizeof(Tile) == sizeof(E)) {
                        tile_words<E, N>(&tile[s][n][at(n, t)], w, nullptr);
                    } else {
                        tile_words<E, 4>(&tile[s][n][at(n, t)], w, scale ? scale + t : nullptr);
                        tile_words<E, 4>(&tile[s][n][at(n, t + 4)], w + 2, scale ? scale + t + 4 : nullptr);
                    }
                }
                const uint4 r = make_uint4(w[0], w[1], w[2], w[3]);
                ((uint4 *)((char *)a.image + (tile0 + part) * a.image_bytes))[unit_place(n0 + n, per_row) ^ (uint32_t)(s * a.p + p)] = r;
            }
        } else {
            char *image = (char *)a.image + tile0 * a.image_bytes;
            if (a.v == 1) small_units<E, SETS, 1>(image, a.image_bytes, parts, tile, at, n0, n_end, units, a.rows, scale);
            else if (a.v == 2) small_units<E, SETS, 2>(image, a.image_bytes, parts, tile, at, n0, n_end, units, a.rows, scale);
            else small_units<E, SETS, (N > 4 ? 4 : 2)>(image, a.image_bytes, parts, tile, at, n0, n_end, units, a.rows, scale);
        }
    }
    if (a.columns) {
        // columns (n, s) are rows of token_stride one after another
        constexpr int STEP = kPackThreads / (64 / G);
        const int t = threadIdx.x % (64 / G) * G, q0 = threadIdx.x / (64 / G);
        Tile *to = (Tile *)a.columns + ((int64_t)n0 * SETS + q0) * a.token_stride + t0 + t;
#pragma unroll
        for (int q = 0; q < SETS * 64; q += STEP, to += STEP * a.token_stride) {
            const int n = (q + q0) / SETS, s = (q + q0) % SETS;
            if (n0 + n < a.rows) *(uint4 *)to = *(const uint4 *)&tile[s][n][at(n, t)];
        }
    }
}

constexpr int kScaleThreads = 512;

// The power of two that brings the largest finite |d| of a token into [2^14, 2^15): what fp16 holds of it is off by half a step, or by 2^-39 of the
// largest where that is more.  2^126 at most, whose reciprocal is a normal number.  One block per token; bringing in what the image is made of, once
// more, is what bounds it (1024 tokens x 16384, both sets: 39 us for 168 MB with four neurons a lane, 43 with eight; 97 tokens: 12 us with 512 threads, 16 with
// 256).
template <int SETS>
__global__ void __launch_bounds__(kScaleThreads) token_scale_kernel(const __grid_constant__ PackArgs a, float *scales) {
    __shared__ uint32_t tops[kScaleThreads / 32];
    const int t = gridDim.x - 1 - blockIdx.x;         // the tokens that prepare_kernel begins with come last, and are still in L2 then
    uint32_t top = 0;           // bits of magnitudes are ordered as they are
    if (t < a.tokens)
        for (int col = threadIdx.x * 4; col < a.rows; col += kScaleThreads * 4) {
            float d[2][4];
            gradient_part<__half, SETS, 4>(a, t, col, d[0], d[1]);
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t m = __float_as_uint(d[s][k]) & 0x7fffffffu;
                    top = max(top, m < 0x7f800000u ? m : 0u);
                }
        }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int w = 1; w < kScaleThreads / 32; ++w) top = max(top, tops[w]);
    scales[t] = __uint_as_float((127 + 14 + 127 - max(top >> 23, 15u)) << 23);
}

// 1 / a power of two between 2^-126 and 2^126
__device__ __forceinline__ float reciprocal(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }

struct OrderArgs {
    Matrix w0, w1;
    const uint32_t *idx, *src;  // the gather table (topology.h)
    int64_t entries;
    int slots;
    int values, p;              // the image's values and units per neuron
    int whole, wide;            // its units are 16 bytes; indexes are 32 bits (image in global memory)
    void *weights, *index;      // [quads][32][4][sets], [quads][32][4]
};

// Bits of the weight at canonical position s, as W.  A caller's matrix has W's type or is microscaled.  Where its rows follow one another
// without gaps the position is the address; the division is for the others.
template <class W> __device__ __forceinline__ uint32_t weight_bits(const Matrix &m, uint32_t s, int slots) {
    if (s == 0xffffffffu) return 0u;
    if (m.type == MX4) {
        uint32_t c = s / (uint32_t)slots, j = s - c * (uint32_t)slots;
        const float v = mx4_value((const uint8_t *)m.data, m.scales, m.stride, c, (int)j);
        if constexpr (sizeof(W) == 4) return __float_as_uint(v);
        else return pair_bits<W>(v, 0.0f) & 0xffffu;
    }
    int64_t at = s;
    if (m.stride != slots) {
        const uint32_t c = s / (uint32_t)slots;
        at = (int64_t)c * m.stride + (s - c * (uint32_t)slots);
    }
    if constexpr (sizeof(W) == 4) return __ldg((const uint32_t *)m.data + at);
    else return __ldg((const uint16_t *)m.data + at);
}

// The gather table as a call's gather reads it: the weights in its order, and the place of every gathered neuron in the image.  Padding
// gets the weight zero, whatever the caller's matrix holds where a neuron has no connection.  A thread has the four connections of a quad.
template <class W, int SETS>
__device__ __forceinline__ void order_block(const OrderArgs &a, unsigned block) {
    const int64_t quad = (int64_t)block * kPackThreads + threadIdx.x;
    if (quad * 4 >= a.entries) return;
    const uint4 src4 = __ldg((const uint4 *)a.src + quad), idx4 = __ldg((const uint4 *)a.idx + quad);
    const uint32_t src[4] = {src4.x, src4.y, src4.z, src4.w}, idx[4] = {idx4.x, idx4.y, idx4.z, idx4.w};
    uint32_t w[4 * SETS], place[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int s = 0; s < SETS; ++s) w[k * SETS + s] = weight_bits<W>(s ? a.w1 : a.w0, src[k], a.slots);
        place[k] = a.whole ? unit_place(idx[k], (uint32_t)(a.values * a.p)) : idx[k];
    }
    if constexpr (sizeof(W) == 4) {
#pragma unroll
        for (int k = 0; k < SETS; ++k) ((uint4 *)a.weights)[quad * SETS + k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    } else if constexpr (SETS == 2) {
        ((uint4 *)a.weights)[quad] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    } else {
        ((uint2 *)a.weights)[quad] = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    }
    if (a.wide) ((uint4 *)a.index)[quad] = make_uint4(place[0], place[1], place[2], place[3]);
    else ((uint2 *)a.index)[quad] = make_uint2(place[0] | place[1] << 16, place[2] | place[3] << 16);
}

struct OrderBlocksArgs {
    Matrix w0, w1;
    const uint32_t *src;        // the block table (topology.h)
    int64_t chunks;
    int slots;
    void *weights;
};

// The weights of a block table as mma.m16n8k16 takes them for its second operand: of a chunk, per step of 16 rows and per set 16 bytes a
// lane, the fragments of the block's neurons 0-7 and 8-15; the table's sources are in that order.  SPREAD (backward): the sets are
// planes of their own.
template <class W, int SETS, bool SPREAD>
__device__ __forceinline__ void order_blocks_block(const OrderBlocksArgs &a, unsigned block) {
    const int64_t e = (int64_t)block * kPackThreads + threadIdx.x;        // lane of a step
    if (e >= a.chunks * 64) return;
    const uint4 lo = __ldg((const uint4 *)a.src + e * 2), hi = __ldg((const uint4 *)a.src + e * 2 + 1);
    const uint32_t src[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int set = 0; set < SETS; ++set) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = weight_bits<W>(set ? a.w1 : a.w0, src[k], a.slots);
        const int64_t to = SPREAD ? set * a.chunks * 64 + e : ((e >> 5) * SETS + set) * 32 + (e & 31);
        ((uint4 *)a.weights)[to] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
}

// Everything that a call lays out, in one launch (a launch takes longer than most of these blocks): the table, then image and columns
// of the gathered values, then (backward) the columns of x.  Measured: 4096 tokens x 4096, bf16, and a table of 524288 connections 21 us (34 MB in, 37
// out); dL/dz of 4096 x 4096, both sets, with 4096 x 1024 of x 75 us (176 MB in, 210 out: 5.1 TB/s).
struct PrepareArgs {
    OrderArgs order;
    OrderBlocksArgs blocks;
    PackArgs main, x;
    int by_blocks;                          // the gather goes by blocks: their weights are ordered, not the gather table's
    unsigned order_blocks, main_blocks;     // the rest are x's
};

// Of gradients five blocks an SM (six of fp32) need no spills: left to itself the compiler took 60 registers for four blocks and 79 and 97 us where these
// take 75 and 88 (4096 tokens x 4096, bf16; 1024 x 16384, fp16; both sets).
template <class E, class W, int SETS, bool GRADIENT>
__global__ void __launch_bounds__(kPackThreads, GRADIENT ? (sizeof(E) == 2 ? 5 : 6) : 0) prepare_kernel(const __grid_constant__ PrepareArgs a) {
    constexpr int MAIN = pack_tile_bytes<E, GRADIENT ? SETS : 1, GRADIENT>(), X = pack_tile_bytes<E, 1, false>();
    __shared__ __align__(16) unsigned char shared[MAIN > X ? MAIN : X];
    if (blockIdx.x < a.order_blocks) {
        if (!a.by_blocks) order_block<W, SETS>(a.order, blockIdx.x);
        else if constexpr (sizeof(W) == 2) order_blocks_block<W, SETS, GRADIENT>(a.blocks, blockIdx.x);
    } else if (blockIdx.x - a.order_blocks < a.main_blocks) pack_block<E, GRADIENT ? SETS : 1, GRADIENT>(a.main, blockIdx.x - a.order_blocks, shared);
    else if (GRADIENT) {
        const unsigned block = blockIdx.x - a.order_blocks - a.main_blocks;
        pack_block<E, 1, false>(a.x, block, shared);
        if (block == 0 && threadIdx.x == 0) *(uint4 *)((E *)a.x.columns + a.x.rows * a.x.token_stride) = make_uint4(0, 0, 0, 0);
    }
}

// ---- the gather ----------------------------------------------------------------------------------

struct GatherArgs {
    const void *image;          // tiles of image_bytes
    int64_t image_bytes;
    const uint32_t *slice_ptr;  // the gather table (topology.h)
    const void *index;          // order_block's: uint16_t (image in shared memory) or uint32_t
    const void *weights;
    int outs, tokens, splits;
    const float *bias0, *bias1; // or nullptr
    void *y;
    float *z0, *z1;             // pre-activations, or nullptr
    int64_t y_stride, z_stride;
    int y_type;
    int act;
    float clip;
    const float *scale;         // of the image's tokens (PackArgs), or nullptr; fp16 only
};

// Units a lane reads per gathered value, and threads per block.  Two units halve what index, weights and the loop cost per fma; with more sums
// than 16 in registers a block of 1024 threads would spill (4096 tokens 1024 -> 4096, gated: two units 90 us, one 129; 768 threads 90, 1024 97).
__host__ __device__ constexpr int lane_units(int P) { return P < 2 ? P : 2; }
__host__ __device__ constexpr int gather_threads(int sums) { return sums <= 16 ? 1024 : 768; }

// Brings `bytes` (a multiple of 16) from global to shared memory, 16 bytes per thread and copy, none of them through registers.
__device__ __forceinline__ void copy_in(void *dst, const void *src, uint32_t bytes) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    for (uint32_t at = threadIdx.x * 16u; at < bytes; at += blockDim.x * 16u)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + at), "l"((const char *)src + at) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
}

// Four connections of a lane's neuron.
template <class W, int SETS, bool WIDE> struct Quad {
    static constexpr int kWords = SETS * (int)sizeof(W);     // 32-bit words of 4 x SETS weights
    uint32_t index[WIDE ? 4 : 2];
    uint32_t weight[kWords];
    __device__ __forceinline__ void load(const GatherArgs &a, size_t at) {
        if constexpr (WIDE) {
            const uint4 r = __ldg((const uint4 *)a.index + at);
            index[0] = r.x; index[1] = r.y; index[2] = r.z; index[3] = r.w;
        } else {
            const uint2 r = __ldg((const uint2 *)a.index + at);
            index[0] = r.x; index[1] = r.y;
        }
        if constexpr (kWords == 2) {
            const uint2 r = __ldg((const uint2 *)a.weights + at);
            weight[0] = r.x; weight[1] = r.y;
        } else {
#pragma unroll
            for (int k = 0; k < kWords / 4; ++k) {
                const uint4 r = __ldg((const uint4 *)a.weights + at * (kWords / 4) + k);
                weight[4 * k] = r.x; weight[4 * k + 1] = r.y; weight[4 * k + 2] = r.z; weight[4 * k + 3] = r.w;
            }
        }
    }
    // bits of weight `set` of connection `k`
    __device__ __forceinline__ uint32_t bits(int k, int set) const {
        const int e = k * SETS + set;
        if constexpr (sizeof(W) == 4) return weight[e];
        else return e & 1 ? weight[e >> 1] >> 16 : weight[e >> 1] & 0xffffu;
    }
};

// One block: the image of one tile of T = V P tokens, and a range of the gathering neurons.  Unit of work of a warp: 32 / L neurons, L
// lanes each with NV units of V tokens.  S = 1: one gathered value for G sums (forward).  S = 2: two gathered values for one
// sum (backward of the gated block).  GLOBAL: the image stays in global memory (it does not fit on the SM).
//
// The table (index and weights of a quad: up to 24 bytes a lane) comes from L2, where a load takes longer than the arithmetic of a
// quad: each is requested while the one before it is worked on, the first of a unit before the last of the one before it.
//
// Measured: 4096 tokens, 4096 -> 16384, gated, bf16 (T = 16) 265 us = 16.2 T fma/s, 0.43 of the FP32 pipe; issue slots 76 % busy, LSU pipe 73 %.  1024
// tokens, 16384 -> 16384, fp16 (T = 4) 114 us without and 124 with pre-activations; its dx (T = 2, two values a connection) 234 us (222 without the
// factors of the tokens), LSU pipe 79 %.
template <class E, class W, int V, int P, int S, int G, bool GLOBAL>
__global__ void __launch_bounds__(gather_threads(V * lane_units(P) * G)) gather_kernel(const __grid_constant__ GatherArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int SETS = S > G ? S : G;
    constexpr int UB = V * (int)sizeof(E);
    constexpr bool WHOLE = UB == 16;
    constexpr int NV = lane_units(P), L = P / NV;
    constexpr int WARPS = gather_threads(V * NV * G) / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const char *image = (const char *)a.image + (int64_t)tile * a.image_bytes;
    const int j = lane % L;
    const int64_t units = (int64_t)((a.outs + 31) / 32) * L;
    const int64_t last = units * (split + 1) / a.splits;
    int64_t unit = units * split / a.splits + warp;
    uint32_t q0 = 0, q1 = 0;
    if (unit < last) { q0 = __ldg(a.slice_ptr + unit / L); q1 = __ldg(a.slice_ptr + unit / L + 1); }
    const auto in_slice = [&](int64_t u) { return (int)(u % L) * (32 / L) + lane / L; };
    // The tokens of a lane are the same in every unit; where they are many, their factors would take its registers.  Two sets always have factors.
    constexpr bool SCALED = std::is_same<E, __half>::value && std::is_same<W, __half>::value && G == 1, KEPT = SCALED && S == 2 && NV * V <= 4;
    const auto factor = [&](int k) { return reciprocal(__ldg(a.scale + (int64_t)tile * (V * P) + j * V + k / V * (L * V) + k % V)); };
    float kept[KEPT ? NV * V : 1];
    if (KEPT)
#pragma unroll
        for (int k = 0; k < NV * V; ++k) kept[k] = factor(k);
    Quad<W, SETS, GLOBAL> cur, ahead;
    if (q0 < q1) cur.load(a, (size_t)q0 * 32 + in_slice(unit));
    if constexpr (!GLOBAL) copy_in(smem, image, (uint32_t)a.image_bytes);
    while (unit < last) {
        const int64_t next = unit + WARPS;
        uint32_t n0 = 0, n1 = 0;
        if (next < last) { n0 = __ldg(a.slice_ptr + next / L); n1 = __ldg(a.slice_ptr + next / L + 1); }
        float acc[G][NV * V];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int k = 0; k < NV * V; ++k) acc[g][k] = 0.0f;
        const auto work = [&](const Quad<W, SETS, GLOBAL> &quad) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    Raw<E, V * (WHOLE ? 1 : S)> x[WHOLE ? S : 1];     // a neuron of few tokens: both values in one load
                    if constexpr (GLOBAL) {
#pragma unroll
                        for (int s = 0; s < S; ++s) x[s].load(image + (((size_t)quad.index[k] * 16u) ^ ((uint32_t)(s * P + i * L + j) * 16u)));
                    } else {
                        const uint32_t w = quad.index[k >> 1];
                        if constexpr (WHOLE) {
#pragma unroll
                            for (int s = 0; s < S; ++s) x[s].load(smem + (((k & 1 ? w >> 12 : w << 4) & 0xffff0u) ^ ((uint32_t)(s * P + i * L + j) * 16u)));
                        } else {
                            x[0].load(smem + (k & 1 ? w >> 16 : w & 0xffffu) * (uint32_t)(S * UB));
                        }
                    }
#pragma unroll
                    for (int s = 0; s < S; ++s)
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const uint32_t w = quad.bits(k, S > 1 ? s : g);
#pragma unroll
                            for (int v = 0; v < V; ++v)
                                acc[g][i * V + v] = fma_bits<E, W>(WHOLE ? x[WHOLE ? s : 0].bits(v) : x[0].bits(s * V + v), w, acc[g][i * V + v]);
                        }
                }
        };
        if (q0 < q1) {
            size_t at = (size_t)q0 * 32 + in_slice(unit);
            const size_t end = (size_t)(q1 - 1) * 32;
#pragma unroll 2
            for (; at < end; at += 32) {
                ahead.load(a, at + 32);
                work(cur);
                cur = ahead;
            }
            if (n0 < n1) ahead.load(a, (size_t)n0 * 32 + in_slice(next));
            work(cur);
            cur = ahead;
        } else if (n0 < n1) {
            cur.load(a, (size_t)n0 * 32 + in_slice(next));
        }
        const int c = (int)(unit / L) * 32 + in_slice(unit);
        if (c < a.outs) {
            const float b0 = a.bias0 ? __ldg(a.bias0 + c) : 0.0f, b1 = G == 2 && a.bias1 ? __ldg(a.bias1 + c) : 0.0f;
#pragma unroll
            for (int k = 0; k < NV * V; ++k) {
                acc[0][k] += b0;
                if (G == 2) acc[G - 1][k] += b1;
            }
            const int64_t t0 = (int64_t)tile * (V * P) + j * V;
            // token k of the lane is t0 + (k / V) L V + k % V
            if (SCALED && (S == 2 || a.scale))
#pragma unroll
                for (int k = 0; k < NV * V; ++k) acc[0][k] *= KEPT ? kept[KEPT ? k : 0] : factor(k);
            const auto store = [&](auto *to, int64_t stride, const auto &value) {
                to += t0 * stride + c;
                const int left = (int)min((int64_t)(P * V), (int64_t)a.tokens - t0);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (left >= i * L * V + V) {
#pragma unroll
                        for (int v = 0; v < V; ++v) to[v * stride] = value(i * V + v);
                    } else {
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            if (i * L * V + v < left) to[v * stride] = value(i * V + v);
                    }
                    to += L * V * stride;
                }
            };
            if (a.z0) {
                store(a.z0, a.z_stride, [&](int k) { return acc[0][k]; });
                if (G == 2) store(a.z1, a.z_stride, [&](int k) { return acc[G - 1][k]; });
            }
            if (S == 1) {
                with_activation(a.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < NV * V; ++k) acc[0][k] = activate<sizeof(E) == 2>(acc[0][k], act.value, a.clip);
                });
                if (G == 2)
#pragma unroll
                    for (int k = 0; k < NV * V; ++k) acc[0][k] *= acc[G - 1][k];
            }
            if (a.y_type == F32) store((float *)a.y, a.y_stride, [&](int k) { return acc[0][k]; });
            else if (a.y_type == F16) store((__half *)a.y, a.y_stride, [&](int k) { return __float2half_rn(acc[0][k]); });
            else store((bf16 *)a.y, a.y_stride, [&](int k) { return __float2bfloat16_rn(acc[0][k]); });
        }
        unit = next; q0 = n0; q1 = n1;
    }
}

// ---- gradients of the weights by blocks ----------------------------------------------------------------

struct DwBlockArgs {
    const void *x;               // [inputs][token_stride]
    const float *d;              // [outputs][sets][token_stride]
    const uint32_t *chunk_ptr, *rows, *src;   // the forward direction's block table
    const int32_t *members;
    const uint32_t *chunk_block; // block of every chunk
    int64_t token_stride;
    int inputs;
    float *dw0, *dw1;            // [outputs][slots]
    float *db0, *db1;            // or nullptr
};

constexpr int kDwBlockThreads = 256;

__device__ __forceinline__ void mma_16x8x8_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One block of threads: a chunk (16 outputs over 32 inputs); its warps take 32 tokens each in turn and are joined at the end, in a fixed
// order.  dw[j][k] = sum_t d[j][t] x[k][t]: both factors lie along tokens, so a lane's 16 bytes of a row are its part of four steps of eight
// tokens (which tokens make a step is free as long as both factors agree), and no shared memory is needed to feed the tensor cores.  x (16
// bits) is exact in tf32; d is the sum of two tf32 numbers, 22 bits, and takes two products.  The
// second has d's sign and is zero for a d of zero only (where nothing is left it is 2^-30 of d; below 2^-96 it may vanish), and an infinite d itself:
// so an infinity of x or of d goes through both products as it goes through one.  The tensor cores cut sums off instead
// of rounding them: they add up 32 tokens only, the rest is added in float32.  Measured: 4096 tokens, 1024 -> 4096, both sets, bf16: 53 us (dw_kernel:
// 119) for 143 MB from HBM; what bounds it is the latency of those loads (128 registers a thread leave 16 warps an SM).
template <class E, int G>
__global__ void __launch_bounds__(kDwBlockThreads, 2) dw_block_kernel(const __grid_constant__ DwBlockArgs a) {
    constexpr int WARPS = kDwBlockThreads / 32;
    __shared__ float sums[WARPS][G][16][33];
    __shared__ float bias_sums[WARPS][G][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t chunk = blockIdx.x, block = __ldg(a.chunk_block + chunk);
    // rows g, g + 8, ...; outputs g and g + 8.  What is not there reads row or output 0, and its sum is dropped.
    const E *x[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const uint32_t row = __ldg(a.rows + (size_t)chunk * 32 + n * 8 + g);
        x[n] = (const E *)a.x + (row < (uint32_t)a.inputs ? row : 0u) * a.token_stride + t * 8;
    }
    const float *d[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) d[h] = a.d + (int64_t)max(__ldg(a.members + (size_t)block * 16 + h * 8 + g), 0) * G * a.token_stride + t * 8;
    float total[G][4][4], bias[G][2];
#pragma unroll
    for (int s = 0; s < G; ++s) {
        bias[s][0] = bias[s][1] = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[s][n][i] = 0.0f;
    }
    for (int64_t at = warp * 32; at < a.token_stride; at += WARPS * 32) {
        Raw<E, 8> xv[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) xv[n].load(x[n] + at);
#pragma unroll
        for (int s = 0; s < G; ++s) {
            float4 dv[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    dv[h][i] = __ldg((const float4 *)(d[h] + s * a.token_stride + at) + i);
                    bias[s][h] += (dv[h][i].x + dv[h][i].y) + (dv[h][i].z + dv[h][i].w);
                }
            float part[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[n][i] = 0.0f;
#pragma unroll
            for (int step = 0; step < 4; ++step) {         // tokens 8 t + 2 step and the next
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 &q = dv[k & 1][step >> 1];
                    const float v = step & 1 ? (k < 2 ? q.z : q.w) : (k < 2 ? q.x : q.y);
                    hi[k] = __float_as_uint(v) & 0xffffe000u;
                    const float rest = fmaf(v, 0x1p-30f, v - __uint_as_float(hi[k]));
                    lo[k] = __float_as_uint(fabsf(v) < __int_as_float(0x7f800000) ? rest : v);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t b0 = __float_as_uint(bits_to_float<E>(xv[n].bits(2 * step))), b1 = __float_as_uint(bits_to_float<E>(xv[n].bits(2 * step + 1)));
                    mma_16x8x8_tf32(part[n], hi, b0, b1);
                    mma_16x8x8_tf32(part[n], lo, b0, b1);
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) total[s][n][i] += part[n][i];
        }
    }
    // total[s][n][i]: output g + 8 (i / 2), row 8 n + 2 t + i % 2
#pragma unroll
    for (int s = 0; s < G; ++s)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[warp][s][g + 8 * (i >> 1)][n * 8 + 2 * t + (i & 1)] = total[s][n][i];
#pragma unroll
    for (int s = 0; s < G; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v = bias[s][h];
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            if (t == 0) bias_sums[warp][s][g + 8 * h] = v;
        }
    __syncthreads();
    // every block has a first chunk: there the biases' gradients, the sums of d, are written
    if (chunk == __ldg(a.chunk_ptr + block) && threadIdx.x < 16 * G) {
        const int s = threadIdx.x >> 4, j = threadIdx.x & 15, c = __ldg(a.members + (size_t)block * 16 + j);
        float *db = s ? a.db1 : a.db0;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += bias_sums[w][s][j];
        if (c >= 0 && db) db[c] = sum;
    }
    for (int e = threadIdx.x; e < 512; e += kDwBlockThreads) {
        // e counts the table's order: lane, half, v of a step (topology.h, fragment)
        const int v = e & 3, half = e >> 2 & 1, l = e >> 3 & 31, step = e >> 8;
        const int k = step * 16 + (l & 3) * 2 + (v & 1) + (v >> 1) * 8, j = half * 8 + (l >> 2);
        const uint32_t to = __ldg(a.src + (size_t)chunk * 512 + e);
        if (to == 0xffffffffu) continue;
#pragma unroll
        for (int s = 0; s < G; ++s) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += sums[w][s][j][k];
            (s ? a.dw1 : a.dw0)[to] = sum;
        }
    }
}

// ---- a few tokens ----------------------------------------------------------------------------------

struct FewArgs {
    Matrix x, w0, w1;
    const void *rows;          // canonical rows [outputs][stride] of the topology: uint16_t where inputs < 65536, else int32_t; `inputs` = none
    int row_stride;            // slots rounded up to a multiple of 4
    int slots, inputs, outputs, tokens;
    const float *bias0, *bias1;
    void *y;
    float *z0, *z1;
    int64_t y_stride, z_stride;
    int y_type, act;
    float clip;
    int vector_x, vector_w;    // every row of x on 16 bytes; every row of the weights on four elements
};

constexpr int kFewThreads = 512;

// Four weights of a row, from slot j on (a multiple of 4), as floats; zeros behind the last slot.
template <class W, bool MX>
__device__ __forceinline__ void four_weights(const Matrix &m, bool vector, int c, int j, int slots, float (&w)[4]) {
    if constexpr (MX) {
        const int64_t b = (int64_t)c * m.stride + (j >> 5);
        const float scale = e8m0_value(__ldg(m.scales + b));
        e2m1_values(__ldg((const uint16_t *)((const uint8_t *)m.data + b * 16 + ((j & 31) >> 1))), w);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] *= scale;
    } else {
        const W *from = (const W *)m.data + (int64_t)c * m.stride + j;
        if (vector && j + 4 <= slots) {
            Raw<W, 4> r;
            r.load(from);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = bits_to_float<W>(r.bits(k));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = j + k < slots ? to_float(from[k]) : 0.0f;
        }
    }
}

// Forward pass of up to T tokens in one launch that reads the caller's operands as they are: with few tokens the latency of a call is what
// counts, and laying out image and weights first would take longer than the sums (one token, 4096 -> 16384, gated, bf16: 3.7 us for 3.1 MB of
// weights and rows; 11.7 in the launches of the images' way when this was written).  Eight lanes share a neuron, four connections
// of 32 each; the tokens' activations lie in shared memory [inputs + 1][T] (the last row zeros, where missing connections point).
template <class E, class W, bool MX, int T, int G>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const __grid_constant__ FewArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    E *x = (E *)smem;
    const int t0 = blockIdx.y * T;
    constexpr int N = 16 / (int)sizeof(E);
    const int tokens = min(T, a.tokens - t0);
    for (int i = threadIdx.x; i < (a.inputs + N) / N; i += kFewThreads) {
        E e[T][N];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float v[N];
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = 0.0f;
            if (t < tokens && i * N < a.inputs) load_row_part<N>(a.x, a.vector_x, t0 + t, i * N, a.inputs, v);
#pragma unroll
            for (int k = 0; k < N; ++k) e[t][k] = from_float<E>(v[k]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i * N + k <= a.inputs) {
#pragma unroll
                for (int t = 0; t < T; ++t) x[(i * N + k) * T + t] = e[t][k];
            }
    }
    __syncthreads();
    const int j0 = (threadIdx.x & 7) * 4;
    // every lane of a warp stays for the shuffles: neurons behind the last are computed as the last one and not stored
    for (int first = blockIdx.x * (kFewThreads / 8); first < a.outputs; first += gridDim.x * (kFewThreads / 8)) {
        const int mine = first + (threadIdx.x >> 3), c = min(mine, a.outputs - 1);
        float acc[G][T];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int t = 0; t < T; ++t) acc[g][t] = 0.0f;
        for (int j = j0; j < a.slots; j += 32) {
            uint32_t row[4];
            if (a.inputs < 65536) {
                const uint2 r = __ldg((const uint2 *)((const uint16_t *)a.rows + (int64_t)c * a.row_stride + j));
                row[0] = r.x & 0xffffu; row[1] = r.x >> 16; row[2] = r.y & 0xffffu; row[3] = r.y >> 16;
            } else {
                const uint4 r = __ldg((const uint4 *)((const int32_t *)a.rows + (int64_t)c * a.row_stride + j));
                row[0] = r.x; row[1] = r.y; row[2] = r.z; row[3] = r.w;
            }
            float w[G][4];
            four_weights<W, MX>(a.w0, a.vector_w, c, j, a.slots, w[0]);
            if (G == 2) four_weights<W, MX>(a.w1, a.vector_w, c, j, a.slots, w[G - 1]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                Raw<E, T> v;
                v.load(x + row[k] * T);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    // a missing connection's weight is whatever the matrix holds there
                    const float one = row[k] == (uint32_t)a.inputs ? 0.0f : w[g][k];
#pragma unroll
                    for (int t = 0; t < T; ++t) acc[g][t] = fmaf(bits_to_float<E>(v.bits(t)), one, acc[g][t]);
                }
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int s = 4; s; s >>= 1) acc[g][t] += __shfl_xor_sync(0xffffffffu, acc[g][t], s);
        // lane t of the eight stores token t
        float g = acc[0][0], u = acc[G - 1][0];
#pragma unroll
        for (int t = 1; t < T; ++t)
            if ((threadIdx.x & 7) == t) { g = acc[0][t]; u = acc[G - 1][t]; }
        const int t = threadIdx.x & 7;
        if (mine >= a.outputs || t >= tokens) continue;
        const int64_t token = t0 + t;
        g += a.bias0 ? __ldg(a.bias0 + c) : 0.0f;
        if (G == 2) u += a.bias1 ? __ldg(a.bias1 + c) : 0.0f;
        if (a.z0) {
            a.z0[token * a.z_stride + c] = g;
            if (G == 2) a.z1[token * a.z_stride + c] = u;
        }
        float y = activate<sizeof(E) == 2>(g, a.act, a.clip);
        if (G == 2) y *= u;
        store_from_float(a.y, a.y_type, token * a.y_stride + c, y);
    }
}

// ---- the gather by blocks ---------------------------------------------------------------------------

struct BlockArgs {
    const void *image;           // tiles of 64 tokens: rows of 128 bytes per neuron and value
    int64_t image_bytes;
    const uint32_t *chunk_ptr, *rows;   // the block table
    const int32_t *members;
    const void *weights;         // order_blocks_block's
    int64_t chunks;
    int blocks, tokens;
    const float *bias0, *bias1;
    void *y;
    float *z0, *z1;
    int64_t y_stride, z_stride;
    int y_type, act;
    float clip;
    const float *scale;          // of the image's tokens (PackArgs), or nullptr; fp16 only
    int whole_y, whole_z;        // rows of y, of z begin on 16 bytes: blocks of 16 neighbours are stored in whole sectors
};

// 16 warps of two stages (1024 tokens of the butterfly 16384, gated: 32 us) rather than 12 of three (38) or 8 of four (43).
constexpr int kBlockWarps = 16, kBlockStages = 2;
__host__ __device__ constexpr int block_stage_bytes(int G) { return 32 * 128 + 1024 * G; }

// Stores 64 tokens x 16 neighbouring neurons of a warp's fragments (value(m, half, i), laid out as block_kernel's accumulators) in a 16-bit type
// through 2 KB of shared memory of its own, 16 bytes a lane: fragments hold two neighbours of eight tokens, an eighth of a sector each.
template <class T, class F>
__device__ __forceinline__ void store_block(unsigned char *stage, T *to, int64_t stride, int tokens, const F &value) {
    const int lane = threadIdx.x & 31;
    // halves of a token's 32 bytes, turned against each other for neighbouring tokens to meet on fewer banks
    const auto place = [](int token, int half) { return token * 32 + ((half ^ (token >> 2 & 1)) * 16); };
    __syncwarp();
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *(uint32_t *)(stage + place(m * 16 + i * 8 + lane / 4, half) + (lane & 3) * 4) = pair_bits<T>(value(m, half, 2 * i), value(m, half, 2 * i + 1));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int token = i * 16 + lane / 2, half = lane & 1;
        if (token < tokens) *(uint4 *)((char *)(to + token * stride) + half * 16) = *(const uint4 *)(stage + place(token, half));
    }
}

template <class E> __device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<E, bf16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy_16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// A warp takes 64 tokens of a block (16 neurons over the same rows) at a time: a chunk of 32 rows x 64 tokens and its weights come into the warp's
// own stages with cp.async, a chunk ahead; ldmatrix.trans turns 16 rows x 16 tokens into a fragment of tokens x rows, wherever the rows
// came from, and the products (16 tokens x 8 neurons x 16 rows) run on the tensor cores.  One gathered value serves 16 neurons and
// both sets, where gather_kernel's serves one: what is left is bringing the rows in (each is used by as many blocks as list it) and the results
// out.  The contraction is 16 wide: mma.sync, not tcgen05, whose tile of 128 tokens and its round trip through tensor memory would have the
// same bytes to move, and those bound this kernel.
template <class E, int S, int G>
__global__ void __launch_bounds__(kBlockWarps * 32) block_kernel(const __grid_constant__ BlockArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int STAGE = block_stage_bytes(G);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t stages = (uint32_t)__cvta_generic_to_shared(smem) + warp * kBlockStages * STAGE;
    const unsigned char *stages_ptr = smem + warp * kBlockStages * STAGE;
    const int tiles = (a.tokens + 63) / 64;
    const int64_t units = (int64_t)a.blocks * tiles, warps = (int64_t)gridDim.x * kBlockWarps, me = (int64_t)blockIdx.x * kBlockWarps + warp;
    const int64_t first = units * me / warps, last = units * (me + 1) / warps;

    // where the copies are: unit, chunk of its list, which begins at chunk `begin` and has `count`; S sets one after another
    int64_t ahead = first;
    uint32_t begin = 0, count = 0, at = 0;
    const auto open = [&] {
        if (ahead >= last) return;
        const int b = (int)(ahead / tiles);
        begin = __ldg(a.chunk_ptr + b);
        count = __ldg(a.chunk_ptr + b + 1) - begin;    // at least one
        at = 0;
    };
    open();
    uint32_t row = ahead < last ? __ldg(a.rows + (size_t)begin * 32 + lane) : 0u;
    int fill = 0;
    const auto request = [&] {
        if (ahead < last) {
            const uint32_t set = S == 2 && at >= count ? 1u : 0u, chunk = begin + at - set * count;
            const char *image = (const char *)a.image + (ahead % tiles) * a.image_bytes;
            const uint32_t stage = stages + fill * STAGE;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = i * 4 + lane / 8, q = lane & 7;
                const uint32_t n = __shfl_sync(0xffffffffu, row, k);
                const uint32_t x = (n & 1u) << 2 | (n & 2u) | (n >> 2 & 1u);           // unit_place's turn
                copy_16(stage + k * 128 + q * 16, image + ((size_t)n * S + set) * 128 + (((q ^ (k & 7)) ^ x) * 16));
            }
            const char *w = (const char *)a.weights + ((size_t)set * a.chunks + chunk) * (1024 * G);
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) copy_16(stage + 4096 + (i * 32 + lane) * 16, w + (i * 32 + lane) * 16);
            if (++at == count * S) { ++ahead; open(); }
            if (ahead < last) row = __ldg(a.rows + (size_t)(begin + (S == 2 && at >= count ? at - count : at)) * 32 + lane);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        fill = fill + 1 == kBlockStages ? 0 : fill + 1;
    };
    for (int i = 0; i + 1 < kBlockStages; ++i) request();

    int drain = 0;
    for (int64_t unit = first; unit < last; ++unit) {
        const int b = (int)(unit / tiles);
        const uint32_t chunks = (__ldg(a.chunk_ptr + b + 1) - __ldg(a.chunk_ptr + b)) * S;
        float acc[4][2 * G][4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int f = 0; f < 2 * G; ++f)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[m][f][k] = 0.0f;
        for (uint32_t c = 0; c < chunks; ++c) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kBlockStages - 2) : "memory");
            __syncwarp();
            request();                                 // into the stage that was drained last
            const uint32_t stage = stages + drain * STAGE;
            const unsigned char *w = stages_ptr + drain * STAGE + 4096;
#pragma unroll
            for (int step = 0; step < 2; ++step) {
                uint4 frag[G];
#pragma unroll
                for (int g = 0; g < G; ++g) frag[g] = *(const uint4 *)(w + ((step * G + g) * 32 + lane) * 16);
                const int r = lane & 7, k = step * 16 + (lane >> 4) * 8 + r;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    uint32_t x[4];
                    const int unit_of = m * 2 + (lane >> 3 & 1);
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(stage + k * 128 + ((unit_of ^ r) * 16)) : "memory");
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        mma_16x8x16<E>(acc[m][2 * g], x, frag[g].x, frag[g].y);
                        mma_16x8x16<E>(acc[m][2 * g + 1], x, frag[g].z, frag[g].w);
                    }
                }
            }
            __syncwarp();
            drain = drain + 1 == kBlockStages ? 0 : drain + 1;
        }
        // acc[m][2 g + half][i]: token 16 m + lane / 4 + 8 (i / 2), neuron 8 half + 2 (lane % 4) + i % 2
        const int64_t tile0 = (unit % tiles) * 64;
        const int tokens = (int)min((int64_t)64, a.tokens - tile0);
        const int32_t *members = a.members + (size_t)b * 16;
        const int head = __ldg(members);
        // sixteen neighbours, on 16 bytes of any type
        const bool neighbours = __ldg(members + 15) - head == 15 && head % 8 == 0;
        // the stage that was drained last is free until the next request
        unsigned char *scratch = smem + warp * kBlockStages * STAGE + (drain == 0 ? kBlockStages - 1 : drain - 1) * STAGE;
        int2 c[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            c[half] = __ldg((const int2 *)(members + half * 8) + (lane & 3));
            float b0[2] = {0, 0}, b1[2] = {0, 0};
            if (a.bias0) { if (c[half].x >= 0) b0[0] = __ldg(a.bias0 + c[half].x); if (c[half].y >= 0) b0[1] = __ldg(a.bias0 + c[half].y); }
            if (G == 2 && a.bias1) { if (c[half].x >= 0) b1[0] = __ldg(a.bias1 + c[half].x); if (c[half].y >= 0) b1[1] = __ldg(a.bias1 + c[half].y); }
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[m][half][i] += b0[i & 1];
                    if (G == 2) acc[m][2 * G - 2 + half][i] += b1[i & 1];
                }
        }
        if (std::is_same<E, __half>::value && G == 1 && a.scale)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = reciprocal(__ldg(a.scale + tile0 + m * 16 + i * 8 + lane / 4));
#pragma unroll
                    for (int half = 0; half < 2; ++half) { acc[m][half][2 * i] *= f; acc[m][half][2 * i + 1] *= f; }
                }
        const auto store = [&](auto *to, int64_t stride, bool whole, const auto &value) {
            using T = typename std::remove_pointer<decltype(to)>::type;
            to += tile0 * stride;
            if (whole && neighbours) {
                if constexpr (sizeof(T) == 4) {
                    // four lanes' pairs fill a sector as they are
#pragma unroll
                    for (int m = 0; m < 4; ++m)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int token = m * 16 + i * 8 + lane / 4;
                            if (token >= tokens) continue;
                            T *row = to + token * stride + head + (lane & 3) * 2;
#pragma unroll
                            for (int half = 0; half < 2; ++half) *(float2 *)(row + half * 8) = make_float2(value(m, half, 2 * i), value(m, half, 2 * i + 1));
                        }
                } else {
                    store_block(scratch, to + head, stride, tokens, value);
                }
                return;
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int token = m * 16 + i / 2 * 8 + lane / 4, neuron = i & 1 ? c[half].y : c[half].x;
                        if (token < tokens && neuron >= 0) to[token * stride + neuron] = from_float<T>(value(m, half, i));
                    }
        };
        if (a.z0) {
            store(a.z0, a.z_stride, a.whole_z, [&](int m, int half, int i) { return acc[m][half][i]; });
            if (G == 2) store(a.z1, a.z_stride, a.whole_z, [&](int m, int half, int i) { return acc[m][2 * G - 2 + half][i]; });
        }
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][half][i] = activate<true>(acc[m][half][i], act.value, a.clip);
        });
        if (G == 2)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][half][i] *= acc[m][2 * G - 2 + half][i];
        const auto result = [&](int m, int half, int i) { return acc[m][half][i]; };
        if (a.y_type == F32) store((float *)a.y, a.y_stride, a.whole_y, result);
        else if (a.y_type == F16) store((__half *)a.y, a.y_stride, a.whole_y, result);
        else store((bf16 *)a.y, a.y_stride, a.whole_y, result);
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- gradients of the weights ----------------------------------------------------------------------

struct DwArgs {
    const void *x;            // [inputs][token_stride], and 16 bytes of zeros
    const float *d;           // [outputs][sets][token_stride]
    const int32_t *rows;      // [outputs][slots] canonical, -1 = none
    int64_t token_stride;
    int inputs, outputs, slots, chunks;   // chunks of kDwSlots connections per output
    float *dw0, *dw1;         // [outputs][slots]
    float *db0, *db1;         // or nullptr
};

constexpr int kDwSlots = 16;
constexpr int kDwThreads = 128;

// Sums of `COUNT` (16 or 32) values over the lanes of a warp: lane l returns that of value l mod COUNT.  Every exchange halves the values a
// lane still holds, so it takes COUNT - 1 shuffles (and one) instead of five for each.
template <int COUNT> __device__ __forceinline__ float sum_lanes(float (&v)[COUNT]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int s = COUNT / 2; s; s >>= 1)
#pragma unroll
        for (int i = 0; i < s; ++i) {
            const bool upper = lane & s;
            const float send = upper ? v[i] : v[i + s], keep = upper ? v[i + s] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, s);
        }
    if (COUNT == 16) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
    return v[0];
}

// A warp owns kDwSlots connections of one output: every lane sums its tokens' products in registers, the lanes are joined at the
// end.  Adjacent warps take adjacent outputs, whose inputs are often the same rows (blocks of a butterfly).  What bounds it is bringing
// the rows from L2, so the loads of several are in flight before the first is used.  A connection that is not there reads row 0 and its sum is
// dropped.  Lanes behind the last token read zeros for both factors: an infinity of any other token would make NaN of a gradient of zero.  (They read
// them behind x's columns; a load under a condition took 155 us instead of 125 at 1024 tokens, 16384 -> 16384, and a last step of its own 159.)
template <class E, int G>
__global__ void __launch_bounds__(kDwThreads, G == 1 ? 7 : 4) dw_kernel(const DwArgs a) {
    constexpr int V = 16 / sizeof(E);
    constexpr int PAIRS = V / 2;
    constexpr int BATCH = 4;
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (kDwThreads / 32) + (threadIdx.x >> 5);
    const int c = (int)(unit % a.outputs), chunk = (int)(unit / a.outputs);
    if (chunk >= a.chunks) return;
    const int j0 = chunk * kDwSlots, slots = min(kDwSlots, a.slots - j0);
    const int mine = lane < slots ? __ldg(a.rows + (int64_t)c * a.slots + j0 + lane) : -1;
    f32x2 acc[kDwSlots][G], bias[G];
#pragma unroll
    for (int g = 0; g < G; ++g) bias[g] = 0;
#pragma unroll
    for (int j = 0; j < kDwSlots; ++j)
#pragma unroll
        for (int g = 0; g < G; ++g) acc[j][g] = 0;
    const f32x2 ones = pack2(1.0f, 1.0f);
    const E *x = (const E *)a.x;
    const float *d = a.d + (int64_t)c * G * a.token_stride;
    for (int64_t t0 = 0; t0 < a.token_stride; t0 += 32 * V) {
        const bool inside = t0 + lane * V < a.token_stride;
        const int64_t t = inside ? t0 + lane * V : 0;
        const int least = inside ? 0 : a.inputs;
        f32x2 dv[G][PAIRS];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < PAIRS; i += 2) {
                ulonglong2 part = make_ulonglong2(0, 0);
                if (inside) part = *(const ulonglong2 *)(d + g * a.token_stride + t + 2 * i);
                dv[g][i] = part.x; dv[g][i + 1] = part.y;
            }
#pragma unroll
        for (int j = 0; j < kDwSlots; j += BATCH) {
            Raw<E, V> raw[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const int row = max(__shfl_sync(0xffffffffu, mine, j + k), least);
                raw[k].load(x + (int64_t)row * a.token_stride + t);
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k)
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) {
                    const f32x2 xv = sizeof(E) == 4 ? pack2(__uint_as_float(raw[k].bits(2 * i)), __uint_as_float(raw[k].bits(2 * i + 1)))
                                                    : widen_word<E>(raw[k].w[i]);
#pragma unroll
                    for (int g = 0; g < G; ++g) acc[j + k][g] = fma2(xv, dv[g][i], acc[j + k][g]);
                }
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) bias[g] = fma2(dv[g][i], ones, bias[g]);
    }
    float sums[kDwSlots * G];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < kDwSlots; ++j) {
            float lo, hi;
            unpack2(acc[j][g], lo, hi);
            sums[g * kDwSlots + j] = lo + hi;
        }
    const float sum = sum_lanes(sums);
    const int j = lane & 15, g = lane >> 4;
    const int row = __shfl_sync(0xffffffffu, mine, j);
    if (g < G && j < slots) (g ? a.dw1 : a.dw0)[(int64_t)c * a.slots + j0 + j] = row >= 0 ? sum : 0.0f;
    if (chunk) return;
#pragma unroll
    for (int s = 0; s < G; ++s) {
        float lo, hi;
        unpack2(bias[s], lo, hi);
        float v = lo + hi;
#pragma unroll
        for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        float *db = s ? a.db1 : a.db0;
        if (lane == 0 && db) db[c] = v;
    }
}

}  // namespace ffn
}  // namespace spdnn_impl
