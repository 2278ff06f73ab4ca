// sm_100a kernels of the feed-forward operators: sparse layers on row-major activations [tokens][neurons], plain or gated,
// forward and backward.
//
//   forward    z_s[t,c] = b_s[c] + sum_j w_s[c,j] x[t,r(c,j)]         s = 0 .. G-1 sets of weights over one topology
//              y[t,c]   = act(z_0)            (G = 1)      act(z_0) z_1            (G = 2)
//   backward   d_0 = dy act'(z_0)             (G = 1)      d_0 = dy z_1 act'(z_0), d_1 = dy act(z_0)     (G = 2)
//              dx[t,i]  = sum over connections (c,j) with r(c,j) = i of  sum_s w_s[c,j] d_s[t,c]
//              dw_s[c,j] = sum_t d_s[t,c] x[t,r(c,j)],   db_s[c] = sum_t d_s[t,c]
//
// There is no dense contraction in this: what a multiply-add costs is fetching its activation.  So activations are gathered in
// vectors over TOKENS: an IMAGE holds the values of T tokens of every neuron side by side, one load brings a connection's
// activation for up to eight tokens, and its index and weights are fetched once for all of them.  pack_kernel writes the
// images (and takes in whatever is irregular: strides, types, 4-bit blocks, the last tokens), gather_kernel brings one into
// shared memory and runs a range of neurons on it.
//
// Roundings: all sums, the pre-activations kept for the backward pass and the d that the weights' gradients are made of are in 32 bits.  The
// d that dx gathers is rounded to the activations' type: a gathered value costs what it is wide, in shared memory and in tokens per
// image, and the error (half a step of every term) is that of rounding dx itself.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

// E2M1: twice the magnitude of codes 0..7 is 0 1 2 3 4 6 8 12
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const float m = 0.5f * (float)((0xC8643210u >> (4 * (code & 7u))) & 15u);
    return (code & 8u) ? -m : m;
}

// E8M0: 2^(byte - 127), 255 is NaN; 2^-127 is a subnormal float
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// Element `col` of row `row` of a microscaled matrix: codes [rows][blocks][16], scales [rows][blocks].  The product with the
// power of two is exact (below 2^128; beyond that it is infinite, as a float32 product is).
__device__ __forceinline__ float mx4_value(const uint8_t *codes, const uint8_t *scales, int64_t blocks, int64_t row, int col) {
    const int64_t b = row * blocks + (col >> 5);
    const uint32_t byte = __ldg(codes + b * 16 + ((col & 31) >> 1));
    return e2m1_value((col & 1) ? byte >> 4 : byte & 15u) * e8m0_value(__ldg(scales + b));
}

// ---- activations ------------------------------------------------------------------------------

constexpr float kInvSqrt2 = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluA = 0.79788456080286536f, kGeluB = 0.044715f;

// A NaN stays one (v < 0 is false for it).
__device__ __forceinline__ float activate(float v, int act, float clip) {
    switch (act) {
        case RELU: return v < 0.0f ? 0.0f : v;
        case CLIP: return v < 0.0f ? 0.0f : v > clip ? clip : v;
        case SILU: return v / (1.0f + expf(-v));
        case GELU: return 0.5f * v * (1.0f + erff(v * kInvSqrt2));
        case GELU_TANH: return 0.5f * v * (1.0f + tanhf(kGeluA * (v + kGeluB * v * v * v)));
        default: return v;
    }
}

__device__ __forceinline__ float activate_slope(float v, int act, float clip) {
    switch (act) {
        case RELU: return v > 0.0f ? 1.0f : v != v ? v : 0.0f;
        case CLIP: return v > 0.0f && v < clip ? 1.0f : v != v ? v : 0.0f;
        case SILU: { const float s = 1.0f / (1.0f + expf(-v)); return s * (1.0f + v * (1.0f - s)); }
        case GELU: return 0.5f * (1.0f + erff(v * kInvSqrt2)) + v * kInvSqrt2Pi * expf(-0.5f * v * v);
        case GELU_TANH: {
            const float t = tanhf(kGeluA * (v + kGeluB * v * v * v));
            return 0.5f * (1.0f + t) + 0.5f * v * (1.0f - t * t) * kGeluA * (1.0f + 3.0f * kGeluB * v * v);
        }
        default: return 1.0f;
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
template <class E> __device__ __forceinline__ f32x2 widen(uint32_t w);
template <> __device__ __forceinline__ f32x2 widen<bf16>(uint32_t w) {
    return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ f32x2 widen<__half>(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return pack2(f.x, f.y);
}

// V consecutive values of one neuron as pairs of floats (V = 1: one pair with a zero).
template <class E, int V> struct Values {
    static constexpr int kPairs = (V + 1) / 2;
    f32x2 v[kPairs];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = 0;
    }
    __device__ __forceinline__ void load(const void *p) {
        constexpr int bytes = V * (int)sizeof(E);
        if constexpr (sizeof(E) == 4) {
            if constexpr (bytes == 16) {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(p);
                v[0] = w.x; v[1] = w.y;
            } else if constexpr (bytes == 8) {
                v[0] = *reinterpret_cast<const f32x2 *>(p);
            } else {
                v[0] = pack2(*reinterpret_cast<const float *>(p), 0.0f);
            }
        } else if constexpr (bytes == 16) {
            const uint4 w = *reinterpret_cast<const uint4 *>(p);
            v[0] = widen<E>(w.x); v[1] = widen<E>(w.y); v[2] = widen<E>(w.z); v[3] = widen<E>(w.w);
        } else if constexpr (bytes == 8) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            v[0] = widen<E>(w.x); v[1] = widen<E>(w.y);
        } else if constexpr (bytes == 4) {
            v[0] = widen<E>(*reinterpret_cast<const uint32_t *>(p));
        } else {
            v[0] = pack2(to_float(*reinterpret_cast<const E *>(p)), 0.0f);
        }
    }
};

// ---- images -------------------------------------------------------------------------------------

// An image: rows + 1 neurons (the last one zeros) x SETS values x T = V P tokens, in UNITS of V tokens (16 bytes, or less where a
// neuron's tokens are fewer).  Unit (n, s, p) is number q = (n SETS + s) P + p.  Units of 16 bytes are stored at
// q ^ (q / 8 mod 8): whoever writes an image walks along n, and without it the units of 8 neurons would share banks.
__host__ __device__ __forceinline__ uint32_t image_units(int rows, int per_row) { return ((uint32_t)(rows + 1) * per_row + 7u) & ~7u; }
__host__ __device__ __forceinline__ uint32_t swizzle(uint32_t q) { return q ^ ((q >> 3) & 7u); }

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
    void *columns;         // [rows][sets][token_stride], or nullptr: what dw_kernel reads (gradients as float)
    int64_t token_stride;
    int rows, tokens;
    int v, p;              // the image's unit and units per neuron
    int act;
    float clip;
};

constexpr int kPackThreads = 256;

// One block: 64 neurons x 64 tokens, through shared memory so that reads run along neurons and writes along tokens.
template <class E, int SETS, bool GRADIENT>
__global__ void __launch_bounds__(kPackThreads) pack_kernel(const PackArgs a) {
    __shared__ float tile[SETS][64][65];
    const int blocks_n = (a.rows + 63) / 64;
    const int n0 = (int)(blockIdx.x % blocks_n) * 64;
    const int t0 = (int)(blockIdx.x / blocks_n) * 64;
    for (int i = threadIdx.x; i < 64 * 64; i += kPackThreads) {
        const int t = i >> 6, n = i & 63;
        float d0 = 0.0f, d1 = 0.0f;
        if (t0 + t < a.tokens && n0 + n < a.rows) {
            const int64_t row = t0 + t;
            const int col = n0 + n;
            if (!GRADIENT) {
                d0 = a.x.type == MX4 ? mx4_value((const uint8_t *)a.x.data, a.x.scales, a.x.stride, row, col)
                                     : load_as_float(a.x.data, a.x.type, row * a.x.stride + col);
            } else {
                const float dy = load_as_float(a.x.data, a.x.type, row * a.x.stride + col);
                const float z0 = a.act == NONE && SETS == 1 ? 0.0f : __ldg(a.z0 + row * a.z_stride + col);
                d0 = dy * activate_slope(z0, a.act, a.clip);
                if (SETS == 2) {
                    d0 *= __ldg(a.z1 + row * a.z_stride + col);
                    d1 = dy * activate(z0, a.act, a.clip);
                }
            }
        }
        tile[0][n][t] = d0;
        if (SETS == 2) tile[SETS - 1][n][t] = d1;
    }
    __syncthreads();
    if (a.image) {
        const int T = a.v * a.p, per_row = a.p * SETS;
        const uint32_t units = image_units(a.rows, per_row);
        const bool swizzled = a.v * (int)sizeof(E) == 16;
        const int per_token_block = 64 / a.v;
        const int tiles = (a.tokens + T - 1) / T;
        // the last block along n also writes the row of zeros and the units behind it
        const int n_end = n0 + 64 >= a.rows ? (int)((units + per_row - 1) / per_row) - n0 : 64;
        for (int i = threadIdx.x; i < n_end * SETS * per_token_block; i += kPackThreads) {
            // along tokens first within a tile, then along n
            const int p = i % a.p, rest = i / a.p;
            const int s = rest % SETS, rest2 = rest / SETS;
            const int n = rest2 % n_end, part = rest2 / n_end;
            const int t = (part * a.p + p) * a.v;
            const int tile_index = (t0 + t) / T;
            const uint32_t q = ((uint32_t)(n0 + n) * SETS + s) * a.p + p;
            if (tile_index >= tiles || q >= units) continue;
            E *to = (E *)((char *)a.image + (int64_t)tile_index * a.image_bytes) + (size_t)(swizzled ? swizzle(q) : q) * a.v;
            const bool real = n < 64 && n0 + n < a.rows;
            for (int k = 0; k < a.v; ++k) to[k] = from_float<E>(real ? tile[s][n & 63][t + k] : 0.0f);
        }
    }
    if (a.columns) {
        for (int i = threadIdx.x; i < SETS * 64 * 64; i += kPackThreads) {
            const int t = i & 63, n = (i >> 6) & 63, s = i >> 12;
            if (n0 + n >= a.rows) continue;
            const int64_t at = ((int64_t)(n0 + n) * SETS + s) * a.token_stride + t0 + t;
            if (GRADIENT) ((float *)a.columns)[at] = tile[s][n][t];
            else ((E *)a.columns)[at] = from_float<E>(tile[s][n][t]);
        }
    }
}

// The weights of a gather table in its order: [quads][32][4][sets].  Padding gets zero, whatever the caller's matrix holds
// where a neuron has no connection.
template <class W, int SETS>
__global__ void __launch_bounds__(256) order_weights_kernel(const Matrix w0, const Matrix w1, const uint32_t *__restrict__ src, int slots,
                                                            int64_t entries, W *__restrict__ out) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= entries) return;
    const uint32_t s = __ldg(src + e);
    const uint32_t c = s / (uint32_t)slots, j = s % (uint32_t)slots;
    for (int k = 0; k < SETS; ++k) {
        const Matrix &w = k ? w1 : w0;
        float v = 0.0f;
        if (s != 0xffffffffu)
            v = w.type == MX4 ? mx4_value((const uint8_t *)w.data, w.scales, w.stride, c, (int)j)
                              : load_as_float(w.data, w.type, (int64_t)c * w.stride + j);
        out[e * SETS + k] = from_float<W>(v);
    }
}

// ---- the gather ----------------------------------------------------------------------------------

struct GatherArgs {
    const void *image;          // tiles of image_bytes
    int64_t image_bytes;
    const uint32_t *slice_ptr;  // the gather table (topology.h)
    const void *idx;            // uint16_t (image in shared memory) or uint32_t
    const void *weights;        // order_weights_kernel's
    int outs, tokens, rows, splits;
    const float *bias0, *bias1; // or nullptr
    void *y;
    float *z0, *z1;             // pre-activations, or nullptr
    int64_t y_stride, z_stride;
    int y_type;
    int act;
    float clip;
};

constexpr int kGatherThreads = 512;

// Brings `bytes` (a multiple of 16) from global to shared memory, 16 bytes per thread and copy, none of them through registers.
__device__ __forceinline__ void copy_in(void *dst, const void *src, uint32_t bytes) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    for (uint32_t at = threadIdx.x * 16u; at < bytes; at += blockDim.x * 16u)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + at), "l"((const char *)src + at) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
}

// One block: the image of one tile of T = V P tokens, and a range of the gathering neurons.  Unit of work of a warp: 32 / P
// neurons, P lanes each with V tokens.  S = 1: one gathered value for G sums (forward).  S = 2: two gathered values for one sum
// (backward of the gated block).  GLOBAL: the image stays in global memory (it does not fit on the SM).
template <class E, class W, int V, int P, int S, int G, bool GLOBAL>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const GatherArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int PAIRS = Values<E, V>::kPairs;
    constexpr int SETS = S > G ? S : G;
    constexpr bool SWIZZLED = V * sizeof(E) == 16;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const char *image = (const char *)a.image + (int64_t)tile * a.image_bytes;
    if constexpr (!GLOBAL) {
        copy_in(smem, image, (uint32_t)a.image_bytes);
        image = (const char *)smem;
    }
    const int p = lane % P, sub = lane / P;
    const int slices = (a.outs + 31) / 32;
    const int64_t units = (int64_t)slices * P;
    const int64_t last = units * (split + 1) / a.splits;
    for (int64_t unit = units * split / a.splits + warp; unit < last; unit += kGatherThreads / 32) {
        const int slice = (int)(unit / P);
        const int in_slice = (int)(unit % P) * (32 / P) + sub;
        const uint32_t q0 = __ldg(a.slice_ptr + slice), q1 = __ldg(a.slice_ptr + slice + 1);
        f32x2 acc[G][PAIRS];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) acc[g][k] = 0;
        for (uint32_t q = q0; q < q1; ++q) {
            const size_t at = (size_t)q * 32 + in_slice;
            uint32_t rows[4];
            if constexpr (GLOBAL) {
                const uint4 r = __ldg((const uint4 *)a.idx + at);
                rows[0] = r.x; rows[1] = r.y; rows[2] = r.z; rows[3] = r.w;
            } else {
                const uint2 r = __ldg((const uint2 *)a.idx + at);
                rows[0] = r.x & 0xffffu; rows[1] = r.x >> 16; rows[2] = r.y & 0xffffu; rows[3] = r.y >> 16;
            }
            Values<W, 4 * SETS <= 16 / (int)sizeof(W) ? 4 * SETS : 16 / (int)sizeof(W)> w[4 * SETS * sizeof(W) > 16 ? 4 * SETS * sizeof(W) / 16 : 1];
            constexpr int PER = 4 * SETS * sizeof(W) > 16 ? 16 / (int)sizeof(W) : 4 * SETS;
#pragma unroll
            for (int k = 0; k < (int)(4 * SETS / PER); ++k) w[k].load((const char *)a.weights + (at * 4 * SETS + (size_t)k * PER) * sizeof(W));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    Values<E, V> x;
                    const uint32_t unit_in_image = (rows[k] * S + s) * P + p;
                    if constexpr (GLOBAL) {
                        x.load(image + (size_t)(SWIZZLED ? swizzle(unit_in_image) : unit_in_image) * (V * sizeof(E)));
                    } else {
                        x.load(image + (SWIZZLED ? swizzle(unit_in_image) : unit_in_image) * (uint32_t)(V * sizeof(E)));
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const int e = k * SETS + (S > 1 ? s : g);
                        float lo, hi;
                        unpack2(w[e / PER].v[e % PER / 2], lo, hi);
                        const float one = e % 2 ? hi : lo;
                        const f32x2 both = pack2(one, one);
#pragma unroll
                        for (int i = 0; i < PAIRS; ++i) acc[g][i] = fma2(x.v[i], both, acc[g][i]);
                    }
                }
            }
        }
        const int c = slice * 32 + in_slice;
        if (c >= a.outs) continue;
        float z[G][2 * PAIRS];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float *bias = g ? a.bias1 : a.bias0;
            const float b = bias ? __ldg(bias + c) : 0.0f;
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                unpack2(acc[g][k], z[g][2 * k], z[g][2 * k + 1]);
                z[g][2 * k] += b; z[g][2 * k + 1] += b;
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int64_t t = (int64_t)tile * (V * P) + p * V + k;
            if (t >= a.tokens) break;
            float y = activate(z[0][k], a.act, a.clip);
            if (G == 2) y *= z[G - 1][k];
            store_from_float(a.y, a.y_type, t * a.y_stride + c, y);
            if (a.z0) a.z0[t * a.z_stride + c] = z[0][k];
            if (G == 2 && a.z1) a.z1[t * a.z_stride + c] = z[G - 1][k];
        }
    }
}

// ---- gradients of the weights ----------------------------------------------------------------------

struct DwArgs {
    const void *x;            // [inputs][token_stride]
    const float *d;           // [outputs][sets][token_stride]
    const int32_t *rows;      // [outputs][slots] canonical, -1 = none
    int64_t token_stride;
    int outputs, slots, chunks;   // chunks of kDwSlots connections per output
    float *dw0, *dw1;         // [outputs][slots]
    float *db0, *db1;         // or nullptr
};

constexpr int kDwSlots = 16;
constexpr int kDwThreads = 128;

// A warp owns kDwSlots connections of one output: every lane sums its tokens' products in registers, the lanes are joined at the
// end.  Adjacent warps take adjacent outputs, whose inputs are often the same rows (blocks of a butterfly).
template <class E, int G>
__global__ void __launch_bounds__(kDwThreads) dw_kernel(const DwArgs a) {
    constexpr int V = 16 / sizeof(E);
    constexpr int PAIRS = V / 2;
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (kDwThreads / 32) + (threadIdx.x >> 5);
    const int c = (int)(unit % a.outputs), chunk = (int)(unit / a.outputs);
    if (chunk >= a.chunks) return;
    const int j0 = chunk * kDwSlots, slots = min(kDwSlots, a.slots - j0);
    const int32_t *rows = a.rows + (int64_t)c * a.slots + j0;
    const int mine = lane < slots ? __ldg(rows + lane) : -1;
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
        const int64_t t = t0 + lane * V;
        const bool inside = t < a.token_stride;
        f32x2 dv[G][PAIRS];
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int i = 0; i < PAIRS; i += 2) {
                Values<float, 4> part;
                part.zero();
                if (inside) part.load(d + g * a.token_stride + t + 2 * i);
                dv[g][i] = part.v[0]; dv[g][i + 1] = part.v[1];
            }
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) bias[g] = fma2(dv[g][i], ones, bias[g]);
        }
#pragma unroll
        for (int j = 0; j < kDwSlots; ++j) {
            const int row = __shfl_sync(0xffffffffu, mine, j);
            if (row >= 0) {
                Values<E, V> xv;
                xv.zero();
                if (inside) xv.load(x + (int64_t)row * a.token_stride + t);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < PAIRS; ++i) acc[j][g] = fma2(xv.v[i], dv[g][i], acc[j][g]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float *out = (g ? a.dw1 : a.dw0) + (int64_t)c * a.slots + j0;
        float keep = 0.0f;
#pragma unroll
        for (int j = 0; j < kDwSlots; ++j) {
            float lo, hi;
            unpack2(acc[j][g], lo, hi);
            float v = lo + hi;
#pragma unroll
            for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
            if (lane == j) keep = v;
        }
        if (lane < slots) out[lane] = keep;
        float *db = g ? a.db1 : a.db0;
        if (chunk == 0 && db) {
            float lo, hi;
            unpack2(bias[g], lo, hi);
            float v = lo + hi;
#pragma unroll
            for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
            if (lane == 0) db[c] = v;
        }
    }
}

}  // namespace ffn
}  // namespace spdnn_impl
