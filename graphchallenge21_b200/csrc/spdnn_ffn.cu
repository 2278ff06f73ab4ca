// C ABI of the feed-forward operators: topologies, sparse layers on row-major activations (plain and gated, forward and
// backward) and microscaled 4-bit matrices.  Kernels: spdnn_ffn.cuh, spdnn_mx4.cuh; host analysis: topology.h; its tables on the GPU:
// topology_device.h.
//
// A topology is immutable once created, and every call works on buffers of its caller (operands and workspace) on the caller's
// stream, so calls on one topology may overlap, from several threads too.
#include "../../include/spdnn_b200.h"

#include <array>
#include <cmath>
#include <cstdio>
#include <map>
#include <mutex>
#include <new>
#include <string>
#include <tuple>

#include "spdnn_ffn.cuh"
#include "spdnn_mx4.cuh"
#include "topology_device.h"

using namespace spdnn_impl;
using namespace spdnn_impl::ffn;

static_assert((int)SPDNN_F32 == F32 && (int)SPDNN_F16 == F16 && (int)SPDNN_BF16 == BF16 && (int)SPDNN_MX4 == MX4, "types of the header");
static_assert((int)SPDNN_ACT_NONE == NONE && (int)SPDNN_ACT_RELU == RELU && (int)SPDNN_ACT_CLIP == CLIP && (int)SPDNN_ACT_SILU == SILU &&
                  (int)SPDNN_ACT_GELU == GELU && (int)SPDNN_ACT_GELU_TANH == GELU_TANH, "activations of the header");

namespace {

// How a gather runs: the image's unit (v tokens) and units per neuron (p), and how many blocks share a tile.
struct GatherPlan {
    int v = 1, p = 1, splits = 1;
    int64_t tiles = 0, image_bytes = 0;
    bool global = false;
    bool blocks = false;            // by blocks, on the tensor cores: 64 tokens per tile
};

}  // namespace

struct spdnn_topology : DeviceTopology {
    Topology host;
    int device = -1;                // -1: analysis only
    int sm_count = 0;
    int block_count[2] = {0, 0};    // forward, backward
    // plans made so far: functions of the topology and the key, kept because a call may come every few microseconds
    mutable std::mutex plans_lock;
    mutable std::map<std::array<int, 5>, GatherPlan> plans;
};

namespace {

int fail(char *err, int err_len, int code, const char *msg) {
    if (err && err_len > 0) snprintf(err, (size_t)err_len, "%s", msg);
    return code;
}
int fail(char *err, int err_len, int code, const std::string &msg) { return fail(err, err_len, code, msg.c_str()); }

// No exception leaves a C entry point.
template <class F>
int guarded(char *err, int err_len, const F &f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return fail(err, err_len, SPDNN_ERR_MEMORY, "host allocation failed");
    } catch (const std::exception &e) {
        return fail(err, err_len, SPDNN_ERR_MEMORY, e.what());
    }
}

// A failed runtime call: its message, and nothing left for the next caller of cudaGetLastError to find.
int fail_cuda(char *err, int err_len, cudaError_t e) {
    cudaGetLastError();
    return fail(err, err_len, e == cudaErrorMemoryAllocation ? SPDNN_ERR_MEMORY : SPDNN_ERR_CUDA, cudaGetErrorString(e));
}

// A launch whose status is its own (cudaGetLastError would also return what an earlier call of someone else left behind).
template <class... P, class... A>
cudaError_t launch(void (*kernel)(P...), unsigned grid, unsigned block, cudaStream_t stream, const A &...args) {
    std::tuple<P...> values(args...);
    return std::apply([&](P &...v) {
        void *ptrs[] = {(void *)&v...};
        return cudaLaunchKernel((const void *)kernel, dim3(grid), dim3(block), ptrs, 0, stream);
    }, values);
}

constexpr int64_t kSharedLimit = 227 * 1024;

// Lets a kernel have more shared memory than a launch has by default: always as much as there is, never the size of this launch, since another
// thread may be about to launch the same kernel with more.
cudaError_t allow_shared(const void *kernel, size_t shared) {
    return shared > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedLimit) : cudaSuccess;
}

// The device of the topology for the length of a call.
struct OnDevice {
    int before = -1;
    cudaError_t status;
    explicit OnDevice(int device) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device) status = cudaSetDevice(device);
        if (before == device) before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

int type_size(int type) { return type == F32 ? 4 : 2; }
bool is_float(int type) { return type == F32 || type == F16 || type == BF16; }
int64_t aligned(int64_t n) { return (n + 255) & ~255ll; }


int64_t image_size(int rows, int sets, int v, int p, int size) {
    return ((int64_t)image_units(rows, p * sets) * v * size + 127) / 128 * 128;
}

// How many neurons are read at a time by the gather that many tokens of `rows` neurons get (plan_gather), for the order of connections: the
// image's bytes per neuron, and with them the lanes per neuron, do not depend on the type.  Fewer tokens may read more at a time.
int neurons_at_a_time(int rows, int sets) {
    int p = 8;
    while (p > 1 && image_size(rows, sets, 8, p, 2) > kSharedLimit) p /= 2;
    if (image_size(rows, sets, 8, p, 2) > kSharedLimit) return 16;
    return 8 / (p / lane_units(p));
}

// Blocks take 16-bit operands of one type and whole tiles of 64 tokens.  From 17 tokens on they are no more than a microsecond or four slower
// than the gather by connections (1024 neurons, 256 tokens, forward / backward 9.1 / 21.5 and 8.1 / 17.5 us), and soon faster
// (4096 neurons, 256 tokens 9.8 / 27.9 and 11.6 / 36.4).
bool go_by_blocks(const DeviceBlocks &b, int tokens, int image_type, int weight_type) {
    return b.blocks && tokens >= 17 && image_type != F32 && image_type == weight_type;
}

GatherPlan make_plan(const spdnn_topology &top, bool forward, int tokens, int sets, int image_type, int weight_type) {
    const DeviceTable &t = forward ? top.forward : top.backward;
    GatherPlan g;
    const int size = type_size(image_type), full = 16 / size;
    if (go_by_blocks(forward ? top.forward_blocks : top.backward_blocks, tokens, image_type, weight_type)) {
        g.blocks = true;
        g.v = 8; g.p = 8;
        g.image_bytes = image_size(t.rows, forward ? 1 : sets, 8, 8, 2);
        g.tiles = ((int64_t)tokens + 63) / 64;
        return g;
    }
    const int slices = (t.outs + 31) / 32;
    const double quads = std::max(1.0, (double)t.entries / 128.0 / slices);       // of a slice
    const int s_values = forward ? 1 : sets, sums = forward ? sets : 1;
    double best = 0.0;
    const auto consider = [&](int T, bool global) {
        const int v = std::min(T, full), p = T / v, nv = lane_units(p), lanes = p / nv;
        const int64_t bytes = image_size(t.rows, s_values, v, p, size), tiles = ((int64_t)tokens + T - 1) / T, units = (int64_t)slices * lanes;
        const int warps = gather_threads(v * nv * sums) / 32;
        // Clocks, fitted to a sweep of T and splits over 15 sizes (33 to 4096 tokens, 300 to 16384 neurons; the choice is 0.4 % off the best of the
        // sweep in the mean).  A connection of a warp takes the shared memory's wavefronts (1.3 per 128 bytes in the order of topology.h,
        // more where more neurons are read at a time than it was made for) with those of the table, or its instructions on four
        // schedulers; a quad that a warp works on alone, the latency of its loads and instructions.
        const int at_a_time = v * size < 16 ? 16 : 8 / lanes;
        const double conflicts = 1.3 + 0.35 * std::max(0.0, std::log2((double)at_a_time / neurons_at_a_time(t.rows, s_values)));
        const double wavefronts = nv * s_values * v * size * 32 / 128.0 * conflicts + (2 + sets * type_size(weight_type)) / 4.0;
        const double issue = (nv * s_values * (v * sums + 1.5) + 6 + sets) / 4.0;
        const double busy = 4.0 * std::max(wavefronts, issue) * 1.25, alone = 600.0 + 6.0 * (nv * s_values * (v * sums + 4) + 6);
        int64_t tried = 0;
        for (int64_t w = 0; w <= 24; ++w) {
            // splits that fill w waves, and a few between
            const int64_t n = std::max<int64_t>(1, std::min<int64_t>(w * top.sm_count / tiles, (units + 3) / 4));
            if (n == tried) continue;
            tried = n;
            const int64_t waves = (tiles * n + top.sm_count - 1) / top.sm_count, here = (units + n - 1) / n;
            const double work = std::max((double)((here + warps - 1) / warps) * quads * alone, here * quads * busy);
            const double cost = waves * (1500.0 + (global ? 0.0 : bytes / 45.0) + work * (global ? 3.0 : 1.0));
            if (best == 0.0 || cost < best) {
                best = cost;
                g.v = v; g.p = p; g.image_bytes = bytes; g.tiles = tiles; g.splits = (int)n; g.global = global;
            }
        }
    };
    for (int T = full * 8; T >= 1; T /= 2)
        if ((T == 1 || T / 2 < tokens) && t.rows < 65536 && image_size(t.rows, s_values, std::min(T, full), std::max(T / full, 1), size) <= kSharedLimit)
            consider(T, false);
    if (best == 0.0) consider(tokens > full ? full * 8 : full, true);     // nothing fits: the image stays in global memory
    return g;
}

GatherPlan plan_gather(const spdnn_topology &top, bool forward, int tokens, int sets, int image_type, int weight_type) {
    const std::array<int, 5> key{forward, tokens, sets, image_type, weight_type};
    std::lock_guard<std::mutex> lock(top.plans_lock);
    const auto found = top.plans.find(key);
    if (found != top.plans.end()) return found->second;
    const GatherPlan g = make_plan(top, forward, tokens, sets, image_type, weight_type);
    if (top.plans.size() >= 4096) top.plans.clear();
    top.plans.emplace(key, g);
    return g;
}

template <class E, class W, int S, int G>
const void *gather_variant(const GatherPlan &g) {
    constexpr int F = 16 / (int)sizeof(E);
    if (g.global) return g.p == 8 ? (const void *)gather_kernel<E, W, F, 8, S, G, true> : (const void *)gather_kernel<E, W, F, 1, S, G, true>;
    if (g.v == F) {
        switch (g.p) {
            case 8: return (const void *)gather_kernel<E, W, F, 8, S, G, false>;
            case 4: return (const void *)gather_kernel<E, W, F, 4, S, G, false>;
            case 2: return (const void *)gather_kernel<E, W, F, 2, S, G, false>;
            default: return (const void *)gather_kernel<E, W, F, 1, S, G, false>;
        }
    }
    if constexpr (F == 8) {
        if (g.v == 4) return (const void *)gather_kernel<E, W, 4, 1, S, G, false>;
    }
    return g.v == 2 ? (const void *)gather_kernel<E, W, 2, 1, S, G, false> : (const void *)gather_kernel<E, W, 1, 1, S, G, false>;
}

template <class E, class W>
const void *gather_variant(const GatherPlan &g, int s, int sets) {
    if (s == 2) return gather_variant<E, W, 2, 1>(g);
    return sets == 2 ? gather_variant<E, W, 1, 2>(g) : gather_variant<E, W, 1, 1>(g);
}

// image_type: E; weight_type: W.  s: values gathered per connection, sets: sums per neuron.
cudaError_t launch_gather(const GatherPlan &g, GatherArgs a, int image_type, int weight_type, int s, int sets, cudaStream_t stream) {
    const void *kernel = image_type == F32 ? gather_variant<float, float>(g, s, sets)
                         : image_type == BF16 ? gather_variant<bf16, bf16>(g, s, sets)
                         : weight_type == F16 ? gather_variant<__half, __half>(g, s, sets)
                                              : gather_variant<__half, bf16>(g, s, sets);
    a.splits = g.splits;
    a.image_bytes = g.image_bytes;
    const size_t shared = g.global ? 0 : (size_t)g.image_bytes;
    if (const cudaError_t e = allow_shared(kernel, shared)) return e;
    void *args[] = {&a};
    const int threads = gather_threads(g.v * lane_units(g.p) * (s == 2 ? 1 : sets));
    return cudaLaunchKernel(kernel, dim3((unsigned)(g.tiles * g.splits)), dim3(threads), args, shared, stream);
}

// The same gather by blocks; of `a` what is not the gather table's.
cudaError_t launch_blocks(const spdnn_topology &top, const GatherPlan &g, const DeviceBlocks &b, const GatherArgs &a, int image_type, int s, int sets,
                          cudaStream_t stream) {
    BlockArgs k{};
    k.image = a.image; k.image_bytes = g.image_bytes; k.chunk_ptr = b.chunk_ptr; k.rows = b.rows; k.members = b.members; k.weights = a.weights;
    k.chunks = b.chunks; k.blocks = b.blocks; k.tokens = a.tokens; k.bias0 = a.bias0; k.bias1 = a.bias1;
    k.y = a.y; k.z0 = a.z0; k.z1 = a.z1; k.y_stride = a.y_stride; k.z_stride = a.z_stride; k.y_type = a.y_type; k.act = a.act; k.clip = a.clip; k.scale = a.scale;
    k.whole_y = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_stride * type_size(a.y_type) % 16 == 0;
    k.whole_z = (reinterpret_cast<uintptr_t>(a.z0) | reinterpret_cast<uintptr_t>(a.z1)) % 16 == 0 && a.z_stride % 4 == 0;
    const auto of = [&](auto e) {
        using E = decltype(e);
        return s == 2 ? block_kernel<E, 2, 1> : sets == 2 ? block_kernel<E, 1, 2> : block_kernel<E, 1, 1>;
    };
    const auto kernel = image_type == BF16 ? of(bf16()) : of(__half());
    const int shared = kBlockWarps * kBlockStages * block_stage_bytes(s == 2 ? 1 : sets);
    if (const cudaError_t e = allow_shared((const void *)kernel, (size_t)shared)) return e;
    const int64_t want = ((int64_t)b.blocks * g.tiles + kBlockWarps - 1) / kBlockWarps;
    void *args[] = {&k};
    return cudaLaunchKernel((const void *)kernel, dim3((unsigned)std::min<int64_t>(want, top.sm_count)), dim3(kBlockWarps * 32), args, (size_t)shared, stream);
}

unsigned pack_blocks(const PackArgs &a) { return (unsigned)((int64_t)((a.rows + 63) / 64) * ((a.tokens + 63) / 64)); }

// What a call's gather (and dw_kernel) read.  gradient: the backward call, whose gathered values are dL/dz.
cudaError_t launch_prepare(const PrepareArgs &args, int x_blocks, int sets, bool gradient, int image_type, int weight_type, cudaStream_t stream) {
    const int64_t grid = (int64_t)args.order_blocks + args.main_blocks + x_blocks;
    if (!grid) return cudaSuccess;
    const auto run = [&](auto e, auto w) {
        using E = decltype(e);
        using W = decltype(w);
        if (gradient) {
            if constexpr (std::is_same<E, W>::value)
                return sets == 2 ? launch(prepare_kernel<E, W, 2, true>, (unsigned)grid, kPackThreads, stream, args)
                                 : launch(prepare_kernel<E, W, 1, true>, (unsigned)grid, kPackThreads, stream, args);
            return cudaErrorInvalidValue;
        }
        return sets == 2 ? launch(prepare_kernel<E, W, 2, false>, (unsigned)grid, kPackThreads, stream, args)
                         : launch(prepare_kernel<E, W, 1, false>, (unsigned)grid, kPackThreads, stream, args);
    };
    if (image_type == F32) return run(float(), float());
    if (image_type == BF16) return run(bf16(), bf16());
    return weight_type == F16 ? run(__half(), __half()) : run(__half(), bf16());
}

// The part of it that orders a table.
void order_part(PrepareArgs &args, const GatherPlan &g, const Matrix &w0, const Matrix &w1, const DeviceTable &t, const DeviceBlocks &b, int slots,
                int values, int image_type, void *weights, void *index) {
    if (g.blocks) {
        args.by_blocks = 1;
        args.blocks = OrderBlocksArgs{w0, w1, b.src, b.chunks, slots, weights};
        args.order_blocks = (unsigned)((b.chunks * 64 + kPackThreads - 1) / kPackThreads);
        return;
    }
    OrderArgs &a = args.order;
    a.w0 = w0; a.w1 = w1; a.idx = t.idx; a.src = t.src; a.entries = t.entries; a.slots = slots; a.values = values; a.p = g.p;
    a.whole = g.v * type_size(image_type) == 16; a.wide = g.global;
    a.weights = weights; a.index = index;
    args.order_blocks = (unsigned)((t.entries / 4 + kPackThreads - 1) / kPackThreads);
}

// The type activations have in an image, and weights in a gather table's order.  Microscaled values are exact in bf16 (two bits of
// magnitude, the exponents of float32), not in fp16.
int image_type(int x_type) { return x_type == MX4 ? BF16 : x_type; }
int ordered_type(int x_type, int w_type) { return x_type == F32 ? F32 : w_type == MX4 ? BF16 : w_type; }

const char *check_types(int x_type, int w_type, bool backward) {
    if (!is_float(x_type) && x_type != MX4) return "unknown type of the activations";
    if (!is_float(w_type) && w_type != MX4) return "unknown type of the weights";
    if (backward && (x_type == MX4 || w_type == MX4)) return "microscaled operands have no backward pass";
    if (w_type != MX4 && w_type != (x_type == MX4 ? BF16 : x_type))
        return "the weights must be microscaled or have the activations' type (bf16 for microscaled activations)";
    return nullptr;
}

struct Workspace {
    int64_t weights = 0, index = 0, image = 0, x_columns = 0, d_columns = 0, scale = 0, total = 0;
};

// Layout of a call's workspace.  The plan is a function of the topology, the device and the arguments.
Workspace layout(const spdnn_topology &top, const GatherPlan &g, const DeviceTable &t, int tokens, int sets, int image, int weight, bool backward) {
    Workspace w;
    int64_t at = 0;
    const DeviceBlocks &b = backward ? top.backward_blocks : top.forward_blocks;
    w.weights = at; at += aligned((g.blocks ? b.chunks * 512 : t.entries) * sets * type_size(weight));
    w.index = at; at += g.blocks ? 0 : aligned(t.entries * (g.global ? 4 : 2));
    w.image = at; at += aligned(g.tiles * g.image_bytes);
    if (backward) {
        const int64_t stride = (tokens + 63) / 64 * 64;
        w.x_columns = at; at += aligned(stride * top.host.inputs * type_size(image) + 16);
        w.d_columns = at; at += aligned(stride * top.host.outputs * sets * 4);
        w.scale = at; at += image == F16 ? aligned(stride * 4) : 0;
    }
    w.total = std::max<int64_t>(at, 256);
    return w;
}

struct Call {            // what linear and gated share
    const spdnn_topology *top;
    int tokens, sets, act;
    float clip;
    const spdnn_operand_t *x, *w[2], *y, *z[2];
    void *workspace;
    int64_t workspace_bytes;
    cudaStream_t stream;
    char *err;
    int err_len;
};

Matrix matrix(const spdnn_operand_t *o) {
    Matrix m{nullptr, nullptr, 0, F32};
    if (o) { m.data = o->data; m.scales = o->scales; m.stride = o->stride; m.type = o->type; }
    return m;
}

// Whether every row begins on 16 bytes (microscaled rows always do as far as the kernels load them).
bool on_16_bytes(const spdnn_operand_t *o) {
    return !o || o->type == MX4 || (reinterpret_cast<uintptr_t>(o->data) % 16 == 0 && o->stride * type_size(o->type) % 16 == 0);
}

// nullptr, or what is wrong with an operand of `rows` x `cols` values
const char *check_operand(const spdnn_operand_t *o, int64_t rows, int64_t cols, bool may_be_mx4) {
    if (!o) return "a required operand is null";
    if (!is_float(o->type) && !(may_be_mx4 && o->type == MX4)) return "an operand has a type that it cannot have";
    if (rows == 0) return nullptr;
    if (!o->data) return "an operand has no data";
    if (o->type == MX4 && !o->scales) return "a microscaled operand has no scales";
    const int64_t least = o->type == MX4 ? (cols + 31) / 32 : cols;
    if (o->stride < least) return "an operand's stride is less than its row";
    if (o->stride > (1ll << 40)) return "an operand's stride is out of range";
    if (reinterpret_cast<uintptr_t>(o->data) % (o->type == MX4 ? 4 : type_size(o->type))) return "an operand is not aligned to its type (codes: 4 bytes)";
    return nullptr;
}

bool off_4_bytes(const void *p) { return reinterpret_cast<uintptr_t>(p) % 4 != 0; }

int check_call(const Call &c, bool backward) {
    if (!c.top) return fail(c.err, c.err_len, SPDNN_ERR_ARG, "null topology");
    if (c.tokens < 0 || c.tokens > SPDNN_MAX_TOKENS) return fail(c.err, c.err_len, SPDNN_ERR_ARG, "tokens must be in [0, 2^26]");
    if (c.act < SPDNN_ACT_NONE || c.act > SPDNN_ACT_GELU_TANH) return fail(c.err, c.err_len, SPDNN_ERR_ARG, "unknown activation");
    if (c.act == SPDNN_ACT_CLIP && !(c.clip > 0.0f)) return fail(c.err, c.err_len, SPDNN_ERR_ARG, "clip must be positive");
    const Topology &h = c.top->host;
    const char *bad = check_operand(c.x, c.tokens, h.inputs, !backward);
    for (int s = 0; s < c.sets && !bad; ++s) bad = check_operand(c.w[s], h.outputs, h.slots, !backward);
    if (!bad && c.sets == 2 && c.w[0]->type != c.w[1]->type) bad = "both sets of weights must have one type";
    if (!bad) bad = check_types(c.x->type, c.w[0]->type, backward);
    if (bad) return fail(c.err, c.err_len, SPDNN_ERR_ARG, bad);
    return SPDNN_OK;
}

constexpr const char *kAnalysisOnly = "the topology was created for analysis only (device -1)";

int check_run(const Call &c, int64_t need) {
    if (!c.workspace || c.workspace_bytes < need)
        return fail(c.err, c.err_len, SPDNN_ERR_ARG, "the workspace is smaller than spdnn_layer_workspace asks for: " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(c.workspace) % 256) return fail(c.err, c.err_len, SPDNN_ERR_ARG, "the workspace must be aligned to 256 bytes");
    return SPDNN_OK;
}

int check_blocks(const Call &c, const GatherPlan &g) {
    const int64_t pack = (int64_t)((std::max(c.top->host.inputs, c.top->host.outputs) + 63) / 64) * ((c.tokens + 63) / 64);
    if (pack > 0x3fffffffll || g.tiles * g.splits > 0x7fffffffll)
        return fail(c.err, c.err_len, SPDNN_ERR_LIMIT, "tokens times neurons is too large for one call: split the tokens");
    return SPDNN_OK;
}

// Tokens that one launch of few_kernel takes at a time, or 0: the images' way.  Up to about 2^21 multiply-adds a set its one launch takes no
// longer than their two (us on the GPU, few_kernel and images: 4096 -> 16384, 32 connections, 4 tokens 7 and 11, 8 tokens 11 and 11;
// 4096 -> 4096, 17 tokens 14 and 8), in at most four groups of tokens.
int few_tokens(const spdnn_topology &top, int tokens, int x_type) {
    const int64_t row = (int64_t)(top.host.inputs + 1) * type_size(image_type(x_type));
    if (tokens * (int64_t)top.host.outputs * top.host.slots > 1ll << 21 && tokens > 1) return 0;
    int T = tokens <= 1 ? 1 : tokens <= 2 ? 2 : tokens <= 4 ? 4 : 8;
    if (x_type == F32) T = std::min(T, 4);
    while (T > 1 && row * T > kSharedLimit / 2) T /= 2;
    return row * T <= kSharedLimit && (tokens + T - 1) / T <= 4 ? T : 0;
}

template <class E, class W, bool MX, int G>
const void *few_variant(int T) {
    switch (T) {
        case 1: return (const void *)few_kernel<E, W, MX, 1, G>;
        case 2: return (const void *)few_kernel<E, W, MX, 2, G>;
        case 4: return (const void *)few_kernel<E, W, MX, 4, G>;
        default:
            if constexpr (sizeof(E) == 2) return (const void *)few_kernel<E, W, MX, 8, G>;
            else return nullptr;
    }
}

cudaError_t launch_few(const Call &c, int T, const float *b0, const float *b1) {
    const Topology &h = c.top->host;
    FewArgs a{};
    a.x = matrix(c.x); a.w0 = matrix(c.w[0]); a.w1 = matrix(c.w[1]);
    a.rows = c.top->few_rows; a.row_stride = few_stride(h.slots); a.slots = h.slots; a.inputs = h.inputs; a.outputs = h.outputs; a.tokens = c.tokens;
    a.bias0 = b0; a.bias1 = b1;
    a.y = const_cast<void *>(c.y->data); a.y_stride = c.y->stride; a.y_type = c.y->type; a.act = c.act; a.clip = c.clip;
    if (c.z[0]) { a.z0 = (float *)const_cast<void *>(c.z[0]->data); a.z_stride = c.z[0]->stride; }
    if (c.z[1]) a.z1 = (float *)const_cast<void *>(c.z[1]->data);
    a.vector_x = on_16_bytes(c.x);
    a.vector_w = 1;
    for (int s = 0; s < c.sets; ++s)
        a.vector_w &= reinterpret_cast<uintptr_t>(c.w[s]->data) % (4 * type_size(c.w[s]->type)) == 0 && c.w[s]->stride % 4 == 0;
    const int it = image_type(c.x->type), w = c.w[0]->type;
    const auto of = [&](auto e) {
        using E = decltype(e);
        if (w == MX4) return c.sets == 2 ? few_variant<E, bf16, true, 2>(T) : few_variant<E, bf16, true, 1>(T);
        return c.sets == 2 ? few_variant<E, E, false, 2>(T) : few_variant<E, E, false, 1>(T);
    };
    const void *kernel = it == F32 ? of(float()) : it == F16 ? of(__half()) : of(bf16());
    const size_t shared = (size_t)(h.inputs + 1) * T * type_size(it);
    if (const cudaError_t e = allow_shared(kernel, shared)) return e;
    const int64_t want = (h.outputs + kFewThreads / 8 - 1) / (kFewThreads / 8);
    const int per_sm = shared > (size_t)kSharedLimit / 4 ? 1 : 4;
    void *args[] = {&a};
    return cudaLaunchKernel(kernel, dim3((unsigned)std::min<int64_t>(want, (int64_t)per_sm * c.top->sm_count), (unsigned)((c.tokens + T - 1) / T)),
                            dim3(kFewThreads), args, shared, c.stream);
}

int run_forward(const Call &c, const float *b0, const float *b1) {
    int rc = check_call(c, false);
    if (rc) return rc;
    const Topology &h = c.top->host;
    const char *bad = check_operand(c.y, c.tokens, h.outputs, false);
    for (int s = 0; s < c.sets && !bad; ++s)
        if (c.z[s]) {
            bad = check_operand(c.z[s], c.tokens, h.outputs, false);
            if (!bad && c.z[s]->type != F32) bad = "pre-activations are saved as fp32";
        }
    if (!bad && c.sets == 2 && !c.z[0] != !c.z[1]) bad = "save both pre-activations or none";
    if (!bad && c.sets == 2 && c.z[0] && c.z[0]->stride != c.z[1]->stride) bad = "both pre-activations must have one stride";
    if (!bad && (off_4_bytes(b0) || off_4_bytes(b1))) bad = "a bias is not aligned to 4 bytes";
    if (bad) return fail(c.err, c.err_len, SPDNN_ERR_ARG, bad);
    if (c.top->device < 0) return fail(c.err, c.err_len, SPDNN_ERR_STATE, kAnalysisOnly);
    if (c.tokens == 0) return SPDNN_OK;
    if (const int T = few_tokens(*c.top, c.tokens, c.x->type)) {
        OnDevice guard(c.top->device);
        const cudaError_t e = guard.status == cudaSuccess ? launch_few(c, T, b0, b1) : guard.status;
        return e == cudaSuccess ? SPDNN_OK : fail_cuda(c.err, c.err_len, e);
    }
    const DeviceTable &t = c.top->forward;
    const int it = image_type(c.x->type), wt = ordered_type(c.x->type, c.w[0]->type);
    const GatherPlan g = plan_gather(*c.top, true, c.tokens, c.sets, it, wt);
    const Workspace ws = layout(*c.top, g, t, c.tokens, c.sets, it, wt, false);
    if ((rc = check_run(c, ws.total)) || (rc = check_blocks(c, g))) return rc;
    OnDevice guard(c.top->device);
    if (guard.status != cudaSuccess) return fail_cuda(c.err, c.err_len, guard.status);
    char *base = (char *)c.workspace;
    PrepareArgs prep{};
    order_part(prep, g, matrix(c.w[0]), matrix(c.w[1]), t, c.top->forward_blocks, h.slots, 1, it, base + ws.weights, base + ws.index);
    PackArgs &p = prep.main;
    p.x = matrix(c.x); p.image = base + ws.image; p.image_bytes = g.image_bytes;
    p.rows = h.inputs; p.tokens = c.tokens; p.v = g.v; p.p = g.p; p.vector = on_16_bytes(c.x); p.same = p.vector && c.x->type == it;
    prep.main_blocks = pack_blocks(p);
    cudaError_t e = launch_prepare(prep, 0, c.sets, false, it, wt, c.stream);
    if (e == cudaSuccess) {
        GatherArgs a{};
        a.image = base + ws.image; a.slice_ptr = t.slice_ptr; a.index = base + ws.index;
        a.weights = base + ws.weights; a.outs = t.outs; a.tokens = c.tokens;
        a.bias0 = b0; a.bias1 = b1; a.act = c.act; a.clip = c.clip;
        a.y = const_cast<void *>(c.y->data); a.y_stride = c.y->stride; a.y_type = c.y->type;
        if (c.z[0]) { a.z0 = (float *)const_cast<void *>(c.z[0]->data); a.z_stride = c.z[0]->stride; }
        if (c.z[1]) a.z1 = (float *)const_cast<void *>(c.z[1]->data);
        e = g.blocks ? launch_blocks(*c.top, g, c.top->forward_blocks, a, it, 1, c.sets, c.stream) : launch_gather(g, a, it, wt, 1, c.sets, c.stream);
    }
    if (e != cudaSuccess) return fail_cuda(c.err, c.err_len, e);
    return SPDNN_OK;
}

// Whether dL/dz of fp16 operands may leave fp16's range or be rounded: not where it is dy or zero.
bool needs_scale(const Call &c) { return c.x->type == F16 && (c.sets == 2 || (c.act != NONE && c.act != RELU && c.act != CLIP)); }

struct Gradients {
    const spdnn_operand_t *dy, *dx;
    float *dw[2], *db[2];
};

cudaError_t launch_dw(const Call &c, const Gradients &d, int type, const void *x_columns, const float *d_columns, int64_t stride) {
    const Topology &h = c.top->host;
    DwArgs a{};
    a.x = x_columns; a.d = d_columns; a.rows = c.top->rows; a.token_stride = stride;
    a.inputs = h.inputs; a.outputs = h.outputs; a.slots = h.slots; a.chunks = (h.slots + kDwSlots - 1) / kDwSlots;
    a.dw0 = d.dw[0]; a.dw1 = d.dw[1]; a.db0 = d.db[0]; a.db1 = d.db[1];
    const int per_block = kDwThreads / 32;
    const unsigned grid = (unsigned)(((int64_t)a.outputs * a.chunks + per_block - 1) / per_block);
    const auto run = [&](auto v) {
        using E = decltype(v);
        return c.sets == 2 ? launch(dw_kernel<E, 2>, grid, kDwThreads, c.stream, a) : launch(dw_kernel<E, 1>, grid, kDwThreads, c.stream, a);
    };
    return type == F32 ? run(float()) : type == F16 ? run(__half()) : run(bf16());
}

cudaError_t launch_dw_blocks(const Call &c, const Gradients &d, const DeviceBlocks &b, int type, const void *x_columns, const float *d_columns, int64_t stride) {
    const Topology &h = c.top->host;
    cudaError_t e = cudaSuccess;
    // the kernel writes the connections there are
    if (h.connections < (int64_t)h.outputs * h.slots)
        for (int s = 0; s < c.sets && e == cudaSuccess; ++s) e = cudaMemsetAsync(d.dw[s], 0, sizeof(float) * (size_t)h.outputs * h.slots, c.stream);
    if (e != cudaSuccess) return e;
    DwBlockArgs a{};
    a.x = x_columns; a.d = d_columns; a.chunk_ptr = b.chunk_ptr; a.rows = b.rows; a.src = b.src; a.members = b.members; a.chunk_block = b.chunk_block;
    a.token_stride = stride; a.inputs = h.inputs; a.dw0 = d.dw[0]; a.dw1 = d.dw[1]; a.db0 = d.db[0]; a.db1 = d.db[1];
    const auto run = [&](auto v) {
        using E = decltype(v);
        return c.sets == 2 ? launch(dw_block_kernel<E, 2>, (unsigned)b.chunks, kDwBlockThreads, c.stream, a)
                           : launch(dw_block_kernel<E, 1>, (unsigned)b.chunks, kDwBlockThreads, c.stream, a);
    };
    return type == F16 ? run(__half()) : run(bf16());
}

int run_backward(const Call &c, const Gradients &d) {
    int rc = check_call(c, true);
    if (rc) return rc;
    const Topology &h = c.top->host;
    const int type = c.x->type;
    const char *bad = check_operand(d.dy, c.tokens, h.outputs, false);
    if (!bad && d.dy->type != type) bad = "dy must have the activations' type";
    for (int s = 0; s < c.sets && !bad; ++s) {
        if (c.sets == 1 && c.act == NONE) break;      // the slope is 1 everywhere: nothing saved is read
        bad = check_operand(c.z[s], c.tokens, h.outputs, false);
        if (!bad && c.z[s]->type != F32) bad = "pre-activations are saved as fp32";
    }
    if (!bad && c.sets == 2 && c.z[0]->stride != c.z[1]->stride) bad = "both pre-activations must have one stride";
    if (!bad && d.dx) {
        bad = check_operand(d.dx, c.tokens, h.inputs, false);
        if (!bad && d.dx->type != type) bad = "dx must have the activations' type";
    }
    if (!bad && c.sets == 2 && !d.dw[0] != !d.dw[1]) bad = "ask for the gradients of both sets of weights or of none";
    for (int s = 0; s < 2 && !bad; ++s)
        if (off_4_bytes(d.dw[s]) || off_4_bytes(d.db[s])) bad = "a gradient is not aligned to 4 bytes";
    if (!bad && !d.dw[0] && (d.db[0] || d.db[1])) bad = "the gradients of the biases come with those of the weights";
    if (bad) return fail(c.err, c.err_len, SPDNN_ERR_ARG, bad);
    if (c.top->device < 0) return fail(c.err, c.err_len, SPDNN_ERR_STATE, kAnalysisOnly);
    const DeviceTable &t = c.top->backward;
    const GatherPlan g = plan_gather(*c.top, false, std::max(c.tokens, 1), c.sets, type, type);
    const Workspace ws = layout(*c.top, g, t, c.tokens, c.sets, type, type, true);
    if ((rc = check_run(c, ws.total)) || (rc = check_blocks(c, g))) return rc;
    OnDevice guard(c.top->device);
    cudaError_t e = guard.status;
    char *base = (char *)c.workspace;
    const int64_t stride = ((int64_t)c.tokens + 63) / 64 * 64;
    if (c.tokens > 0 && e == cudaSuccess) {
        PrepareArgs prep{};
        if (d.dx) order_part(prep, g, matrix(c.w[0]), matrix(c.w[1]), t, c.top->backward_blocks, h.slots, c.sets, type, base + ws.weights, base + ws.index);
        PackArgs &p = prep.main;
        p.x = matrix(d.dy);
        if (c.z[0]) { p.z0 = (const float *)c.z[0]->data; p.z_stride = c.z[0]->stride; }
        if (c.z[1]) p.z1 = (const float *)c.z[1]->data;
        p.vector = on_16_bytes(d.dy) && on_16_bytes(c.z[0]) && on_16_bytes(c.z[1]);
        p.rows = h.outputs; p.tokens = c.tokens; p.v = g.v; p.p = g.p; p.act = c.act; p.clip = c.clip;
        p.image = d.dx ? base + ws.image : nullptr; p.image_bytes = g.image_bytes;
        p.columns = d.dw[0] ? base + ws.d_columns : nullptr; p.token_stride = stride;
        prep.main_blocks = p.image || p.columns ? pack_blocks(p) : 0;
        if (p.image && needs_scale(c)) {
            e = launch(c.sets == 2 ? token_scale_kernel<2> : token_scale_kernel<1>, (unsigned)stride, kScaleThreads, c.stream, p, (float *)(base + ws.scale));
            p.scale = (const float *)(base + ws.scale);
        }
        PackArgs &x = prep.x;
        x.x = matrix(c.x); x.rows = h.inputs; x.tokens = c.tokens; x.v = x.p = 1; x.vector = on_16_bytes(c.x); x.same = x.vector;
        x.columns = base + ws.x_columns; x.token_stride = stride;
        if (e == cudaSuccess) e = launch_prepare(prep, d.dw[0] ? pack_blocks(x) : 0, c.sets, true, type, type, c.stream);
    }
    if (c.tokens > 0 && d.dx && e == cudaSuccess) {
        GatherArgs a{};
        a.image = base + ws.image; a.slice_ptr = t.slice_ptr; a.index = base + ws.index;
        a.weights = base + ws.weights; a.outs = t.outs; a.tokens = c.tokens;
        a.y = const_cast<void *>(d.dx->data); a.y_stride = d.dx->stride; a.y_type = type;
        if (needs_scale(c)) a.scale = (const float *)(base + ws.scale);
        e = g.blocks ? launch_blocks(*c.top, g, c.top->backward_blocks, a, type, c.sets, 1, c.stream) : launch_gather(g, a, type, type, c.sets, 1, c.stream);
    }
    if (d.dw[0] && e == cudaSuccess) {
        const DeviceBlocks &b = c.top->forward_blocks;
        const char *x_columns = base + ws.x_columns;
        const float *d_columns = (const float *)(base + ws.d_columns);
        e = go_by_blocks(b, c.tokens, type, type) ? launch_dw_blocks(c, d, b, type, x_columns, d_columns, stride)
                                                  : launch_dw(c, d, type, x_columns, d_columns, stride);
    }
    if (e != cudaSuccess) return fail_cuda(c.err, c.err_len, e);
    return SPDNN_OK;
}

}  // namespace

// ---- topologies ------------------------------------------------------------------------------------

extern "C" int spdnn_topology_create(spdnn_topology_t **out, int device, int inputs, int outputs, int slots, const int32_t *col_ptr,
                                     const int32_t *row_idx, char *err, int err_len) {
    if (!out) return fail(err, err_len, SPDNN_ERR_ARG, "null handle pointer");
    *out = nullptr;
    spdnn_topology *t = nullptr;
    try {
        t = new spdnn_topology();
        const std::string why = build_topology(inputs, outputs, slots, col_ptr, row_idx, neurons_at_a_time(std::max(inputs, 1), 1),
                                               neurons_at_a_time(std::max(outputs, 1), 2), t->host);
        if (!why.empty()) {
            delete t;
            return fail(err, err_len, SPDNN_ERR_ARG, why);
        }
        t->block_count[0] = t->host.forward_blocks.blocks;
        t->block_count[1] = t->host.backward_blocks.blocks;
        if (device < 0) {
            *out = t;
            return SPDNN_OK;
        }
        OnDevice guard(device);
        cudaError_t e = guard.status;
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&t->sm_count, cudaDevAttrMultiProcessorCount, device);
        if (e == cudaSuccess) e = upload(*t, t->host);
        if (e != cudaSuccess) {
            delete t;
            return fail_cuda(err, err_len, e);
        }
        t->device = device;
        // the tables are on the device: only the canonical rows are asked for again
        t->host.forward = GatherTable();
        t->host.backward = GatherTable();
        t->host.forward_blocks = BlockTable();
        t->host.backward_blocks = BlockTable();
        *out = t;
        return SPDNN_OK;
    } catch (const std::bad_alloc &) {
        spdnn_topology_destroy(t);
        return fail(err, err_len, SPDNN_ERR_MEMORY, "host allocation failed");
    } catch (...) {
        spdnn_topology_destroy(t);
        return fail(err, err_len, SPDNN_ERR_MEMORY, "topology analysis failed");
    }
}

extern "C" void spdnn_topology_destroy(spdnn_topology_t *top) {
    if (!top) return;
    if (top->device >= 0) {
        OnDevice guard(top->device);
        release(*top);
    }
    delete top;
}

extern "C" int spdnn_topology_info(const spdnn_topology_t *top, int *inputs, int *outputs, int *slots, int *fan_out, int64_t *connections) {
    if (!top) return SPDNN_ERR_ARG;
    if (inputs) *inputs = top->host.inputs;
    if (outputs) *outputs = top->host.outputs;
    if (slots) *slots = top->host.slots;
    if (fan_out) *fan_out = top->host.fan_out;
    if (connections) *connections = top->host.connections;
    return SPDNN_OK;
}

extern "C" int spdnn_topology_blocks(const spdnn_topology_t *top, int *forward, int *backward) {
    if (!top) return SPDNN_ERR_ARG;
    if (forward) *forward = top->block_count[0];
    if (backward) *backward = top->block_count[1];
    return SPDNN_OK;
}

extern "C" int spdnn_topology_rows(const spdnn_topology_t *top, int32_t *rows, int64_t capacity) {
    if (!top || !rows || capacity < (int64_t)top->host.rows.size()) return SPDNN_ERR_ARG;
    std::copy(top->host.rows.begin(), top->host.rows.end(), rows);
    return SPDNN_OK;
}

// ---- layers ------------------------------------------------------------------------------------------

extern "C" int spdnn_layer_workspace(const spdnn_topology_t *top, int tokens, int sets, int x_type, int w_type, int backward, int64_t *bytes) {
    if (!top || !bytes || tokens < 0 || tokens > SPDNN_MAX_TOKENS || (sets != 1 && sets != 2)) return SPDNN_ERR_ARG;
    if (check_types(x_type, w_type, backward != 0)) return SPDNN_ERR_ARG;
    if (top->device < 0) return SPDNN_ERR_STATE;
    const int it = image_type(x_type), wt = ordered_type(x_type, w_type);
    return guarded(nullptr, 0, [&] {
        if (!backward && few_tokens(*top, tokens, x_type)) {
            *bytes = 0;
            return (int)SPDNN_OK;
        }
        const DeviceTable &t = backward ? top->backward : top->forward;
        const GatherPlan g = plan_gather(*top, !backward, std::max(tokens, 1), sets, it, wt);
        *bytes = layout(*top, g, t, tokens, sets, it, wt, backward != 0).total;
        return (int)SPDNN_OK;
    });
}

extern "C" int spdnn_linear(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *x, const spdnn_operand_t *w, const float *bias,
                            int activation, float clip, const spdnn_operand_t *y, const spdnn_operand_t *z, void *workspace,
                            int64_t workspace_bytes, void *cuda_stream, char *err, int err_len) {
    const Call c{top, tokens, 1, activation, clip, x, {w, nullptr}, y, {z, nullptr}, workspace, workspace_bytes,
                 static_cast<cudaStream_t>(cuda_stream), err, err_len};
    return guarded(err, err_len, [&] { return run_forward(c, bias, nullptr); });
}

extern "C" int spdnn_gated(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *x, const spdnn_operand_t *w_gate,
                           const spdnn_operand_t *w_up, const float *bias_gate, const float *bias_up, int activation, float clip,
                           const spdnn_operand_t *y, const spdnn_operand_t *z_gate, const spdnn_operand_t *z_up, void *workspace,
                           int64_t workspace_bytes, void *cuda_stream, char *err, int err_len) {
    const Call c{top, tokens, 2, activation, clip, x, {w_gate, w_up}, y, {z_gate, z_up}, workspace, workspace_bytes,
                 static_cast<cudaStream_t>(cuda_stream), err, err_len};
    return guarded(err, err_len, [&] { return run_forward(c, bias_gate, bias_up); });
}

extern "C" int spdnn_linear_backward(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *dy, const spdnn_operand_t *x,
                                     const spdnn_operand_t *w, const spdnn_operand_t *z, int activation, float clip, const spdnn_operand_t *dx,
                                     float *dw, float *dbias, void *workspace, int64_t workspace_bytes, void *cuda_stream, char *err,
                                     int err_len) {
    const Call c{top, tokens, 1, activation, clip, x, {w, nullptr}, nullptr, {z, nullptr}, workspace, workspace_bytes,
                 static_cast<cudaStream_t>(cuda_stream), err, err_len};
    return guarded(err, err_len, [&] { return run_backward(c, Gradients{dy, dx, {dw, nullptr}, {dbias, nullptr}}); });
}

extern "C" int spdnn_gated_backward(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *dy, const spdnn_operand_t *x,
                                    const spdnn_operand_t *w_gate, const spdnn_operand_t *w_up, const spdnn_operand_t *z_gate,
                                    const spdnn_operand_t *z_up, int activation, float clip, const spdnn_operand_t *dx, float *dw_gate,
                                    float *dw_up, float *dbias_gate, float *dbias_up, void *workspace, int64_t workspace_bytes,
                                    void *cuda_stream, char *err, int err_len) {
    const Call c{top, tokens, 2, activation, clip, x, {w_gate, w_up}, nullptr, {z_gate, z_up}, workspace, workspace_bytes,
                 static_cast<cudaStream_t>(cuda_stream), err, err_len};
    return guarded(err, err_len, [&] { return run_backward(c, Gradients{dy, dx, {dw_gate, dw_up}, {dbias_gate, dbias_up}}); });
}

// ---- microscaled matrices ------------------------------------------------------------------------------

namespace {

const char *check_mx4(const void *codes, const uint8_t *scales, int64_t rows, int cols, const spdnn_operand_t *m) {
    if (rows < 0 || cols <= 0 || cols > (1 << 30) || rows > (1ll << 40) / cols) return "a microscaled matrix has rows >= 0, cols in [1, 2^30], fewer than 2^40 values";
    if (rows && (!codes || !scales)) return "null device pointer";
    if (reinterpret_cast<uintptr_t>(codes) % 4) return "codes must be aligned to 4 bytes";
    return check_operand(m, rows, cols, false);
}

unsigned mx4_grid(int64_t groups, int batch) { return (unsigned)std::min<int64_t>((groups + kMx4Threads * batch - 1) / (kMx4Threads * batch), 1 << 20); }

// Groups of a thread: several, whose loads are in flight together, where that leaves the GPU full (8191 x 4100 bf16 28.4 us with one, 24.0
// with four; 16384 x 32 fp32 2.0 and 2.9).
bool mx4_batched(int64_t groups) { return groups >= 1 << 20; }

template <class E>
cudaError_t quantize(const spdnn_operand_t *x, int64_t rows, int cols, uint8_t *codes, uint8_t *scales, cudaStream_t stream) {
    const int blocks = (cols + 31) / 32;
    const uintptr_t both = reinterpret_cast<uintptr_t>(x->data) | (uintptr_t)(x->stride * (int64_t)sizeof(E));
    const int64_t groups = rows * blocks * 4;
    const auto choose = [&](auto batch) {
        constexpr int B = decltype(batch)::value;
        return both % 16 == 0  ? mx4_quantize_kernel<E, 16, B>
               : both % 8 == 0 ? mx4_quantize_kernel<E, 8, B>
               : both % 4 == 0 ? mx4_quantize_kernel<E, 4, B>
                               : mx4_quantize_kernel<E, (int)sizeof(E), B>;
    };
    const int batch = mx4_batched(groups) ? kMx4Batch : 1;
    const auto kernel = batch == 1 ? choose(std::integral_constant<int, 1>()) : choose(std::integral_constant<int, kMx4Batch>());
    return launch(kernel, mx4_grid(groups, batch), kMx4Threads, stream, (const E *)x->data, x->stride, rows, cols, blocks, (uint32_t *)codes,
                  scales);
}

template <class E>
cudaError_t dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int cols, const spdnn_operand_t *y, cudaStream_t stream) {
    const int blocks = (cols + 31) / 32;
    const bool vector = reinterpret_cast<uintptr_t>(y->data) % (4 * sizeof(E)) == 0 && y->stride % 4 == 0;
    const int64_t groups = rows * ((cols + 3) / 4);
    const int batch = mx4_batched(groups) ? kMx4Batch : 1;
    const auto kernel = batch == 1 ? (vector ? mx4_dequantize_kernel<E, true, 1> : mx4_dequantize_kernel<E, false, 1>)
                                   : (vector ? mx4_dequantize_kernel<E, true, kMx4Batch> : mx4_dequantize_kernel<E, false, kMx4Batch>);
    return launch(kernel, mx4_grid(groups, batch), kMx4Threads, stream,
                  codes, scales, rows, cols, blocks, (E *)const_cast<void *>(y->data), y->stride);
}

}  // namespace

extern "C" int spdnn_mx4_quantize(const spdnn_operand_t *x, int64_t rows, int cols, uint8_t *codes, uint8_t *scales, void *cuda_stream,
                                  char *err, int err_len) {
    const char *bad = check_mx4(codes, scales, rows, cols, x);
    if (bad) return fail(err, err_len, SPDNN_ERR_ARG, bad);
    if (!rows) return SPDNN_OK;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = x->type == F32   ? quantize<float>(x, rows, cols, codes, scales, stream)
                          : x->type == F16 ? quantize<__half>(x, rows, cols, codes, scales, stream)
                                         : quantize<bf16>(x, rows, cols, codes, scales, stream);
    return e == cudaSuccess ? SPDNN_OK : fail_cuda(err, err_len, e);
}

extern "C" int spdnn_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int cols, const spdnn_operand_t *y,
                                    void *cuda_stream, char *err, int err_len) {
    const char *bad = check_mx4(codes, scales, rows, cols, y);
    if (bad) return fail(err, err_len, SPDNN_ERR_ARG, bad);
    if (!rows) return SPDNN_OK;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = y->type == F32   ? dequantize<float>(codes, scales, rows, cols, y, stream)
                          : y->type == F16 ? dequantize<__half>(codes, scales, rows, cols, y, stream)
                                         : dequantize<bf16>(codes, scales, rows, cols, y, stream);
    return e == cudaSuccess ? SPDNN_OK : fail_cuda(err, err_len, e);
}
