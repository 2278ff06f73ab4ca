/*
 * spdnn_b200 -- C ABI of the B200 (sm_100a) sparse-DNN inference path
 *     Y_{l+1} = min(clip, ReLU(Y_l W_l + bias)),  l = 0 .. L-1
 * with Y a batch x N activation matrix and every W_l an N x N sparse matrix
 * (Graph Challenge networks: 32 non-zeros per column, all 0.0625).
 *
 * It replaces, behind plain pointers and sizes, the GPU execution functions of the
 * reference (paths relative to the reference's project root):
 *   ftxj::test_benchmark_graph_challenge            src/microbenchmark/header.h:16-19,
 *                                                   defined src/microbenchmark/all_network.cu:207-526
 *                                                   (64-bit/streaming variant src/microbenchmark/out_memory.cu:208)
 *   ftxj::test_benchmark_multi_gpu_graph_challenge  src/microbenchmark/multi_gpu/header.h:5-14,
 *                                                   defined src/microbenchmark/multi_gpu/multi_gpu.cu:207
 * and the CUDA plumbing they use (ftxj::GpuEnv, src/gpu_lib/gpu_env.h:11-89; Safe_Call,
 * src/gpu_lib/gpu_runtime.h:6-17).  Those functions take the output of the reference's
 * inspector, which carries no sparsity pattern beyond its block assumptions, so the seam
 * here is one step earlier: the data the drivers load -- one COO/CSC matrix per layer
 * (src/utils/matrix.h:255-282) and the input images (src/network.cpp:33-54).
 *
 * Conventions: every function returns SPDNN_OK (0) or a negative status and never exits
 * the process (the reference's Safe_Call does); spdnn_last_error() gives the message.
 * Host buffers that describe LAYERS are borrowed for the duration of the call.  Host buffers that hold
 * INPUT images are copied with cudaMemcpyAsync on the context's stream: from pageable memory the
 * copy has read the buffer when the call returns, from page-locked (pinned) memory it may still be
 * reading it, so keep a pinned input buffer unchanged until the next call that waits for the stream
 * (spdnn_infer, spdnn_sync, spdnn_get_*) has returned.  All device memory belongs to
 * the context and is released by spdnn_destroy().  One context drives one GPU; different
 * contexts may be used from different host threads concurrently (no mutable state is shared
 * between contexts), one context must not be used by two threads at once.
 */
#ifndef SPDNN_B200_H
#define SPDNN_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct spdnn spdnn_t;

enum {
    SPDNN_OK = 0,
    SPDNN_ERR_ARG = -1,      /* bad argument (shape, range, null pointer, order of calls) */
    SPDNN_ERR_CUDA = -2,     /* a CUDA runtime call failed; message holds the CUDA error */
    SPDNN_ERR_MEMORY = -3,   /* host or device allocation failed */
    SPDNN_ERR_STATE = -4,    /* call made before its prerequisites (layers/input missing) */
    SPDNN_ERR_DEVICE = -5,   /* a kernel reported an internal inconsistency */
    SPDNN_ERR_LIMIT = -6     /* a fixed capacity of the library was exceeded */
};

/* Largest number of images one spdnn_layer_static call accepts (its scratch is a fixed array). */
#define SPDNN_STATIC_MAX_IMAGES 2097152

/* Filled by spdnn_infer / spdnn_sync. */
typedef struct spdnn_stats {
    int32_t layers;             /* layers executed */
    int32_t batch;              /* images the input held */
    int64_t survivors;          /* images alive after the last layer */
    float prepare_ms;           /* device time of the input layout conversion of the last set_input */
    float infer_ms;             /* device time of the layer loop incl. on-device compaction (CUDA events) */
    double algorithmic_bytes;   /* sum over layers of 4N(live_in + live_out) + bytes of W_l as CSC */
    int64_t kernel_launches;    /* kernels of this library launched by the last infer (+ last set_input) */
    int32_t loop_launches;      /* of those, launches of the layer loop (1 per layer, or 1 per chunk of layers) */
    int32_t resident_group;     /* images per block of the shared-memory-resident kernel, 0 = per-layer kernel */
} spdnn_stats_t;

/* Replaces GpuEnv::GpuEnv(gpu_id) + the allocations of all_network.cu:283-303.
 * clip is 32 in the reference (all_network.cu:8-10). */
int spdnn_create(spdnn_t **ctx, int device, int neurons, int layers, float bias, float clip);

/* Layer `layer` (0-based) as CSC: column c = output neuron c holds input neurons
 * row_idx[col_ptr[c] .. col_ptr[c+1]) with weights val[...] (val == NULL: every weight is
 * 0.0625, the constant the reference's inspector assumes, src/inspector/matrix_block_container.h:218).
 * Rows of a column may come in any order; they are summed in ascending row order, the
 * order of the reference's CPU loop (src/utils/cpu_spmm.h:12-43).  Replaces the per-layer
 * upload all_network.cu:296-303 and the inspector pass src/network.cpp:97-121. */
int spdnn_set_layer_csc(spdnn_t *ctx, int layer, const int32_t *col_ptr, const int32_t *row_idx, const float *val);

/* Same layer given as the triplets of the reference's layer file: line `a b v` means
 * W[a][b] = v, a = input neuron, b = output neuron, index_base = 1 in the files
 * (src/utils/matrix.h:255-282 with T == false). */
int spdnn_set_layer_coo(spdnn_t *ctx, int layer, int64_t nnz, const int32_t *in_neuron, const int32_t *out_neuron,
                        const float *val, int index_base);

/* Layer `layer` is the same matrix as `other_layer`, which was set before: both share one device
 * copy and the host-side preparation is not repeated.  (spdnn_set_layer_csc finds equal layers by
 * content as well, but only after canonicalising the new one.)  The reference uploads every layer
 * separately (all_network.cu:296-303); networks whose layers repeat with a short period -- its
 * stride table all_network.cu:316-327 cycles -- make this the cheap way to declare 1920 of them. */
int spdnn_set_layer_same_as(spdnn_t *ctx, int layer, int other_layer);

/* Input images, dense batch x N row-major fp32 in HOST memory (the reference's `input`
 * vectors flattened, all_network.cu:240-248, 283-284).  Image i gets the global number
 * first_global_id + i.  Replaces the H2D upload of A_d. */
int spdnn_set_input_dense(spdnn_t *ctx, const float *y0, int batch, int first_global_id);

/* Same, from a DEVICE buffer on the context's GPU (inputs already resident in HBM).  The buffer
 * may be read in place by the inference pass that follows (when its first launch can take a
 * row-major matrix; otherwise it is converted to the internal layout here): keep it unchanged
 * until that pass has finished (spdnn_infer returned, or spdnn_sync after spdnn_infer_async).
 * It is never written. */
int spdnn_set_input_dense_device(spdnn_t *ctx, const float *y0_dev, int batch, int first_global_id);

/* Input images as the triplets of the reference's input file: `img neuron val`
 * (src/network.cpp:33-54; index_base = 1 in the file).  img is relative to this shard:
 * img - index_base in [0, batch). */
int spdnn_set_input_coo(spdnn_t *ctx, int64_t nnz, const int32_t *img, const int32_t *neuron, const float *val,
                        int batch, int first_global_id, int index_base);

/* Input images as a bit matrix in HOST memory: image i is row i of `row_bytes` bytes, bit (n & 7) of byte
 * n >> 3 set = neuron n of the image is 1.0, clear = 0.0 (numpy: packbits(y0 != 0, axis=1, bitorder="little")).
 * row_bytes is a multiple of 4 and at least ceil(neurons / 8).  The challenge's inputs are binary -- every
 * entry of the reference's input file carries the value 1 (src/network.cpp:49-51 logs anything else) -- so this
 * is the same information as spdnn_set_input_coo's triplets or spdnn_set_input_dense's matrix in 1/32 of the
 * dense bytes; it replaces the same H2D upload of A_d (all_network.cu:283-284).  The _device form takes the
 * matrix from a 4-byte aligned buffer on the context's GPU. */
int spdnn_set_input_bits(spdnn_t *ctx, const uint8_t *bits, int64_t row_bytes, int batch, int first_global_id);
int spdnn_set_input_bits_device(spdnn_t *ctx, const uint8_t *bits_dev, int64_t row_bytes, int batch, int first_global_id);

/* The layer loop of all_network.cu:333-519: all layers on the images of the last
 * set_input, with dead images removed on the device after every layer.  Blocks until the
 * result is on the device and fills *stats (may be NULL).  Consumes the input. */
int spdnn_infer(spdnn_t *ctx, spdnn_stats_t *stats);

/* Asynchronous form: enqueue on the context's stream and return; spdnn_sync waits and
 * fills the statistics.  A set_input call made while a pass is in flight does not wait: the
 * new input is ordered behind that pass on the stream and the pass's unfetched results are
 * dropped, so passes can be queued back to back and only the last one synchronised. */
int spdnn_infer_async(spdnn_t *ctx);
int spdnn_sync(spdnn_t *ctx, spdnn_stats_t *stats);

/* Use the caller's CUDA stream (a cudaStream_t passed as void*) for everything the context
 * enqueues from now on; NULL restores the context's own stream.  Replaces
 * GpuEnv::get_stream (gpu_env.h:85-87). */
int spdnn_set_stream(spdnn_t *ctx, void *cuda_stream);

/* live[l] = images alive after layer l: the numbers of the reference's
 * "layer l, batch = k" lines (all_network.cu:508).  capacity >= layers. */
int spdnn_get_layer_live(spdnn_t *ctx, int32_t *live, int capacity);

/* Ascending global image numbers alive after the last layer (the challenge's category
 * list; the reference prints only the count). */
int spdnn_get_categories(spdnn_t *ctx, int32_t *ids, int capacity, int *count);

/* Final activations of the survivors, count x N row-major fp32 in host memory, rows in the
 * order of spdnn_get_categories (the reference copies C back at all_network.cu:521). */
int spdnn_get_activations(spdnn_t *ctx, float *y, int64_t capacity_rows);

/* What the last pass left out because it could not change the result: retired_images = survivors taken off the
 * work list once every activation was clip and every later layer keeps that; skipped_layers = layers of periodic
 * networks behind a fixed point of the saturated activations, summed over the blocks that found one.  For tests
 * and for judging a schedule; either pointer may be NULL. */
int spdnn_get_shortcuts(spdnn_t *ctx, int64_t *retired_images, int64_t *skipped_layers);

/* How the library stored layer `layer`: classes = number of distinct columns (columns with
 * identical rows and weights are computed once), k = padded non-zeros per column,
 * uniform = 1 when all weights are one power-of-two constant.  Any pointer may be NULL. */
int spdnn_get_layer_info(spdnn_t *ctx, int layer, int *classes, int *k, int *uniform);

/* The layer preparation alone, on the host, without a context or a GPU: how a CSC layer of
 * `neurons` columns would be stored (same outputs as spdnn_get_layer_info).  Returns
 * SPDNN_ERR_ARG for a malformed layer.  It takes the place of running the reference's
 * inspector stand-alone (src/main.cpp:57-92). */
int spdnn_inspect_layer_csc(int neurons, const int32_t *col_ptr, const int32_t *row_idx, const float *val,
                            int *classes, int *k, int *uniform);

/* The analysis of a whole network, on the host, without a context or a GPU: for every layer the
 * number of classes when it is expressed in the value ids of the layer before it, the number of
 * value ids it reads (v_in[l] == classes[l-1], or `neurons` where the layer before has no
 * repeated columns) and the table form the resident kernel would use (0 = K gathers per class,
 * 1 = alternating pair).  Layer l is given as CSC through col_ptr[l], row_idx[l], val[l]
 * (val or val[l] may be NULL: all weights 0.0625).  Output arrays hold `layers` entries and
 * may be NULL. */
int spdnn_inspect_network_csc(int neurons, int layers, const int32_t *const *col_ptr, const int32_t *const *row_idx,
                              const float *const *val, int32_t *classes, int32_t *v_in, int32_t *form);

/* One layer, for callers that cannot allocate device memory when they run it (a plugin inside
 * another runtime's memory pool, a callback where cudaMalloc's implicit synchronisation is
 * forbidden, a process whose footprint is frozen after start-up).  This entry point has no
 * counterpart in the reference; it runs the same layer arithmetic as spdnn_infer on buffers
 * the caller owns and keeps its own scratch (survivor ballots, block counters) in a fixed
 * array inside the loaded module, so it calls no cudaMalloc / cudaFree and needs no context.
 *
 *   yin, yout      device, tile layout: tile t holds images 32t..32t+31 as [neurons + 1][32]
 *                  floats (row r = neuron r for the 32 images, row `neurons` = zeros, used
 *                  as padding target); yout must not alias yin
 *   live_in        images to process; image j is read from position in_positions[j] of yin
 *                  (device array, or NULL for j) and written to position j of yout
 *   off            device [neurons][k]: for output neuron c the k input rows times 32,
 *                  ascending; pad short columns with neurons * 32.  k: multiple of 4
 *   vals           device [neurons][k] weights, or NULL: every weight is w (a power of two)
 *   survivors      device out, capacity live_in: ascending positions in yout of the images
 *                  with a non-zero activation; survivor_count: device out, their number
 *   cuda_stream    cudaStream_t as void* (NULL = default stream); the call only enqueues
 *   err, err_len   optional host buffer that receives the message of a failure
 *
 * What a caller that chains calls must know: positions live_in .. 32 * ceil(live_in / 32) - 1 of yout (the
 * unused lanes of the last tile) are overwritten with a copy of that tile's first image; row `neurons`
 * of yout is never written, so a buffer that is fed back as yin must have that row zeroed once by its
 * owner; live_in == 0 is valid (survivor_count becomes 0, nothing else is written).
 *
 * Limits: neurons < 2^26; at most SPDNN_STATIC_MAX_IMAGES images per call (SPDNN_ERR_LIMIT beyond that: split
 * the batch).  The scratch array (about 264 KB) is held by every GPU that loads the library
 * until the process exits and is shared by all calls on that GPU: calls that overlap on the
 * device race, so keep them on one stream or order them with events.  The first call on a
 * device also looks up the array's device address and the launch shape; make that call
 * before any stream capture. */
int spdnn_layer_static(const float *yin, float *yout, int neurons, int live_in, const int32_t *in_positions,
                       const int32_t *off, const float *vals, int k, float w, float bias, float clip,
                       int32_t *survivors, int32_t *survivor_count, void *cuda_stream, char *err, int err_len);

/* ---- Feed-forward operators -------------------------------------------------------------------
 *
 * Sparse layers on row-major activations [tokens][neurons] in device memory of the caller, with trained weights: the plain
 * layer y = act(x W + b) and the gated block y = act(x Wg + bg) * (x Wu + bu), forward and backward, in fp32, fp16 or
 * bf16; and microscaled 4-bit matrices, which weights and activations of the forward calls may be.  They have no counterpart
 * in the reference, whose layers carry one constant weight (src/inspector/matrix_block_container.h:218); like
 * spdnn_layer_static they work on buffers the caller owns, enqueue on the caller's stream (a cudaStream_t as void*, NULL =
 * default stream), allocate nothing, may be captured into a graph, and put the message of a failure into the optional host
 * buffer err (err_len bytes).
 *
 * A TOPOLOGY says which inputs every output neuron is connected to; the weights are arguments of the calls.  It does not change
 * once created: calls on one topology may overlap, on several streams and from several threads, each with a workspace of
 * its own.  Destroy it when no call on it is in flight and no graph that holds one will be replayed.
 *
 * A set of weights is a matrix [outputs][slots] in CANONICAL order: connection j of a neuron is its j-th smallest input
 * (spdnn_topology_rows).  What a matrix holds where a neuron has no j-th connection is never read; gradients are zero there.
 * Sums are held in float32, in no order that callers may rely on (the tensor cores, which take 16-bit neurons that share their connections, cut
 * off what they add at a time instead of rounding it); results are rounded once.  Activations are computed in float32 (of 16-bit operands with the
 * hardware's exponential, also where the result is float32), within (20 + 12 |z| + 2 z^2 + |z|^3) 2^-24 of the value, or 2^-120. */
typedef struct spdnn_topology spdnn_topology_t;

enum { SPDNN_F32 = 0, SPDNN_F16 = 1, SPDNN_BF16 = 2, SPDNN_MX4 = 3 };

/* NONE v, RELU max(v, 0), CLIP min(max(v, 0), clip), SILU v / (1 + e^-v), GELU v Phi(v), GELU_TANH its tanh approximation */
enum {
    SPDNN_ACT_NONE = 0, SPDNN_ACT_RELU = 1, SPDNN_ACT_CLIP = 2, SPDNN_ACT_SILU = 3, SPDNN_ACT_GELU = 4, SPDNN_ACT_GELU_TANH = 5
};

#define SPDNN_MAX_TOKENS (1 << 26)   /* of one call */

/* A matrix in device memory.  F32, F16, BF16: row i begins at data + i * stride elements; any stride not less than a row, any
 * alignment of the type.  MX4: data = codes [rows][stride][16] on 4 bytes, scales [rows][stride] (stride in blocks of 32 columns). */
typedef struct spdnn_operand {
    const void *data;         /* written where the call says so */
    const uint8_t *scales;    /* MX4 only */
    int64_t stride;
    int32_t type;             /* SPDNN_F32 ... */
    int32_t reserved;
} spdnn_operand_t;

/* Topology as CSC: output c is connected to inputs row_idx[col_ptr[c] .. col_ptr[c+1]), in any order (at most 4096; repeated
 * entries stay separate connections).  slots: columns of a weight matrix, at least the connections of every output; 0 = as many as
 * the output with most has (1 if none has any).  Host arrays, borrowed for the call.  device -1: analysis only, for
 * spdnn_topology_info and _rows, without a GPU.  Call it outside stream captures (it allocates). */
int spdnn_topology_create(spdnn_topology_t **top, int device, int inputs, int outputs, int slots, const int32_t *col_ptr,
                          const int32_t *row_idx, char *err, int err_len);
void spdnn_topology_destroy(spdnn_topology_t *top);

/* slots: columns of a weight matrix; fan_out: most outputs that one input feeds.  Pointers may be NULL. */
int spdnn_topology_info(const spdnn_topology_t *top, int *inputs, int *outputs, int *slots, int *fan_out, int64_t *connections);

/* Blocks of up to 16 neurons with equal lists of connections (outputs over the same inputs; inputs read by the same outputs), which 16-bit calls of
 * 17 tokens or more take to the tensor cores.  0: too few neurons share their list, and connections are gathered one by one.  It does not
 * depend on how the neurons are numbered.  Pointers may be NULL. */
int spdnn_topology_blocks(const spdnn_topology_t *top, int *forward, int *backward);

/* The canonical order, to host memory: rows[outputs][slots] = inputs of every output ascending, -1 behind the last one. */
int spdnn_topology_rows(const spdnn_topology_t *top, int32_t *rows, int64_t capacity);

/* Bytes of device workspace (aligned to 256) that a call needs: sets 1 = spdnn_linear, 2 = spdnn_gated, or their backward calls.
 * Its contents need not be kept between calls; calls that may overlap need one each.  0 (forward calls of few tokens): none is
 * needed, workspace may be NULL. */
int spdnn_layer_workspace(const spdnn_topology_t *top, int tokens, int sets, int x_type, int w_type, int backward, int64_t *bytes);

/* y[tokens][outputs] = act(x W + bias).  x [tokens][inputs] and w [outputs][slots]: one float type, or w MX4 with any x, or x
 * MX4 with w MX4 or BF16.  bias: fp32 [outputs] or NULL.  y: any float type, written.  z: x W + bias for the backward call, written in
 * fp32, or NULL.  Outputs must not overlap inputs. */
int spdnn_linear(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *x, const spdnn_operand_t *w, const float *bias,
                 int activation, float clip, const spdnn_operand_t *y, const spdnn_operand_t *z, void *workspace,
                 int64_t workspace_bytes, void *cuda_stream, char *err, int err_len);

/* y = act(x w_gate + bias_gate) * (x w_up + bias_up), both projections over one topology in one pass; both z of one stride, or none. */
int spdnn_gated(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *x, const spdnn_operand_t *w_gate,
                const spdnn_operand_t *w_up, const float *bias_gate, const float *bias_up, int activation, float clip,
                const spdnn_operand_t *y, const spdnn_operand_t *z_gate, const spdnn_operand_t *z_up, void *workspace,
                int64_t workspace_bytes, void *cuda_stream, char *err, int err_len);

/* Gradients from dy = dL/dy and what the forward call read and saved; dy, x, w and dx have one float type.  dx
 * [tokens][inputs] or NULL; dw, dbias in fp32 ([outputs][slots] without gaps, [outputs]), overwritten, or NULL (dbias only with dw).
 * z may be NULL for SPDNN_ACT_NONE (linear).  The slope of RELU at 0 is 0, of CLIP at 0 and clip too.  Every sum has a fixed order: the same call
 * gives the same bits.  On its way to dx dL/dz is rounded to the operands' type; in fp16 after a token's values were multiplied by the power of two
 * that brings the largest into [2^14, 2^15) (the sums are divided by it), so that they keep half a step, or 2^-39 of the token's largest.  On its way to dw it is
 * not rounded, but of 16-bit neurons that share their connections 22 bits of it are multiplied. */
int spdnn_linear_backward(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *dy, const spdnn_operand_t *x,
                          const spdnn_operand_t *w, const spdnn_operand_t *z, int activation, float clip, const spdnn_operand_t *dx,
                          float *dw, float *dbias, void *workspace, int64_t workspace_bytes, void *cuda_stream, char *err,
                          int err_len);
int spdnn_gated_backward(const spdnn_topology_t *top, int tokens, const spdnn_operand_t *dy, const spdnn_operand_t *x,
                         const spdnn_operand_t *w_gate, const spdnn_operand_t *w_up, const spdnn_operand_t *z_gate,
                         const spdnn_operand_t *z_up, int activation, float clip, const spdnn_operand_t *dx, float *dw_gate,
                         float *dw_up, float *dbias_gate, float *dbias_up, void *workspace, int64_t workspace_bytes,
                         void *cuda_stream, char *err, int err_len);

/* Microscaled 4-bit floats: rows in blocks of 32 columns, a block one power of two (E8M0) and 32 values of E2M1 (0, 0.5, 1, 1.5,
 * 2, 3, 4, 6 and their negatives).  Scale 2^(floor(log2 max) - 2), from 2^-127 on; values rounded half to even, above 6 to
 * 6.  A block with a NaN or an infinity becomes NaN.  codes [rows][ceil(cols/32)][16] (even element in the low half of a byte;
 * zeros behind the last column), scales [rows][ceil(cols/32)]; codes aligned to 4 bytes.  On the current device. */
int spdnn_mx4_quantize(const spdnn_operand_t *x, int64_t rows, int cols, uint8_t *codes, uint8_t *scales, void *cuda_stream,
                       char *err, int err_len);
int spdnn_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int cols, const spdnn_operand_t *y,
                         void *cuda_stream, char *err, int err_len);

const char *spdnn_last_error(const spdnn_t *ctx);
void spdnn_destroy(spdnn_t *ctx);

/* Library version string. */
const char *spdnn_version(void);

#ifdef __cplusplus
}
#endif
#endif /* SPDNN_B200_H */
