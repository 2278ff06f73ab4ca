// The tables of a topology (topology.h) on a GPU.
#pragma once

#include <cuda_runtime_api.h>

#include "topology.h"

namespace spdnn_impl {

struct DeviceTable {
    uint32_t *slice_ptr = nullptr, *idx = nullptr, *src = nullptr;
    int64_t entries = 0;
    int outs = 0, rows = 0;
};

struct DeviceBlocks {
    uint32_t *chunk_ptr = nullptr, *rows = nullptr, *src = nullptr, *chunk_block = nullptr;
    int32_t *members = nullptr;
    int blocks = 0;                 // 0: this direction has none
    int64_t chunks = 0;
};

struct DeviceTopology {
    DeviceTable forward, backward;
    DeviceBlocks forward_blocks, backward_blocks;
    int32_t *rows = nullptr;        // canonical
    void *few_rows = nullptr;       // canonical as few_kernel reads them: uint16_t where inputs < 65536, else int32_t
};

template <class T>
inline cudaError_t upload(T **to, const std::vector<T> &from) {
    cudaError_t e = cudaMalloc((void **)to, std::max<size_t>(from.size(), 1) * sizeof(T));
    if (e != cudaSuccess) return e;
    return cudaMemcpy(*to, from.data(), from.size() * sizeof(T), cudaMemcpyHostToDevice);
}

inline cudaError_t upload(DeviceTable &d, const GatherTable &t) {
    d.outs = t.outs; d.rows = t.rows; d.entries = (int64_t)t.idx.size();
    cudaError_t e = upload(&d.slice_ptr, t.slice_ptr);
    if (e == cudaSuccess) e = upload(&d.idx, t.idx);
    if (e == cudaSuccess) e = upload(&d.src, t.src);
    return e;
}

inline cudaError_t upload(DeviceBlocks &d, const BlockTable &t) {
    if (!t.blocks) return cudaSuccess;
    d.blocks = t.blocks; d.chunks = (int64_t)t.chunk_ptr.back();
    cudaError_t e = upload(&d.chunk_ptr, t.chunk_ptr);
    if (e == cudaSuccess) e = upload(&d.rows, t.rows);
    if (e == cudaSuccess) e = upload(&d.src, t.src);
    if (e == cudaSuccess) e = upload(&d.members, t.members);
    if (e == cudaSuccess) e = upload(&d.chunk_block, t.chunk_block);
    return e;
}

inline void release(DeviceBlocks &d) {
    cudaFree(d.chunk_ptr); cudaFree(d.rows); cudaFree(d.src); cudaFree(d.members); cudaFree(d.chunk_block);
    d = DeviceBlocks();
}

inline void release(DeviceTable &d) {
    cudaFree(d.slice_ptr); cudaFree(d.idx); cudaFree(d.src);
    d = DeviceTable();
}

inline int few_stride(int slots) { return (slots + 3) / 4 * 4; }

template <class T>
inline cudaError_t upload_few_rows(const Topology &host, T **to) {
    const int stride = few_stride(host.slots);
    std::vector<T> rows((size_t)host.outputs * stride, (T)host.inputs);
    for (int c = 0; c < host.outputs; ++c)
        for (int k = 0; k < host.slots; ++k) {
            const int32_t r = host.rows[(size_t)c * host.slots + k];
            if (r >= 0) rows[(size_t)c * stride + k] = (T)r;
        }
    return upload(to, rows);
}

inline void release(DeviceTopology &d) {
    release(d.forward);
    release(d.backward);
    release(d.forward_blocks);
    release(d.backward_blocks);
    cudaFree(d.rows);
    cudaFree(d.few_rows);
    d = DeviceTopology();
}

inline cudaError_t upload_all(DeviceTopology &d, const Topology &host) {
    cudaError_t e = upload(d.forward, host.forward);
    if (e == cudaSuccess) e = upload(d.backward, host.backward);
    if (e == cudaSuccess) e = upload(d.forward_blocks, host.forward_blocks);
    if (e == cudaSuccess) e = upload(d.backward_blocks, host.backward_blocks);
    if (e == cudaSuccess) e = upload(&d.rows, host.rows);
    if (e == cudaSuccess) e = host.inputs < 65536 ? upload_few_rows(host, (uint16_t **)&d.few_rows) : upload_few_rows(host, (int32_t **)&d.few_rows);
    // A copy from pageable memory may return when it is staged, before it is on the GPU, and the first call on the topology may come on a
    // stream that does not wait for this one.
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    return e;
}

// On the current device.  What fails, with a status or an exception, leaves nothing behind.
inline cudaError_t upload(DeviceTopology &d, const Topology &host) {
    cudaError_t e;
    try {
        e = upload_all(d, host);
    } catch (...) {
        release(d);
        throw;
    }
    if (e != cudaSuccess) release(d);
    return e;
}

}  // namespace spdnn_impl
