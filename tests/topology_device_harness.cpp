// Runs the upload of a topology's tables (csrc/topology_device.h) against a CUDA runtime of its own that only counts.
//
//   ordered      prints how many copies from pageable memory nothing has waited for when the upload returns
//   calls        prints how many allocations on the GPU and on the host an upload makes
//   device N     the Nth allocation on the GPU fails; prints what is left of the others
//   host N       the Nth allocation on the host throws; the same
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "topology_device.h"

using namespace spdnn_impl;

static int live = 0, pending = 0;
static int device_calls = 0, host_calls = 0, failing_device = 0, failing_host = 0;
static bool counting = false;

void *operator new(size_t n) {
    if (counting && ++host_calls == failing_host) throw std::bad_alloc();
    if (void *p = malloc(n)) return p;
    throw std::bad_alloc();
}
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }

extern "C" {
cudaError_t cudaMalloc(void **p, size_t n) {
    if (++device_calls == failing_device) return cudaErrorMemoryAllocation;
    *p = malloc(n);
    ++live;
    return cudaSuccess;
}
cudaError_t cudaFree(void *p) {
    if (p) --live;
    free(p);
    return cudaSuccess;
}
cudaError_t cudaMemcpy(void *to, const void *from, size_t n, cudaMemcpyKind) {
    memcpy(to, from, n);
    ++pending;
    return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t stream) {
    if (!stream) pending = 0;
    return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() {
    pending = 0;
    return cudaSuccess;
}
}

int main(int argc, char **argv) {
    // a butterfly: gather tables and blocks in both directions
    constexpr int N = 256, K = 32;
    std::vector<int32_t> col_ptr(N + 1), row_idx(N * K);
    for (int c = 0; c <= N; ++c) col_ptr[c] = c * K;
    for (int c = 0; c < N; ++c)
        for (int k = 0; k < K; ++k) row_idx[c * K + k] = (c / 16 * 16 + k / 16 * 128 + k % 16) % N;
    Topology host;
    const std::string why = build_topology(N, N, 0, col_ptr.data(), row_idx.data(), 8, 8, host);
    if (!why.empty() || !host.forward_blocks.blocks || !host.backward_blocks.blocks) return 2;
    if (argc == 2 && !strcmp(argv[1], "ordered")) {
        DeviceTopology d;
        if (upload(d, host) != cudaSuccess) return 3;
        printf("%d\n", pending);
        release(d);
        return live ? 4 : 0;
    }
    if (argc == 2 && !strcmp(argv[1], "calls")) {
        DeviceTopology d;
        counting = true;
        if (upload(d, host) != cudaSuccess) return 3;
        counting = false;
        printf("%d %d\n", device_calls, host_calls);
        return 0;
    }
    if (argc == 3) {
        (strcmp(argv[1], "host") ? failing_device : failing_host) = atoi(argv[2]);
        DeviceTopology d;
        bool failed;
        counting = true;
        try {
            failed = upload(d, host) != cudaSuccess;
        } catch (const std::bad_alloc &) {
            failed = true;
        }
        counting = false;
        printf("%d %d\n", (int)failed, live);
        return 0;
    }
    return 1;
}
