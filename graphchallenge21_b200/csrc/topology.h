// Host-side preparation of a topology (which inputs every output neuron reads) for the feed-forward operators.
//
// A topology is the sparsity pattern of a layer without its weights: they change from step to step when a network is trained,
// the pattern does not.  In canonical order (the order of every weight matrix a caller passes) connection j of a neuron is its
// j-th smallest input, as in canonicalize_layer.  The kernels read their connections through GATHER TABLES, one for the forward direction (outputs
// gather inputs) and one for the backward direction (inputs gather outputs).
#pragma once

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <new>
#include <string>
#include <thread>
#include <vector>

namespace spdnn_impl {

constexpr uint32_t kNoSource = 0xffffffffu;

// The connections of `outs` gathering neurons in slices of 32 (lane = neuron of the slice).  A slice is as long as its longest
// neuron, rounded up to whole quads of four connections; quad q of a slice holds 32 x 4 entries, so that a lane fetches its four
// in one load.  Slices of their own length rather than one length for all: of a random topology an input neuron feeds 32 +- 6
// outputs, the longest of 16384 more than 58.
struct GatherTable {
    int outs = 0;                      // gathering neurons
    int rows = 0;                      // gathered neurons; row `rows` is a row of zeros, the target of padding
    std::vector<uint32_t> slice_ptr;   // [slices + 1] first quad of a slice
    std::vector<uint32_t> idx;         // [quads][32][4] gathered row
    std::vector<uint32_t> src;         // [quads][32][4] position in the canonical weights, kNoSource = padding
};

struct Topology {
    int inputs = 0, outputs = 0;
    int slots = 0;                     // connections per output neuron, at least 1
    int fan_out = 0;                   // most outputs one input feeds
    int64_t connections = 0;
    std::vector<int32_t> rows;         // [outputs][slots] ascending input per output, -1 behind the last
    GatherTable forward, backward;
};

// Most entries of a gather table (4 bytes of index, 4 of source): a slice is as long as its longest neuron.
constexpr int64_t kMostEntries = 1ll << 30;
constexpr int kMostSlots = 4096;       // as canonicalize_layer

// Orders the connections of 16 neighbouring neurons, whose lanes read their k-th connections at the same time, so that those fall on
// different banks: of the sixteen (eight aligned, four, two) neurons the gathered rows should differ in the bits 0 to 3 (0 to 2, 0 and 1, 0)
// of their numbers; spdnn_ffn.cuh says why.  Step by step and neuron by neuron the connection with the fewest meetings, of equals
// one from the class (the four bits) that has most left.  Without it 2.1 wavefronts of shared memory a load where 1 would do.
class BankOrder {
public:
    struct Entry { uint32_t row, source; };
    std::vector<Entry> lists[16];      // of every neuron, in any order; run() puts them in the order of the steps
    void run() {
        size_t longest = 0;
        for (int l = 0; l < 16; ++l) {
            longest = std::max(longest, lists[l].size());
            std::fill(left_[l], left_[l] + 16, 0);
            for (const Entry &e : lists[l]) ++left_[l][e.row & 15];
            uint32_t at = 0;
            for (int c = 0; c < 16; ++c) { next_[l][c] = at; at += left_[l][c]; }
            sorted_[l].resize(lists[l].size());
            for (const Entry &e : lists[l]) sorted_[l][next_[l][e.row & 15]++] = e;
            lists[l].clear();
        }
        for (size_t k = 0; k < longest; ++k) {
            uint32_t pair[8][2] = {}, quad[4][4] = {}, oct[2][8] = {}, hex[16] = {};
            for (int l = 0; l < 16; ++l) {
                if (lists[l].size() + 1 > sorted_[l].size()) continue;
                int best = -1;
                uint32_t best_cost = 0;
                for (int c = 0; c < 16; ++c) {
                    const uint32_t meetings = hex[c] + oct[l / 8][c & 7] + quad[l / 4][c & 3] + pair[l / 2][c & 1];
                    const uint32_t cost = 4096u * meetings + 4095u - std::min<uint32_t>(left_[l][c], 4095u);
                    if (left_[l][c] && (best < 0 || cost < best_cost)) { best = c; best_cost = cost; }
                }
                ++hex[best]; ++oct[l / 8][best & 7]; ++quad[l / 4][best & 3]; ++pair[l / 2][best & 1];
                --left_[l][best];
                lists[l].push_back(sorted_[l][--next_[l][best]]);
            }
        }
    }
private:
    std::vector<Entry> sorted_[16];
    uint32_t left_[16][16], next_[16][16];
};

// Runs f(begin, end) over [0, n) in a few host threads (large topologies: 16384 neurons of 32 connections take 15 ms in one).
template <class F>
inline void in_threads(int n, int64_t work, const F &f) {
    const int threads = (int)std::min<int64_t>(std::min<int64_t>(std::max(1u, std::thread::hardware_concurrency()), 8), work / 32768 + 1);
    std::vector<std::thread> more;
    int begun = 0;
    try {
        for (; begun + 1 < threads; ++begun) more.emplace_back(f, (int)((int64_t)n * begun / threads), (int)((int64_t)n * (begun + 1) / threads));
    } catch (...) {                    // no more threads to be had: the rest is done here
    }
    f((int)((int64_t)n * begun / threads), n);
    for (std::thread &t : more) t.join();
}

// lists(i, emit) calls emit(row, source) for the connections of gathering neuron i
template <class Lists>
inline std::string build_gather_table(int outs, int rows, const std::vector<uint32_t> &count, const Lists &lists, GatherTable &t) {
    t.outs = outs; t.rows = rows;
    const int slices = (outs + 31) / 32;
    t.slice_ptr.assign((size_t)slices + 1, 0);
    int64_t quads = 0;
    for (int s = 0; s < slices; ++s) {
        uint32_t longest = 0;
        for (int i = s * 32; i < std::min(outs, s * 32 + 32); ++i) longest = std::max(longest, count[i]);
        quads += (longest + 3) / 4;
        if (quads * 128 > kMostEntries) return "the topology's gather table would pass 2^30 entries";
        t.slice_ptr[s + 1] = (uint32_t)quads;
    }
    t.idx.assign((size_t)quads * 128, (uint32_t)rows);
    t.src.assign((size_t)quads * 128, kNoSource);
    std::atomic<bool> failed{false};
    in_threads(slices * 2, quads * 128, [&](int begin, int end) {
        try {
            BankOrder order;
            for (int group = begin; group < end; ++group) {
                const int first = group * 16;
                for (int l = 0; l < 16; ++l)
                    if (first + l < outs) lists(first + l, [&](uint32_t row, uint32_t source) { order.lists[l].push_back({row, source}); });
                order.run();
                for (int l = 0; l < 16; ++l) {
                    const size_t at = (size_t)t.slice_ptr[first / 32] * 128 + (size_t)((first + l) % 32) * 4;
                    for (size_t k = 0; k < order.lists[l].size(); ++k) {
                        const size_t e = at + k / 4 * 128 + k % 4;
                        t.idx[e] = order.lists[l][k].row; t.src[e] = order.lists[l][k].source;
                    }
                    order.lists[l].clear();
                }
            }
        } catch (...) { failed = true; }
    });
    if (failed) throw std::bad_alloc();
    return "";
}

// Returns an empty string on success, else the reason the topology is rejected.
inline std::string build_topology(int inputs, int outputs, const int32_t *col_ptr, const int32_t *row_idx, Topology &t) {
    if (inputs <= 0 || outputs <= 0 || inputs >= (1 << 26) || outputs >= (1 << 26)) return "inputs and outputs must be in [1, 2^26)";
    if (!col_ptr) return "col_ptr is null";
    if (col_ptr[0] != 0) return "col_ptr[0] must be 0";
    int most = 1;
    for (int c = 0; c < outputs; ++c) {
        const int64_t n = (int64_t)col_ptr[c + 1] - col_ptr[c];
        if (n < 0) return "col_ptr must be non-decreasing";
        if (n > kMostSlots) return "more than 4096 connections of one output are not supported";
        most = std::max(most, (int)n);
    }
    const int64_t nnz = col_ptr[outputs];
    if (nnz && !row_idx) return "row_idx is null";
    if ((int64_t)outputs * most >= (1ll << 31)) return "outputs times connections per output must stay below 2^31";
    t.inputs = inputs; t.outputs = outputs; t.slots = most; t.connections = nnz;
    t.rows.assign((size_t)outputs * most, -1);
    std::vector<uint32_t> in_count((size_t)outputs), out_count((size_t)inputs, 0);
    for (int c = 0; c < outputs; ++c) {
        const int n = col_ptr[c + 1] - col_ptr[c];
        int32_t *r = t.rows.data() + (size_t)c * most;
        bool ascending = true;
        for (int k = 0; k < n; ++k) {
            const int32_t v = row_idx[col_ptr[c] + k];
            if (v < 0 || v >= inputs) return "row index out of range in column " + std::to_string(c);
            ascending &= k == 0 || r[k - 1] <= v;
            r[k] = v;
            ++out_count[v];
        }
        if (!ascending) std::sort(r, r + n);
        in_count[c] = (uint32_t)n;
    }
    t.fan_out = (int)*std::max_element(out_count.begin(), out_count.end());
    std::string why = build_gather_table(outputs, inputs, in_count, [&](int c, auto emit) {
        const int32_t *r = t.rows.data() + (size_t)c * most;
        for (uint32_t k = 0; k < in_count[c]; ++k) emit((uint32_t)r[k], (uint32_t)((size_t)c * most + k));
    }, t.forward);
    if (!why.empty()) return why;
    // the transposed lists, outputs ascending
    std::vector<size_t> start((size_t)inputs + 1, 0);
    for (int i = 0; i < inputs; ++i) start[i + 1] = start[i] + out_count[i];
    std::vector<uint32_t> by_input((size_t)nnz);
    std::vector<size_t> at(start.begin(), start.end() - 1);
    for (int c = 0; c < outputs; ++c)
        for (uint32_t k = 0; k < in_count[c]; ++k) {
            const size_t p = (size_t)c * most + k;
            by_input[at[t.rows[p]]++] = (uint32_t)p;
        }
    return build_gather_table(inputs, outputs, out_count, [&](int i, auto emit) {
        for (size_t e = start[i]; e < start[i + 1]; ++e) emit(by_input[e] / (uint32_t)most, by_input[e]);
    }, t.backward);
}

}  // namespace spdnn_impl
