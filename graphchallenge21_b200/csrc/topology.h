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
#include <unordered_map>
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

// Gathering neurons that gather the SAME rows (the 16 outputs of a butterfly's block), up to 16 to a block: a small dense product, which the
// tensor cores take.  Rows in chunks of 32, chunk by chunk.
struct BlockTable {
    int blocks = 0;                    // 0: not worth it (too few neurons share their rows)
    std::vector<uint32_t> chunk_ptr;   // [blocks + 1] first chunk of a block
    std::vector<uint32_t> rows;        // [chunks][32] gathered row, padding = the row of zeros
    std::vector<uint32_t> src;         // [chunks][2][32][8] position in the canonical weights, kNoSource = padding: see fragment()
    std::vector<int32_t> members;      // [blocks][16] gathering neuron, -1 = none
    std::vector<uint32_t> chunk_block; // [chunks]
};

// Where the weight of row `k` and neuron `j` of a chunk is: in the order of the tensor cores' second operand (16 rows x 8 neurons: lane 4 (j mod 8) +
// (k mod 8) / 2 holds the rows 2 (lane mod 4) + {0, 1, 8, 9}), a lane's eight for the neurons 0-7 and 8-15 together.
inline size_t fragment(int k, int j) {
    const int lane = j % 8 * 4 + k % 8 / 2, v = k % 2 + k % 16 / 8 * 2;
    return (size_t)((k / 16 * 32 + lane) * 8 + j / 8 * 4 + v);
}

struct Topology {
    int inputs = 0, outputs = 0;
    int slots = 0;                     // connections per output neuron, at least 1
    int fan_out = 0;                   // most outputs one input feeds
    int64_t connections = 0;
    std::vector<int32_t> rows;         // [outputs][slots] ascending input per output, -1 behind the last
    GatherTable forward, backward;
    BlockTable forward_blocks, backward_blocks;
};

// Most entries of a gather table (4 bytes of index, 4 of source): a slice is as long as its longest neuron.
constexpr int64_t kMostEntries = 1ll << 30;
constexpr int kMostSlots = 4096;       // as canonicalize_layer
// Blocks are used where their products have at most this many times the connections (1024 tokens, 4096 neurons, 32 connections, bf16, gated, us
// forward / backward by blocks: 15 / 66 where 16 neurons share their rows, 27 / 88 where 8 do, 44 / 129 where 4 do; by connections 27 / 97).
constexpr int64_t kBlockWaste = 2;

// Orders the connections of `lanes` (2, 4, 8 or 16) neighbouring neurons, whose lanes read their k-th connections at the same time, so
// that those fall on different banks: into steps in which the gathered rows belong to different CLASSES, row mod `lanes` (spdnn_ffn.cuh
// says why these).  Every neuron has a connection in every step, so as long as no class has more connections left than there are
// steps, a matching of neurons to classes exists in which no class occurs twice (an edge colouring of the bipartite multigraph
// of neurons and classes); where one has more, steps in which classes occur twice take the surplus off all such
// classes at once.  Of a random topology (8 lanes, 32 connections) that leaves 1.25 wavefronts per load of eight lanes, 2.6 in any order.
class BankOrder {
public:
    struct Entry { uint32_t row, source; };
    explicit BankOrder(int lanes) : lanes_(lanes) {}
    std::vector<Entry> lists[16];      // of every neuron, in any order; run() puts them in the order of the steps
    void run() {
        int steps = 0;
        std::fill(total_, total_ + lanes_, 0);
        for (int l = 0; l < lanes_; ++l) {
            steps = std::max(steps, (int)lists[l].size());
            std::fill(left_[l], left_[l] + lanes_, 0);
            for (const Entry &e : lists[l]) ++left_[l][e.row & (lanes_ - 1)];
            int at = 0;
            for (int c = 0; c < lanes_; ++c) { next_[l][c] = at; at += left_[l][c]; total_[c] += left_[l][c]; }
            sorted_[l].resize(lists[l].size());
            for (const Entry &e : lists[l]) sorted_[l][next_[l][e.row & (lanes_ - 1)]++] = e;
            lists[l].clear();
        }
        for (; steps > 0; --steps) {
            int by_total[16];
            for (int c = 0; c < lanes_; ++c) by_total[c] = c;
            std::sort(by_total, by_total + lanes_, [&](int x, int y) { return total_[x] != total_[y] ? total_[x] > total_[y] : x < y; });
            std::fill(class_of_, class_of_ + 16, -1);
            std::fill(used_, used_ + 16, 0);
            cap_ = total_[by_total[0]] > steps ? 2 : 1;
            // classes without slack first: they must occur in this step (twice where they have a surplus) ...
            for (int i = 0; i < lanes_ && total_[by_total[i]] >= steps; ++i)
                for (int k = total_[by_total[i]] > steps ? 2 : 1; k > 0; --k) {
                    std::fill(seen_, seen_ + 16, false);
                    if (!give_class(by_total[i])) break;
                }
            // ... then every neuron a class; where none is free, the least used of its own
            for (int l = 0; l < lanes_; ++l) {
                if (class_of_[l] >= 0 || lists[l].size() == sorted_[l].size()) continue;
                std::fill(seen_, seen_ + 16, false);
                if (!give_neuron(l, by_total)) {
                    int best = -1;
                    for (int i = 0; i < lanes_; ++i) {
                        const int c = by_total[i];
                        if (left_[l][c] && (best < 0 || used_[c] < used_[best])) best = c;
                    }
                    class_of_[l] = best; ++used_[best];
                }
            }
            for (int l = 0; l < lanes_; ++l) {
                const int c = class_of_[l];
                if (c < 0) continue;
                --left_[l][c]; --total_[c];
                lists[l].push_back(sorted_[l][--next_[l][c]]);
            }
        }
    }
private:
    // augmenting paths; a neuron or class that was served stays served
    bool give_class(int c) {
        for (int l = 0; l < lanes_; ++l)
            if (class_of_[l] < 0 && left_[l][c]) { class_of_[l] = c; ++used_[c]; return true; }
        seen_[c] = true;
        for (int l = 0; l < lanes_; ++l) {
            const int other = class_of_[l];
            if (other < 0 || seen_[other] || !left_[l][c]) continue;
            if (!give_class(other)) continue;          // another neuron takes `other` on
            --used_[other]; class_of_[l] = c; ++used_[c];
            return true;
        }
        return false;
    }
    bool give_neuron(int l, const int *order) {
        for (int i = 0; i < lanes_; ++i)
            if (left_[l][order[i]] && used_[order[i]] < cap_) { class_of_[l] = order[i]; ++used_[order[i]]; return true; }
        for (int i = 0; i < lanes_; ++i) {
            const int c = order[i];
            if (!left_[l][c] || seen_[c]) continue;
            seen_[c] = true;
            for (int m = 0; m < lanes_; ++m) {
                if (class_of_[m] != c) continue;
                if (!give_neuron(m, order)) continue;  // it moved to another class and left its place in this one
                --used_[c]; class_of_[l] = c; ++used_[c];
                return true;
            }
        }
        return false;
    }
    int lanes_, cap_ = 1;
    std::vector<Entry> sorted_[16];
    int left_[16][16], next_[16][16], total_[16], class_of_[16], used_[16];
    bool seen_[16];
};

// Runs f(begin, end) over [0, n) in a few host threads (large topologies: 16384 neurons of 32 connections take 86 ms in one, 20 in eight, with all else).
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

// lists(i, emit) calls emit(row, source) for the connections of gathering neuron i; lanes: see BankOrder
template <class Lists>
inline std::string build_gather_table(int outs, int rows, const std::vector<uint32_t> &count, const Lists &lists, int lanes, GatherTable &t) {
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
    in_threads(slices * 32 / lanes, quads * 128, [&](int begin, int end) {
        try {
            BankOrder order(lanes);
            for (int group = begin; group < end; ++group) {
                const int first = group * lanes;
                for (int l = 0; l < lanes; ++l)
                    if (first + l < outs) lists(first + l, [&](uint32_t row, uint32_t source) { order.lists[l].push_back({row, source}); });
                order.run();
                for (int l = 0; l < lanes; ++l) {
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

// The blocks of a gather: neuron i gathers row(i, k) for k < length(i), with the weight at source(i, k).
template <class Length, class Row, class Source>
inline void build_block_table(int outs, int rows, int64_t entries, const Length &length, const Row &row, const Source &source, BlockTable &t) {
    std::unordered_map<uint64_t, int> newest;          // hash of a list -> the class that was opened last for it
    std::vector<int> first, older;                     // of a class: its first neuron; the class before it with the same hash
    std::vector<std::vector<int32_t>> members;
    const auto same = [&](int i, int j) {
        if (length(i) != length(j)) return false;
        for (size_t k = 0; k < length(i); ++k)
            if (row(i, k) != row(j, k)) return false;
        return true;
    };
    int64_t chunks = 0, blocks = 0;
    for (int i = 0; i < outs; ++i) {
        uint64_t h = 0x9E3779B97F4A7C15ull ^ length(i);
        for (size_t k = 0; k < length(i); ++k) h = (h ^ row(i, k)) * 0xBF58476D1CE4E5B9ull, h ^= h >> 29;
        const auto found = newest.find(h);
        int c = found == newest.end() ? -1 : found->second;
        while (c >= 0 && !same(first[c], i)) c = older[c];
        if (c < 0) {
            c = (int)first.size();
            first.push_back(i);
            older.push_back(found == newest.end() ? -1 : found->second);
            members.emplace_back();
            newest[h] = c;
        }
        // They only grow, so it does not matter in which order the neurons come; of a random topology an eighth of them is read.
        if (members[c].size() % 16 == 0) {
            ++blocks;
            chunks += (int64_t)std::max<size_t>(1, (length(i) + 31) / 32);
            if (chunks * 512 > entries * kBlockWaste) return;
        }
        members[c].push_back(i);
    }
    t.blocks = (int)blocks;
    t.chunk_ptr.assign(1, 0);
    t.chunk_ptr.reserve(blocks + 1);
    t.rows.assign((size_t)chunks * 32, (uint32_t)rows);
    t.src.assign((size_t)chunks * 512, kNoSource);
    t.members.assign((size_t)blocks * 16, -1);
    size_t block = 0, chunk = 0;
    for (size_t c = 0; c < first.size(); ++c)
        for (size_t m = 0; m < members[c].size(); m += 16, ++block) {
            const size_t n = length(first[c]);
            for (size_t k = 0; k < n; ++k) {
                t.rows[chunk * 32 + k] = row(first[c], k);
                for (size_t j = m; j < std::min(m + 16, members[c].size()); ++j)
                    t.src[(chunk + k / 32) * 512 + fragment((int)(k % 32), (int)(j - m))] = source(members[c][j], k);
            }
            for (size_t j = m; j < std::min(m + 16, members[c].size()); ++j) t.members[block * 16 + (j - m)] = members[c][j];
            chunk += std::max<size_t>(1, (n + 31) / 32);        // neurons without connections have a chunk of padding
            t.chunk_block.resize(chunk, (uint32_t)block);
            t.chunk_ptr.push_back((uint32_t)chunk);
        }
}

// Returns an empty string on success, else the reason the topology is rejected.  slots: width of a weight matrix, 0 = as many as the output with
// most connections has.  forward_lanes, backward_lanes: see BankOrder.
inline std::string build_topology(int inputs, int outputs, int slots, const int32_t *col_ptr, const int32_t *row_idx, int forward_lanes, int backward_lanes,
                                  Topology &t) {
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
    if (slots < 0 || slots > kMostSlots || (slots > 0 && slots < most)) return "slots must be 0, or at least an output's connections and at most 4096";
    if (slots) most = slots;
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
    }, forward_lanes, t.forward);
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
    build_block_table(outputs, inputs, nnz, [&](int c) { return (size_t)in_count[c]; },
                      [&](int c, size_t k) { return (uint32_t)t.rows[(size_t)c * most + k]; },
                      [&](int c, size_t k) { return (uint32_t)((size_t)c * most + k); }, t.forward_blocks);
    build_block_table(inputs, outputs, nnz, [&](int i) { return (size_t)out_count[i]; },
                      [&](int i, size_t k) { return by_input[start[i] + k] / (uint32_t)most; },
                      [&](int i, size_t k) { return by_input[start[i] + k]; }, t.backward_blocks);
    return build_gather_table(inputs, outputs, out_count, [&](int i, auto emit) {
        for (size_t e = start[i]; e < start[i + 1]; ++e) emit(by_input[e] / (uint32_t)most, by_input[e]);
    }, backward_lanes, t.backward);
}

}  // namespace spdnn_impl
