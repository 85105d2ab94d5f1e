// What the kernels of drafted trees share: who sees whom, where a cached row lies, how the work is split and joined.
//
// Node i of a sequence sees the cached rows 0 .. lengths[b]-1 and, of the drafted ones, itself and its ancestors.  A node
// whose chain of parents does not end at -1 (a place that is not used) sees nothing; its output is zero.
#pragma once

#include "sa2_causal_common.h"

namespace sa2 {
namespace {

// Bit j: node `lane` sees node j.  Six rounds of taking over one's ancestor's ancestors reach all 64.
__device__ __forceinline__ uint64_t tree_ancestors(const Tree& p, int b) {
    const int lane = threadIdx.x & 63;
    int up = -2;
    if (lane < p.T) {
        const int parent = p.parents ? p.parents[(int64_t)b * p.T + lane] : lane - 1;
        if (parent >= -1 && parent < lane) up = parent;
    }
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
    for (int round = 0; round < 6; ++round) {
        const int from = up < 0 ? lane : up;
        const uint32_t l2 = __shfl(lo, from), h2 = __shfl(hi, from);
        const int u2 = __shfl(up, from);
        lo |= l2;
        hi |= h2;
        up = up < 0 ? up : u2;
    }
    return up == -1 ? (uint64_t)hi << 32 | lo : 0u;
}

// Cached rows of sequence b
__device__ __forceinline__ int tree_held(const Tree& p, int b) {
    const int64_t room = p.cache.table ? (int64_t)p.cache.width * p.cache.page_size : p.cache.page_size;
    const int n = p.cache.lengths[b];
    return n < 0 ? 0 : n > room ? (int)room : n;
}
// Page and place of cached row r; false where the table names no page of the cache
__device__ __forceinline__ bool tree_place(const Cache& c, int b, int r, int& page, int& at) {
    if (!c.table) {
        page = b;
        at = r;
        return true;
    }
    const int i = (unsigned)r / (unsigned)c.page_size;
    page = c.table[(int64_t)b * c.width + i];
    at = r - i * c.page_size;
    return page >= 0 && page < c.pages;
}

// How the workgroups of a key head are dealt to the sequences: a unit is one share of one sequence's keys.  Either every sequence has
// nsplit of them, or (`dealt`) of nsplit * B units every sequence gets one and its part of the others by its keys, at most 64 in
// all.  Lengths lie in device memory, so every wavefront counts for itself, which takes about 4 us of a call: dealt are the shares
// of the kernels whose time is products, and from eight per sequence on (one empty cache and three of 33000 to 65000 rows, 48
// nodes: 160 us with 16 each, 130 dealt; single tokens of 8 x 4096 rows 22.6 us with 8 each, 23.2 dealt; of 32 x 2048 rows, two
// each, 37 and 49).
struct TreeShare {
    int b, split, count, first;                            // sequence, which of its shares, how many it has, the first one's unit
};
// A lane counts for one sequence: with eight shares each there are 32 at most (tree_splits).
template <class F>
__device__ __forceinline__ bool tree_deal(const Tree& p, F&& is, TreeShare& s) {
    const int lane = threadIdx.x & 63;
    const double keys = lane < p.B ? (double)tree_held(p, lane) + p.T : 0.0;
    double total = keys;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    // (a little less than its part, so that rounding never deals more units than there are)
    const double each = (double)(p.nsplit - 1) * p.B / total * (1.0 - 1e-9);
    int mine = 1 + (int)(keys * each);
    mine = lane >= p.B ? 0 : mine < 64 ? mine : 64;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o);
        if (lane >= o) sum += up;
    }
    const uint64_t hit = __ballot(mine > 0 && is(lane, sum - mine, sum));
    if (!hit) return false;
    s.b = __ffsll((unsigned long long)hit) - 1;
    s.count = __builtin_amdgcn_readfirstlane(__shfl(mine, s.b));
    s.first = __builtin_amdgcn_readfirstlane(__shfl(sum - mine, s.b));
    s.split = 0;
    return true;
}
// The share that a unit is; false: none
__device__ __forceinline__ bool tree_share(const Tree& p, int unit, TreeShare& s) {
    if (!p.dealt) {
        const int b = unit / p.nsplit;
        s = TreeShare{b, unit - b * p.nsplit, p.nsplit, b * p.nsplit};
        return true;
    }
    const bool any = tree_deal(p, [&](int, int from, int to) { return from <= unit && unit < to; }, s);
    s.split = unit - s.first;
    return any;
}
// The shares of a sequence
__device__ __forceinline__ void tree_shares_of(const Tree& p, int b, TreeShare& s) {
    if (!p.dealt) s = TreeShare{b, 0, p.nsplit, b * p.nsplit};
    else tree_deal(p, [&](int i, int, int) { return i == b; }, s);
}

// Partial result of a row of a unit: `sum` and values in units of e^top
struct TreePart {
    float top, sum;
};
__device__ __forceinline__ TreePart* tree_stat(const Tree& p, int unit, int hk, int row) {
    return (TreePart*)p.part + ((int64_t)unit * p.HK + hk) * (p.T * p.G) + row;
}
__device__ __forceinline__ float* tree_values(const Tree& p, int unit, int hk, int row, int width) {
    const int64_t R = p.T * p.G, slots = (int64_t)p.nsplit * p.B * p.HK * R;
    return p.part + 2 * slots + (((int64_t)unit * p.HK + hk) * R + row) * width;
}

}  // namespace

int launch_tree_join(const Tree& p, int dtype, hipStream_t st);

}  // namespace sa2
