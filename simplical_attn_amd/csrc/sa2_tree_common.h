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

// Result (nsplit 1) or partial result of a row: `sum` and values in units of e^top
struct TreePart {
    float top, sum;
};
__device__ __forceinline__ TreePart* tree_stat(const Tree& p, int split, int64_t stream, int row) {
    const int R = p.T * p.G;
    return (TreePart*)p.part + ((int64_t)split * p.B * p.HK + stream) * R + row;
}
__device__ __forceinline__ float* tree_values(const Tree& p, int split, int64_t stream, int row, int width) {
    const int64_t R = p.T * p.G, rows = (int64_t)p.B * p.HK * R;
    return p.part + 2 * rows * p.nsplit + ((int64_t)split * rows + stream * R + row) * width;
}

}  // namespace

int launch_tree_join(const Tree& p, int dtype, hipStream_t st);

}  // namespace sa2
