// What the causal attention kernels share: which rows a workgroup has, products in which a hidden row may hold anything.
#pragma once

#include "sa2_layer_common.h"

namespace sa2 {
namespace {

// The sequence of a workgroup: its batch entry, first row and length, and the block of rows that the workgroup has.
// fill: rows of no sequence, first .. first + len - 1 of them
struct Span {
    int b, first, len, block;
    bool fill;
};
// Workgroups that tiles of `rows` rows need, per head
inline int64_t count_tiles(const Rows& r, int rows) {
    return r.cu ? (int64_t)r.N / rows + r.sequences + 2 : ((int64_t)r.N + rows - 1) / rows;
}
// The `tile`-th one; false: none.  Packed sequences are counted by every wavefront for itself, 64 at a time: a prefix sum of
// their tiles, no launch and no table before the kernel (about 1 us where 64 lanes hold all sequences).  Rows that no
// sequence holds come last.  Tiles are numbered sequence by sequence: callers put the longest of a sequence first, but a long
// sequence behind others starts late.
__device__ __forceinline__ bool find_tile(const Rows& r, int b, int tile, int rows, Span& s) {
    if (!r.cu) {
        s = Span{b, 0, r.N, tile, false};
        return true;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    auto bound = [&](int i) { const int x = r.cu[i]; return x < 0 ? 0 : x > r.N ? r.N : x; };
    for (int c = 0; c < r.sequences; c += 64) {
        const int i = c + lane;
        int first = 0, len = 0;
        if (i < r.sequences) {
            first = bound(i);
            len = bound(i + 1) - first;
            len = len < 0 ? 0 : len;
        }
        const int mine = (len + rows - 1) / rows;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(sum, o);
            if (lane >= o) sum += up;
        }
        const uint64_t past = __ballot(before + sum > tile);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s.b = 0;
            s.first = __builtin_amdgcn_readfirstlane(__shfl(first, l));
            s.len = __builtin_amdgcn_readfirstlane(__shfl(len, l));
            s.block = __builtin_amdgcn_readfirstlane(tile - before - __shfl(sum - mine, l));
            s.fill = false;
            return true;
        }
        before += __builtin_amdgcn_readfirstlane(__shfl(sum, 63));
    }
    tile -= before;
    const int head = bound(0), tail = bound(r.sequences), head_tiles = (head + rows - 1) / rows;
    s.b = 0;
    s.fill = true;
    s.block = 0;
    const int t = tile < head_tiles ? tile : tile - head_tiles, lo = tile < head_tiles ? 0 : tail, hi = tile < head_tiles ? head : r.N;
    s.first = lo + t * rows;
    s.len = hi - s.first < rows ? hi - s.first : rows;
    return s.len > 0;
}
// Workgroup pid of streams * tiles: a stream is a (batch entry, head) pair.  Tiles run in the outer order, so that in a batch the longest
// ones, which callers put first, start first (packed: each sequence's, one sequence after the other); with a multiple of eight streams every XCD keeps its own (its L2 their keys).
__device__ __forceinline__ void order(int pid, int streams, int& stream, int& tile) {
    if (streams % 8 == 0) {
        const int each = streams / 8, i = pid >> 3;
        stream = (pid & 7) * each + i % each;
        tile = i / each;
    } else {
        stream = pid % streams;
        tile = pid / streams;
    }
}

// Rows of a tile: offset of the row at place `at` of the sequence
__device__ __forceinline__ int64_t row_offset(const Tensor& t, const Span& s, int at, int h) { return t.off(s.b, s.first + at, h); }

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

}  // namespace
}  // namespace sa2
