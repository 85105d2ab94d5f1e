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

// Tiles of SIZE keys that queries first .. last see any of, numbered from 0 on: those of the first keys, then those of the window
template <bool BAND, int SIZE>
struct KeyTiles {
    int head, start, count;
    __device__ __forceinline__ KeyTiles(const Band& band, int first, int last) {
        head = start = 0;
        if constexpr (BAND) {
            start = (first < band.window ? 0 : first - band.window + 1) / SIZE;
            head = (band.sinks + SIZE - 1) / SIZE;
            head = head < start ? head : start;
        }
        count = head + last / SIZE + 1 - start;
    }
    // the first key of tile t
    __device__ __forceinline__ int at(int t) const { return (!BAND || t < head ? t : t - head + start) * SIZE; }
};
// Bits 0 .. n-1 of 32
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
// What query i sees of the keys j0 .. j0+31, and which of the queries i0 .. i0+31 see key j (`sink`: one of the first ones), bit by bit
__device__ __forceinline__ uint32_t band_keys(const Band& b, int i, int j0) { return bits_below(i - j0 + 1) & (~bits_below(i - b.window + 1 - j0) | bits_below(b.sinks - j0)); }
__device__ __forceinline__ uint32_t band_queries(const Band& b, int j, int i0, bool sink) { return ~bits_below(j - i0) & (sink ? ~0u : bits_below(j - i0 + b.window)); }
// Of such queries or keys, those whose gradients count: a query that sees its own key only has one weight, 1, whose gradient is zero
__device__ __forceinline__ uint32_t band_counted(const Band& b, uint32_t queries, int i0) { return i0 + 31 <= b.alone ? 0u : i0 == 0 ? queries & ~1u : queries; }
// Whether queries i0 .. i1 see all of the keys j0 .. j1
__device__ __forceinline__ bool band_full(const Band& b, int i0, int i1, int j0, int j1) { return j1 <= i0 && (i1 - j0 < b.window || j1 < b.sinks); }
// Keys j0 .. j0+rows-1 of a workgroup and the queries lo .. hi-1 that it takes for them: with a band, those of the window of keys behind the
// first ones (`extra` < 0), or a chunk of the sequence for the first keys.  The workgroups of these come in groups, of which `extra` is the
// number in the group: a group has a chunk (`s` is the `tile`-th of them), its members a block of the first keys each; or (by_rows) a group
// of two a block of `rows` rows, and its members two of the sequence's pairs of a chunk and a block of first keys (which are never more than that).
// false: none, or nothing that it has to leave
struct KeyWork {
    int j0, lo, hi;
    int64_t sink;                                           // the chunk's first row of sums, or -1
};
template <bool BAND>
__device__ __forceinline__ bool key_work(const Causal& p, const Span& s, int rows, int tile, int extra, KeyWork& w) {
    w = KeyWork{s.block * rows, s.block * rows, s.len, -1};
    if constexpr (BAND) {
        if (extra < 0) {
            if (w.j0 + rows <= p.band.sinks) return false;
            const int64_t end = (int64_t)w.j0 + rows - 1 + p.band.window;
            w.hi = end < s.len ? (int)end : s.len;
        } else {
            int chunk = s.block;
            w.j0 = extra * rows;
            w.sink = s.b * (p.band.sink_rows / p.rows.B) + (int64_t)tile * p.band.sinks;
            if (p.band.by_rows) {
                const int held = p.band.sinks < s.len ? p.band.sinks : s.len, blocks = (held + rows - 1) / rows;
                const int64_t pair = 2 * (int64_t)s.block + extra;
                chunk = (int)(pair / blocks);
                w.j0 = (int)(pair % blocks) * rows;
                w.sink = 2 * (int64_t)s.first + (int64_t)chunk * held;
            }
            const int64_t from = (int64_t)chunk * p.band.chunk;
            if (from >= s.len) return false;
            w.lo = from > w.j0 ? (int)from : w.j0;
            w.hi = s.len - from < p.band.chunk ? s.len : (int)from + p.band.chunk;
            return w.j0 < s.len && w.lo < w.hi;
        }
    }
    return true;
}
// Sums of the first key j of a key head over the chunk whose rows begin at `sink`; which: 0 dK, 1 dV
__device__ __forceinline__ float* sink_row(const Causal& p, int which, int64_t sink, int hk, int j) {
    return p.sink_part + (((int64_t)which * p.HK + hk) * p.band.sink_rows + sink + j) * p.D;
}
// Members of a group of workgroups of the first keys, and the groups, of a key head
inline int sink_members(const Causal& p, int rows) { return p.band.by_rows ? 2 : (p.band.sinks + rows - 1) / rows; }
inline int64_t sink_groups(const Causal& p, int rows) { return (int64_t)p.rows.B * count_tiles(p.rows, p.band.by_rows ? rows : p.band.chunk); }
// Windows: query heads that a workgroup's four wavefronts have, and whether a wavefront has two blocks of 32 queries (as causal16_two)
inline int window_heads(const Causal& p) { return p.G % 4 == 0 ? 4 : p.G % 2 == 0 ? 2 : 1; }
inline bool window_two(const Causal& p, int heads) { return (int64_t)p.rows.B * (p.H / heads) * count_tiles(p.rows, 256 / heads) >= 2 * CUS; }

// Whether the exponent x c - at c of a score near the reference point `at` is not to be had from at c, whose rounding, half a unit of 2^-24 of it, is more
// than half a power of two: x - at comes first then
__device__ __forceinline__ bool far_from_zero(float at, float c) { return fabsf(at) * c > 16777216.f; }
__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

}  // namespace
}  // namespace sa2
