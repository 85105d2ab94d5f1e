// What the kernels of keys' weights share: the stream of queries of a block of keys, its shares, where a sum goes.
#pragma once

#include "sa2_causal_common.h"

namespace sa2 {
namespace {

// Queries lo .. hi-1 of every head are the stream of the keys j0 .. j0+rows-1: `per` tiles of `tile` each
struct KeyStream {
    int lo, hi, per;
};
__device__ __forceinline__ KeyStream key_stream(const KeySums& p, const Span& s, int j0, int rows, int tile) {
    KeyStream k{j0, s.len, 0};
    if (p.band.window && j0 >= p.band.sinks) {
        const int64_t end = (int64_t)j0 + rows - 1 + p.band.window;
        k.hi = end < s.len ? (int)end : s.len;
    }
    k.per = (k.hi - k.lo + tile - 1) / tile;
    return k;
}
// Which of the queries i0 .. i0+31 see key j, bit by bit
__device__ __forceinline__ uint32_t key_seen_by(const KeySums& p, const Span& s, int j, int i0) {
    return ~bits_below(j - i0) & bits_below(s.len - i0) & (p.band.window && j >= p.band.sinks ? bits_below(j - i0 + p.band.window) : ~0u);
}
// Whether all of the queries i0 .. i1 see all of the keys j0 .. j1
__device__ __forceinline__ bool key_all_seen(const KeySums& p, const Span& s, int i0, int i1, int j0, int j1) {
    return i0 >= j1 && i1 < s.len && (!p.band.window || i1 - j0 < p.band.window || j1 < p.band.sinks);
}
// The sum of key `at` of the sequence
__device__ __forceinline__ void put_key_sum(const KeySums& p, const Span& s, int hk, int at, float sum) {
    if (!p.lengths) {
        p.out[s.b * p.sb + hk * p.sh + s.first + at] = sum;
        return;
    }
    if (s.fill) return;
    const int b = p.rows.cu ? sequence_of(p.rows, s.first) : s.b;
    if (b < 0) return;                                      // (bounds out of order)
    const int held = p.lengths[b];
    if (held >= 0 && (int64_t)held + at < p.places) p.out[b * p.sb + hk * p.sh + held + at] += sum;
}

// A workgroup's block of keys, and the share of its stream; sums go to to[key], or where they belong (nullptr).  The first workgroups have the
// first keys' blocks: with the shares of the others, a block whose stream is the whole sequence is the last to end (8192 queries of 16 heads,
// window 512, 4 first keys: 84 us instead of 62; 131072 queries take 670, 500 without first keys)
struct KeyBlock {
    Span s;
    int hk, share, chunk;
    float* to;
};
__device__ __forceinline__ bool key_block(const KeySums& p, int pid, int block, KeyBlock& w) {
    if (pid < p.front_grid) {
        const int blocks = p.front / block, sequences = p.rows.cu ? p.rows.sequences : p.rows.B;
        w.share = pid % p.front_shares;
        pid /= p.front_shares;
        w.hk = pid % p.HK;
        pid /= p.HK;
        const int at = pid % blocks, sequence = pid / blocks;
        if (sequence >= sequences) return false;            // (the grid of these is a multiple of eight)
        w.s = Span{sequence, 0, p.rows.N, at, false};
        if (p.rows.cu) {
            const auto bound = [&](int i) { const int x = p.rows.cu[i]; return x < 0 ? 0 : x > p.rows.N ? p.rows.N : x; };
            w.s.b = 0;
            w.s.first = __builtin_amdgcn_readfirstlane(bound(sequence));
            w.s.len = __builtin_amdgcn_readfirstlane(bound(sequence + 1)) - w.s.first;
        }
        w.chunk = p.front_chunk;
        w.to = p.front_shares > 1 ? p.front_part + (((int64_t)w.share * sequences + sequence) * p.HK + w.hk) * p.front : nullptr;
        return (int64_t)at * block < w.s.len;
    }
    int stream, tile;
    order(pid - p.front_grid, p.rows.B * p.HK, stream, tile);            // (a block's shares behind each other, so that no XCD has only late, empty ones)
    w.share = tile % p.shares;
    w.hk = stream % p.HK;
    w.chunk = p.chunk;
    if (!find_tile(p.rows, stream / p.HK, tile / p.shares, block, w.s)) return false;
    w.to = p.shares > 1 ? p.part + (((int64_t)w.share * p.rows.B + w.s.b) * p.HK + w.hk) * p.rows.N + w.s.first : nullptr;
    return w.s.fill || (int64_t)w.s.block * block >= p.front;
}
inline int64_t key_blocks(const KeySums& p, int block) { return (int64_t)p.rows.B * p.HK * p.shares * count_tiles(p.rows, block); }

}  // namespace
}  // namespace sa2
