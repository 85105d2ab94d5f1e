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
    const int b = p.rows.cu ? sequence_of(p.rows, s.first) : s.b, held = p.lengths[b];
    if (held >= 0 && (int64_t)held + at < p.places) p.out[b * p.sb + hk * p.sh + held + at] += sum;
}

}  // namespace
}  // namespace sa2
