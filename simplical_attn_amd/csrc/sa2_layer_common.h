// Shared declarations of the kernels of ordinary attention layers (rotary positions, causal attention over prompts,
// cache rows, drafted trees).
#pragma once

#include <initializer_list>

#include "sa2_common.h"
#include "sa2_mfma_common.h"

namespace sa2 {

// Rows of a problem: B sequences of N rows each, or (cu != nullptr) B = 1 and `sequences` packed ones, sequence s in
// the rows cu[s] .. cu[s+1]-1 of the N.  The bounds lie in device memory: kernels clamp them to 0 .. N.
struct Rows {
    int B, N;
    const int32_t* cu;
    int sequences;
};

// What queries see besides the causal mask (window 0: every key before them): the last `window` keys up to their own, and the first
// `sinks` ones of the sequence.  Gradients of the first keys, which all queries see, are made by workgroups of their own, each with
// `chunk` queries of a sequence (of all heads that share the keys), whose fp32 sums meet in a last launch.  A chunk has `sinks` rows of sums,
// or (`by_rows`), where those of many short packed sequences would be more than twice the tensors' rows, as many as its sequence has first keys: chunk c
// of the sequence whose rows begin at n has those from 2 n + c min(sinks, its length) on.  (chunk is sinks or more, so that 2 len rows are enough.)
struct Band {
    int window, sinks;
    int alone;                                 // queries up to this number see their own key only
    int chunk;
    bool by_rows;
    int64_t sink_rows;                         // in all, of a key head
};

// One call of causal attention.  H query heads share HK heads of keys and values, G = H / HK neighbours one.
struct Causal {
    Rows rows;
    int H, HK, G, D;
    float scale;
    Tensor q, k, v, out, dout, dq, dk, dv;     // gradients with p == nullptr: not requested
    void* out_low;                             // laid out as out, or nullptr: what rounding out to 16 bits left
    float* lse;                                // [B,H,N]
    float* delta;                              // [B,H,N]  sum_d dout*(out + out_low)
    float* part;                               // partial sums (path specific)
    Band band;
    float* sink_part;                          // [dK, dV][HK][sink_rows][D]: the first keys' sums
};

struct Rotary {
    Rows rows;
    int H, HK, D, rot;
    Tensor q, k, q_out, k_out;
    const double* frequencies;                 // [rot / 2], radians per position
    const void* positions;                     // [B,N] of position_bytes each, or nullptr: the row's place in its sequence
    int position_bytes;
    float amplitude;
    int interleaved, inverse;
};

// A cache of keys and values: `pages` pieces of `page_size` rows (sn: from row to row, sb: from page to page).  Row r of
// sequence b lies in page table[b * width + r / page_size], or without a table in page b.
struct Cache {
    Tensor k, v;
    const int32_t* table;
    const int32_t* lengths;                    // [B] rows that are there
    int page_size, pages, width;
};

struct Append {
    Cache cache;
    Rows rows;                                 // of the new rows
    int HK, D;
    Tensor k, v;
    const int32_t* chosen;                     // [B, nchosen] rows of the sequence's N to take, or nullptr: all
    int nchosen;
};

// Nodes of drafted trees over a cache: the G query heads of a key head and the T nodes make R = T * G rows that read the
// same keys; row r is node r / G, head r % G of the G.  The keys of the B sequences are cut into shares, nsplit * B units in all
// (sa2_tree_common.h), whose outputs, not yet divided by their sums, lie in `part`: [units][HK][R] pairs (reference point, sum),
// then [units][HK][R][width] values.
struct Tree {
    Cache cache;
    int B, T, H, HK, G, D;
    float scale;
    Tensor q, k, v, out;
    const int32_t* parents;                    // [B,T], or nullptr: a chain
    float* part;
    int nsplit;
    bool dealt;                                // shares by the sequences' lengths
    // Kernels with BAND only.  A node sees of the cached rows and of its ancestors the last `window` up to itself, and the first `sinks`
    // ones; where `weights` are wanted (trees of one node), the scores of all rows go to `scores`, [B][HK][R][span] by the numbers
    // that the sweep gives the rows, and a second launch adds what they weigh to weights[b, hk, place].
    int window, sinks;
    float *weights, *scores;
    int64_t weights_sb, weights_sh, span;
};
__host__ __device__ constexpr int tree_width(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
inline size_t tree_part_bytes(int B, int T, int H, int D, int nsplit, bool always = false) {
    return nsplit > 1 || always ? (size_t)nsplit * B * T * H * (tree_width(D) + 2) * sizeof(float) : 0;
}

// What each key of a prompt got from the queries that see it: sums of e^(scale q k - lse) over them and over the G query heads.  The stream
// of a block of keys, tiles of queries of one head after the other, is cut into shares of `chunk` tiles, whose sums lie in `part`:
// [share][B][HK][N].
struct KeySums {
    Rows rows;
    int H, HK, G, D;
    float scale;
    Tensor q, k;
    const float* lse;                          // [B,H,N]
    Band band;                                 // (window, sinks)
    float* part;
    int shares, chunk;
    // With a window, the blocks of the first keys, which all queries see: `front` keys of every sequence, in shares of their own
    int front, front_shares, front_chunk;
    float* front_part;                         // [front_shares][sequence][HK][front]
    int front_grid;
    // out[b * sb + hk * sh + n]; or with `lengths`, added to place lengths[b] + (n in its sequence b) where that is below `places`
    float* out;
    int64_t sb, sh;
    const int32_t* lengths;
    int64_t places;
};

// Rows of a cache that stay: kept[b, head, i] (ascending, -1 behind them) goes to place i.  One choice for each key head, or (heads 1) one for
// all of them.
struct Evict {
    Cache cache;
    int B, HK, heads, D;
    const float* weights;                      // [B][heads][..places], strides sb, sh
    int64_t sb, sh, places;
    float* left;                               // [B][heads][places]: of the rows that stay, zeros behind
    int32_t* kept;                             // [B][heads][keep]
    int keep, first, recent;
};

constexpr int KEY_SUMS16_BLOCK = 256;                      // keys of a workgroup
bool key_sums16_supported(const KeySums& p, int dtype);
int launch_key_sums16(const KeySums& p, int dtype, hipStream_t st);
int launch_key_sums_f32(const KeySums& p, int dtype, hipStream_t st);
int launch_key_sums_join(const KeySums& p, int block, int tile, hipStream_t st);
int launch_evict(const Evict& p, int dtype, hipStream_t st);
int launch_rotary(const Rotary& p, int dtype, hipStream_t st);
int launch_append(const Append& p, int dtype, hipStream_t st);
int launch_causal_f32_fwd(const Causal& p, int dtype, hipStream_t st);
int launch_causal_f32_bwd(const Causal& p, int dtype, hipStream_t st);
// with p.band
int launch_window_f32_fwd(const Causal& p, int dtype, hipStream_t st);
int launch_window_f32_bwd(const Causal& p, int dtype, hipStream_t st);
int launch_window_f32_narrow_fwd(const Causal& p, int dtype, bool wide, hipStream_t st);
int launch_window_f32_narrow_bwd(const Causal& p, int dtype, bool wide, hipStream_t st);
size_t sink_part_bytes(const Causal& p);
int launch_sink_sums(const Causal& p, int dtype, hipStream_t st);
// the same, head_dim up to 128: the four wavefronts of a workgroup share its 32 rows and divide what these see
int launch_causal_f32_narrow_fwd(const Causal& p, int dtype, bool wide, hipStream_t st);
int launch_causal_f32_narrow_bwd(const Causal& p, int dtype, bool wide, hipStream_t st);
// bf16 and fp16 with a head_dim up to 128 that is a multiple of 8, rows on the 16-byte grid
bool causal16_supported(int D, int dtype);
bool causal16_layout(const Causal& p, std::initializer_list<const Tensor*> ts);
// whether a wavefront owns two blocks of 32 queries (forward, dQ)
bool causal16_two(const Causal& p);
int launch_causal16_fwd(const Causal& p, int dtype, hipStream_t st);
int launch_window16_fwd(const Causal& p, int dtype, hipStream_t st);
// Their backward.  Row terms: p.delta receives -delta; fp16: the Euclidean norms of rows bound dS
struct Causal16Terms {
    float* minus_lse;                          // [B,H,N]  -lse / scale; fp16: what weights are lifted by added (sa2_causal_dkv16.h)
    float* dout;                               // [B,H,N]  |dout|, fp16 only
    float* v;                                  // [B,HK,N] |v|, fp16 only
    float *queries, *keys;                     // [B,H,N], [B,HK,N]: the factors of rows of dQ and of keys (sa2_causal16.h), fp16 with a band only
};
int causal16_splits(int B, int N, int HK, int G);
size_t causal16_part_bytes(int B, int N, int HK, int G, int D);
int launch_causal16_bwd(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st);
int launch_causal16_dq(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st);
// rows of the cache that a sequence's nodes see at most
inline int64_t tree_reach(int64_t capacity, int T, int window, int sinks) {
    const int64_t reach = (int64_t)window + sinks + T;
    return window && reach < capacity ? reach : capacity;
}
// With p.band: shares of the key blocks' streams, the largest number of their sums' bytes; the whole backward
int window16_splits(const Causal& p);
size_t window16_part_bytes(const Causal& p);
int launch_window16_bwd(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st);
int launch_tree_f32(const Tree& p, int dtype, hipStream_t st);
int launch_window_tree_f32(const Tree& p, int dtype, hipStream_t st);
int launch_window_tree16(const Tree& p, int dtype, hipStream_t st);
int launch_window_tree_rows16(const Tree& p, int dtype, hipStream_t st);
// 16-bit kernels: rows that a workgroup has of R; up to 64 its wavefronts share them and divide the keys, beyond it is the other
// way round (16/4 heads, 4 x 65536 cached rows, head_dim 128, 192 rows: 398 us dividing keys, 161 dividing rows).  From 33 to 64
// it is the other way round too where a CU has 1024 keys or more (64 rows of head_dim 128: 4 x 65536 rows 148 us and 98, 32 x 2048
// 63 and 54; 8 x 2048 26.5 and 27.6, 512 rows 19 and 23).  `keys`: those that the cache may hold, of all sequences and key heads.
inline int tree16_rows(int R, int64_t keys) { return R <= 32 ? 32 : R <= 64 && keys < 1024 * CUS ? 64 : R <= 128 ? 128 : 256; }
inline int tree16_rows(const Tree& p) { return tree16_rows(p.T * p.G, (int64_t)p.B * p.HK * tree_reach((int64_t)p.cache.page_size * p.cache.width, p.T, p.window, p.sinks)); }
constexpr int TREE16_ENTRIES = 4096;                       // of the page table that a workgroup keeps in LDS
int launch_tree_rows16(const Tree& p, int dtype, hipStream_t st);
bool tree16_layout(const Tree& p, int dtype);
bool tree16_supported(const Tree& p, int dtype);
int launch_tree16(const Tree& p, int dtype, hipStream_t st);

namespace {

// The memory of V elements as 32-bit floats and back
template <class T, int V>
__device__ __forceinline__ void load_floats(const T* p, float (&x)[V]) {
    if constexpr (V * sizeof(T) == 16 && sizeof(T) == 4) {
        const float4 u = *(const float4*)p;
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else if constexpr (V * sizeof(T) == 16) {
        union { uint4 u; T e[8]; } w;
        w.u = *(const uint4*)p;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_float(w.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_float(p[i]);
    }
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, bf16_t*) { return ElemBF16::pack(a, b); }
__device__ __forceinline__ uint32_t pack_pair(float a, float b, f16_t*) { return ElemF16::pack(a, b); }
template <class T, int V>
__device__ __forceinline__ void store_floats(T* p, const float (&x)[V]) {
    if constexpr (V * sizeof(T) == 16 && sizeof(T) == 4) {
        *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    } else if constexpr (V * sizeof(T) == 16) {
        *(uint4*)p = make_uint4(pack_pair(x[0], x[1], p), pack_pair(x[2], x[3], p), pack_pair(x[4], x[5], p), pack_pair(x[6], x[7], p));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) from_float(x[i], p + i);
    }
}

// The sequence of packed row n, -1 where none holds it (cu is non-decreasing)
__device__ __forceinline__ int sequence_of(const Rows& r, int n) {
    int lo = 0, hi = r.sequences;                       // cu[lo] <= n < cu[hi], once both are checked
    if (n < r.cu[0] || n >= r.cu[hi]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (r.cu[mid] <= n) lo = mid;
        else hi = mid;
    }
    return lo;
}
// The place of packed row n in that sequence (a first bound below zero, down to the smallest int, is zero)
__device__ __forceinline__ int place_of(const Rows& r, int sequence, int n) {
    const int first = r.cu[sequence];
    return first < 0 ? n : n - first;
}

// All pointers and strides that a kernel's 16-byte accesses need
inline bool aligned16(const Tensor& t, int64_t size, bool batched) {
    return !((uintptr_t)t.p & 15u) && (t.sn * size) % 16 == 0 && (t.sh * size) % 16 == 0 && (!batched || (t.sb * size) % 16 == 0);
}

template <class F>
int for_type(int dtype, F&& f) {
    return dtype == SA2_F32 ? f((float*)nullptr) : dtype == SA2_BF16 ? f((bf16_t*)nullptr) : f((f16_t*)nullptr);
}

}  // namespace
}  // namespace sa2
