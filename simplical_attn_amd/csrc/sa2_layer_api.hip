// extern "C" boundary of the operators of ordinary attention layers: argument validation and kernel choice.
// No allocation, no synchronisation, no state.
#include <math.h>
#include <string.h>

#include "sa2_causal_common.h"

using namespace sa2;

namespace {

bool valid_dtype(int dtype) { return dtype == SA2_F32 || dtype == SA2_BF16 || dtype == SA2_F16; }

Tensor tensor(const void* p, const int64_t* strides, int which) {
    return Tensor{const_cast<void*>(p), strides[3 * which], strides[3 * which + 1], strides[3 * which + 2]};
}

// a size-1 axis may carry any stride; otherwise strides must be positive
bool stride_ok(const Tensor& t, int B, int N, int H) { return (B <= 1 || t.sb > 0) && (N <= 1 || t.sn > 0) && (H <= 1 || t.sh > 0); }

int check_rows(int B, int N, int H, int D, const int32_t* cu, int sequences, int dtype) {
    if (!valid_dtype(dtype)) return SA2_ERR_BAD_DTYPE;
    if (B < 1 || N < 1 || H < 1 || D < 1 || D > 256) return SA2_ERR_BAD_SHAPE;
    if (cu && (B != 1 || sequences < 1)) return SA2_ERR_BAD_SHAPE;
    if ((int64_t)B * H * N > 0x7fffffffLL || (int64_t)N + sequences > 0x7fffffffLL) return SA2_ERR_TOO_LARGE;
    return SA2_OK;
}

int make_causal(Causal& p, const int32_t* cu, int sequences, int B, int N, int H, int HK, int D, float scale, int dtype) {
    const int rc = check_rows(B, N, H, D, cu, sequences, dtype);
    if (rc != SA2_OK) return rc;
    if (HK < 1 || H % HK) return SA2_ERR_BAD_HEADS;
    memset(&p, 0, sizeof(p));
    p.rows = Rows{B, N, cu, sequences};
    p.H = H; p.HK = HK; p.G = H / HK; p.D = D;
    p.scale = scale;
    return SA2_OK;
}
// Rows that the kernels of windows and of keys' weights take: row numbers up to two blocks of 256 behind the last row fit 31 bits
constexpr int BAND_ROWS = 0x7fffffff - 1023;
// window 0: none
int make_band(Causal& p, int window, int sinks) {
    if (window < 0 || sinks < 0) return SA2_ERR_BAD_WINDOW;
    if (window == 0 || window >= p.rows.N) return SA2_OK;                  // (every key of the sequence is in reach)
    p.band.window = window;
    p.band.sinks = sinks < p.rows.N ? sinks : p.rows.N;
    p.band.alone = window == 1 && sinks == 0 ? 0x7fffffff : 0;
    if (p.rows.N > BAND_ROWS || p.band.sinks > 65535) return SA2_ERR_TOO_LARGE;
    // (where the first keys are many, longer chunks, so that their sums stay of the tensors' size; of many short sequences: see Band)
    p.band.chunk = 128 * (p.band.sinks > 128 ? (p.band.sinks + 127) / 128 : 1);
    const int64_t chunks = sink_groups(p, 0), rows = 2 * (int64_t)p.rows.B * p.rows.N;
    p.band.by_rows = chunks * p.band.sinks > rows;         // (of a batch never: ceil(N / chunk) sinks <= N + sinks)
    p.band.sink_rows = p.band.by_rows ? rows : chunks * p.band.sinks;
    return SA2_OK;
}
size_t row_bytes(const Causal& p, int heads) { return ((size_t)p.rows.B * heads * p.rows.N * sizeof(float) + 255) / 256 * 256; }
size_t delta_bytes(const Causal& p) { return row_bytes(p, p.H); }

int check_tree(int B, int T, int H, int HK, int D, int dtype) {
    const int rc = check_rows(B, T, H, D, nullptr, 0, dtype);
    if (rc != SA2_OK) return rc;
    if (HK < 1 || H % HK) return SA2_ERR_BAD_HEADS;
    return T > SA2_TREE_NODES ? SA2_ERR_BAD_TREE : SA2_OK;
}
// Workgroups that share a sequence's keys: as many as are on the chip at once, one per CU, each with at least four tiles of 32
// keys (one per wavefront; eight where the wavefronts share them) of what a sequence may hold, at most 64 (how many it does hold is known on the device only)
int tree_splits(int B, int T, int H, int HK, int D, int page_size, int table_width, int window, int sinks, int dtype) {
    const int64_t reach = tree_reach((int64_t)page_size * table_width, T, window, sinks), keys = (int64_t)B * HK * reach;
    const int rows = T * (H / HK), block = dtype == SA2_F32 ? 32 : tree16_rows(rows, keys), least = block > 64 ? 8 : 4;
    const int64_t streams = (int64_t)B * HK * ((rows + block - 1) / block), tiles = (reach + 31) / 32;
    int64_t n = CUS / streams;
    if (n > tiles / least) n = tiles / least;
    return n < 1 ? 1 : n > 64 ? 64 : (int)n;
}

// Prompts; window 0: every key up to the query's own
int prompt_forward(const void* q, const void* k, const void* v, void* out, void* out_low, float* lse,
                   const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                   const int64_t* strides, int window, int sinks, float scale, int dtype, unsigned flags, void* hip_stream) {
    if (!q || !k || !v || !out || !lse || !strides) return SA2_ERR_NULL_POINTER;
    Causal p;
    int rc = make_causal(p, cu_seqlens, sequences, B, N, H, HK, D, scale, dtype);
    if (rc == SA2_OK) rc = make_band(p, window, sinks);
    if (rc != SA2_OK) return rc;
    p.q = tensor(q, strides, 0);
    p.k = tensor(k, strides, 1);
    p.v = tensor(v, strides, 2);
    p.out = tensor(out, strides, 3);
    p.out_low = dtype == SA2_F32 ? nullptr : out_low;
    p.lse = lse;
    if (!stride_ok(p.q, B, N, H) || !stride_ok(p.out, B, N, H) || !stride_ok(p.k, B, N, HK) || !stride_ok(p.v, B, N, HK)) return SA2_ERR_BAD_STRIDE;
    const hipStream_t st = (hipStream_t)hip_stream;
    const bool narrow = !(flags & SA2_FLAG_FORCE_GENERIC) && causal16_supported(D, dtype) && causal16_layout(p, {&p.q, &p.k, &p.v, &p.out}) && !((uintptr_t)out_low & 15u);
    if (p.band.window) return narrow ? launch_window16_fwd(p, dtype, st) : launch_window_f32_fwd(p, dtype, st);
    return narrow ? launch_causal16_fwd(p, dtype, st) : launch_causal_f32_fwd(p, dtype, st);
}

size_t prompt_workspace(int sequences, int B, int N, int H, int HK, int D, int window, int sinks, int dtype, unsigned flags) {
    Causal p;
    static const int32_t packed = 0;                       // (only whether there are packed sequences counts here)
    if (make_causal(p, sequences > 0 ? &packed : nullptr, sequences, B, N, H, HK, D, 1.f, dtype) != SA2_OK || make_band(p, window, sinks) != SA2_OK) return 0;
    if (p.band.window) {
        const bool narrow = !(flags & SA2_FLAG_FORCE_GENERIC) && causal16_supported(D, dtype);
        const size_t terms = narrow ? delta_bytes(p) + (dtype == SA2_F16 ? 2 * delta_bytes(p) + 2 * row_bytes(p, HK) : 0) + window16_part_bytes(p) : 0;
        return (delta_bytes(p) + terms + sink_part_bytes(p) + 255) / 256 * 256;
    }
    if ((flags & SA2_FLAG_FORCE_GENERIC) || !causal16_supported(D, dtype)) return delta_bytes(p);
    return 2 * delta_bytes(p) + (dtype == SA2_F16 ? delta_bytes(p) + row_bytes(p, HK) : 0) + causal16_part_bytes(B, N, HK, p.G, D);
}

int prompt_backward(const void* q, const void* k, const void* v, const void* out, const void* out_low, const void* dout, const float* lse,
                    void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                    const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                    const int64_t* strides, int window, int sinks, float scale, int dtype, unsigned flags, void* hip_stream) {
    if (!q || !k || !v || !out || !dout || !lse || !workspace || !strides) return SA2_ERR_NULL_POINTER;
    Causal p;
    int rc = make_causal(p, cu_seqlens, sequences, B, N, H, HK, D, scale, dtype);
    if (rc == SA2_OK) rc = make_band(p, window, sinks);
    if (rc != SA2_OK) return rc;
    Tensor* const t[8] = {&p.q, &p.k, &p.v, &p.out, &p.dout, &p.dq, &p.dk, &p.dv};
    const void* const at[8] = {q, k, v, out, dout, dq, dk, dv};
    for (int i = 0; i < 8; ++i) {
        *t[i] = tensor(at[i], strides, i);
        if (at[i] && !stride_ok(*t[i], B, N, i == 1 || i == 2 || i > 5 ? HK : H)) return SA2_ERR_BAD_STRIDE;
    }
    if (((uintptr_t)workspace & 255u) || workspace_bytes < prompt_workspace(cu_seqlens ? sequences : 0, B, N, H, HK, D, window, sinks, dtype, flags)) return SA2_ERR_WORKSPACE_TOO_SMALL;
    p.out_low = dtype == SA2_F32 ? nullptr : const_cast<void*>(out_low);
    p.lse = const_cast<float*>(lse);
    p.delta = (float*)workspace;
    const hipStream_t st = (hipStream_t)hip_stream;
    if (!dq && !dk && !dv) return SA2_OK;
    char* behind = (char*)workspace + delta_bytes(p);
    auto next = [&](size_t bytes) { char* const here = behind; behind += bytes; return (float*)here; };
    // (-lse / scale is one of the 16-bit kernels' operands)
    const bool narrow = !(flags & SA2_FLAG_FORCE_GENERIC) && causal16_supported(D, dtype) && causal16_layout(p, {&p.q, &p.k, &p.v, &p.out, &p.dout, &p.dq, &p.dk, &p.dv}) &&
                        fabsf(scale) > 1e-20f && !((uintptr_t)out_low & 15u);
    if (p.band.window) {
        Causal16Terms terms{};
        if (narrow) {
            terms.minus_lse = next(delta_bytes(p));
            if (dtype == SA2_F16) {
                terms.dout = next(delta_bytes(p));
                terms.queries = next(delta_bytes(p));
                terms.v = next(row_bytes(p, HK));
                terms.keys = next(row_bytes(p, HK));
            }
            p.part = next(window16_part_bytes(p));
        }
        p.sink_part = next(0);
        return narrow ? launch_window16_bwd(p, dtype, terms, st) : launch_window_f32_bwd(p, dtype, st);
    }
    if (narrow) {
        Causal16Terms terms{next(delta_bytes(p)), nullptr, nullptr};
        if (dtype == SA2_F16) {
            terms.dout = next(delta_bytes(p));
            terms.v = next(row_bytes(p, HK));
        }
        p.part = next(0);
        return launch_causal16_bwd(p, dtype, terms, st);
    }
    return launch_causal_f32_bwd(p, dtype, st);
}

// Tiles of 32 scores that a row of query leaves at most, its own node's among them
int64_t tree_span(int page_size, int table_width, int window, int sinks) {
    const int64_t all = ((int64_t)page_size * table_width + 31) / 32, seen = ((int64_t)window + sinks) / 32 + 4;
    return 32 * ((window && seen < all ? seen : all) + 1);
}
// A window that every cached row is in is none
int tree_window_of(int T, int page_size, int table_width, int window) { return window >= (int64_t)page_size * table_width + T ? 0 : window; }
size_t tree_parts(int B, int T, int H, int D, int nsplit, bool weighted) { return (tree_part_bytes(B, T, H, D, nsplit, weighted) + 255) / 256 * 256; }

size_t tree_workspace(int B, int T, int H, int HK, int D, int page_size, int table_width, int window, int sinks, bool weighted, int dtype) {
    if (check_tree(B, T, H, HK, D, dtype) != SA2_OK || page_size < 1 || table_width < 1 || window < 0 || sinks < 0 || (weighted && T != 1)) return 0;
    window = tree_window_of(T, page_size, table_width, window);
    const int nsplit = tree_splits(B, T, H, HK, D, page_size, table_width, window, sinks, dtype);
    if (!weighted) return tree_part_bytes(B, T, H, D, nsplit);
    return tree_parts(B, T, H, D, nsplit, true) + (size_t)B * H * tree_span(page_size, table_width, window, sinks) * sizeof(float);
}

// window 0: none; weights: wanted or nullptr, with their strides behind those of the tensors
int tree_attention(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache, void* out, float* weights,
                   const int32_t* parents, const int32_t* lengths, const int32_t* page_table,
                   void* workspace, size_t workspace_bytes, int B, int T, int H, int HK, int D,
                   int page_size, int pages, int table_width, const int64_t* strides, int window, int sinks, float scale,
                   int dtype, unsigned flags, void* hip_stream) {
    if (!q || !k || !v || !k_cache || !v_cache || !out || !lengths || !strides) return SA2_ERR_NULL_POINTER;
    const int rc = check_tree(B, T, H, HK, D, dtype);
    if (rc != SA2_OK) return rc;
    if (weights && T != 1) return SA2_ERR_BAD_TREE;
    if (page_size < 1 || pages < 1 || table_width < 1 || (!page_table && (pages < B || table_width != 1)) || (int64_t)page_size * table_width > 0x7fffffff - 64)
        return SA2_ERR_BAD_CACHE;
    window = tree_window_of(T, page_size, table_width, window);
    Tree p;
    memset(&p, 0, sizeof(p));
    p.B = B; p.T = T; p.H = H; p.HK = HK; p.G = H / HK; p.D = D;
    p.scale = scale;
    p.q = tensor(q, strides, 0);
    p.k = tensor(k, strides, 1);
    p.v = tensor(v, strides, 2);
    p.cache = Cache{tensor(k_cache, strides, 3), tensor(v_cache, strides, 4), page_table, lengths, page_size, pages, table_width};
    p.out = tensor(out, strides, 5);
    if (!stride_ok(p.q, B, T, H) || !stride_ok(p.out, B, T, H) || !stride_ok(p.k, B, T, HK) || !stride_ok(p.v, B, T, HK) ||
        !stride_ok(p.cache.k, pages, page_size, HK) || !stride_ok(p.cache.v, pages, page_size, HK))
        return SA2_ERR_BAD_STRIDE;
    p.parents = parents;
    p.nsplit = tree_splits(B, T, H, HK, D, page_size, table_width, window, sinks, dtype);
    p.part = (float*)workspace;
    const bool banded = window > 0 || weights;
    const size_t need = tree_workspace(B, T, H, HK, D, page_size, table_width, window, sinks, weights != nullptr, dtype);
    if (need && (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < need)) return SA2_ERR_WORKSPACE_TOO_SMALL;
    if (banded) {
        p.window = window > 0 ? window : 0x7fffffff;
        p.sinks = window > 0 ? sinks : 0;
    }
    if (weights) {
        p.weights = weights;
        p.weights_sb = strides[18];
        p.weights_sh = strides[19];
        if ((B > 1 && p.weights_sb < 1) || (HK > 1 && p.weights_sh < 1)) return SA2_ERR_BAD_STRIDE;
        p.scores = (float*)((char*)workspace + tree_parts(B, T, H, D, p.nsplit, true));
        p.span = tree_span(page_size, table_width, window, sinks);
        if ((int64_t)B * HK * ((p.span + 1023) / 1024) > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    }
    const bool narrow = !(flags & SA2_FLAG_FORCE_GENERIC) && (banded ? tree16_layout(p, dtype) : tree16_supported(p, dtype));
    p.dealt = B > 1 && p.nsplit >= 8 && (!narrow || (tree16_rows(p) > 64 && !weights));      // (sa2_tree16.h takes equal shares; 32 sequences at most)
    const hipStream_t st = (hipStream_t)hip_stream;
    if (banded) return narrow ? launch_window_tree16(p, dtype, st) : launch_window_tree_f32(p, dtype, st);
    return narrow ? launch_tree16(p, dtype, st) : launch_tree_f32(p, dtype, st);
}

// Shares of the streams of blocks of `block` keys in tiles of `tile` queries: about `all` of them, of `least` tiles or more.  Short prompts in many
// short shares: 512 queries of 16 heads over 4 key heads (head_dim 128) take 16 us with 4 tiles of 64 and 24 with 8, in fp32 23 with 2 tiles of
// 32 and 52 with 16; below these numbers the workgroups' starts and the join cost as much as they save.
void key_shares(KeySums& p, int block, int tile, int all, int least) {
    const int64_t N = p.rows.N, streams = (int64_t)p.rows.B * p.HK, longest = p.band.window && p.band.window + block < N ? p.band.window + block : N;
    const auto cut = [&](int64_t tiles, int64_t each) { return (int)(each < least ? least : each < tiles ? each : tiles); };
    const auto shares = [](int64_t tiles, int chunk) { return (int)((tiles + chunk - 1) / chunk); };
    const int64_t tiles = (longest + tile - 1) / tile * p.G, work = streams * ((N + block - 1) / block) * tiles / (p.band.window ? 1 : 2);
    p.chunk = cut(tiles, (work + all - 1) / all);
    p.shares = shares(tiles, p.chunk);
    p.front_shares = 1;
    if (!p.band.sinks) return;
    // (a block of the first keys: of every sequence, whatever its length)
    const int64_t blocks = (p.band.sinks + block - 1) / block, whole = (N + tile - 1) / tile * p.G, of_all = (int64_t)(p.rows.sequences ? p.rows.sequences : p.rows.B) * p.HK * blocks;
    p.front = (int)(blocks * block);
    p.front_chunk = cut(whole, (streams * blocks * whole + 1023) / 1024);
    p.front_shares = shares(whole, p.front_chunk);
    if (of_all * p.front_shares > 65536) {
        p.front_shares = of_all >= 65536 ? 1 : (int)(65536 / of_all);
        p.front_chunk = shares(whole, p.front_shares);
    }
    const int64_t grid = (of_all * p.front_shares + 7) / 8 * 8;
    p.front_grid = grid > 0x7fffffff ? -1 : (int)grid;
}
size_t key_part_bytes(const KeySums& p) { return p.shares > 1 ? ((size_t)p.shares * p.rows.B * p.HK * p.rows.N * sizeof(float) + 255) / 256 * 256 : 0; }
size_t key_parts_bytes(const KeySums& p) {
    return key_part_bytes(p) + (p.front_shares > 1 ? (size_t)p.front_shares * (p.rows.sequences ? p.rows.sequences : p.rows.B) * p.HK * p.front * sizeof(float) : 0);
}

int make_key_sums(KeySums& p, const int32_t* cu, int sequences, int B, int N, int H, int HK, int D, int window, int sinks, float scale, int dtype) {
    Causal c;
    int rc = make_causal(c, cu, sequences, B, N, H, HK, D, scale, dtype);
    if (rc != SA2_OK) return rc;
    if (window < 0 || sinks < 0) return SA2_ERR_BAD_WINDOW;
    if (N > BAND_ROWS) return SA2_ERR_TOO_LARGE;
    memset(&p, 0, sizeof(p));
    p.rows = c.rows;
    p.H = H; p.HK = HK; p.G = c.G; p.D = D;
    p.scale = scale;
    p.band.window = window < N ? window : 0;
    p.band.sinks = p.band.window ? (sinks < N ? sinks : N) : 0;
    if (p.band.sinks > 65535) return SA2_ERR_TOO_LARGE;
    key_shares(p, 128, 32, 1024, 2);
    return SA2_OK;
}
// for the kernels on the 16-bit MFMA.  4096 shares are more than fit on the card at once, so that the short ones of packed prompts fill the gaps:
// six of 8100 queries in all 97 us (1024: 158, 2048: 112)
KeySums narrow_sums(KeySums p) {
    key_shares(p, KEY_SUMS16_BLOCK, 64, 4096, 4);
    return p;
}
size_t key_sums_workspace(const KeySums& p, int dtype, unsigned flags) {
    const size_t wide = key_parts_bytes(p), narrow = causal16_supported(p.D, dtype) && !(flags & SA2_FLAG_FORCE_GENERIC) ? key_parts_bytes(narrow_sums(p)) : 0;
    return wide > narrow ? wide : narrow;                  // (which it is goes by the tensors' alignment)
}

}  // namespace

extern "C" {

int sa2_rotary(const void* q, const void* k, void* q_out, void* k_out, const double* frequencies,
               const void* positions, int position_bytes, const int32_t* cu_seqlens, int sequences,
               int B, int N, int H, int HK, int D, int rotary_dim, const int64_t* strides,
               float amplitude, int interleaved, int inverse, int dtype, void* hip_stream) {
    if (!q || !q_out || !frequencies || !strides || (HK > 0 && (!k || !k_out))) return SA2_ERR_NULL_POINTER;
    const int rc = check_rows(B, N, H, D, cu_seqlens, sequences, dtype);
    if (rc != SA2_OK) return rc;
    if (HK < 0) return SA2_ERR_BAD_SHAPE;
    if ((int64_t)B * N * HK > 0x7fffffffLL) return SA2_ERR_TOO_LARGE;
    if (rotary_dim < 2 || rotary_dim > D || (rotary_dim & 1) || (positions && position_bytes != 4 && position_bytes != 8))
        return SA2_ERR_BAD_ROTARY;
    Rotary p;
    memset(&p, 0, sizeof(p));
    p.rows = Rows{B, N, cu_seqlens, sequences};
    p.H = H; p.HK = HK; p.D = D; p.rot = rotary_dim;
    p.q = tensor(q, strides, 0);
    p.k = tensor(k, strides, 1);
    p.q_out = tensor(q_out, strides, 2);
    p.k_out = tensor(k_out, strides, 3);
    for (const Tensor* t : {&p.q, &p.q_out})
        if (!stride_ok(*t, B, N, H)) return SA2_ERR_BAD_STRIDE;
    for (const Tensor* t : {&p.k, &p.k_out})
        if (HK > 0 && !stride_ok(*t, B, N, HK)) return SA2_ERR_BAD_STRIDE;
    p.frequencies = frequencies;
    p.positions = positions;
    p.position_bytes = position_bytes;
    p.amplitude = amplitude;
    p.interleaved = interleaved;
    p.inverse = inverse;
    return launch_rotary(p, dtype, (hipStream_t)hip_stream);
}

int sa2_cache_append(const void* k, const void* v, void* k_cache, void* v_cache, const int32_t* lengths,
                     const int32_t* page_table, const int32_t* rows, int nrows,
                     const int32_t* cu_seqlens, int sequences, int B, int N, int HK, int D,
                     int page_size, int pages, int table_width, const int64_t* strides, int dtype, void* hip_stream) {
    if (!k || !v || !k_cache || !v_cache || !lengths || !strides) return SA2_ERR_NULL_POINTER;
    const int rc = check_rows(B, N, HK, D, cu_seqlens, sequences, dtype);
    if (rc != SA2_OK) return rc;
    if (rows && (nrows < 1 || cu_seqlens)) return SA2_ERR_BAD_SHAPE;
    if (page_size < 1 || pages < 1 || (page_table ? table_width < 1 : pages < (cu_seqlens ? sequences : B))) return SA2_ERR_BAD_CACHE;
    Append p;
    memset(&p, 0, sizeof(p));
    p.cache.k = tensor(k_cache, strides, 2);
    p.cache.v = tensor(v_cache, strides, 3);
    p.cache.table = page_table;
    p.cache.lengths = lengths;
    p.cache.page_size = page_size;
    p.cache.pages = pages;
    p.cache.width = table_width;
    p.rows = Rows{B, N, cu_seqlens, sequences};
    p.HK = HK; p.D = D;
    p.k = tensor(k, strides, 0);
    p.v = tensor(v, strides, 1);
    p.chosen = rows;
    p.nchosen = nrows;
    for (const Tensor* t : {&p.k, &p.v})
        if (!stride_ok(*t, B, N, HK)) return SA2_ERR_BAD_STRIDE;
    for (const Tensor* t : {&p.cache.k, &p.cache.v})
        if (!stride_ok(*t, pages, page_size, HK)) return SA2_ERR_BAD_STRIDE;
    return launch_append(p, dtype, (hipStream_t)hip_stream);
}

int sa2_causal_forward(const void* q, const void* k, const void* v, void* out, void* out_low, float* lse,
                       const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                       const int64_t* strides, float scale, int dtype, unsigned flags, void* hip_stream) {
    return prompt_forward(q, k, v, out, out_low, lse, cu_seqlens, sequences, B, N, H, HK, D, strides, 0, 0, scale, dtype, flags, hip_stream);
}
int sa2_window_forward(const void* q, const void* k, const void* v, void* out, void* out_low, float* lse,
                       const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                       const int64_t* strides, int window, int sinks, float scale, int dtype, unsigned flags, void* hip_stream) {
    if (window < 1) return SA2_ERR_BAD_WINDOW;
    return prompt_forward(q, k, v, out, out_low, lse, cu_seqlens, sequences, B, N, H, HK, D, strides, window, sinks, scale, dtype, flags, hip_stream);
}

size_t sa2_causal_bwd_workspace_bytes(int B, int N, int H, int HK, int D, int dtype, unsigned flags) {
    return prompt_workspace(0, B, N, H, HK, D, 0, 0, dtype, flags);
}
size_t sa2_window_bwd_workspace_bytes(int sequences, int B, int N, int H, int HK, int D, int window, int sinks, int dtype, unsigned flags) {
    return window < 1 ? 0 : prompt_workspace(sequences, B, N, H, HK, D, window, sinks, dtype, flags);
}

int sa2_causal_backward(const void* q, const void* k, const void* v, const void* out, const void* out_low, const void* dout, const float* lse,
                        void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                        const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                        const int64_t* strides, float scale, int dtype, unsigned flags, void* hip_stream) {
    return prompt_backward(q, k, v, out, out_low, dout, lse, dq, dk, dv, workspace, workspace_bytes, cu_seqlens, sequences, B, N, H, HK, D, strides, 0, 0, scale, dtype, flags, hip_stream);
}
int sa2_window_backward(const void* q, const void* k, const void* v, const void* out, const void* out_low, const void* dout, const float* lse,
                        void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                        const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                        const int64_t* strides, int window, int sinks, float scale, int dtype, unsigned flags, void* hip_stream) {
    if (window < 1) return SA2_ERR_BAD_WINDOW;
    return prompt_backward(q, k, v, out, out_low, dout, lse, dq, dk, dv, workspace, workspace_bytes, cu_seqlens, sequences, B, N, H, HK, D, strides, window, sinks, scale, dtype, flags, hip_stream);
}

size_t sa2_tree_workspace_bytes(int B, int T, int H, int HK, int D, int page_size, int table_width, int dtype, unsigned flags) {
    return tree_workspace(B, T, H, HK, D, page_size, table_width, 0, 0, false, dtype);
}
size_t sa2_window_tree_workspace_bytes(int B, int T, int H, int HK, int D, int page_size, int table_width, int window, int sinks, int weighted, int dtype, unsigned flags) {
    return tree_workspace(B, T, H, HK, D, page_size, table_width, window, sinks, weighted != 0, dtype);
}

int sa2_tree_attention(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache, void* out,
                       const int32_t* parents, const int32_t* lengths, const int32_t* page_table,
                       void* workspace, size_t workspace_bytes, int B, int T, int H, int HK, int D,
                       int page_size, int pages, int table_width, const int64_t* strides, float scale,
                       int dtype, unsigned flags, void* hip_stream) {
    return tree_attention(q, k, v, k_cache, v_cache, out, nullptr, parents, lengths, page_table, workspace, workspace_bytes, B, T, H, HK, D, page_size, pages, table_width, strides, 0, 0, scale, dtype,
                          flags, hip_stream);
}
int sa2_window_tree_attention(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache, void* out, float* weights,
                              const int32_t* parents, const int32_t* lengths, const int32_t* page_table,
                              void* workspace, size_t workspace_bytes, int B, int T, int H, int HK, int D,
                              int page_size, int pages, int table_width, const int64_t* strides, int window, int sinks, float scale,
                              int dtype, unsigned flags, void* hip_stream) {
    if (window < 0 || sinks < 0) return SA2_ERR_BAD_WINDOW;
    return tree_attention(q, k, v, k_cache, v_cache, out, weights, parents, lengths, page_table, workspace, workspace_bytes, B, T, H, HK, D, page_size, pages, table_width, strides, window, sinks,
                          scale, dtype, flags, hip_stream);
}

size_t sa2_key_weights_workspace_bytes(int sequences, int B, int N, int H, int HK, int D, int window, int sinks, int dtype, unsigned flags) {
    KeySums p;
    static const int32_t packed = 0;                       // (only whether there are packed sequences counts here)
    return make_key_sums(p, sequences > 0 ? &packed : nullptr, sequences, B, N, H, HK, D, window, sinks, 1.f, dtype) == SA2_OK ? key_sums_workspace(p, dtype, flags) : 0;
}
int sa2_key_weights(const void* q, const void* k, const float* lse, float* weights, const int32_t* lengths, int64_t places, void* workspace, size_t workspace_bytes,
                    const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D, const int64_t* strides, int window, int sinks, float scale,
                    int dtype, unsigned flags, void* hip_stream) {
    if (!q || !k || !lse || !weights || !strides) return SA2_ERR_NULL_POINTER;
    KeySums p;
    const int rc = make_key_sums(p, cu_seqlens, sequences, B, N, H, HK, D, window, sinks, scale, dtype);
    if (rc != SA2_OK) return rc;
    p.q = tensor(q, strides, 0);
    p.k = tensor(k, strides, 1);
    p.lse = lse;
    p.out = weights;
    p.sb = strides[6];
    p.sh = strides[7];
    p.lengths = lengths;
    p.places = places;
    const int outer = cu_seqlens && lengths ? sequences : B;
    if (!stride_ok(p.q, B, N, H) || !stride_ok(p.k, B, N, HK) || (outer > 1 && p.sb < 1) || (HK > 1 && p.sh < 1)) return SA2_ERR_BAD_STRIDE;
    if (lengths && places < 1) return SA2_ERR_BAD_SHAPE;
    const size_t need = key_sums_workspace(p, dtype, flags);
    if (need && (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < need)) return SA2_ERR_WORKSPACE_TOO_SMALL;
    const bool narrow = !(flags & SA2_FLAG_FORCE_GENERIC) && key_sums16_supported(p, dtype);
    if (narrow) p = narrow_sums(p);
    if (p.front_grid < 0) return SA2_ERR_TOO_LARGE;
    p.part = (float*)workspace;
    p.front_part = (float*)((char*)workspace + key_part_bytes(p));
    if (narrow) return launch_key_sums16(p, dtype, (hipStream_t)hip_stream);
    return launch_key_sums_f32(p, dtype, (hipStream_t)hip_stream);
}

int sa2_cache_evict(void* k_cache, void* v_cache, const float* weights, float* left, int32_t* kept, const int32_t* lengths, const int32_t* page_table,
                    int B, int HK, int heads, int D, int page_size, int pages, int table_width, int64_t places, int keep, int first, int recent,
                    const int64_t* strides, int dtype, void* hip_stream) {
    if (!k_cache || !v_cache || !weights || !left || !kept || !lengths || !strides) return SA2_ERR_NULL_POINTER;
    if (!valid_dtype(dtype)) return SA2_ERR_BAD_DTYPE;
    if (B < 1 || HK < 1 || D < 1 || D > 256) return SA2_ERR_BAD_SHAPE;
    if (heads != HK && heads != 1) return SA2_ERR_BAD_HEADS;
    if (page_size < 1 || pages < 1 || table_width < 1 || (!page_table && (pages < B || table_width != 1)) || (int64_t)page_size * table_width > 0x7fffffff - 64) return SA2_ERR_BAD_CACHE;
    if (keep < 1 || first < 0 || recent < 0 || (int64_t)first + recent > keep || places < (int64_t)page_size * table_width) return SA2_ERR_BAD_EVICTION;
    Evict p;
    memset(&p, 0, sizeof(p));
    p.cache = Cache{tensor(k_cache, strides, 0), tensor(v_cache, strides, 1), page_table, lengths, page_size, pages, table_width};
    if (!stride_ok(p.cache.k, pages, page_size, HK) || !stride_ok(p.cache.v, pages, page_size, HK)) return SA2_ERR_BAD_STRIDE;
    p.B = B; p.HK = HK; p.heads = heads; p.D = D;
    p.weights = weights;
    p.sb = strides[6];
    p.sh = strides[7];
    if ((B > 1 && p.sb < 1) || (heads > 1 && p.sh < 1)) return SA2_ERR_BAD_STRIDE;
    p.places = places;
    p.left = left;
    p.kept = kept;
    p.keep = keep; p.first = first; p.recent = recent;
    return launch_evict(p, dtype, (hipStream_t)hip_stream);
}

}  // extern "C"
