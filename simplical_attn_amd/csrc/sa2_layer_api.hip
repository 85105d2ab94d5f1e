// extern "C" boundary of the operators of ordinary attention layers: argument validation and kernel choice.
// No allocation, no synchronisation, no state.
#include <math.h>
#include <string.h>

#include "sa2_layer_common.h"

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
int tree_splits(int B, int T, int H, int HK, int D, int page_size, int table_width, int dtype) {
    const int64_t keys = (int64_t)B * HK * page_size * table_width;
    const int rows = T * (H / HK), block = dtype == SA2_F32 ? 32 : tree16_rows(rows, keys), least = block > 64 ? 8 : 4;
    const int64_t streams = (int64_t)B * HK * ((rows + block - 1) / block), tiles = ((int64_t)page_size * table_width + 31) / 32;
    int64_t n = CUS / streams;
    if (n > tiles / least) n = tiles / least;
    return n < 1 ? 1 : n > 64 ? 64 : (int)n;
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
    if (!q || !k || !v || !out || !lse || !strides) return SA2_ERR_NULL_POINTER;
    Causal p;
    const int rc = make_causal(p, cu_seqlens, sequences, B, N, H, HK, D, scale, dtype);
    if (rc != SA2_OK) return rc;
    p.q = tensor(q, strides, 0);
    p.k = tensor(k, strides, 1);
    p.v = tensor(v, strides, 2);
    p.out = tensor(out, strides, 3);
    p.out_low = dtype == SA2_F32 ? nullptr : out_low;
    p.lse = lse;
    if (!stride_ok(p.q, B, N, H) || !stride_ok(p.out, B, N, H) || !stride_ok(p.k, B, N, HK) || !stride_ok(p.v, B, N, HK)) return SA2_ERR_BAD_STRIDE;
    if (!(flags & SA2_FLAG_FORCE_GENERIC) && causal16_supported(D, dtype) && causal16_layout(p, {&p.q, &p.k, &p.v, &p.out}) && !((uintptr_t)out_low & 15u))
        return launch_causal16_fwd(p, dtype, (hipStream_t)hip_stream);
    return launch_causal_f32_fwd(p, dtype, (hipStream_t)hip_stream);
}

size_t sa2_causal_bwd_workspace_bytes(int B, int N, int H, int HK, int D, int dtype, unsigned flags) {
    Causal p;
    if (make_causal(p, nullptr, 0, B, N, H, HK, D, 1.f, dtype) != SA2_OK) return 0;
    if ((flags & SA2_FLAG_FORCE_GENERIC) || !causal16_supported(D, dtype)) return delta_bytes(p);
    return 2 * delta_bytes(p) + (dtype == SA2_F16 ? delta_bytes(p) + row_bytes(p, HK) : 0) + causal16_part_bytes(B, N, HK, p.G, D);
}

int sa2_causal_backward(const void* q, const void* k, const void* v, const void* out, const void* out_low, const void* dout, const float* lse,
                        void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                        const int32_t* cu_seqlens, int sequences, int B, int N, int H, int HK, int D,
                        const int64_t* strides, float scale, int dtype, unsigned flags, void* hip_stream) {
    if (!q || !k || !v || !out || !dout || !lse || !workspace || !strides) return SA2_ERR_NULL_POINTER;
    Causal p;
    const int rc = make_causal(p, cu_seqlens, sequences, B, N, H, HK, D, scale, dtype);
    if (rc != SA2_OK) return rc;
    Tensor* const t[8] = {&p.q, &p.k, &p.v, &p.out, &p.dout, &p.dq, &p.dk, &p.dv};
    const void* const at[8] = {q, k, v, out, dout, dq, dk, dv};
    for (int i = 0; i < 8; ++i) {
        *t[i] = tensor(at[i], strides, i);
        if (at[i] && !stride_ok(*t[i], B, N, i == 1 || i == 2 || i > 5 ? HK : H)) return SA2_ERR_BAD_STRIDE;
    }
    if (((uintptr_t)workspace & 255u) || workspace_bytes < sa2_causal_bwd_workspace_bytes(B, N, H, HK, D, dtype, flags)) return SA2_ERR_WORKSPACE_TOO_SMALL;
    p.out_low = dtype == SA2_F32 ? nullptr : const_cast<void*>(out_low);
    p.lse = const_cast<float*>(lse);
    p.delta = (float*)workspace;
    const hipStream_t st = (hipStream_t)hip_stream;
    if (!dq && !dk && !dv) return SA2_OK;
    // (-lse / scale is one of the 16-bit kernels' operands)
    if (!(flags & SA2_FLAG_FORCE_GENERIC) && causal16_supported(D, dtype) && causal16_layout(p, {&p.q, &p.k, &p.v, &p.out, &p.dout, &p.dq, &p.dk, &p.dv}) &&
        fabsf(scale) > 1e-20f && !((uintptr_t)out_low & 15u)) {
        char* at = (char*)workspace + delta_bytes(p);
        auto next = [&](size_t bytes) { char* const here = at; at += bytes; return (float*)here; };
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

size_t sa2_tree_workspace_bytes(int B, int T, int H, int HK, int D, int page_size, int table_width, int dtype, unsigned flags) {
    if (check_tree(B, T, H, HK, D, dtype) != SA2_OK || page_size < 1 || table_width < 1) return 0;
    return tree_part_bytes(B, T, H, D, tree_splits(B, T, H, HK, D, page_size, table_width, dtype));
}

int sa2_tree_attention(const void* q, const void* k, const void* v, const void* k_cache, const void* v_cache, void* out,
                       const int32_t* parents, const int32_t* lengths, const int32_t* page_table,
                       void* workspace, size_t workspace_bytes, int B, int T, int H, int HK, int D,
                       int page_size, int pages, int table_width, const int64_t* strides, float scale,
                       int dtype, unsigned flags, void* hip_stream) {
    if (!q || !k || !v || !k_cache || !v_cache || !out || !lengths || !strides) return SA2_ERR_NULL_POINTER;
    const int rc = check_tree(B, T, H, HK, D, dtype);
    if (rc != SA2_OK) return rc;
    if (page_size < 1 || pages < 1 || table_width < 1 || (!page_table && (pages < B || table_width != 1)) || (int64_t)page_size * table_width > 0x7fffffff - 64)
        return SA2_ERR_BAD_CACHE;
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
    p.nsplit = tree_splits(B, T, H, HK, D, page_size, table_width, dtype);
    p.part = (float*)workspace;
    if (p.nsplit > 1 && (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < tree_part_bytes(B, T, H, D, p.nsplit)))
        return SA2_ERR_WORKSPACE_TOO_SMALL;
    const bool narrow = !(flags & SA2_FLAG_FORCE_GENERIC) && tree16_supported(p, dtype);
    p.dealt = B > 1 && p.nsplit >= 8 && (!narrow || tree16_rows(p) > 64);      // (sa2_tree16.hip takes equal shares; 32 sequences at most)
    if (narrow) return launch_tree16(p, dtype, (hipStream_t)hip_stream);
    return launch_tree_f32(p, dtype, (hipStream_t)hip_stream);
}

}  // extern "C"
