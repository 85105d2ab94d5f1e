// extern "C" boundary of the operators of ordinary attention layers: argument validation and kernel choice.
// No allocation, no synchronisation, no state.
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

}  // extern "C"
