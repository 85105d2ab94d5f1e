// New rows of keys and values into a cache: row a of what sequence b brings goes to place lengths[b] + a.
//
// Bound by memory, or for the few rows of a decoding step by the launch: each thread moves one 16-byte chunk of a key and
// the same of a value (8100 rows of four heads of 128: 8.2 us, 4000 GB/s; 16 x 8 accepted rows 4.3 us).  A row whose place lies
// beyond the table or whose page is not one of the cache's is left out.
#include "sa2_layer_common.h"

namespace sa2 {
namespace {

constexpr int THREADS = 256;

// UNIT: the bytes that a thread moves of a row; `chunks` of them in the HK * D elements of one
template <class UNIT>
__global__ __launch_bounds__(THREADS) void append_kernel(Append p, int size, int per_head) {
    const int chunks = p.HK * per_head;
    const int64_t it = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const int64_t item = it / chunks;
    const int ch = (int)(it - item * chunks), h = ch / per_head;
    const int per = p.chosen ? p.nchosen : p.rows.N;
    if (item >= (int64_t)p.rows.B * per) return;
    int b = (int)(item / per), a = (int)(item - (int64_t)b * per), n = a, held;
    int64_t sb = b;
    if (p.rows.cu) {                                  // packed: B is 1, the sequence is the row's
        n = a;
        b = sequence_of(p.rows, n);
        if (b < 0) return;
        a = place_of(p.rows, b, n);
        sb = 0;
    } else if (p.chosen) {
        n = p.chosen[item];
        if (n < 0 || n >= p.rows.N) return;
    }
    held = p.cache.lengths[b];
    if (held < 0) return;
    const int64_t place = (int64_t)held + a;
    int64_t page = b;
    int at = (int)place;
    if (p.cache.table) {
        const int64_t i = place / p.cache.page_size;
        if (i >= p.cache.width) return;
        page = p.cache.table[(int64_t)b * p.cache.width + i];
        if (page < 0 || page >= p.cache.pages) return;
        at = (int)(place - i * p.cache.page_size);
    } else if (place >= p.cache.page_size) {
        return;
    }
    const int64_t byte = (int64_t)(ch - h * per_head) * sizeof(UNIT);
    auto from = [&](const Tensor& t) { return (const UNIT*)((const char*)t.p + (sb * t.sb + (int64_t)n * t.sn + (int64_t)h * t.sh) * size + byte); };
    auto to = [&](const Tensor& t) { return (UNIT*)((char*)t.p + (page * t.sb + (int64_t)at * t.sn + (int64_t)h * t.sh) * size + byte); };
    const UNIT x = *from(p.k), y = *from(p.v);
    *to(p.cache.k) = x;
    *to(p.cache.v) = y;
}

}  // namespace

int launch_append(const Append& p, int dtype, hipStream_t st) {
    const int size = dtype == SA2_F32 ? 4 : 2;
    bool wide = (p.D * size) % 16 == 0;
    for (const Tensor* t : {&p.k, &p.v, &p.cache.k, &p.cache.v}) wide = wide && aligned16(*t, size, true);
    const int per_head = wide ? p.D * size / 16 : p.D;
    const int64_t items = (int64_t)p.rows.B * (p.chosen ? p.nchosen : p.rows.N) * p.HK * per_head;
    const int64_t blocks = (items + THREADS - 1) / THREADS;
    if (blocks > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    const dim3 grid((unsigned)blocks), block(THREADS);
    if (wide) append_kernel<uint4><<<grid, block, 0, st>>>(p, size, per_head);
    else if (size == 4) append_kernel<uint32_t><<<grid, block, 0, st>>>(p, size, per_head);
    else append_kernel<uint16_t><<<grid, block, 0, st>>>(p, size, per_head);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace sa2
