// Windowed attention, gradients, bf16 and fp16 on the 16-bit MFMA: the kernels of sa2_causal_dkv16.h and sa2_causal_dq16.h with a band, in one
// launch, and fp16's factors before it.
//
// The keys behind the first ones are seen by the queries of their windows, a stream of (window + 127) rows per head and block of 128; the
// first keys by all queries, in chunks of these whose fp32 sums meet in a last launch.
// 16 heads over 4 key heads, 8192 queries, head_dim 128, bf16, window 512 with 4 first keys: dQ 145 us, dK and dV 135 (0.35 and 0.50 PFLOP/s of the
// three and four products that each forms), row terms 20 (memory), the first keys' sums 12.  Ten tiles per workgroup, so that starts and ends weigh as
// much as the sweep.  8 heads, batch 2, 2048 queries, head_dim 64, window 512: 42 us in one launch of 512 workgroups, half of them for dQ, of which a
// CU has one at a time: two rounds of such chains.  fp16: 46 us more than bf16 in the first case (all gradients 340 us and 294), factors and row terms;
// with many first keys the factors cost more, since every row goes through all of these.
#include "sa2_causal_dkv16.h"

namespace sa2 {
namespace {

// ---- fp16: factors of the rows of dQ and of the keys (sa2_causal16.h), from the rows that meet there alone --------------------------------
constexpr int FACTOR_ROWS = 256;

// max of x(n - window + 1) .. x(n) for the lane's n = n0 + threadIdx.x; x(i) is 0 where i < 0.  `lds`: 2 * FACTOR_ROWS floats, and every
// thread calls it.  Windows up to 256 double up to the largest power of two, two of which overlap; longer ones are the 256 up to n, the
// 256 from the window's start, and what all windows of the block share between them.
template <class X>
__device__ __forceinline__ float window_max(X&& x, int n0, int window, float* lds) {
    const int t = threadIdx.x;
    int power = 0;
    while (power < 8 && 2 << power <= window) ++power;
    // lds[i]: the maximum of 2^power values up to place `from` + i
    auto doubled = [&](int from) {
        __syncthreads();
        float* const y = lds;
        y[t] = x(from + t);
        y[FACTOR_ROWS + t] = x(from + FACTOR_ROWS + t);
        __syncthreads();
        for (int s = 0; s < power; ++s) {
            const int o = 1 << s;
            const float a = t >= o ? fmaxf(y[t], y[t - o]) : y[t], b = fmaxf(y[FACTOR_ROWS + t], y[FACTOR_ROWS + t - o]);
            __syncthreads();
            y[t] = a;
            y[FACTOR_ROWS + t] = b;
            __syncthreads();
        }
    };
    doubled(n0 - FACTOR_ROWS);                              // place n is FACTOR_ROWS + t
    float most = lds[FACTOR_ROWS + t];
    if (window <= FACTOR_ROWS) {
        const int back = window - (1 << power);
        return fmaxf(most, lds[FACTOR_ROWS + t - back]);
    }
    // 256 values from the window's start: up to n - window + 256
    const int64_t start = (int64_t)n0 - window;
    doubled(start < -2 * FACTOR_ROWS ? -2 * FACTOR_ROWS : (int)start);
    // (the block's first window starts at n0 - window + 1: place FACTOR_ROWS + t is n - window + 256)
    if (start >= -2 * FACTOR_ROWS) most = fmaxf(most, lds[FACTOR_ROWS + t]);
    float shared = 0.f;
    const int first = start + FACTOR_ROWS < 0 ? 0 : (int)start + FACTOR_ROWS;
    for (int i = first + t; i <= n0; i += FACTOR_ROWS) shared = fmaxf(shared, x(i));
    shared = wave_max(shared);
    __syncthreads();
    if ((t & 63) == 0) lds[t >> 6] = shared;
    __syncthreads();
    for (int w = 0; w < FACTOR_ROWS / 64; ++w) most = fmaxf(most, lds[w]);
    return most;
}

__global__ __launch_bounds__(FACTOR_ROWS) void window_factors_kernel(Causal p, Causal16Terms terms) {
    __shared__ float lds[2 * FACTOR_ROWS];
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.HK, stream, tile);
    const int b = stream / p.HK, hk = stream % p.HK;
    Span s;
    if (!find_tile(p.rows, b, tile, FACTOR_ROWS, s) || s.fill) return;
    const int n0 = s.block * FACTOR_ROWS, n = n0 + threadIdx.x;
    const int64_t key0 = ((int64_t)s.b * p.HK + hk) * p.rows.N + s.first, query0 = ((int64_t)s.b * p.H + hk * p.G) * p.rows.N + s.first;
    // queries: values that they see
    auto value = [&](int i) { return i >= 0 && i < s.len ? finite_or_zero(terms.v[key0 + i]) : 0.f; };
    float seen = window_max(value, n0, p.band.window, lds);
    if (p.band.sinks > 0) {
        const int end = n + 1 < p.band.sinks ? n + 1 : p.band.sinks;
        // (all threads of a block behind the first keys go through the same ones)
        for (int i = 0; i < end; ++i) seen = fmaxf(seen, value(i));
    }
    if (n < s.len)
        for (int g = 0; g < p.G; ++g) {
            const int64_t at = query0 + (int64_t)g * p.rows.N + n;
            terms.queries[at] = gradient_factor(fmaf(terms.dout[at], seen, fabsf(p.delta[at])));
        }
    // keys behind the first ones: gradients of the outputs that see them, the same from the other end of the sequence
    auto over = [&](const float* x) {
        return [&, x](int i) {
            const int row = s.len - 1 - i;
            float most = 0.f;
            if (row >= 0 && row < s.len)
                for (int g = 0; g < p.G; ++g) most = fmaxf(most, finite_or_zero(x[query0 + (int64_t)g * p.rows.N + row]));
            return most;
        };
    };
    const float dout = window_max(over(terms.dout), n0, p.band.window, lds), delta = window_max(over(p.delta), n0, p.band.window, lds);
    const int key = s.len - 1 - n;
    if (key >= 0) terms.keys[key0 + key] = gradient_factor(fmaf(dout, terms.v[key0 + key], delta));
}

// `queries` workgroups for dQ, then those for dK and dV
template <class E, int D, int NQ>
__global__ __launch_bounds__(THREADS, 1) void window_bwd16_kernel(Causal p, Causal16Terms terms, int nsplit, int queries, int heads, int main, int members, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if ((int)blockIdx.x < queries) queries_gradient16<E, D, NQ, true>(p, terms, padded, blockIdx.x, lds, heads);
    else keys_gradients16<E, D, true>(p, terms, nsplit, padded, blockIdx.x - queries, lds, main, members);
}
// At head_dim 128 one launch after the other, and two blocks of queries per wavefront whatever their number: dQ's sums and operands beside
// the masks and the other kernel's needs left no registers (with one block, its operands moved between the files in front of the MFMAs)
template <class E, int D>
__global__ __launch_bounds__(THREADS, 1) void window_dkv16_kernel(Causal p, Causal16Terms terms, int nsplit, int main, int members, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    keys_gradients16<E, D, true>(p, terms, nsplit, padded, blockIdx.x, lds, main, members);
}
template <class E, int D, int NQ>
__global__ __launch_bounds__(THREADS, 1) void window_dq16_kernel(Causal p, Causal16Terms terms, int heads, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    queries_gradient16<E, D, NQ, true>(p, terms, padded, blockIdx.x, lds, heads);
}

template <class E, int D, int NQ>
int launch_of(const Causal& p, const Causal16Terms& terms, int heads, hipStream_t st) {
    const bool any = p.dk.p || p.dv.p, sink = any && p.band.sinks > 0, padded = p.D != D;
    const int nsplit = window16_splits(p);
    const int64_t queries = p.dq.p ? (int64_t)p.rows.B * (p.H / heads) * count_tiles(p.rows, 32 * NQ * WAVES / heads) : 0;
    const int64_t main = any ? (int64_t)p.rows.B * p.HK * nsplit * count_tiles(p.rows, BLOCK) : 0;
    const int members = sink ? sink_members(p, BLOCK) : 1;
    const int64_t keys = main + (sink ? sink_groups(p, BLOCK) * members * p.HK : 0);
    constexpr int LDS = BUFFERS * (Buffer<D>::BYTES + STATS), QUERY_LDS = QUERY_BUFFERS<NQ, true> * Buffer<D>::BYTES;
    static_assert(LDS >= QUERY_LDS, "");
    if (queries + keys > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    const dim3 block(THREADS);
    if constexpr (D == 64) {
        const auto kernel = window_bwd16_kernel<E, D, NQ>;
        if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
        kernel<<<dim3((unsigned)(queries + keys)), block, LDS, st>>>(p, terms, nsplit, (int)queries, heads, (int)main, members, padded);
    } else {
        const auto to_keys = window_dkv16_kernel<E, D>;
        const auto to_queries = window_dq16_kernel<E, D, NQ>;
        if (!allow_full_lds((const void*)to_keys) || !allow_full_lds((const void*)to_queries)) return SA2_ERR_LAUNCH_FAILED;
        if (keys) to_keys<<<dim3((unsigned)keys), block, LDS, st>>>(p, terms, nsplit, (int)main, members, padded);
        if (queries) to_queries<<<dim3((unsigned)queries), block, QUERY_LDS, st>>>(p, terms, heads, padded);
    }
    if (hipGetLastError() != hipSuccess) return SA2_ERR_LAUNCH_FAILED;
    if (any && nsplit > 1) {
        const int rc = launch_sums<E>(p, nsplit, st);
        if (rc != SA2_OK) return rc;
    }
    return sink ? launch_sink_sums(p, E::DTYPE, st) : SA2_OK;
}

template <class E>
int launch(const Causal& p, const Causal16Terms& terms, hipStream_t st) {
    const int rc = launch_terms<E>(p, terms, st);
    if (rc != SA2_OK) return rc;
    if constexpr (E::DTYPE == SA2_F16) {
        const int64_t grid = (int64_t)p.rows.B * p.HK * count_tiles(p.rows, FACTOR_ROWS);
        if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
        window_factors_kernel<<<dim3((unsigned)grid), dim3(FACTOR_ROWS), 0, st>>>(p, terms);
        if (hipGetLastError() != hipSuccess) return SA2_ERR_LAUNCH_FAILED;
    }
    const int heads = window_heads(p);
    const bool two = window_two(p, heads);
    if (p.D <= 64) return two ? launch_of<E, 64, 2>(p, terms, heads, st) : launch_of<E, 64, 1>(p, terms, heads, st);
    return launch_of<E, 128, 2>(p, terms, heads, st);
}

}  // namespace

// Shares of a key block's stream: a workgroup per CU, where the stream is long enough for eight tiles each
int window16_splits(const Causal& p) {
    const int64_t blocks = (int64_t)p.rows.B * p.HK * ((p.rows.N + BLOCK - 1) / BLOCK), tiles = (int64_t)p.G * ((p.band.window + BLOCK + TILE_ROWS - 1) / TILE_ROWS);
    int64_t n = CUS / blocks;
    if (n > tiles / 8) n = tiles / 8;
    return n < 1 ? 1 : n > 16 ? 16 : (int)n;
}
size_t window16_part_bytes(const Causal& p) {
    const int n = window16_splits(p);
    return n > 1 ? ((size_t)n * 2 * p.rows.B * p.HK * p.rows.N * p.D * sizeof(float) + 255) / 256 * 256 : 0;
}

int launch_window16_bwd(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st) {
    return dtype == SA2_F16 ? launch<ElemF16>(p, terms, st) : launch<ElemBF16>(p, terms, st);
}

}  // namespace sa2
