// Launches of the gradients of causal attention, bf16 and fp16 (sa2_causal_dkv16.h, sa2_causal_dq16.h).
#include "sa2_causal_dkv16.h"

namespace sa2 {
namespace {

template <class E, int D>
__global__ __launch_bounds__(THREADS, 1) void causal_dkv16_kernel(Causal p, Causal16Terms terms, int nsplit, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    keys_gradients16<E, D>(p, terms, nsplit, padded, blockIdx.x, lds);
}
// All gradients in one launch where there are few workgroups, so that one's fill the CUs that the other's short ones leave: `queries`
// workgroups for dQ, whose longest chains are the longest of all, then those for dK and dV (B2 N2048 H8 D64 80 us apart, 57 together; B4 N1024
// H16/4 D128 133 and 121; with as many blocks of 256 queries as would give every CU two, B1 N8192 H16/4 D128, 921 and 967: there
// a wavefront with 64 queries saves more).
template <class E, int D>
__global__ __launch_bounds__(THREADS, 1) void causal_bwd16_kernel(Causal p, Causal16Terms terms, int nsplit, int queries, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if ((int)blockIdx.x < queries) queries_gradient16<E, D, 1>(p, terms, padded, blockIdx.x, lds);
    else keys_gradients16<E, D>(p, terms, nsplit, padded, blockIdx.x - queries, lds);
}

template <class E>
int launch(const Causal& p, const Causal16Terms& terms, hipStream_t st) {
    const int first = launch_terms<E>(p, terms, st);
    if (first != SA2_OK) return first;
    const bool together = p.dq.p && (p.dk.p || p.dv.p) && !causal16_two(p);
    if (p.dk.p || p.dv.p) {
        const int nsplit = causal16_splits(p.rows.B, p.rows.N, p.HK, p.G);
        auto of = [&](auto w) {
            constexpr int D = decltype(w)::value;
            const int64_t keys = (int64_t)p.rows.B * p.HK * nsplit * count_tiles(p.rows, BLOCK), queries = together ? (int64_t)p.rows.B * p.H * count_tiles(p.rows, BLOCK) : 0;
            constexpr int LDS = BUFFERS * (Buffer<D>::BYTES + STATS);
            static_assert(LDS >= DQ_BUFFERS * Buffer<D>::BYTES, "");
            if (keys + queries > 0x7fffffff) return (int)SA2_ERR_TOO_LARGE;
            const dim3 grid((unsigned)(keys + queries)), block(THREADS);
            if (!allow_full_lds(together ? (const void*)causal_bwd16_kernel<E, D> : (const void*)causal_dkv16_kernel<E, D>)) return (int)SA2_ERR_LAUNCH_FAILED;
            if (together) causal_bwd16_kernel<E, D><<<grid, block, LDS, st>>>(p, terms, nsplit, (int)queries, p.D != D);
            else causal_dkv16_kernel<E, D><<<grid, block, LDS, st>>>(p, terms, nsplit, p.D != D);
            return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
        };
        const int rc = p.D <= 64 ? of(std::integral_constant<int, 64>{}) : of(std::integral_constant<int, 128>{});
        if (rc != SA2_OK) return rc;
        if (nsplit > 1) {
            const int sums = launch_sums<E>(p, nsplit, st);
            if (sums != SA2_OK) return sums;
        }
    }
    return p.dq.p && !together ? launch_causal16_dq(p, E::DTYPE, terms, st) : SA2_OK;
}

}  // namespace

// Shares of a key block's stream: two workgroups per CU over the chip, where the stream is that long (packed sequences: as if
// they were one, the bound that the host knows)
int causal16_splits(int B, int N, int HK, int G) {
    const int64_t blocks = (int64_t)B * HK * ((N + BLOCK - 1) / BLOCK), tiles = (int64_t)G * ((N + TILE_ROWS - 1) / TILE_ROWS);
    int64_t n = (2 * CUS + blocks - 1) / blocks;
    if (n > tiles / 8) n = tiles / 8;
    return n < 1 ? 1 : n > 16 ? 16 : (int)n;
}
size_t causal16_part_bytes(int B, int N, int HK, int G, int D) {
    const int n = causal16_splits(B, N, HK, G);
    return n > 1 ? (size_t)n * 2 * B * HK * N * D * sizeof(float) : 0;
}

int launch_causal16_bwd(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st) {
    return dtype == SA2_F16 ? launch<ElemF16>(p, terms, st) : launch<ElemBF16>(p, terms, st);
}

}  // namespace sa2
