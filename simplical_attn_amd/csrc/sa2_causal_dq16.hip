// Launches of the gradient of the queries by itself (sa2_causal_dq16.h), bf16 and fp16.
#include "sa2_causal_dq16.h"

namespace sa2 {
namespace {

template <class E, int D, int NQ>
__global__ __launch_bounds__(THREADS, 1) void causal_dq16_kernel(Causal p, Causal16Terms terms, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    queries_gradient16<E, D, NQ>(p, terms, padded, blockIdx.x, lds);
}

template <class E, int D, int NQ>
int launch(const Causal& p, const Causal16Terms& terms, hipStream_t st) {
    const auto kernel = causal_dq16_kernel<E, D, NQ>;
    const int64_t grid = (int64_t)p.rows.B * p.H * count_tiles(p.rows, 32 * NQ * WAVES);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), DQ_BUFFERS * Buffer<D>::BYTES, st>>>(p, terms, p.D != D);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

// Two blocks of queries per wavefront halve what LDS has to deliver, one makes twice as many workgroups with half the chain: two where
// every CU has two workgroups all the same (forward, head_dim 128: B1 N8192 H16/4 306 us with two, 350 with one; B4 N1024 43 and 37).
// Packed rows are counted as count_tiles bounds them, with a workgroup more for every sequence: many short sequences have two.
bool causal16_two(const Causal& p) { return (int64_t)p.rows.B * p.H * count_tiles(p.rows, 64 * WAVES) >= 2 * CUS; }

int launch_causal16_dq(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        const bool two = causal16_two(p);
        if (p.D <= 64) return two ? launch<E, 64, 2>(p, terms, st) : launch<E, 64, 1>(p, terms, st);
        return two ? launch<E, 128, 2>(p, terms, st) : launch<E, 128, 1>(p, terms, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace sa2
