// Launches of windowed attention with fp32 products (sa2_causal_f32.h), and the sums of the first keys' gradients.
#include "sa2_causal_f32.h"

namespace sa2 {
namespace {

// A workgroup adds up a row of 32 first keys over a sequence's chunks, in their order: it is the one whose chunk is the sequence's
// first.  (Chunks that end before a key's block of 32 to 128 have left nothing for it.)
template <class T>
__global__ __launch_bounds__(THREADS) void sink_sums_kernel(Causal p, int64_t slots) {
    const int64_t each = slots / p.rows.B;
    const int slot = blockIdx.x / p.HK, hk = blockIdx.x % p.HK, j0 = blockIdx.y * TILE, b = (int)(slot / each), tile = (int)(slot - b * each);
    Span s;
    if (!find_tile(p.rows, b, tile, p.band.chunk, s) || s.fill || s.block) return;
    const int end = p.band.sinks < s.len ? p.band.sinks : s.len, chunks = (s.len + p.band.chunk - 1) / p.band.chunk;
    for (int i = threadIdx.x; i < TILE * p.D; i += THREADS) {
        const int j = j0 + i / p.D, d = i % p.D;
        if (j >= end) return;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const Tensor& t = which ? p.dv : p.dk;
            if (!t.p) continue;
            const float* const from = sink_row(p, slots, which, slot, hk, j) + d;
            const int64_t step = (int64_t)p.HK * p.band.sinks * p.D;
            float sum = 0.f;
            for (int c = j / p.band.chunk; c < chunks; ++c) sum += from[c * step];
            from_float(sum, (T*)t.p + row_offset(t, s, j, hk) + d);
        }
    }
}

}  // namespace

size_t sink_part_bytes(const Causal& p) { return p.band.sinks > 0 ? (size_t)2 * sink_slots(p) * p.HK * p.band.sinks * p.D * sizeof(float) : 0; }

int launch_sink_sums(const Causal& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        const int64_t slots = sink_slots(p);
        const dim3 grid((unsigned)(slots * p.HK), (p.band.sinks + TILE - 1) / TILE);
        sink_sums_kernel<T><<<grid, dim3(THREADS), 0, st>>>(p, slots);
        return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
    });
}

int launch_window_f32_fwd(const Causal& p, int dtype, hipStream_t st) { return f32_forward<true>(p, dtype, st); }
int launch_window_f32_bwd(const Causal& p, int dtype, hipStream_t st) { return f32_backward<true>(p, dtype, st); }

}  // namespace sa2
