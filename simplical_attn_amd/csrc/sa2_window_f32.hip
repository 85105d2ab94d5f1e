// Launches of windowed attention with fp32 products (sa2_causal_f32.h), and the sums of the first keys' gradients.
#include "sa2_causal_f32.h"

namespace sa2 {
namespace {

// A workgroup adds up one first key over a sequence's chunks: it is the one whose chunk is the sequence's first.  Eight groups of threads
// have every eighth chunk each, with eight reads under way (one thread per value, one read after the other, took 61 us for 64 chunks);
// the groups are added in order.  (Chunks that end before a key's block of 32 to 128 have left nothing for it.)
constexpr int SUM_GROUPS = 8;
template <class T>
__global__ __launch_bounds__(512) void sink_sums_kernel(Causal p, int64_t slots) {
    __shared__ float sums[SUM_GROUPS][64];
    const int64_t each = slots / p.rows.B;
    const int slot = blockIdx.x / p.HK, hk = blockIdx.x % p.HK, j = blockIdx.y, b = (int)(slot / each), tile = (int)(slot - b * each);
    Span s;
    if (!find_tile(p.rows, b, tile, p.band.chunk, s) || s.fill || s.block || j >= s.len) return;
    const int chunks = (s.len + p.band.chunk - 1) / p.band.chunk, group = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t step = (int64_t)p.HK * p.band.sinks * p.D;
    for (int it = 0; it < 2 * ((p.D + 63) / 64); ++it) {
        const int which = it % 2, d = it / 2 * 64 + lane;
        const Tensor& t = which ? p.dv : p.dk;
        if (!t.p) continue;
        float sum = 0.f;
        if (d < p.D) {
            const float* const from = sink_row(p, slots, which, slot, hk, j) + d;
            for (int c = j / p.band.chunk + group; c < chunks; c += 8 * SUM_GROUPS) {
                float x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] = c + u * SUM_GROUPS < chunks ? from[(c + u * SUM_GROUPS) * step] : 0.f;
#pragma unroll
                for (int u = 0; u < 8; ++u) sum += x[u];
            }
        }
        __syncthreads();
        sums[group][lane] = sum;
        __syncthreads();
        if (group == 0 && d < p.D) {
#pragma unroll
            for (int g = 1; g < SUM_GROUPS; ++g) sum += sums[g][lane];
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
        const dim3 grid((unsigned)(slots * p.HK), p.band.sinks);
        sink_sums_kernel<T><<<grid, dim3(512), 0, st>>>(p, slots);
        return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
    });
}

int launch_window_f32_fwd(const Causal& p, int dtype, hipStream_t st) { return f32_forward<true>(p, dtype, st); }
int launch_window_f32_bwd(const Causal& p, int dtype, hipStream_t st) { return f32_backward<true>(p, dtype, st); }

}  // namespace sa2
