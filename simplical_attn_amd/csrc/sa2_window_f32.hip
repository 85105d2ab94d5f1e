// Launches of windowed attention with fp32 products (sa2_causal_f32.h), and the sums of the first keys' gradients.
#include "sa2_causal_f32.h"

namespace sa2 {
namespace {

// A workgroup adds up one first key over a sequence's chunks: it is the one whose chunk is the sequence's first.  Eight groups of threads
// have every eighth chunk each, with eight reads under way (one thread per value, one read after the other, took 61 us for 64 chunks);
// the groups are added in order.  (Chunks that end before a key's block of 32 to 128 have left nothing for it.)
constexpr int SUM_GROUPS = 8;
template <class T>
__global__ __launch_bounds__(64 * SUM_GROUPS) void sink_sums_kernel(Causal p, int64_t slots) {
    __shared__ float sums[SUM_GROUPS][64];
    const int64_t each = slots / p.rows.B, step = (int64_t)p.band.sinks * p.D;
    const int group = threadIdx.x / 64, lane = threadIdx.x % 64, j = blockIdx.y;
    for (int64_t item = blockIdx.x; item < slots * p.HK; item += gridDim.x) {
        const int64_t slot = item / p.HK;
        const int hk = (int)(item - slot * p.HK), b = (int)(slot / each), tile = (int)(slot - b * each);
        Span s;
        if (!find_tile(p.rows, b, tile, p.band.chunk, s) || s.fill || s.block || j >= s.len) continue;
        const int chunks = (s.len + p.band.chunk - 1) / p.band.chunk;
        for (int it = 0; it < 2 * ((p.D + 63) / 64); ++it) {
            const int which = it % 2, d = it / 2 * 64 + lane;
            const Tensor& t = which ? p.dv : p.dk;
            if (!t.p) continue;
            float sum = 0.f;
            if (d < p.D) {
                const float* const from = sink_row(p, which, slot * p.band.sinks, hk, j) + d;
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
}
// The same for packed sequences (Band::by_rows), 64 threads for a row of a key head: most sequences have a chunk or two
template <class T>
__global__ __launch_bounds__(64 * SUM_GROUPS) void sink_sums_by_rows_kernel(Causal p) {
    const int lane = threadIdx.x % 64;
    for (int64_t item = (int64_t)blockIdx.x * SUM_GROUPS + threadIdx.x / 64; item < (int64_t)p.rows.N * p.HK; item += (int64_t)gridDim.x * SUM_GROUPS) {
        const int n = (int)(item / p.HK), hk = (int)(item % p.HK), sequence = sequence_of(p.rows, n);
        if (sequence < 0) continue;
        const auto bound = [&](int i) { const int x = p.rows.cu[i]; return x < 0 ? 0 : x > p.rows.N ? p.rows.N : x; };
        Span s{0, bound(sequence), 0, 0, false};
        s.len = bound(sequence + 1) - s.first;
        const int j = n - s.first, held = p.band.sinks < s.len ? p.band.sinks : s.len;
        if (j >= held) continue;
        const int chunks = (s.len + p.band.chunk - 1) / p.band.chunk;
        const int64_t step = (int64_t)held * p.D;
        for (int it = 0; it < 2 * ((p.D + 63) / 64); ++it) {
            const int which = it % 2, d = it / 2 * 64 + lane;
            const Tensor& t = which ? p.dv : p.dk;
            if (!t.p || d >= p.D) continue;
            const float* const from = sink_row(p, which, 2 * (int64_t)s.first, hk, j) + d;
            float sums[SUM_GROUPS] = {};
            for (int c = j / p.band.chunk; c < chunks; c += SUM_GROUPS) {
                float x[SUM_GROUPS];
#pragma unroll
                for (int g = 0; g < SUM_GROUPS; ++g) x[g] = c + g < chunks ? from[(c + g) * step] : 0.f;
#pragma unroll
                for (int g = 0; g < SUM_GROUPS; ++g) sums[g] += x[g];
            }
#pragma unroll
            for (int g = 1; g < SUM_GROUPS; ++g) sums[0] += sums[g];
            from_float(sums[0], (T*)t.p + row_offset(t, s, j, hk) + d);
        }
    }
}

}  // namespace

size_t sink_part_bytes(const Causal& p) { return p.band.sinks > 0 ? (size_t)2 * p.HK * p.band.sink_rows * p.D * sizeof(float) : 0; }

int launch_sink_sums(const Causal& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        const dim3 block(64 * SUM_GROUPS);
        const auto grid = [](int64_t items) { return (unsigned)(items < 65536 ? items : 65536); };
        const int64_t slots = sink_groups(p, 0);
        if (p.band.by_rows) sink_sums_by_rows_kernel<T><<<dim3(grid(((int64_t)p.rows.N * p.HK + SUM_GROUPS - 1) / SUM_GROUPS)), block, 0, st>>>(p);
        else sink_sums_kernel<T><<<dim3(grid(slots * p.HK), p.band.sinks), block, 0, st>>>(p, slots);
        return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
    });
}

int launch_window_f32_fwd(const Causal& p, int dtype, hipStream_t st) { return f32_forward<true>(p, dtype, st); }
int launch_window_f32_bwd(const Causal& p, int dtype, hipStream_t st) { return f32_backward<true>(p, dtype, st); }

}  // namespace sa2
