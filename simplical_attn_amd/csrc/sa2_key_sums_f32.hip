// What each key of a prompt got from the queries that see it, with fp32 products (v_mfma_f32_32x32x2_f32): fp32 tensors, and 16-bit ones
// that sa2_key_sums16.hip does not take.  And the sums of the shares.
//
//   w_j = sum over heads g and queries i that see j of e^(scale q_gi k_j - lse_gi)
//
// A wavefront owns 32 keys, whose products with a tile of 32 queries in LDS leave a lane one key and 16 queries: its sum is arithmetic
// within the lane.  4096 queries of 16 heads over 4 key heads, head_dim 128: 460 us, 75 TFLOP/s of the 154 that a large product reaches.  An MFMA
// has the matrix pipe for 64 cycles (two columns of 32 x 32 products); a tile's chain of them, its exponentials and masks, and the two barriers
// around the next tile's way to LDS stand one after the other, which only other wavefronts fill.  Short prompts are bound by the start of workgroups and the second launch (217 queries, 4 heads: 11.6 us).
#include "sa2_f32_tiles.h"
#include "sa2_key_sums.h"

namespace sa2 {
namespace {

constexpr int THREADS = 256, WAVES = 4, BLOCK = TILE * WAVES;

template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(THREADS) void key_sums_f32_kernel(KeySums p) {
    constexpr int PER = DP / 32;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float* const stats = lds + TILE * Pitch<DP>::value;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    KeyBlock w;
    if (!key_block(p, blockIdx.x, BLOCK, w)) return;
    const Span& s = w.s;
    const int hk = w.hk, share = w.share;
    if (s.fill) {
        if (share == 0)
            for (int i = threadIdx.x; i < s.len; i += THREADS) put_key_sum(p, s, hk, i, 0.f);
        return;
    }
    const int j0 = s.block * BLOCK, mine = j0 + wave * TILE, key = mine + (lane & 31);
    const KeyStream of = key_stream(p, s, j0, BLOCK, TILE);
    const int64_t all = (int64_t)of.per * p.G;
    const int lo = share * w.chunk, hi = all - lo < w.chunk ? (int)all : lo + w.chunk;
    if (lo >= hi) return;
    float k[DP / 2];
    own_rows<T, DP>(k, p.k, s, mine, hk, p.D, WIDE, 1.f);
    const float c = p.scale * LOG2E;
    float4 x[PER];
    float stat = 0.f, sum = 0.f;
    auto load = [&](int it) {
        const int h = hk * p.G + it / of.per, q0 = of.lo + it % of.per * TILE;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int ch = i * THREADS + threadIdx.x, r = ch / (DP / 4), d = ch % (DP / 4) * 4;
            x[i] = load4((const T*)p.q.p + row_offset(p.q, s, q0 + r < s.len ? q0 + r : 0, h), d, p.D, WIDE, q0 + r < s.len);
        }
        if (threadIdx.x < TILE) {
            const int at = q0 + threadIdx.x;
            stat = at < s.len ? p.lse[((int64_t)s.b * p.H + h) * p.rows.N + s.first + at] * LOG2E : 0.f;
        }
    };
    load(lo);
    for (int it = lo; it < hi; ++it) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int ch = i * THREADS + threadIdx.x, r = ch / (DP / 4), d = ch % (DP / 4) * 4;
            *(float4*)(lds + r * Pitch<DP>::value + d) = x[i];
        }
        if (threadIdx.x < TILE) stats[threadIdx.x] = stat;
        __syncthreads();
        if (it + 1 < hi) load(it + 1);
        const int q0 = of.lo + it % of.per * TILE;
        const uint32_t seen = key_all_seen(p, s, q0, q0 + TILE - 1, mine, mine + TILE - 1) ? ~0u : key_seen_by(p, s, key, q0);
        if (!__any(seen != 0)) continue;
        const floatx16 x = tile_product<DP>(lds, k);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 l = *(const float4*)(stats + 8 * g + 4 * half);
            const float* const ls = &l.x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = exp2f(fmaf(x[4 * g + r], c, -ls[r]));
                sum += seen >> (8 * g + 4 * half + r) & 1 ? e : 0.f;
            }
        }
    }
    sum += other_half(sum);
    if (half || key >= s.len) return;
    if (w.to) w.to[key] = sum;
    else put_key_sum(p, s, hk, key, sum);
}

// The sums of the shares, in their order: a thread per key
__global__ __launch_bounds__(THREADS) void key_sums_join_kernel(KeySums p, int block, int tile) {
    int stream, at;
    order(blockIdx.x, p.rows.B * p.HK, stream, at);
    const int b = stream / p.HK, hk = stream % p.HK;
    Span s;
    if (!find_tile(p.rows, b, at, THREADS, s) || s.fill) return;
    const int key = s.block * THREADS + threadIdx.x;
    if (key >= s.len) return;
    const bool front = key < p.front;
    if ((front ? p.front_shares : p.shares) == 1) return;   // (is where it belongs)
    const int64_t all = (int64_t)key_stream(p, s, key / block * block, block, tile).per * p.G;
    const int chunk = front ? p.front_chunk : p.chunk, n = (int)((all + chunk - 1) / chunk);
    int64_t step = (int64_t)p.rows.B * p.HK * p.rows.N;
    const float* from = p.part + ((int64_t)s.b * p.HK + hk) * p.rows.N + s.first + key;
    if (front) {
        const int sequence = p.rows.cu ? sequence_of(p.rows, s.first) : s.b;
        if (sequence < 0) return;
        step = (int64_t)(p.rows.cu ? p.rows.sequences : p.rows.B) * p.HK * p.front;
        from = p.front_part + ((int64_t)sequence * p.HK + hk) * p.front + key;
    }
    float sum = 0.f;
    for (int i = 0; i < n; i += 8) {                        // (eight reads under way, added in order)
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = i + j < n ? from[(i + j) * step] : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += x[j];
    }
    put_key_sum(p, s, hk, key, sum);
}

}  // namespace

int launch_key_sums_join(const KeySums& p, int block, int tile, hipStream_t st) {
    const int64_t grid = (int64_t)p.rows.B * p.HK * count_tiles(p.rows, THREADS);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    key_sums_join_kernel<<<dim3((unsigned)grid), dim3(THREADS), 0, st>>>(p, block, tile);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

int launch_key_sums_f32(const KeySums& p, int dtype, hipStream_t st) {
    const int rc = for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        constexpr int BYTES = 4 * sizeof(T);
        bool wide = p.D % 4 == 0;
        for (const Tensor* t : {&p.q, &p.k}) wide = wide && (uintptr_t)t->p % BYTES == 0 && t->sn % 4 == 0 && t->sh % 4 == 0 && (p.rows.B == 1 || t->sb % 4 == 0);
        return for_width(p.D, [&](auto w) {
            constexpr int DP = decltype(w)::value;
            const int64_t grid = p.front_grid + key_blocks(p, BLOCK);
            if (grid > 0x7fffffff) return (int)SA2_ERR_TOO_LARGE;
            const auto kernel = wide ? key_sums_f32_kernel<T, DP, true> : key_sums_f32_kernel<T, DP, false>;
            if (!allow_full_lds((const void*)kernel)) return (int)SA2_ERR_LAUNCH_FAILED;
            kernel<<<dim3((unsigned)grid), dim3(THREADS), (TILE * Pitch<DP>::value + TILE) * sizeof(float), st>>>(p);
            return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
        });
    });
    return rc == SA2_OK && (p.shares > 1 || p.front_shares > 1) ? launch_key_sums_join(p, BLOCK, TILE, st) : rc;
}

}  // namespace sa2
