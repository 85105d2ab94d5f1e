// What each key of a prompt got from the queries that see it, bf16 and fp16 on the 16-bit MFMA: head_dim a multiple of 8 up to 128, rows on the
// 16-byte grid.
//
//   w_j = sum over heads g and queries i that see j of e^(scale q_gi k_j - lse_gi)
//
// A wavefront owns KB blocks of 32 keys: S = Q K^T leaves lane l with key l % 32 and 16 of 32 queries, so that a key's sum is arithmetic within the
// lane.  Q comes by direct global->LDS loads in tiles of 64 rows, which the four wavefronts and their blocks share; the operands of
// a product are read once for KB of them.  Scores, exponentials and sums are fp32.
// Bound by issue: a 32 x 32 of scores (head_dim 128) takes 8 MFMAs, 16 exponentials, 16 products with the scale and 16 additions, which run beside
// each other only where wavefronts share a SIMD; three do (168 registers).  16 heads over 4 key heads, 8192 queries, head_dim 128, bf16: 190 us
// without a window (0.7 PFLOP/s), 43 us with one of 512.  Tried: both blocks' chains of MFMAs side by side (191 us; 216 where that leaves two
// wavefronts on a SIMD), requests two tiles ahead (no change).
#include "sa2_causal16.h"
#include "sa2_key_sums.h"

namespace sa2 {
namespace {

constexpr int RING = 2;
template <int D>
struct QueryTile {                                          // 64 rows of Q, and their lse
    static constexpr int STATS = 2 * QuadTile<D>::BYTES, BYTES = STATS + TILE_ROWS * 4;
};

template <class E, int D, int KB>
__global__ __launch_bounds__(THREADS, 3) void key_sums16_kernel(KeySums p, bool padded) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    constexpr int KK = D / 16, INSTR = TILE_ROWS / T::RPW / WAVES, BLOCK = 32 * KB * WAVES;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t base = lds_address(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    KeyBlock w;
    if (!key_block(p, blockIdx.x, BLOCK, w)) return;
    const Span& s = w.s;
    const int hk = w.hk, share = w.share;
    if (s.fill) {
        if (share == 0)
            for (int i = threadIdx.x; i < s.len; i += THREADS) put_key_sum(p, s, hk, i, 0.f);
        return;
    }
    const int j0 = s.block * BLOCK, mine = j0 + wave * 32 * KB;
    const KeyStream of = key_stream(p, s, j0, BLOCK, TILE_ROWS);
    const int64_t all = (int64_t)of.per * p.G;
    const int lo = share * w.chunk, hi = all - lo < w.chunk ? (int)all : lo + w.chunk;
    if (lo >= hi) return;

    // tiles of the stream to LDS, each wavefront a quarter
    const int chunk = T::dma_chunk(lane);
    const bool pad = chunk * 8 >= p.D;
    int g = lo / of.per, t = lo - g * of.per;
    auto request = [&](uint32_t to) {
        const int q0 = of.lo + t * TILE_ROWS, h = hk * p.G + g;
        const char* const row0 = (const char*)p.q.p + row_offset(p.q, s, q0, h) * 2 + chunk * 16;
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
            const int group = wave * INSTR + i, row = group * T::RPW + T::dma_row(lane);
            const bool there = q0 + row < s.len && !(padded && pad);
            lds_request(there ? (const void*)(row0 + (int64_t)row * p.q.sn * 2) : (const void*)zero_chunk, to + group * T::GROUP);
        }
        if (wave == 0) {
            const float* const lse = p.lse + ((int64_t)s.b * p.H + h) * p.rows.N + s.first + q0 + lane;
            lds_request4(q0 + lane < s.len ? (const void*)lse : (const void*)zero_chunk, to + QueryTile<D>::STATS);
        }
        if (++t == of.per) {
            t = 0;
            ++g;
        }
    };
    request(base);

    X8 k[KB][KK];
#pragma unroll
    for (int n = 0; n < KB; ++n) {
        const int key = mine + 32 * n + (lane & 31);
        const uint16_t* const row = (const uint16_t*)p.k.p + row_offset(p.k, s, key < s.len ? key : 0, hk);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int col = 16 * kk + 8 * half;
            union { uint4 u; X8 x; } word;
            word.u = make_uint4(0, 0, 0, 0);
            if (key < s.len && col < p.D) word.u = *(const uint4*)(row + col);
            k[n][kk] = word.x;
        }
    }
    const float c = p.scale * LOG2E;
    const uint32_t row_lane = T::row_lane(lane);
    float sum[KB];
#pragma unroll
    for (int n = 0; n < KB; ++n) sum[n] = 0.f;
    for (int it = lo; it < hi; ++it) {
        const uint32_t here = base + (uint32_t)((it - lo) % RING) * QueryTile<D>::BYTES;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (it + 1 < hi) request(base + (uint32_t)((it + 1 - lo) % RING) * QueryTile<D>::BYTES);
        const int q0 = of.lo + it % of.per * TILE_ROWS;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            const int i0 = q0 + 32 * sub;
            if (i0 + 31 < mine) continue;                   // (before the wavefront's keys)
            float lse[16];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 l = *(const float4*)(lds + (here - base) + QueryTile<D>::STATS + (32 * sub + 8 * r + 4 * half) * 4);
                lse[4 * r] = l.x * LOG2E; lse[4 * r + 1] = l.y * LOG2E; lse[4 * r + 2] = l.z * LOG2E; lse[4 * r + 3] = l.w * LOG2E;
            }
            X8 q[KK];
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) q[kk] = lds_read_x8<X8>(here + (uint32_t)(sub * T::BYTES) + row_lane + (uint32_t)(kk / 2 * T::BLOCK + kk % 2 * 32));
            const bool whole = key_all_seen(p, s, i0, i0 + 31, mine, mine + 32 * KB - 1);
#pragma unroll
            for (int n = 0; n < KB; ++n) {
                floatx16 x;
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) x = E::mfma(q[kk], k[n][kk], x, 0, 0, 0);
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                if (whole) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) part[r % 4] += fast_exp2(fmaf(x[r], c, -lse[r]));
                } else {
                    const uint32_t seen = key_seen_by(p, s, mine + 32 * n + (lane & 31), i0) >> 4 * half;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float e = fast_exp2(fmaf(x[r], c, -lse[r]));
                        part[r % 4] += seen >> (8 * (r / 4) + r % 4) & 1 ? e : 0.f;
                    }
                }
                sum[n] += (part[0] + part[1]) + (part[2] + part[3]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < KB; ++n) {
        const float both = sum[n] + other_half(sum[n]);
        const int key = mine + 32 * n + (lane & 31);
        if (half || key >= s.len) continue;
        if (w.to) w.to[key] = both;
        else put_key_sum(p, s, hk, key, both);
    }
}

template <class E, int D, int KB>
int launch(const KeySums& p, hipStream_t st) {
    const auto kernel = key_sums16_kernel<E, D, KB>;
    const int64_t grid = p.front_grid + key_blocks(p, 32 * KB * WAVES);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), RING * QueryTile<D>::BYTES, st>>>(p, p.D != D);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

// 16-byte rows
bool key_sums16_supported(const KeySums& p, int dtype) {
    return causal16_supported(p.D, dtype) && aligned16(p.q, 2, p.rows.B > 1) && aligned16(p.k, 2, p.rows.B > 1);
}

int launch_key_sums16(const KeySums& p, int dtype, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        return p.D <= 64 ? launch<E, 64, KEY_SUMS16_BLOCK / 128>(p, st) : launch<E, 128, KEY_SUMS16_BLOCK / 128>(p, st);
    };
    const int rc = dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
    return rc == SA2_OK && (p.shares > 1 || p.front_shares > 1) ? launch_key_sums_join(p, KEY_SUMS16_BLOCK, TILE_ROWS, st) : rc;
}

}  // namespace sa2
