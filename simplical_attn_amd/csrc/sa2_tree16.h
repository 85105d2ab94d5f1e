// Attention of drafted tokens (or single ones) over a cache, bf16 and fp16 on the 16-bit MFMA: head_dim a multiple of 8 up to 128,
// rows on the 16-byte grid.
//
// The G query heads of a key head and the T nodes are R = T G rows over the same keys: 32 NQ of them per workgroup, which sweeps
// its share of the sequence's cached rows and drafted nodes in tiles of 32 keys.  S^T = K Q^T leaves lane l with row l % 32 and 16
// of the keys, which are, as weights, the second operand of O^T = V^T P^T as they are.  Wavefronts take tiles in turn, each with
// two LDS buffers of its own that direct global->LDS loads fill one tile ahead: no barrier in the sweep, 64 KB of a CU's reads under
// way at head_dim 128 (a CU's share of the memory rate times its latency is 26 KB).  They meet at the end.
// Bound by the cache's bytes where they are many (16 x 16384 rows, 16/4 heads of 128: 105 us, 5100 GB/s), elsewhere by the start of
// a call and the latency of its chain: length, page numbers, rows, join (8 x 4096: 25.6 us, of which the bytes take 14; 512 rows 14.5).  Workgroups that read the same keys for other
// rows follow each other on one XCD, whose L2 serves all but the first.
#pragma once

#include "sa2_causal16.h"
#include "sa2_tree_common.h"

namespace sa2 {
namespace {

// With a band, the pages of a share are in two parts: those of the window, then those of the first rows; where that is more than LDS has
// room for, they are read from the table each time.
template <class E, int D, int NQ, bool BAND>
__global__ __launch_bounds__(THREADS, 1) void tree16_kernel(Tree p, int blocks) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    constexpr int KK = D / 16, DT = D / 32, ROWS = 32 * NQ, STAGE = 2 * T::BYTES, PITCH = D + 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const uint32_t mine = lds_address(lds) + wave * 2 * STAGE;
    int32_t* const pages = (int32_t*)(lds + WAVES * 2 * STAGE);
    const int R = p.T * p.G;
    // the blocks of rows of a unit's key head on one XCD
    const int all_units = p.nsplit * p.B * p.HK, group = blockIdx.x / (8 * blocks), in = blockIdx.x - group * 8 * blocks;
    const int left = all_units - 8 * group < 8 ? all_units - 8 * group : 8, block = in / left, id = 8 * group + in - block * left;
    const int unit = id / p.HK, hk = id % p.HK, b = unit / p.nsplit, split = unit - b * p.nsplit;
    // (a short table as a whole: its reads do not wait for the sequence's length)
    const bool whole = !BAND && p.cache.width <= 4 * THREADS;
    if (p.cache.table && whole)
        for (int i = threadIdx.x; i < p.cache.width; i += THREADS) pages[i] = p.cache.table[(int64_t)b * p.cache.width + i];
    const TreeRows<BAND, 32> cache(p, b);
    const int held = cache.held, cached = cache.cached, all = cached + (p.T + 31) / 32;
    const int lo = (int)((int64_t)all * split / p.nsplit), hi = (int)((int64_t)all * (split + 1) / p.nsplit);

    // the share's part of the page table
    const int page_size = p.cache.page_size;
    int page0 = 0, near_pages = 0;                                         // (near_pages: of the first part)
    bool kept = true;
    if (BAND && p.cache.table) {
        page0 = (int)((unsigned)(cache.edge * 32) / (unsigned)page_size);
        near_pages = held > cache.edge * 32 ? (int)((unsigned)(held - 1) / (unsigned)page_size) - page0 + 1 : 0;
        const int head = cached - cache.near - (cache.whole - cache.edge), first_pages = (int)(((unsigned)(head * 32) + page_size - 1) / page_size);
        kept = (int64_t)near_pages + first_pages <= TREE16_ENTRIES;
        if (kept)
            for (int i = threadIdx.x; i < near_pages + first_pages; i += THREADS) {
                const int at = i < near_pages ? page0 + i : i - near_pages;
                pages[i] = at < p.cache.width ? p.cache.table[(int64_t)b * p.cache.width + at] : -1;
            }
        __syncthreads();
    } else if (p.cache.table) {
        if (!whole) {
            page0 = (int)((unsigned)(lo * 32) / (unsigned)page_size);
            const int end = (hi < cached ? hi * 32 : held) - 1, last = end < 0 ? -1 : (int)((unsigned)end / (unsigned)page_size);
            for (int i = threadIdx.x; page0 + i <= last; i += THREADS) pages[i] = p.cache.table[(int64_t)b * p.cache.width + page0 + i];
        }
        __syncthreads();
    }
    // K and V rows of tile t to a buffer; returns which of its 32 rows are there (the others are zeros).  One instruction brings RPW
    // rows; where these lie in one page, one behind the other, their address is scalar arithmetic, elsewhere every lane asks the
    // lane that found its row.
    const int chunk = T::dma_chunk(lane), sub = T::dma_row(lane);
    const bool pad = chunk * 8 >= p.D, together = p.D == D && (!p.cache.table || page_size % T::RPW == 0);
    auto request = [&](int t, uint32_t to) __attribute__((always_inline)) {
        const bool drafted = t >= cached;
        const int first = drafted ? (t - cached) * 32 : cache.row(t), r = first + (lane & 31);
        const Tensor &K = drafted ? p.k : p.cache.k, &V = drafted ? p.v : p.cache.v;
        int page = b, at = r;
        bool there = r < (drafted ? p.T : held);
        if (!drafted && p.cache.table && there) {
            const int i = (int)((unsigned)r / (unsigned)page_size);
            if (!BAND) page = pages[i - page0];
            else if (kept) page = pages[first >= cache.edge * 32 ? i - page0 : near_pages + i];
            else page = p.cache.table[(int64_t)b * p.cache.width + i];
            at = r - i * page_size;
            there = page >= 0 && page < p.cache.pages;
        }
        const uint32_t mask = (uint32_t)__ballot(there);
        const uint32_t koff = (uint32_t)(sub * K.sn * 2) + chunk * 16, voff = (uint32_t)(sub * V.sn * 2) + chunk * 16;
        const char *kb = (const char*)K.p + (int64_t)hk * K.sh * 2, *vb = (const char*)V.p + (int64_t)hk * V.sh * 2;
#pragma unroll
        for (int g = 0; g < T::NGROUP; ++g) {
            constexpr uint32_t FULL = (1u << T::RPW) - 1;
            const uint32_t kto = to + g * T::GROUP, vto = kto + T::BYTES;
            if (together && (mask >> (g * T::RPW) & FULL) == FULL) {
                const int64_t pg = __builtin_amdgcn_readlane(page, g * T::RPW), row = __builtin_amdgcn_readlane(at, g * T::RPW);
                lds_request(kb + (pg * K.sb + row * K.sn) * 2, koff, kto);
                lds_request(vb + (pg * V.sb + row * V.sn) * 2, voff, vto);
            } else {
                const int from = g * T::RPW + sub;
                const int64_t pg = __shfl(page, from), row = __shfl(at, from);
                const bool ok = (mask >> from & 1) && !pad;
                lds_request(ok ? (const void*)(kb + (pg * K.sb + row * K.sn) * 2 + chunk * 16) : (const void*)zero_chunk, kto);
                lds_request(ok ? (const void*)(vb + (pg * V.sb + row * V.sn) * 2 + chunk * 16) : (const void*)zero_chunk, vto);
            }
        }
        return mask;
    };
    int t = lo + wave;
    uint32_t there[2] = {0, 0};
    auto begin = [&]() __attribute__((always_inline)) {
        if (t < hi) there[0] = request(t, mine);
        if (t + WAVES < hi) there[1] = request(t + WAVES, mine + STAGE);
    };
    begin();

    // what the lane's rows are and see
    uint64_t ancestors = tree_ancestors(p, b);
    const int depth = BAND ? __popcll(ancestors) - 1 : 0;
    if (BAND) ancestors = tree_banded(p, held, ancestors);
    int64_t place[NQ];                                                     // of the lane's nodes
    uint64_t seen[NQ];
    X8 q[NQ][KK];
    const float c = fabsf(p.scale) * LOG2E;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int row = block * ROWS + 32 * n + (lane & 31), node = row < R ? row / p.G : 0, h = hk * p.G + (row < R ? row - node * p.G : 0);
        seen[n] = (uint64_t)(uint32_t)__shfl((int)(ancestors >> 32), node) << 32 | (uint32_t)__shfl((int)ancestors, node);
        if (row >= R) seen[n] = 0;
        place[n] = BAND ? (int64_t)held + __shfl(depth, node) : 0;
        const uint16_t* src = (const uint16_t*)p.q.p + p.q.off(b, node, h);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            union { uint4 u; X8 x; } w;
            w.u = make_uint4(0, 0, 0, 0);
            const int col = 16 * kk + 8 * half;
            if (row < R && col < p.D) w.u = *(const uint4*)(src + col);
            w.u.x ^= flip; w.u.y ^= flip; w.u.z ^= flip; w.u.w ^= flip;
            q[n][kk] = w.x;
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) stays(q[n][kk]);                   // (their wait is here and not in the sweep)
    floatx16 o[NQ][DT];
    float m[NQ], l[NQ];
    bool look[NQ] = {};                                                    // some row's m is far from zero (the same in all lanes)
    float farthest = 0.f;                                                  // of the reference points that the lane's rows have had
    auto nothing_yet = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[n][d][i] = 0.f;
        }
    };
    nothing_yet();
    const uint32_t row_lane = T::row_lane(lane), column_lane = T::column_lane(lane);
    // FAR: scores less their reference point come first (far_from_zero): 0 never, 1 always, 2 where one is far from zero
    auto tile = [&](uint32_t at, bool drafted, int first, uint32_t here, int number, auto FAR) __attribute__((always_inline)) {
        X8 kf[KK], vf[2][DT];
        uint32_t ka = at + row_lane, va = at + T::BYTES + column_lane;
        stays(ka);
        stays(va);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) kf[kk] = lds_read_x8<X8>(ka + (uint32_t)(kk / 2 * T::BLOCK + kk % 2 * 32));
        floatx16 x[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[n][i] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) x[n] = E::mfma(kf[kk], q[n][kk], x[n], 0, 0, 0);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[ks][d] = quad_tile_column<D, X8>(va, 0, d, ks);
        // (with a band, cached rows that some node does not see are in this tile)
        const bool edge = BAND && !drafted && number >= cache.near;
        uint32_t bits = 0;
        if (drafted || edge) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int d = 0; d < DT; ++d) bits |= odd_bits<E>(vf[ks][d]);
        }
        const bool odd = any_odd(bits);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            uint32_t sees = drafted ? (uint32_t)(seen[n] >> first) & here : seen[n] ? here : 0u;
            if (edge) sees &= tree_window(p, place[n], first);
            const bool masked = drafted || edge || here != ~0u || __any(!seen[n]);
            float top = -INFINITY;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[n][i] = sees >> (8 * (i / 4) + 4 * half + i % 4) & 1 ? x[n][i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, x[n][i]);
            if (BAND && p.scores && block * ROWS + 32 * n + (lane & 31) < R) {
                float* const to = p.scores + (((int64_t)b * p.HK + hk) * R + block * ROWS + 32 * n + (lane & 31)) * p.span + (int64_t)number * 32 + 4 * half;
#pragma unroll
                for (int i = 0; i < 4; ++i) *(float4*)(to + 8 * i) = make_float4(x[n][4 * i], x[n][4 * i + 1], x[n][4 * i + 2], x[n][4 * i + 3]);
            }
            top = fmaxf(top, other_half(top));
            const float m2 = fmaxf(m[n], top), ref = m2 == -INFINITY ? 0.f : m2;
            if (__any(m2 != m[n])) {
                const float f = m[n] == -INFINITY ? 0.f : exp2f((m[n] - ref) * c);
                l[n] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[n][d][i] *= f;
                m[n] = m2;
                if (decltype(FAR)::value == 2) look[n] = __any(far_from_zero(ref, c));
                if (decltype(FAR)::value == 0) farthest = fmaxf(farthest, fabsf(ref));
            }
            union { uint32_t u[8]; X8 v[2]; } w;
            // (fp16: weights of up to 2^15 instead of 1, in all shares alike, so that many far below the largest are not lost)
            constexpr float lift = E::DTYPE == SA2_F16 ? 15.f : 0.f;
            float off = fmaf(-ref, c, lift);
            if (decltype(FAR)::value == 1 || (decltype(FAR)::value == 2 && look[n])) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[n][i] -= ref;
                off = lift;
            }
            float part[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float e[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = 2 * i + j;
                    e[j] = fast_exp2(fmaf(x[n][r], c, off));
                    if (masked) e[j] = sees >> (8 * (r / 4) + 4 * half + r % 4) & 1 ? e[j] : 0.f;
                    part[j] += e[j];
                }
                w.u[i] = pack2<E>(e[0], e[1]);
            }
            l[n] += part[0] + part[1];
            if (odd) {
                // an infinity or NaN among the drafted values: one node at a time, into the rows that see it
#pragma unroll 1
                for (int key = 0; key < 32; ++key) {
                    const int ks = key / 16, slot = key % 4 + 4 * (key % 16 / 8);
                    const bool own = (key / 4 & 1) == half, sees_it = sees >> key & 1;
                    auto only = [&](const X8& a, const X8& z) {
                        union { X8 v; uint32_t u[4]; } s, y;
                        s.v = a;
                        y.v = z;
#pragma unroll
                        for (int i = 0; i < 4; ++i) s.u[i] = own && slot / 2 == i ? (ks ? y.u[i] : s.u[i]) & (slot & 1 ? 0xffff0000u : 0xffffu) : 0u;
                        return s.v;
                    };
                    const X8 weight = only(w.v[0], w.v[1]);
                    floatx16 zero;
#pragma unroll
                    for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const floatx16 one = E::mfma(only(vf[0][d], vf[1][d]), weight, zero, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[n][d][i] = sees_it ? o[n][d][i] + one[i] : o[n][d][i];
                    }
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[n][d] = E::mfma(vf[ks][d], w.v[ks], o[n][d], 0, 0, 0);
            }
        }
    };
    auto sweep = [&](auto FAR) __attribute__((always_inline)) {
        for (int s = 0; t < hi; t += WAVES, s ^= 1) {
            if (t + WAVES < hi) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * T::NGROUP) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            tile(mine + s * STAGE, t >= cached, t >= cached ? (t - cached) * 32 : BAND ? cache.row(t) : 0, s ? there[1] : there[0], t, FAR);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (t + 2 * WAVES < hi) {
                const uint32_t next = request(t + 2 * WAVES, mine + s * STAGE);
                if (s) there[1] = next;
                else there[0] = next;
            }
        }
    };
    // A wavefront with a row that was so far from zero that its weights are not to be had the short way sweeps its tiles again: a look in every tile takes
    // 1.6 % of a call (16 x 16384 rows, 108 us).  Two blocks of 128 columns look all the same (48 rows over 8 x 2048: 25.9 -> 26.4 us), because a second
    // sweep's code takes registers that they lack (27.4).
    if constexpr (D * NQ > 128) {
        sweep(std::integral_constant<int, 2>{});
    } else {
        sweep(std::integral_constant<int, 0>{});
        if (__any(far_from_zero(farthest, c))) {
            t = lo + wave;
            begin();
            nothing_yet();
            sweep(std::integral_constant<int, 1>{});
        }
    }

    // the wavefronts' results meet, 32 rows at a time: [row][D] in their buffers
    float* const stats = (float*)(lds + WAVES * 2 * STAGE);                // (over the page table)
    static_assert(32 * PITCH * 4 <= 2 * STAGE, "32 rows of fp32 fit a wavefront's buffers");
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float sum = l[n] + other_half(l[n]);
        __syncthreads();
        float* const own = (float*)(lds + wave * 2 * STAGE) + (lane & 31) * PITCH;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(float4*)(own + 32 * d + 8 * g + 4 * half) = make_float4(o[n][d][4 * g], o[n][d][4 * g + 1], o[n][d][4 * g + 2], o[n][d][4 * g + 3]);
        if (half == 0) {
            stats[wave * 64 + lane] = m[n];
            stats[wave * 64 + 32 + lane] = sum;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * (D / 4); i += THREADS) {
            const int col = i / (D / 4), d = i % (D / 4) * 4, to = block * ROWS + 32 * n + col;
            if (to >= R) continue;
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int x = 0; x < WAVES; ++x) top = fmaxf(top, stats[x * 64 + col]);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < WAVES; ++x) {
                const float mx = stats[x * 64 + col], sx = stats[x * 64 + 32 + col];
                if (sx == 0.f) continue;                                   // nothing seen: its values may be anything
                const float f = mx == -INFINITY ? 1.f : exp2f((mx - top) * c);
                const float4 z = *(const float4*)((const float*)(lds + x * 2 * STAGE) + col * PITCH + d);
                total += f * sx;
                y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
            }
            if (p.nsplit > 1 || (BAND && p.scores)) {
                if (d == 0) *tree_stat(p, unit, hk, to) = TreePart{top, total};
                *(float4*)(tree_values(p, unit, hk, to, D) + d) = y;
            } else if (d < p.D) {
                const float f = total == 0.f ? 0.f : 1.f / total;
                *(uint2*)((uint16_t*)p.out.p + p.out.off(b, to / p.G, hk * p.G + to % p.G) + d) = make_uint2(pack2<E>(y.x * f, y.y * f), pack2<E>(y.z * f, y.w * f));
            }
        }
    }
}

template <class E, int D, int NQ, bool BAND>
int launch(const Tree& p, hipStream_t st) {
    const auto kernel = tree16_kernel<E, D, NQ, BAND>;
    const int blocks = (p.T * p.G + 32 * NQ - 1) / (32 * NQ);
    const int64_t grid = (int64_t)blocks * p.nsplit * p.B * p.HK;
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), WAVES * 4 * QuadTile<D>::BYTES + TREE16_ENTRIES * 4, st>>>(p, blocks);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

template <bool BAND>
int launch_tree16_of(const Tree& p, int dtype, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        const bool two = p.T * p.G > 32;
        if (p.D <= 64) return two ? launch<E, 64, 2, BAND>(p, st) : launch<E, 64, 1, BAND>(p, st);
        return two ? launch<E, 128, 2, BAND>(p, st) : launch<E, 128, 1, BAND>(p, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace
}  // namespace sa2
