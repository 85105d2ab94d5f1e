// Large drafted trees over a cache, bf16 and fp16: more than 64 rows (nodes times query heads per key head) read the same keys, or
// more than 32 many of them (tree16_rows).
//
// The sweep of causal attention (sa2_sweep16.h): four wavefronts own 32 or 64 rows each and share tiles of 64 keys, which come from
// the pages into LDS once for up to 256 rows.  All tiles but the last cached and the drafted one are seen whole by all rows.
// Bound by MFMAs and exponentials (48 nodes of 4 heads per key head over 65536 rows: the cache's bytes take half of the
// time: four ragged caches of up to 65536 rows 105 us and the join 12, MFMAs busy 29 %, with a quarter of the 256 rows empty; full ones
// 178).
#pragma once

#include "sa2_sweep16.h"
#include "sa2_tree_common.h"

namespace sa2 {
namespace {

template <int D, int NQ, bool BAND>
struct TreeKeys {
    static constexpr bool SLIDING = false;                 // (all tiles but the leading ones go piece by piece)
    using T = QuadTile<D>;
    const Tree& p;
    const int32_t* pages;                                  // of the share, the first of them page0 (with a band: see sa2_tree16.h)
    const TreeRows<BAND, TILE_ROWS> rows;
    const char *kc, *vc, *kd, *vd;                         // cache and drafted rows of the key head
    int b, page0, near_pages, held, cached, lo, tiles, full, pieces, chunk, sub;
    float lower;
    bool pad, together, kept;
    int64_t place[NQ];                                     // of the lane's nodes
    uint64_t seen[NQ];                                     // drafted nodes that the lane's rows see (0: a row that is not there)

    // the page and the place of row r, in a tile that starts at `first`; false: it is not there
    __device__ __forceinline__ bool find(int first, int r, int& page, int& at) const {
        page = b;
        at = r;
        bool there = r < held;
        if (p.cache.table && there) {
            const int i = (int)((unsigned)r / (unsigned)p.cache.page_size);
            if (!BAND) page = pages[i - page0];
            else if (kept) page = pages[first >= rows.edge * TILE_ROWS ? i - page0 : near_pages + i];
            else page = p.cache.table[(int64_t)b * p.cache.width + i];
            at = r - i * p.cache.page_size;
            there = page >= 0 && page < p.cache.pages;
        }
        return there;
    }
    __device__ __forceinline__ void request(int t, uint32_t to) const {
        constexpr int INSTR = TILE_ROWS / T::RPW / WAVES;
        constexpr uint64_t GROUP_ROWS = (1u << T::RPW) - 1;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const bool drafted = lo + t >= cached;
        const Tensor &K = drafted ? p.k : p.cache.k, &V = drafted ? p.v : p.cache.v;
        const char *kb = drafted ? kd : kc, *vb = drafted ? vd : vc;
        int page = b, at = lane;
        const int first = drafted ? 0 : rows.row(lo + t);
        const bool there = drafted ? lane < p.T : find(first, first + lane, page, at);
        const uint64_t mask = __ballot(there);
        const uint32_t koff = (uint32_t)(sub * K.sn * 2) + chunk * 16, voff = (uint32_t)(sub * V.sn * 2) + chunk * 16;
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
            const int g = wave * INSTR + i;
            const uint32_t kto = to + Buffer<D>::FIRST + g * T::GROUP, vto = to + Buffer<D>::SECOND + g * T::GROUP;
            if (together && (mask >> (g * T::RPW) & GROUP_ROWS) == GROUP_ROWS) {
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
    }
    // (cached rows that are not there are zeros in LDS)
    __device__ __forceinline__ bool guarded(int piece) const { return lo + piece / 2 >= (BAND ? rows.near : cached); }
    __device__ __forceinline__ uint32_t sees(int n, int piece) const {
        if (lo + piece / 2 >= cached) return (uint32_t)(seen[n] >> (32 * (piece & 1)));
        int page, at;
        const int first = rows.row(lo + piece / 2), r0 = first + piece % 2 * SUB;
        uint32_t there = (uint32_t)__ballot(find(first, r0 + (int)(threadIdx.x & 31), page, at));
        if (BAND && lo + piece / 2 >= rows.near) there &= tree_window(p, place[n], r0);
        return seen[n] ? there : 0u;
    }
};

template <class E, int D, int NQ, bool BAND>
__global__ __launch_bounds__(THREADS, 1) void tree_rows16_kernel(Tree p, int blocks) {
    using T = QuadTile<D>;
    using L = SweepRegs<D, NQ>;
    constexpr int KK = D / 16, DT = D / 32, ROWS = 32 * NQ, BLOCK = ROWS * WAVES;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int32_t* const pages = (int32_t*)(lds + BUFFERS * Buffer<D>::BYTES);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, R = p.T * p.G;
    // the blocks of rows of a unit's key head on one XCD
    const int all_units = p.nsplit * p.B * p.HK, group = blockIdx.x / (8 * blocks), in = blockIdx.x - group * 8 * blocks;
    const int left = all_units - 8 * group < 8 ? all_units - 8 * group : 8, block = in / left, id = 8 * group + in - block * left;
    const int unit = id / p.HK, hk = id % p.HK;
    TreeShare share;
    if (!tree_share(p, unit, share)) return;
    const auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };       // in all lanes, which the compiler does not see
    const int b = same(share.b);
    TreeRows<BAND, TILE_ROWS> rows(p, b);
    rows.held = same(rows.held); rows.whole = same(rows.whole); rows.edge = same(rows.edge); rows.near = same(rows.near); rows.cached = same(rows.cached);
    const int held = rows.held, cached = rows.cached, all = cached + 1;
    const int lo = same((int)((int64_t)all * share.split / share.count)), hi = same((int)((int64_t)all * (share.split + 1) / share.count));

    TreeKeys<D, NQ, BAND> keys{p, pages, rows};
    keys.b = b;
    keys.held = held;
    keys.cached = cached;
    keys.lo = lo;
    keys.tiles = hi - lo;
    keys.pieces = 2 * keys.tiles;
    keys.kc = (const char*)p.cache.k.p + (int64_t)hk * p.cache.k.sh * 2;
    keys.vc = (const char*)p.cache.v.p + (int64_t)hk * p.cache.v.sh * 2;
    keys.kd = (const char*)p.k.p + (int64_t)hk * p.k.sh * 2;
    keys.vd = (const char*)p.v.p + (int64_t)hk * p.v.sh * 2;
    keys.chunk = T::dma_chunk(lane);
    keys.sub = T::dma_row(lane);
    keys.pad = keys.chunk * 8 >= p.D;
    keys.together = p.D == D && (!p.cache.table || p.cache.page_size % T::RPW == 0);
    keys.page0 = keys.near_pages = 0;
    keys.kept = true;
    bool bad = false;                                                      // a page of the share is none of the cache's
    if (BAND && p.cache.table) {
        const unsigned page_size = p.cache.page_size;
        keys.page0 = (int)((unsigned)(rows.edge * TILE_ROWS) / page_size);
        keys.near_pages = held > rows.edge * TILE_ROWS ? (int)((unsigned)(held - 1) / page_size) - keys.page0 + 1 : 0;
        const int head = cached - rows.near - (rows.whole - rows.edge), first_pages = (int)((head * TILE_ROWS + page_size - 1) / page_size), all_pages = keys.near_pages + first_pages;
        keys.kept = all_pages <= TREE16_ENTRIES;
        for (int i = threadIdx.x; i < all_pages; i += THREADS) {
            const int at = i < keys.near_pages ? keys.page0 + i : i - keys.near_pages;
            const int x = at < p.cache.width ? p.cache.table[(int64_t)b * p.cache.width + at] : -1;
            if (keys.kept) pages[i] = x;
            bad = bad || x < 0 || x >= p.cache.pages;
        }
    } else if (p.cache.table) {
        keys.page0 = (int)((unsigned)(lo * TILE_ROWS) / (unsigned)p.cache.page_size);
        const int end = (hi < cached ? hi * TILE_ROWS : held) - 1, last = end < 0 ? -1 : (int)((unsigned)end / (unsigned)p.cache.page_size);
        for (int i = threadIdx.x; keys.page0 + i <= last; i += THREADS) {
            const int x = p.cache.table[(int64_t)b * p.cache.width + keys.page0 + i];
            pages[i] = x;
            bad = bad || x < 0 || x >= p.cache.pages;
        }
    }
    bad = __syncthreads_or(bad);
    // (with a band the last rows' tile, which may not be full, is the last of those before the window's start)
    const int leading = BAND ? held / TILE_ROWS - rows.whole : held / TILE_ROWS, whole = leading < hi ? leading : hi;
    keys.full = bad || whole < lo ? 0 : whole - lo;

    uint64_t ancestors = tree_ancestors(p, b);
    const int depth = BAND ? __popcll(ancestors) - 1 : 0;
    if (BAND) ancestors = tree_banded(p, held, ancestors);
    const float c = fabsf(p.scale) * LOG2E;
    keys.lower = lowered_by<E>(held + p.T, c);
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    int node[NQ], head[NQ];
    static_for<NQ>([&](auto N) __attribute__((always_inline)) {
        constexpr int n = decltype(N)::value;
        const int row = block * BLOCK + wave * ROWS + 32 * n + (lane & 31);
        node[n] = row < R ? row / p.G : 0;
        head[n] = hk * p.G + (row < R ? row - node[n] * p.G : 0);
        keys.seen[n] = (uint64_t)(uint32_t)__shfl((int)(ancestors >> 32), node[n]) << 32 | (uint32_t)__shfl((int)ancestors, node[n]);
        if (row >= R) keys.seen[n] = 0;
        keys.place[n] = BAND ? (int64_t)held + __shfl(depth, node[n]) : 0;
        const uint16_t* src = (const uint16_t*)p.q.p + p.q.off(b, node[n], head[n]);
        uint4 x[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int col = 16 * kk + 8 * half;
            x[kk] = make_uint4(0, 0, 0, 0);
            // (rows that see nothing: zeros, whatever stands there)
            if (keys.seen[n] && col < p.D) x[kk] = *(const uint4*)(src + col);
        }
        static_for<KK>([&](auto K) __attribute__((always_inline)) {
            constexpr int kk = decltype(K)::value;
            L::template set_regs<L::Q0 + (n * KK + kk) * 4>(x[kk].x ^ flip, x[kk].y ^ flip, x[kk].z ^ flip, x[kk].w ^ flip);
        });
    });
    float m[NQ], l[NQ];
    if (keys.tiles > 0) {
        sweep16<E, D, NQ>(keys, lds_address(lds), c, m, l);
    } else {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
        }
    }
    static_for<NQ>([&](auto N) __attribute__((always_inline)) {
        constexpr int n = decltype(N)::value;
        const int row = block * BLOCK + wave * ROWS + 32 * n + (lane & 31);
        const float both = l[n] + other_half(l[n]);
        const bool any = keys.seen[n] && keys.tiles > 0 && both != 0.f;
        const float sum = any ? both : 0.f, f = any ? 1.f / sum : 0.f;
        if (row < R) {
            float* const part = p.nsplit > 1 ? tree_values(p, unit, hk, row, D) : nullptr;
            uint16_t* const out = (uint16_t*)p.out.p + p.out.off(b, node[n], head[n]);
            static_for<4 * DT>([&](auto X) __attribute__((always_inline)) {
                constexpr int x = decltype(X)::value;
                float4 o = L::template get_regs<L::O0 + n * DT * 16 + 4 * x>();
                if (!any) o = make_float4(0.f, 0.f, 0.f, 0.f);             // (its registers may hold anything)
                const int col = 8 * x + 4 * half;
                if (part) *(float4*)(part + col) = o;
                else if (col < p.D) *(uint2*)(out + col) = make_uint2(pack2<E>(o.x * f, o.y * f), pack2<E>(o.z * f, o.w * f));
            });
            if (part && half == 0) *tree_stat(p, unit, hk, row) = TreePart{any ? m[n] : -INFINITY, sum};
        }
    });
}

template <class E, int D, int NQ, bool BAND>
int launch(const Tree& p, hipStream_t st) {
    const auto kernel = tree_rows16_kernel<E, D, NQ, BAND>;
    const int blocks = (p.T * p.G + 32 * NQ * WAVES - 1) / (32 * NQ * WAVES);
    const int64_t grid = (int64_t)blocks * p.nsplit * p.B * p.HK;
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), BUFFERS * Buffer<D>::BYTES + TREE16_ENTRIES * 4, st>>>(p, blocks);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

template <bool BAND>
int launch_tree_rows16_of(const Tree& p, int dtype, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        const bool two = p.T * p.G > 32 * WAVES;
        if (p.D <= 64) return two ? launch<E, 64, 2, BAND>(p, st) : launch<E, 64, 1, BAND>(p, st);
        return two ? launch<E, 128, 2, BAND>(p, st) : launch<E, 128, 1, BAND>(p, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace
}  // namespace sa2
