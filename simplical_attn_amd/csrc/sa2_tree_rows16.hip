// Large drafted trees over a cache, bf16 and fp16: more than 64 rows (nodes times query heads per key head) read the same keys, or
// more than 32 many of them (tree16_rows).
//
// The sweep of causal attention (sa2_sweep16.h): four wavefronts own 32 or 64 rows each and share tiles of 64 keys, which come from
// the pages into LDS once for up to 256 rows.  All tiles but the last cached and the drafted one are seen whole by all rows.
// Bound by MFMAs and exponentials (48 nodes of 4 heads per key head over 65536 rows: the cache's bytes take half of the
// time: four ragged caches of up to 65536 rows 105 us and the join 12, MFMAs busy 29 %, with a quarter of the 256 rows empty; full ones
// 178).
#include "sa2_sweep16.h"
#include "sa2_tree_common.h"

namespace sa2 {
namespace {

template <int D, int NQ>
struct TreeKeys {
    using T = QuadTile<D>;
    const Tree& p;
    const int32_t* pages;                                  // of the share, the first of them page0
    const char *kc, *vc, *kd, *vd;                         // cache and drafted rows of the key head
    int b, page0, held, cached, lo, tiles, full, pieces, chunk, sub;
    float lower;
    bool pad, together;
    uint64_t seen[NQ];                                     // drafted nodes that the lane's rows see (0: a row that is not there)

    // the page and the place of row r; false: it is not there
    __device__ __forceinline__ bool find(int r, int& page, int& at) const {
        page = b;
        at = r;
        bool there = r < held;
        if (p.cache.table && there) {
            const int i = (int)((unsigned)r / (unsigned)p.cache.page_size);
            page = pages[i - page0];
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
        const bool there = drafted ? lane < p.T : find((lo + t) * TILE_ROWS + lane, page, at);
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
    __device__ __forceinline__ bool guarded(int piece) const { return lo + piece / 2 >= cached; }
    __device__ __forceinline__ uint32_t sees(int n, int piece) const {
        if (lo + piece / 2 >= cached) return (uint32_t)(seen[n] >> (32 * (piece & 1)));
        int page, at;
        const uint32_t there = (uint32_t)__ballot(find(lo * TILE_ROWS + piece * SUB + (int)(threadIdx.x & 31), page, at));
        return seen[n] ? there : 0u;
    }
};

template <class E, int D, int NQ>
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
    const int held = same(tree_held(p, b)), cached = (held + TILE_ROWS - 1) / TILE_ROWS, all = cached + 1;
    const int lo = same((int)((int64_t)all * share.split / share.count)), hi = same((int)((int64_t)all * (share.split + 1) / share.count));

    TreeKeys<D, NQ> keys{p, pages};
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
    keys.page0 = 0;
    bool bad = false;                                                      // a page of the share is none of the cache's
    if (p.cache.table) {
        keys.page0 = (int)((unsigned)(lo * TILE_ROWS) / (unsigned)p.cache.page_size);
        const int end = (hi < cached ? hi * TILE_ROWS : held) - 1, last = end < 0 ? -1 : (int)((unsigned)end / (unsigned)p.cache.page_size);
        for (int i = threadIdx.x; keys.page0 + i <= last; i += THREADS) {
            const int x = p.cache.table[(int64_t)b * p.cache.width + keys.page0 + i];
            pages[i] = x;
            bad = bad || x < 0 || x >= p.cache.pages;
        }
    }
    bad = __syncthreads_or(bad);
    const int whole = held / TILE_ROWS < hi ? held / TILE_ROWS : hi;
    keys.full = bad || whole < lo ? 0 : whole - lo;

    const uint64_t ancestors = tree_ancestors(p, b);
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

template <class E, int D, int NQ>
int launch(const Tree& p, hipStream_t st) {
    const auto kernel = tree_rows16_kernel<E, D, NQ>;
    const int blocks = (p.T * p.G + 32 * NQ * WAVES - 1) / (32 * NQ * WAVES);
    const int64_t grid = (int64_t)blocks * p.nsplit * p.B * p.HK;
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), BUFFERS * Buffer<D>::BYTES + TREE16_ENTRIES * 4, st>>>(p, blocks);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

int launch_tree_rows16(const Tree& p, int dtype, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        const bool two = p.T * p.G > 32 * WAVES;
        if (p.D <= 64) return two ? launch<E, 64, 2>(p, st) : launch<E, 64, 1>(p, st);
        return two ? launch<E, 128, 2>(p, st) : launch<E, 128, 1>(p, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace sa2
