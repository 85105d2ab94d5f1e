// Attention of drafted tokens (or single ones) over a cache, with fp32 products.
//
// The G query heads of a key head and the T nodes are R = T G rows over the same keys: 32 of them per workgroup, which sweeps
// its share of the sequence's cached rows and drafted nodes in tiles of 32 keys.  Its wavefronts take tiles in turn, each with
// LDS, running maximum, sum and output of its own: they meet only at the end.
// Bound by the cache's bytes where R is small, by the matrix pipe where it is large (fp32, 4 x 8192 rows, 16/4 heads of 128, single
// tokens: 81 us; the bytes take 28 at a copy's rate, the products, of whose 32 columns four hold rows, 14: the rest is the latency
// of a wavefront's tiles, whose loads start when the tile before is done).
#pragma once

#include "sa2_f32_tiles.h"
#include "sa2_tree_common.h"

namespace sa2 {
namespace {

template <int DP>
constexpr int waves_of() { return DP > 128 ? 2 : 4; }      // (the tiles of four would not fit LDS)

template <class T, int DP, bool WIDE, bool BAND>
__global__ __launch_bounds__(64 * waves_of<DP>()) void tree_f32_kernel(Tree p, int blocks) {
    constexpr bool wide = WIDE;
    constexpr int WAVES = waves_of<DP>(), PITCH = Pitch<DP>::value;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    float *kt = lds + wave * 2 * TILE * PITCH, *vt = kt + TILE * PITCH, *stats = lds + WAVES * 2 * TILE * PITCH;
    const int R = p.T * p.G;
    int id = blockIdx.x;
    const int block = id % blocks;
    id /= blocks;
    const int unit = id / p.HK, hk = id % p.HK;
    TreeShare share;
    if (!tree_share(p, unit, share)) return;
    const int b = share.b;
    const int row = block * TILE + (lane & 31), node = row < R ? row / p.G : 0, h = hk * p.G + (row < R ? row - node * p.G : 0);
    const TreeRows<BAND, TILE> cache(p, b);
    const int held = cache.held, cached = cache.cached, all = cached + (p.T + TILE - 1) / TILE;
    uint64_t seen = tree_ancestors(p, b);
    const int64_t place = BAND ? (int64_t)held + __shfl(__popcll(seen) - 1, node) : 0;      // of the lane's node
    if (BAND) seen = tree_banded(p, held, seen);
    seen = (uint64_t)__shfl((uint32_t)(seen >> 32), node) << 32 | __shfl((uint32_t)seen, node);
    if (row >= R) seen = 0;
    const int lo = (int)((int64_t)all * share.split / share.count), hi = (int)((int64_t)all * (share.split + 1) / share.count);

    float q[DP / 2];
    const float sign = p.scale < 0.f ? -1.f : 1.f, c = fabsf(p.scale) * LOG2E;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
        const float4 v = load4((const T*)p.q.p + p.q.off(b, node, h), 8 * i + 4 * half, p.D, wide, row < R);
        q[4 * i] = v.x * sign; q[4 * i + 1] = v.y * sign; q[4 * i + 2] = v.z * sign; q[4 * i + 3] = v.w * sign;
    }
    floatx16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
    float m = -INFINITY, l = 0.f;
    for (int t = lo + wave; t < hi; t += WAVES) {
        // lane l brings half a row: row l % 32 of the tile
        const bool drafted = t >= cached;
        const int first = drafted ? (t - cached) * TILE : cache.row(t), r = first + (lane & 31);
        const bool edge = BAND && !drafted && t >= cache.near;             // some node does not see all of it
        bool there;
        const T *krow = (const T*)p.q.p, *vrow = krow;                     // (can be read)
        if (drafted) {
            there = r < p.T;
            if (there) {
                krow = (const T*)p.k.p + p.k.off(b, r, hk);
                vrow = (const T*)p.v.p + p.v.off(b, r, hk);
            }
        } else {
            int page, at;
            there = r < held && tree_place(p.cache, b, r, page, at);
            if (there) {
                krow = (const T*)p.cache.k.p + p.cache.k.off(page, at, hk);
                vrow = (const T*)p.cache.v.p + p.cache.v.off(page, at, hk);
            }
        }
        __builtin_amdgcn_wave_barrier();
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const int d = half * (DP / 2) + 4 * i;
            *(float4*)(kt + (lane & 31) * PITCH + d) = load4(krow, d, p.D, wide, there);
            const float4 v = load4(vrow, d, p.D, wide, there);
            if (BAND) bits |= odd_values(v);
            *(float4*)(vt + (lane & 31) * PITCH + d) = v;
        }
        const bool odd = BAND && (drafted || edge) && __any((int)(bits >> 31));
        __threadfence_block();
        __builtin_amdgcn_wave_barrier();
        const uint32_t here = (uint32_t)__ballot(there);
        floatx16 w = tile_product<DP>(kt, q);
        uint32_t sees = drafted ? (uint32_t)(seen >> first) & here : seen ? here : 0u;
        if (edge) sees &= tree_window(p, place, first);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (!(sees >> (8 * (i / 4) + 4 * half + i % 4) & 1)) w[i] = -INFINITY;
            top = fmaxf(top, w[i]);
        }
        if (BAND && p.scores && row < R) {
            float* const to = p.scores + (((int64_t)b * p.HK + hk) * R + row) * p.span + (int64_t)t * TILE + 4 * half;
#pragma unroll
            for (int i = 0; i < 4; ++i) *(float4*)(to + 8 * i) = make_float4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
        top = fmaxf(top, other_half(top));
        const float m2 = fmaxf(m, top), at = m2 == -INFINITY ? 0.f : m2, alpha = m == -INFINITY ? 0.f : exp2f((m - at) * c);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            w[i] = exp2f((w[i] - at) * c);
            if (!(sees >> (8 * (i / 4) + 4 * half + i % 4) & 1)) w[i] = 0.f;
            sum += w[i];
        }
        if (m2 != m) {
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] *= alpha;
        }
        l += sum;
        m = m2;
        auto visible = [&](int j) { return (sees >> j & 1) != 0; };
        if constexpr (BAND) banded_rows<DP, DP>(vt, 0, w, acc, odd, sees);
        else if (drafted) weighted_rows<DP, DP, true>(vt, 0, w, acc, visible);
        else weighted_rows<DP, DP, false>(vt, 0, w, acc, visible);
    }
    l += other_half(l);
    // the wavefronts' results meet: [column][DP] over their tiles
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(float4*)(kt + (lane & 31) * PITCH + 32 * i + 8 * g + 4 * half) = make_float4(acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]);
    if (half == 0) {
        stats[wave * 64 + lane] = m;
        stats[wave * 64 + 32 + lane] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * DP / 4; i += 64 * WAVES) {
        const int col = i / (DP / 4), d = i % (DP / 4) * 4, to = block * TILE + col;
        if (to >= R) continue;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) top = fmaxf(top, stats[x * 64 + col]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < WAVES; ++x) {
            const float mx = stats[x * 64 + col], f = mx == -INFINITY ? (stats[x * 64 + 32 + col] == 0.f ? 0.f : 1.f) : exp2f((mx - top) * c);
            const float4 y = *(const float4*)(lds + x * 2 * TILE * PITCH + col * PITCH + d);
            if (stats[x * 64 + 32 + col] == 0.f) continue;                 // nothing seen: its values may be anything
            sum += f * stats[x * 64 + 32 + col];
            o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w;
        }
        if (p.nsplit > 1 || (BAND && p.scores)) {
            if (d == 0) *tree_stat(p, unit, hk, to) = TreePart{top, sum};
            *(float4*)(tree_values(p, unit, hk, to, tree_width(p.D)) + d) = o;
        } else {
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            store4((T*)p.out.p + p.out.off(b, to / p.G, hk * p.G + to % p.G), d, p.D, wide, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
        }
    }
}

template <class T>
bool wide_tree(const Tree& p) {
    constexpr int BYTES = 4 * sizeof(T);
    bool ok = p.D % 4 == 0;
    for (const Tensor* t : {&p.q, &p.k, &p.v, &p.cache.k, &p.cache.v, &p.out})
        ok = ok && (uintptr_t)t->p % BYTES == 0 && t->sn % 4 == 0 && t->sh % 4 == 0 && t->sb % 4 == 0;
    return ok;
}

template <bool BAND>
int launch_tree_f32_of(const Tree& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        return for_width(p.D <= 64 ? 64 : p.D, [&](auto w) {
            constexpr int DP = decltype(w)::value, WAVES = waves_of<DP>();
            const int blocks = (p.T * p.G + TILE - 1) / TILE;
            const int64_t grid = (int64_t)blocks * p.nsplit * p.B * p.HK;
            if (grid > 0x7fffffff) return (int)SA2_ERR_TOO_LARGE;
            const auto kernel = wide_tree<T>(p) ? tree_f32_kernel<T, DP, true, BAND> : tree_f32_kernel<T, DP, false, BAND>;
            if (!allow_full_lds((const void*)kernel)) return (int)SA2_ERR_LAUNCH_FAILED;
            kernel<<<dim3((unsigned)grid), dim3(64 * WAVES), (WAVES * 2 * TILE * Pitch<DP>::value + WAVES * 64) * sizeof(float), st>>>(p, blocks);
            return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
        });
    });
}

}  // namespace
}  // namespace sa2
