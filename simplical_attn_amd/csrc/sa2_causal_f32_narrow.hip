// Causal attention with fp32 products, head_dim up to 128 (sa2_causal_f32.hip has the mathematics): a workgroup has 32 rows, its
// four wavefronts divide the tiles of 32 rows that these see and bring each its own into LDS; their sums meet at the end.
// Small calls are bound by the longest chain of tiles: a quarter of it here.  Every tile is read by as many workgroups as
// have rows that see it, four times as many as with 128 rows each, from L2.  Against 128 rows per workgroup: 323 rows in four
// sequences, 4/2 heads, head_dim 64, forward and backward 244 -> 80 us (67 with all gradients in one launch); B1 N8192 H4/1 D128 1779 -> 950 us forward (72 TFLOP/s of
// the 153 that a large product reaches: an exponential and its mask for every two columns of products), 14.2 -> 3.9 ms backward.
#include "sa2_f32_tiles.h"

namespace sa2 {
namespace {

constexpr int THREADS = 256, WAVES = 4;

// 32 rows from `first` on on their way to LDS by one wavefront, neighbouring lanes at neighbouring columns (each lane with a row of
// its own, every instruction touches 64 lines of L1)
template <class T, int DP>
struct Half {
    static constexpr int PER = DP / 8, STEP = 256 / DP;                    // chunks per lane, rows per instruction
    float4 x[PER];
    __device__ __forceinline__ void load(const Tensor& t, const Span& s, int first, int h, int D, bool wide) {
        const int lane = threadIdx.x & 63, r = lane / (DP / 4), d = lane % (DP / 4) * 4;
        const T* base = (const T*)t.p + row_offset(t, s, 0, h);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = first + i * STEP + r;
            x[i] = load4(base + (int64_t)(at < s.len ? at : 0) * t.sn, d, D, wide, at < s.len);
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
        const int lane = threadIdx.x & 63;
        float* at = lds + lane / (DP / 4) * Pitch<DP>::value + lane % (DP / 4) * 4;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            *(float4*)(at + i * STEP * Pitch<DP>::value) = x[i];
    }
};
__device__ __forceinline__ void wave_fence() {
    __threadfence_block();
    __builtin_amdgcn_wave_barrier();
}
// the wavefront's sums as rows [own row][DP] of its region
template <int DP>
__device__ __forceinline__ void leave(float* lds, const floatx16 (&acc)[DP / 32]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(float4*)(lds + (lane & 31) * Pitch<DP>::value + 32 * b + 8 * g + 4 * (lane >> 5)) =
                make_float4(acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]);
}
// the sums of all wavefronts, in their order, as rows of t; `at`: where a region has them
template <class T, int DP>
__device__ __forceinline__ void add_up(const float* lds, int region, const Tensor& t, const Span& s, int first, int h, int D, bool wide, float factor) {
    for (int i = threadIdx.x; i < TILE * (DP / 4); i += THREADS) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        if (first + r >= s.len) continue;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float4 x = *(const float4*)(lds + w * region + r * Pitch<DP>::value + d);
            y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
        }
        store4((T*)t.p + row_offset(t, s, first + r, h), d, D, wide, make_float4(y.x * factor, y.y * factor, y.z * factor, y.w * factor));
    }
}
template <class T>
__device__ __forceinline__ void zeros(const Tensor& t, const Span& s, int h, int D) {
    if (!t.p) return;
    for (int i = threadIdx.x; i < s.len * D; i += THREADS) from_float(0.f, (T*)t.p + row_offset(t, s, i / D, h) + i % D);
}

template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(THREADS) void causal_f32_narrow_fwd_kernel(Causal p) {
    constexpr bool wide = WIDE;
    constexpr int REGION = 2 * TILE * Pitch<DP>::value;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    float *kt = lds + wave * REGION, *vt = kt + TILE * Pitch<DP>::value, *stats = lds + WAVES * REGION;
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.H, stream, tile);
    const int b = stream / p.H, h = stream % p.H, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, TILE, s)) return;
    float* lse = p.lse + ((int64_t)s.b * p.H + h) * p.rows.N + s.first;
    if (s.fill) {
        zeros<T>(p.out, s, h, p.D);
        for (int i = threadIdx.x; i < s.len; i += THREADS) lse[i] = -INFINITY;
        return;
    }
    const int q0 = ((s.len + TILE - 1) / TILE - 1 - s.block) * TILE, qi = q0 + (lane & 31);
    const float c = fabsf(p.scale) * LOG2E;
    float q[DP / 2];
    own_rows<T, DP>(q, p.q, s, q0, h, p.D, wide, p.scale < 0.f ? -1.f : 1.f);
    floatx16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
    float m = -INFINITY, l = 0.f;
    Half<T, DP> ks, vs;
    ks.load(p.k, s, wave * TILE, hk, p.D, wide);
    vs.load(p.v, s, wave * TILE, hk, p.D, wide);
    for (int k0 = wave * TILE; k0 <= q0; k0 += WAVES * TILE) {
        __builtin_amdgcn_wave_barrier();
        ks.put(kt);
        vs.put(vt);
        wave_fence();
        if (k0 + WAVES * TILE <= q0) {
            ks.load(p.k, s, k0 + WAVES * TILE, hk, p.D, wide);
            vs.load(p.v, s, k0 + WAVES * TILE, hk, p.D, wide);
        }
        floatx16 w = tile_product<DP>(kt, q);
        const bool masked = k0 == q0;
        auto sees = [&](int j) { return k0 + j <= qi; };
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (masked && !sees(8 * (i / 4) + 4 * half + i % 4)) w[i] = -INFINITY;
            top = fmaxf(top, w[i]);
        }
        top = fmaxf(top, other_half(top));
        const float m2 = fmaxf(m, top), at = m2 == -INFINITY ? 0.f : m2, alpha = m == -INFINITY ? 0.f : exp2f((m - at) * c);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            w[i] = exp2f((w[i] - at) * c);
            if (masked && !sees(8 * (i / 4) + 4 * half + i % 4)) w[i] = 0.f;
            sum += w[i];
        }
        if (m2 != m) {
            l *= alpha;
#pragma unroll
            for (int b2 = 0; b2 < DP / 32; ++b2)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b2][i] *= alpha;
        }
        l += sum;
        m = m2;
        if (masked) weighted_rows<DP, DP, true>(vt, 0, w, acc, sees);
        else weighted_rows<DP, DP, false>(vt, 0, w, acc, sees);
    }
    l += other_half(l);
    __builtin_amdgcn_wave_barrier();
    leave<DP>(kt, acc);
    if (half == 0) {
        stats[wave * 64 + lane] = m;
        stats[wave * 64 + 32 + lane] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * (DP / 4); i += THREADS) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        if (q0 + r >= s.len) continue;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w * 64 + r]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float mw = stats[w * 64 + r], lw = stats[w * 64 + 32 + r], f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : exp2f((mw - top) * c);
            const float4 x = *(const float4*)(lds + w * REGION + r * Pitch<DP>::value + d);
            sum += f * lw;
            y.x += f * x.x; y.y += f * x.y; y.z += f * x.z; y.w += f * x.w;
        }
        const float f = 1.f / sum;
        y.x *= f; y.y *= f; y.z *= f; y.w *= f;
        const int64_t to = row_offset(p.out, s, q0 + r, h);
        store4((T*)p.out.p + to, d, p.D, wide, y);
        if constexpr (sizeof(T) == 2)
            if (p.out_low) {
                float4 z = y;
                float* v = &z.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    T rounded;
                    from_float(v[j], &rounded);
                    v[j] -= to_float(rounded);
                }
                store4((T*)p.out_low + to, d, p.D, wide, z);
            }
        if (d == 0) lse[q0 + r] = fmaf(top, fabsf(p.scale), logf(sum));
    }
}

template <class T, int DP, bool WIDE>
__device__ __forceinline__ void queries_gradient(const Causal& p, int id, float* lds) {
    constexpr bool wide = WIDE;
    constexpr int REGION = 2 * TILE * Pitch<DP>::value;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    float *kt = lds + wave * REGION, *vt = kt + TILE * Pitch<DP>::value;
    int stream, tile;
    order(id, p.rows.B * p.H, stream, tile);
    const int b = stream / p.H, h = stream % p.H, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, TILE, s)) return;
    if (s.fill) return zeros<T>(p.dq, s, h, p.D);
    const int q0 = ((s.len + TILE - 1) / TILE - 1 - s.block) * TILE, qi = q0 + (lane & 31);
    float q[DP / 2], d[DP / 2];
    own_rows<T, DP>(q, p.q, s, q0, h, p.D, wide, 1.f);
    own_rows<T, DP>(d, p.dout, s, q0, h, p.D, wide, 1.f);
    const int64_t at = ((int64_t)s.b * p.H + h) * p.rows.N + s.first + qi;
    const float lse2 = qi < s.len ? p.lse[at] * LOG2E : 0.f, delta = qi < s.len ? p.delta[at] : 0.f, c = p.scale * LOG2E;
    floatx16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
    Half<T, DP> ks, vs;
    ks.load(p.k, s, wave * TILE, hk, p.D, wide);
    vs.load(p.v, s, wave * TILE, hk, p.D, wide);
    for (int k0 = wave * TILE; k0 <= q0; k0 += WAVES * TILE) {
        __builtin_amdgcn_wave_barrier();
        ks.put(kt);
        vs.put(vt);
        wave_fence();
        if (k0 + WAVES * TILE <= q0) {
            ks.load(p.k, s, k0 + WAVES * TILE, hk, p.D, wide);
            vs.load(p.v, s, k0 + WAVES * TILE, hk, p.D, wide);
        }
        floatx16 w = tile_product<DP>(kt, q);
        const floatx16 dp = tile_product<DP>(vt, d);
        const bool masked = k0 == q0;
        auto sees = [&](int j) { return k0 + j <= qi && qi > 0; };         // (a first query: see sa2_causal_f32.hip)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            w[i] = exp2f(fmaf(w[i], c, -lse2)) * (dp[i] - delta);
            if (masked && !sees(8 * (i / 4) + 4 * half + i % 4)) w[i] = 0.f;
        }
        if (masked) weighted_rows<DP, DP, true>(kt, 0, w, acc, sees);
        else weighted_rows<DP, DP, false>(kt, 0, w, acc, sees);
    }
    __builtin_amdgcn_wave_barrier();
    leave<DP>(kt, acc);
    __syncthreads();
    add_up<T, DP>(lds, REGION, p.dq, s, q0, h, p.D, wide, p.scale);
}

// KEYS, VALUES: which of dK and dV a workgroup makes
template <class T, int DP, bool WIDE, bool KEYS, bool VALUES>
__device__ __forceinline__ void keys_gradients(const Causal& p, int id, float* lds) {
    constexpr bool wide = WIDE;
    constexpr int REGION = 2 * TILE * Pitch<DP>::value;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    float *qt = lds + wave * REGION, *dt = qt + TILE * Pitch<DP>::value, *stats = lds + WAVES * REGION + wave * 64;
    int stream, tile;
    order(id, p.rows.B * p.HK, stream, tile);
    const int b = stream / p.HK, hk = stream % p.HK;
    Span s;
    if (!find_tile(p.rows, b, tile, TILE, s)) return;
    if (s.fill) {
        if (KEYS) zeros<T>(p.dk, s, hk, p.D);
        if (VALUES) zeros<T>(p.dv, s, hk, p.D);
        return;
    }
    const int j0 = s.block * TILE, ki = j0 + (lane & 31), per = (s.len - j0 + TILE - 1) / TILE;
    float k[DP / 2], v[DP / 2];
    own_rows<T, DP>(k, p.k, s, j0, hk, p.D, wide, 1.f);
    if constexpr (KEYS) own_rows<T, DP>(v, p.v, s, j0, hk, p.D, wide, 1.f);
    const float c = p.scale * LOG2E;
    floatx16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = zero16();
    Half<T, DP> qs, ds;
    float stat = 0.f;
    auto load = [&](int it) {
        const int h = hk * p.G + it / per, q0 = j0 + it % per * TILE, i0 = q0 + (lane & 31);
        const int64_t at = ((int64_t)s.b * p.H + h) * p.rows.N + s.first + i0;
        qs.load(p.q, s, q0, h, p.D, wide);
        ds.load(p.dout, s, q0, h, p.D, wide);
        stat = i0 >= s.len ? 0.f : half ? p.delta[at] : p.lse[at] * LOG2E;
    };
    if (wave < per * p.G) load(wave);
    for (int it = wave; it < per * p.G; it += WAVES) {
        const int q0 = j0 + it % per * TILE;
        __builtin_amdgcn_wave_barrier();
        qs.put(qt);
        ds.put(dt);
        stats[lane] = stat;
        wave_fence();
        if (it + WAVES < per * p.G) load(it + WAVES);
        floatx16 w = tile_product<DP>(qt, k);
        const bool masked = q0 == j0;
        auto sees = [&](int i) { return q0 + i >= ki; };
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 8 * (i / 4) + 4 * half + i % 4;
            w[i] = exp2f(fmaf(w[i], c, -stats[row]));
            if (masked && !sees(row)) w[i] = 0.f;
        }
        if constexpr (VALUES) {
            if (masked) weighted_rows<DP, DP, true>(dt, 0, w, dv, sees);
            else weighted_rows<DP, DP, false>(dt, 0, w, dv, sees);
        }
        if constexpr (KEYS) {
            const floatx16 dp = tile_product<DP>(dt, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 8 * (i / 4) + 4 * half + i % 4;
                w[i] *= dp[i] - stats[32 + row];
                if (masked && (!sees(row) || q0 + row == 0)) w[i] = 0.f;
            }
            if (masked) weighted_rows<DP, DP, true>(qt, 0, w, dk, [&](int i) { return sees(i) && q0 + i > 0; });
            else weighted_rows<DP, DP, false>(qt, 0, w, dk, sees);
        }
    }
    __builtin_amdgcn_wave_barrier();
    if constexpr (KEYS) leave<DP>(qt, dk);
    if constexpr (VALUES) leave<DP>(dt, dv);
    __syncthreads();
    if (KEYS && p.dk.p) add_up<T, DP>(lds, REGION, p.dk, s, j0, hk, p.D, wide, p.scale);
    if (VALUES && p.dv.p) add_up<T, DP>(lds + TILE * Pitch<DP>::value, REGION, p.dv, s, j0, hk, p.D, wide, 1.f);
}

// All gradients in one launch, so that one's workgroups fill the CUs that the other's last ones leave (323 rows in four sequences: dK and
// dV 38 us, dQ 19, one after the other): `keys` workgroups for dK and dV (APART: for dK), `values` for dV, the others for dQ.
// APART: dK and dV from workgroups of their own, with the logits twice (five products instead of four).  At head_dim 128 always, because
// keys, values and both sums take 256 registers and what did not fit went to memory (N 8192, 4/1 heads: 5.8 ms together, 4.7 apart);
// below where there are CUs for both (217 rows of 4/2 heads of 64: 41 us together, 32 apart; B2 N1024 H8/8: 156 and 181).
template <class T, int DP, bool WIDE, bool APART>
__global__ __launch_bounds__(THREADS) void causal_f32_narrow_bwd_kernel(Causal p, int keys, int values) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int id = blockIdx.x;
    if (id < keys) keys_gradients<T, DP, WIDE, true, !APART>(p, id, lds);
    else if (APART && id < keys + values) keys_gradients<T, DP, WIDE, false, true>(p, id - keys, lds);
    else queries_gradient<T, DP, WIDE>(p, id - keys - values, lds);
}

template <class K, class... A>
int launch(K kernel, const Causal& p, int64_t streams, int DP, hipStream_t st, A... more) {
    const int64_t grid = (int64_t)p.rows.B * streams * count_tiles(p.rows, TILE);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), (WAVES * 2 * TILE * (DP + 4) + WAVES * 64) * sizeof(float), st>>>(p, more...);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}
template <class F>
int for_narrow_width(int D, F&& f) {
    if (D <= 32) return f(std::integral_constant<int, 32>{});
    if (D <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

}  // namespace

int launch_causal_f32_narrow_fwd(const Causal& p, int dtype, bool wide, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        return for_narrow_width(p.D, [&](auto w) {
            constexpr int DP = decltype(w)::value;
            return launch(wide ? causal_f32_narrow_fwd_kernel<T, DP, true> : causal_f32_narrow_fwd_kernel<T, DP, false>, p, p.H, DP, st);
        });
    });
}

int launch_causal_f32_narrow_bwd(const Causal& p, int dtype, bool wide, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        return for_narrow_width(p.D, [&](auto w) {
            constexpr int DP = decltype(w)::value;
            const int64_t each = (int64_t)p.rows.B * p.HK * count_tiles(p.rows, TILE);
            const bool any = p.dk.p || p.dv.p, apart = DP == 128 || 2 * each <= CUS;
            const int streams = (apart ? (p.dk.p ? p.HK : 0) + (p.dv.p ? p.HK : 0) : any ? p.HK : 0) + (p.dq.p ? p.H : 0);
            const int keys = (apart ? p.dk.p != nullptr : any) ? (int)each : 0, values = apart && p.dv.p ? (int)each : 0;
            if (streams == 0) return (int)SA2_OK;
            if constexpr (DP < 128)
                if (!apart) return launch(wide ? causal_f32_narrow_bwd_kernel<T, DP, true, false> : causal_f32_narrow_bwd_kernel<T, DP, false, false>, p, streams, DP, st, keys, values);
            return launch(wide ? causal_f32_narrow_bwd_kernel<T, DP, true, true> : causal_f32_narrow_bwd_kernel<T, DP, false, true>, p, streams, DP, st, keys, values);
        });
    });
}

}  // namespace sa2
