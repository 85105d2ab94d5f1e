// Causal attention with fp32 products (v_mfma_f32_32x32x2_f32), forward and backward: fp32 tensors, and 16-bit ones that the
// 16-bit kernels do not take (head_dim above 128 or no multiple of 8, rows off the 16-byte grid).  Any head_dim to 256.
//
//   S = scale Q K^T (j <= i), P = softmax(S), O = P V, LSE = log sum e^S
//   dV = P^T dO, dP = dO V^T, dS = P (dP - delta), delta_i = sum_d dO O, dQ = scale dS K, dK = scale dS^T Q
//
// Every product keeps the index that a wavefront owns (32 queries, or 32 keys) in the lane: S^T = K Q^T leaves lane l with
// query l % 32 and the keys 8g + 4(l/32) + r in register 4g + r, so that softmax is arithmetic within a lane and one exchange
// of halves, and these registers are, as they are, the second operand of the next product.
// Here: the kernels for a head_dim above 128, whose accumulators leave no room for a wavefront to have tiles of its own (four share
// each tile and have 32 rows apiece); the row terms; the choice.  Up to 128: sa2_causal_f32_narrow.hip.
// Bound by the matrix pipe: an MFMA takes 64 cycles, for which one LDS read of 4 or 16 bytes per lane is enough.  N4096 H8/2, forward and
// backward: head_dim 256 bf16 2.3 and 15.4 ms, fp32 3.3 and 19.5; 192 (on 256 columns) as long.
#include "sa2_f32_tiles.h"

namespace sa2 {
namespace {

constexpr int THREADS = 256, WAVES = 4, BLOCK = TILE * WAVES;

// 32 rows at `first` of the sequence on their way from memory to LDS: DP / 32 chunks of four columns per thread
template <class T, int DP>
struct Stage {
    static constexpr int PER = DP / 32;
    float4 x[PER];
    __device__ __forceinline__ void load(const Tensor& t, const Span& s, int first, int h, int D, bool wide) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = i * THREADS + threadIdx.x, r = c / (DP / 4), d = c % (DP / 4) * 4;
            x[i] = load4((const T*)t.p + row_offset(t, s, first + r < s.len ? first + r : 0, h), d, D, wide, first + r < s.len);
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = i * THREADS + threadIdx.x, r = c / (DP / 4), d = c % (DP / 4) * 4;
            *(float4*)(lds + r * Pitch<DP>::value + d) = x[i];
        }
    }
};
template <class T, int DO>
__device__ __forceinline__ void store_own(const Tensor& t, const Span& s, int at, int h, int first, int D, bool wide, const floatx16 (&acc)[DO / 32], float factor) {
    const int half = (threadIdx.x & 63) >> 5;
    if (at >= s.len) return;
    T* row = (T*)t.p + row_offset(t, s, at, h);
#pragma unroll
    for (int b = 0; b < DO / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4(row, first + 32 * b + 8 * g + 4 * half, D, wide,
                   make_float4(acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor, acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor));
}
// Rows of no sequence: zeros
template <class T>
__device__ __forceinline__ void fill_rows(const Tensor& t, const Span& s, int h, int D) {
    if (!t.p) return;
    for (int i = threadIdx.x; i < s.len * D; i += THREADS) from_float(0.f, (T*)t.p + row_offset(t, s, i / D, h) + i % D);
}

template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(THREADS) void causal_f32_fwd_kernel(Causal p) {
    constexpr bool wide = WIDE;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *kt = lds, *vt = lds + TILE * Pitch<DP>::value;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.H, stream, tile);
    const int b = stream / p.H, h = stream % p.H, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, BLOCK, s)) return;
    float* lse = p.lse + ((int64_t)s.b * p.H + h) * p.rows.N + s.first;
    if (s.fill) {
        fill_rows<T>(p.out, s, h, p.D);
        for (int i = threadIdx.x; i < s.len; i += THREADS) lse[i] = -INFINITY;
        return;
    }
    const int q0 = ((s.len + BLOCK - 1) / BLOCK - 1 - s.block) * BLOCK, mine = q0 + wave * TILE, qi = mine + (lane & 31);
    const float c = fabsf(p.scale) * LOG2E;
    float q[DP / 2];
    own_rows<T, DP>(q, p.q, s, mine, h, p.D, wide, p.scale < 0.f ? -1.f : 1.f);
    floatx16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
    float m = -INFINITY, l = 0.f;
    const int last = q0 + BLOCK < s.len ? q0 + BLOCK : s.len;             // keys 0 .. last - 1
    Stage<T, DP> ks, vs;
    ks.load(p.k, s, 0, hk, p.D, wide);
    vs.load(p.v, s, 0, hk, p.D, wide);
    for (int k0 = 0; k0 < last; k0 += TILE) {
        __syncthreads();
        ks.put(kt);
        vs.put(vt);
        __syncthreads();
        if (k0 + TILE < last) {
            ks.load(p.k, s, k0 + TILE, hk, p.D, wide);
            vs.load(p.v, s, k0 + TILE, hk, p.D, wide);
        }
        if (k0 > mine + TILE - 1) continue;                               // all keys behind the wavefront's queries
        floatx16 w = tile_product<DP>(kt, q);
        const bool masked = k0 + TILE - 1 > mine;
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
        if (m2 != m) {                                                    // (a lane whose maximum stays has alpha 1)
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
    const float f = l > 0.f || l != l ? 1.f / l : 0.f;
    store_own<T, DP>(p.out, s, qi, h, 0, p.D, wide, acc, f);
    if constexpr (sizeof(T) == 2)
        if (p.out_low) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    T rounded;
                    from_float(acc[i][j] * f, &rounded);
                    acc[i][j] = acc[i][j] * f - to_float(rounded);
                }
            Tensor low = p.out;
            low.p = p.out_low;
            store_own<T, DP>(low, s, qi, h, 0, p.D, wide, acc, 1.f);
        }
    if (half == 0 && qi < s.len) lse[qi] = l == 0.f ? -INFINITY : fmaf(m, fabsf(p.scale), logf(l));
}

// delta = sum_d dO O, O with what its rounding left: a wavefront per row
template <class T>
__global__ __launch_bounds__(THREADS) void causal_f32_delta_kernel(Causal p) {
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (r >= (int64_t)p.rows.B * p.rows.N * p.H) return;
    const int h = (int)(r % p.H), n = (int)(r / p.H % p.rows.N), b = (int)(r / p.H / p.rows.N);
    const int64_t at = p.out.off(b, n, h);
    const T *out = (const T*)p.out.p + at, *low = p.out_low ? (const T*)p.out_low + at : nullptr, *dout = (const T*)p.dout.p + p.dout.off(b, n, h);
    float sum = 0.f;
    for (int d = lane; d < p.D; d += 64) sum = fmaf(to_float(out[d]) + (low ? to_float(low[d]) : 0.f), to_float(dout[d]), sum);
    sum = wave_sum(sum);
    if (lane == 0) p.delta[((int64_t)b * p.H + h) * p.rows.N + n] = sum;
}

// dQ: the wavefront owns 32 queries and sweeps the keys they see
template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(THREADS) void causal_f32_dq_kernel(Causal p) {
    constexpr bool wide = WIDE;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *kt = lds, *vt = lds + TILE * Pitch<DP>::value;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.H, stream, tile);
    const int b = stream / p.H, h = stream % p.H, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, BLOCK, s)) return;
    if (s.fill) return fill_rows<T>(p.dq, s, h, p.D);
    const int q0 = ((s.len + BLOCK - 1) / BLOCK - 1 - s.block) * BLOCK, mine = q0 + wave * TILE, qi = mine + (lane & 31);
    float q[DP / 2], d[DP / 2];
    own_rows<T, DP>(q, p.q, s, mine, h, p.D, wide, 1.f);
    own_rows<T, DP>(d, p.dout, s, mine, h, p.D, wide, 1.f);
    const int64_t at = ((int64_t)s.b * p.H + h) * p.rows.N + s.first + qi;
    const float lse = qi < s.len ? p.lse[at] : 0.f, delta = qi < s.len ? p.delta[at] : 0.f, c = p.scale * LOG2E, lse2 = lse * LOG2E;
    floatx16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = zero16();
    const int last = q0 + BLOCK < s.len ? q0 + BLOCK : s.len;
    Stage<T, DP> ks, vs;
    ks.load(p.k, s, 0, hk, p.D, wide);
    vs.load(p.v, s, 0, hk, p.D, wide);
    for (int k0 = 0; k0 < last; k0 += TILE) {
        __syncthreads();
        ks.put(kt);
        vs.put(vt);
        __syncthreads();
        if (k0 + TILE < last) {
            ks.load(p.k, s, k0 + TILE, hk, p.D, wide);
            vs.load(p.v, s, k0 + TILE, hk, p.D, wide);
        }
        if (k0 > mine + TILE - 1) continue;
        floatx16 w = tile_product<DP>(kt, q);
        const floatx16 dp = tile_product<DP>(vt, d);
        const bool masked = k0 + TILE - 1 > mine || k0 + mine == 0;
        // (the first query of a sequence has one weight, 1, whose gradient is zero: no rounding of dP - delta is left of it)
        auto sees = [&](int j) { return k0 + j <= qi && qi > 0; };
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            w[i] = exp2f(fmaf(w[i], c, -lse2)) * (dp[i] - delta);
            if (masked && !sees(8 * (i / 4) + 4 * half + i % 4)) w[i] = 0.f;
        }
        if (masked) weighted_rows<DP, DP, true>(kt, 0, w, acc, sees);
        else weighted_rows<DP, DP, false>(kt, 0, w, acc, sees);
    }
    store_own<T, DP>(p.dq, s, qi, h, 0, p.D, wide, acc, p.scale);
}

// dK and dV: the wavefront owns 32 keys and sweeps the queries of all G heads that see them.  Columns `first` .. + DO of the
// gradients: at head_dim 256 two workgroups share them, each with all of the two first products (the registers hold no more).
template <class T, int DP, int DO, bool WIDE>
__global__ __launch_bounds__(THREADS) void causal_f32_dkv_kernel(Causal p) {
    constexpr bool wide = WIDE;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *qt = lds, *dt = lds + TILE * Pitch<DP>::value, *stats = dt + TILE * Pitch<DP>::value;     // lse * log2(e), delta
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.HK * (DP / DO), stream, tile);
    const int first = stream % (DP / DO) * DO;
    stream /= DP / DO;
    const int b = stream / p.HK, hk = stream % p.HK;
    Span s;
    if (!find_tile(p.rows, b, tile, BLOCK, s)) return;
    if (s.fill) {
        if (first) return;
        fill_rows<T>(p.dk, s, hk, p.D);
        return fill_rows<T>(p.dv, s, hk, p.D);
    }
    const int j0 = s.block * BLOCK, mine = j0 + wave * TILE, ki = mine + (lane & 31);
    float k[DP / 2], v[DP / 2];
    own_rows<T, DP>(k, p.k, s, mine, hk, p.D, wide, 1.f);
    own_rows<T, DP>(v, p.v, s, mine, hk, p.D, wide, 1.f);
    const float c = p.scale * LOG2E;
    floatx16 dk[DO / 32], dv[DO / 32];
#pragma unroll
    for (int i = 0; i < DO / 32; ++i) dk[i] = dv[i] = zero16();
    Stage<T, DP> qs, ds;
    float stat = 0.f;
    auto load = [&](int g, int q0) {
        const int h = hk * p.G + g;
        qs.load(p.q, s, q0, h, p.D, wide);
        ds.load(p.dout, s, q0, h, p.D, wide);
        if (threadIdx.x < 64) {
            const int i = q0 + (lane & 31);
            const int64_t at = ((int64_t)s.b * p.H + h) * p.rows.N + s.first + i;
            stat = i >= s.len ? 0.f : half ? p.delta[at] : p.lse[at] * LOG2E;
        }
    };
    int g = 0, q0 = j0;
    load(g, q0);
    while (g < p.G) {
        __syncthreads();
        qs.put(qt);
        ds.put(dt);
        if (threadIdx.x < 64) stats[threadIdx.x] = stat;
        __syncthreads();
        const int now = q0;
        q0 += TILE;
        if (q0 >= s.len) {
            q0 = j0;
            ++g;
        }
        if (g < p.G) load(g, q0);
        if (now + TILE - 1 < mine) continue;                              // queries before the wavefront's keys
        floatx16 w = tile_product<DP>(qt, k);
        const floatx16 dp = tile_product<DP>(dt, v);
        const bool masked = now < mine + TILE - 1 || now == 0;
        auto sees = [&](int i) { return now + i >= ki; };
        floatx16 dS;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 8 * (i / 4) + 4 * half + i % 4;
            w[i] = exp2f(fmaf(w[i], c, -stats[row]));
            dS[i] = w[i] * (dp[i] - stats[32 + row]);
            if (masked && !sees(row)) w[i] = 0.f;
            if (masked && (!sees(row) || now + row == 0)) dS[i] = 0.f;    // (a first query has one weight: see the dQ kernel)
        }
        if (masked) {
            weighted_rows<DP, DO, true>(dt, first, w, dv, sees);
            weighted_rows<DP, DO, true>(qt, first, dS, dk, [&](int i) { return sees(i) && now + i > 0; });
        } else {
            weighted_rows<DP, DO, false>(dt, first, w, dv, sees);
            weighted_rows<DP, DO, false>(qt, first, dS, dk, sees);
        }
    }
    if (p.dk.p) store_own<T, DO>(p.dk, s, ki, hk, first, p.D, wide, dk, p.scale);
    if (p.dv.p) store_own<T, DO>(p.dv, s, ki, hk, first, p.D, wide, dv, 1.f);
}

template <class T>
bool wide_rows(const Causal& p, std::initializer_list<const Tensor*> ts, bool batched) {
    constexpr int BYTES = 4 * sizeof(T);
    bool ok = p.D % 4 == 0;
    for (const Tensor* t : ts) {
        if (!t->p) continue;
        ok = ok && (uintptr_t)t->p % BYTES == 0 && t->sn % 4 == 0 && t->sh % 4 == 0 && (!batched || t->sb % 4 == 0);
    }
    return ok;
}
template <class K>
int launch(K kernel, const Causal& p, int64_t streams, int floats, hipStream_t st) {
    const int64_t tiles = count_tiles(p.rows, BLOCK);
    if (streams * tiles > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)(streams * tiles)), dim3(THREADS), floats * sizeof(float), st>>>(p);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

int launch_causal_f32_fwd(const Causal& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        const bool wide = wide_rows<T>(p, {&p.q, &p.k, &p.v, &p.out}, p.rows.B > 1);
        if (p.D <= 128) return launch_causal_f32_narrow_fwd(p, dtype, wide, st);
        return launch(wide ? causal_f32_fwd_kernel<T, 256, true> : causal_f32_fwd_kernel<T, 256, false>, p, (int64_t)p.rows.B * p.H, 2 * TILE * Pitch<256>::value, st);
    });
}

int launch_causal_f32_bwd(const Causal& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        const bool wide = wide_rows<T>(p, {&p.q, &p.k, &p.v, &p.dout, &p.dq, &p.dk, &p.dv}, p.rows.B > 1);
        if (p.dq.p || p.dk.p) {
            const int64_t blocks = ((int64_t)p.rows.B * p.rows.N * p.H + WAVES - 1) / WAVES;
            causal_f32_delta_kernel<T><<<dim3((unsigned)blocks), dim3(THREADS), 0, st>>>(p);
            if (hipGetLastError() != hipSuccess) return (int)SA2_ERR_LAUNCH_FAILED;
        }
        if (p.D <= 128) return launch_causal_f32_narrow_bwd(p, dtype, wide, st);
        int rc = SA2_OK;
        if (p.dk.p || p.dv.p)
            rc = launch(wide ? causal_f32_dkv_kernel<T, 256, 128, true> : causal_f32_dkv_kernel<T, 256, 128, false>, p, (int64_t)p.rows.B * p.HK * 2, 2 * TILE * Pitch<256>::value + 64, st);
        if (rc == SA2_OK && p.dq.p)
            rc = launch(wide ? causal_f32_dq_kernel<T, 256, true> : causal_f32_dq_kernel<T, 256, false>, p, (int64_t)p.rows.B * p.H, 2 * TILE * Pitch<256>::value, st);
        return rc;
    });
}

}  // namespace sa2
