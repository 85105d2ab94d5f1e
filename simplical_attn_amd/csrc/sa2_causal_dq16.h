// Causal attention, gradient of the queries, bf16 and fp16 on the 16-bit MFMA (row terms: sa2_causal_dkv16.hip).
//
//   P = e^(scale q k - lse), dP = dO V^T, dS = P (dP - delta), dQ_i = scale sum_j dS_ij k_j
//
// The forward's sweep (sa2_causal_fwd16.hip) with dP beside the logits and dS K in the place of P V: a wavefront owns NQ blocks of 32
// queries, whose rows of Q and dO and sums of dQ fill the accumulation registers (256 at head_dim 128 and NQ 2).  A piece of keys
// is read three times from LDS: rows of K, rows of V, columns of K.  dS is rounded to 16 bits before the last product (half a step
// of each); fp16: times a power of two of its row's own (sa2_causal16.h).
// Measured: B1 N8192 H16/4 D128 bf16 344 us, 1200 TFLOP/s of its three products, MFMAs busy 59 % of the time at 1.9 GHz.
#pragma once

#include "sa2_causal16.h"

namespace sa2 {
namespace {

constexpr int DQ_BUFFERS = 3;

// The factors of the lane's NQ rows, whose workgroup starts at row q0 of the sequence; `lds`: 2 * WAVES floats.  Every thread calls it
template <int NQ>
__device__ __forceinline__ void query_factors(const Causal& p, const Causal16Terms& terms, const Span& s, int h, int q0, float (&f)[NQ], float* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = q0 + wave * 32 * NQ;
    const float* const v = terms.v + ((int64_t)s.b * p.HK + h / p.G) * p.rows.N + s.first;
    const int64_t stat = ((int64_t)s.b * p.H + h) * p.rows.N + s.first;
    // keys before the block, eight loads under way; those of the block by themselves
    float before = 0.f;
    for (int i = threadIdx.x; i < q0; i += 8 * THREADS)
#pragma unroll
        for (int j = 0; j < 8; ++j) before = fmaxf(before, finite_or_zero(v[i + j * THREADS < q0 ? i + j * THREADS : i]));
    float own[NQ], dout[NQ], delta[NQ], all = 0.f;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int at = mine + 32 * n + (lane & 31);
        own[n] = at < s.len ? finite_or_zero(v[at]) : 0.f;
        all = fmaxf(all, own[n]);
        dout[n] = at < s.len ? terms.dout[stat + at] : 0.f;
        delta[n] = at < s.len ? p.delta[stat + at] : 0.f;
    }
    before = wave_max(before);
    all = wave_max(all);
    if (lane == 0) {
        lds[wave] = before;
        lds[WAVES + wave] = all;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) before = fmaxf(before, fmaxf(lds[w], w < wave ? lds[WAVES + w] : 0.f));
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float seen = fmaxf(before, largest_up_to(own[n]));
        f[n] = gradient_factor(fmaf(dout[n], seen, fabsf(delta[n])));
        before = __shfl(seen, 31, 32);
    }
}

// Workgroup `id`; all of LDS is its own
template <class E, int D, int NQ>
__device__ __forceinline__ void queries_gradient16(const Causal& p, const Causal16Terms& terms, bool padded, int id, char* lds) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    using L = Lone<(D * NQ > 128 ? 256 : D * NQ > 64 ? 192 : 96)>;
    constexpr int KK = D / 16, DT = D / 32, ROWS = 32 * NQ, BLOCK = ROWS * WAVES;
    constexpr int S0 = 0, Q0 = NQ * DT * 16, G0 = Q0 + NQ * KK * 4;        // accumulation registers of dQ, Q and dO
    const uint32_t base = lds_address(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int stream, tile;
    order(id, p.rows.B * p.H, stream, tile);
    const int b = stream / p.H, h = stream % p.H, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, BLOCK, s)) return;
    typedef typename E::scalar scalar;
    if (s.fill) {
        for (int i = threadIdx.x; i < s.len * p.D; i += THREADS) ((scalar*)p.dq.p)[row_offset(p.dq, s, i / p.D, h) + i % p.D] = (scalar)0.f;
        return;
    }
    const int q0 = ((s.len + BLOCK - 1) / BLOCK - 1 - s.block) * BLOCK, mine = q0 + wave * ROWS;
    const int last = q0 + BLOCK < s.len ? q0 + BLOCK : s.len;
    const int tiles = (last + TILE_ROWS - 1) / TILE_ROWS;
    Fetch<D> fetch;
    fetch.init(p.k, p.v, s, hk, p.D);

    const float c = p.scale * LOG2E;
    float lse2[NQ], f[NQ], df[NQ];                                         // f: the rows' factors, df: delta times them
    if constexpr (E::DTYPE == SA2_F16) query_factors<NQ>(p, terms, s, h, q0, f, (float*)lds);
    static_for<2 * NQ>([&](auto N) __attribute__((always_inline)) {
        constexpr int n = decltype(N)::value / 2, grad = decltype(N)::value % 2;
        const Tensor& t = grad ? p.dout : p.q;
        const int at = mine + 32 * n + (lane & 31);
        const uint16_t* row = (const uint16_t*)t.p + row_offset(t, s, at < s.len ? at : 0, h);
        uint4 x[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int col = 16 * kk + 8 * half;
            x[kk] = make_uint4(0, 0, 0, 0);
            if (at < s.len && col < p.D) x[kk] = *(const uint4*)(row + col);
        }
        static_for<KK>([&](auto K) __attribute__((always_inline)) {
            constexpr int kk = decltype(K)::value;
            L::template set_regs<(grad ? G0 : Q0) + (n * KK + kk) * 4>(x[kk].x, x[kk].y, x[kk].z, x[kk].w);
        });
        const int64_t stat = ((int64_t)s.b * p.H + h) * p.rows.N + s.first + at;
        if (grad) df[n] = at < s.len ? -p.delta[stat] * (E::DTYPE == SA2_F16 ? f[n] : 1.f) : 0.f;
        else lse2[n] = at < s.len ? p.lse[stat] * LOG2E : 0.f;
    });
    static_for<NQ * DT * 4>([&](auto X) __attribute__((always_inline)) { L::template set_regs<S0 + 4 * decltype(X)::value>(0u, 0u, 0u, 0u); });

    const uint32_t row_lane = T::row_lane(lane), column_lane = T::column_lane(lane);
    auto after = [&](uint32_t buf) { return buf == base + (DQ_BUFFERS - 1) * Buffer<D>::BYTES ? base : buf + Buffer<D>::BYTES; };
    constexpr int UNITS = 2 * NQ;                                          // of a tile: unit v is piece v / NQ, block v % NQ
    floatx16 st[2], dp[2];
    X8 w[2][2];                                                            // dS
    X8 rows[2 * KK], cols[2 * DT];                                         // K then V; K
    auto rows_at = [&](uint32_t buf, int sub) {
        uint32_t at = buf + row_lane + (uint32_t)(sub * T::BYTES);
        stays(at);
        return at;
    };
    auto cols_at = [&](uint32_t buf, int sub) {
        uint32_t at = buf + column_lane + (uint32_t)(Buffer<D>::FIRST + sub * T::BYTES);
        stays(at);
        return at;
    };
    auto load_row = [&](int a, uint32_t at) {
        const int kk = a % KK;
        rows[a] = lds_read_x8<X8>(at + (uint32_t)((a < KK ? Buffer<D>::FIRST : Buffer<D>::SECOND) + kk / 2 * T::BLOCK + kk % 2 * 32));
    };
    auto load_col = [&](int j, uint32_t at) { cols[j] = quad_tile_column<D, X8>(at, 0, j % DT, j / DT); };
    auto load_rows = [&](uint32_t at) {
#pragma unroll
        for (int a = 0; a < 2 * KK; ++a) load_row(a, at);
    };
    auto load_cols = [&](uint32_t at) {
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) load_col(j, at);
    };
    auto first_mfma = [&](auto N, auto A, floatx16& x, floatx16& y) __attribute__((always_inline)) {
        constexpr int a = decltype(A)::value, at = (a < KK ? Q0 : G0) + (decltype(N)::value * KK + a % KK) * 4;
        if constexpr (a == 0) L::template tile_start<at>(x, rows[a]);
        else if constexpr (a < KK) L::template tile_more<at>(x, rows[a]);
        else if constexpr (a == KK) L::template tile_start<at>(y, rows[a]);
        else L::template tile_more<at>(y, rows[a]);
    };
    auto second_mfma = [&](auto N, auto J, const X8 (&x)[2]) __attribute__((always_inline)) {
        constexpr int j = decltype(J)::value;
        L::template sum_more<S0 + (decltype(N)::value * DT + j % DT) * 16>(cols[j], x[j / DT]);
    };
    auto rest = [&]() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); };
    auto first = [&](auto N, floatx16& x, floatx16& y) __attribute__((always_inline)) {
        static_for<2 * KK>([&](auto A) __attribute__((always_inline)) { first_mfma(N, A, x, y); });
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(x));
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(y));
    };
    auto second = [&](auto N, X8 (&x)[2]) __attribute__((always_inline)) {
        asm volatile("s_nop 3" : "+v"(x[0]), "+v"(x[1]));
        static_for<2 * DT>([&](auto J) __attribute__((always_inline)) { second_mfma(N, J, x); });
        rest();
    };
    // dS of a unit, and what its rounding left (for the pieces of the own tile: see sa2_causal_dkv16.hip); masked: the lane's query sees the piece's keys 0 .. seen
    auto weigh = [&](const floatx16& x, const floatx16& y, int n, X8 (&z)[2], X8 (&rest)[2], auto masked, int seen) {
        union { uint32_t u[8]; X8 v[2]; } o, low;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float e[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 2 * i + j;
                e[j] = fast_exp2(fmaf(x[r], c, -lse2[n])) * (E::DTYPE == SA2_F16 ? fmaf(y[r], f[n], -df[n]) : y[r] - df[n]);
                if constexpr (decltype(masked)::value) e[j] = 8 * (r / 4) + 4 * half + r % 4 <= seen ? e[j] : 0.f;
            }
            o.u[i] = pack2<E>(e[0], e[1]);
            low.u[i] = pack2<E>(e[0] - E::lo(o.u[i]), e[1] - E::hi(o.u[i]));
        }
        z[0] = o.v[0];
        z[1] = o.v[1];
        rest[0] = low.v[0];
        rest[1] = low.v[1];
    };
    // One step: first products of unit V + 2, second product of unit V, dS of unit V + 1; operands of the units after those, as
    // soon as the ones before have been read for the last time (two MFMAs later)
    constexpr int SLOTS = 2 * KK + 2 * DT, LAG = SLOTS - 4;
    auto step = [&](auto VV, uint32_t rat, uint32_t cat) __attribute__((always_inline)) {
        constexpr int V = decltype(VV)::value;
        constexpr bool NEXT_ROWS = (V + 3) % NQ == 0, NEXT_COLS = (V + 1) % NQ == 0;
        constexpr int mid = (V + 1) % NQ;
        const floatx16 &x = st[(V + 1) & 1], &y = dp[(V + 1) & 1];
        float e[16], d[16];
        union { uint32_t u[8]; X8 v[2]; } z;
        static_for<SLOTS>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value, a = 2 * (i / 3) + i % 3;          // two first products, one second, in turn
            if constexpr (i % 3 < 2) {
                first_mfma(LONE_C((V + 2) % NQ), LONE_C(a), st[V & 1], dp[V & 1]);
                if constexpr (NEXT_ROWS && a >= 2) load_row(a - 2, rat);
            } else {
                second_mfma(LONE_C(V % NQ), LONE_C(i / 3), w[V & 1]);
                if constexpr (NEXT_COLS && i / 3 >= 1) load_col(i / 3 - 1, cat);
            }
            deal<16, i - 1, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = fmaf(x[decltype(X)::value], c, -lse2[mid]); });
            deal<16, i - 2, LAG>([&](auto X) __attribute__((always_inline)) {
                e[decltype(X)::value] = fast_exp2(e[decltype(X)::value]);
                if constexpr (E::DTYPE == SA2_F16) d[decltype(X)::value] = fmaf(y[decltype(X)::value], f[mid], -df[mid]);
                else d[decltype(X)::value] = y[decltype(X)::value] - df[mid];
            });
            deal<16, i - 3, LAG>([&](auto X) __attribute__((always_inline)) {
                constexpr int j = decltype(X)::value;
                e[j] *= d[j];
                if constexpr (j % 2) z.u[j / 2] = pack2<E>(e[j - 1], e[j]);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        w[(V + 1) & 1][0] = z.v[0];
        w[(V + 1) & 1][1] = z.v[1];
        stays(w[(V + 1) & 1][0]);
        stays(w[(V + 1) & 1][1]);
        if constexpr (NEXT_ROWS) load_row(2 * KK - 2, rat);
        if constexpr (NEXT_ROWS || NEXT_COLS) asm volatile("s_nop 7" ::: "memory");
        if constexpr (NEXT_ROWS) load_row(2 * KK - 1, rat);
        if constexpr (NEXT_COLS) load_col(2 * DT - 1, cat);
        __builtin_amdgcn_sched_barrier(0);
    };
    int released = -1;                                                     // tiles 0 .. released are in LDS
    uint32_t arriving = base;
    auto request = [&](int t) {
        fetch.request(t * TILE_ROWS, last, arriving, padded);
        arriving = after(arriving);
    };
    auto arrive = [&]() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        ++released;
        if (released + 1 < tiles) request(released + 1);
    };
    auto piece = [&](uint32_t buf, int sub, int from) {
        load_rows(rows_at(buf, sub));
        load_cols(cols_at(buf, sub));
        const bool masked = from + SUB - 1 > mine || from + mine == 0;
        uint32_t bits = 0;
        if (masked) {
#pragma unroll
            for (int j = 0; j < 2 * DT; ++j) bits |= odd_bits<E>(cols[j]);
        }
        const bool odd = any_odd(bits);
        static_for<NQ>([&](auto N) __attribute__((always_inline)) {
            constexpr int n = decltype(N)::value;
            if (from <= mine + 32 * n + 31) {
                // (the first query of a sequence has one weight, 1, whose gradient is zero)
                const int at = mine + 32 * n + (lane & 31), seen = at ? at - from : -1;
                first(N, st[0], dp[0]);
                weigh(st[0], dp[0], n, w[0], w[1], std::true_type{}, seen);
                if (odd) {
                    const uint32_t tile = buf + (uint32_t)(Buffer<D>::FIRST + sub * T::BYTES);
                    guarded_sum<E, L, S0 + n * DT * 16, D>(tile, w[0], [&](int key) { return key <= seen; });
                    guarded_sum<E, L, S0 + n * DT * 16, D>(tile, w[1], [&](int key) { return key <= seen; });
                } else {
                    second(N, w[0]);
                    second(N, w[1]);
                }
            }
        });
    };
    if (E::DTYPE == SA2_F16) __syncthreads();                              // (the factors have left LDS)
    request(0);
    arrive();
    const bool active = mine < s.len;
    const int full = active ? mine / TILE_ROWS : 0;
    constexpr int LOOK = NQ == 1 ? 2 : 1;
    int done = 0;
    uint32_t here = base;
    const std::false_type no{};
    if (full > LOOK) {
        load_rows(rows_at(base, 0));
        first(LONE_C(0), st[0], dp[0]);
        if constexpr (NQ == 1) {
            load_rows(rows_at(base, 1));
            first(LONE_C(0), st[1], dp[1]);
            arrive();
            load_rows(rows_at(after(base), 0));
        } else {
            first(LONE_C(1), st[1], dp[1]);
            load_rows(rows_at(base, 1));
        }
        load_cols(cols_at(base, 0));
        X8 unused[2];
        weigh(st[0], dp[0], 0, w[0], unused, no, 0);
        asm volatile("s_nop 3" : "+v"(w[0][0]), "+v"(w[0][1]));
        int t = 0;
        for (; t + LOOK < full; ++t) {
            const uint32_t next = after(here);
            L::keep_out();
            if constexpr (NQ == 2) {
                step(LONE_C(0), 0u, 0u);
                arrive();
                step(LONE_C(1), rows_at(next, 0), cols_at(here, 1));
                step(LONE_C(2), 0u, 0u);
                step(LONE_C(3), rows_at(next, 1), cols_at(next, 0));
            } else {
                step(LONE_C(0), rows_at(next, 1), cols_at(here, 1));
                arrive();
                step(LONE_C(1), rows_at(after(next), 0), cols_at(next, 0));
            }
            here = next;
        }
        rest();
        second(LONE_C(0), w[0]);
        weigh(st[1], dp[1], NQ - 1, w[1], unused, no, 0);
        if constexpr (NQ == 1) load_cols(cols_at(here, 1));
        second(LONE_C(NQ - 1), w[1]);
        done = 2 * t + (NQ == 1 ? 2 : 1);
        if constexpr (NQ == 1) here = after(here);
    }
    for (int t = done / 2; t < tiles; ++t, here = after(here)) {
        if (t > released) arrive();
        if (active && t <= full) {
#pragma unroll 1
            for (int sub = t == done / 2 ? done % 2 : 0; sub < 2; ++sub) {
                const int from = t * TILE_ROWS + sub * SUB;
                if (from < mine + ROWS) piece(here, sub, from);
            }
        }
    }
    rest();
    static_for<NQ>([&](auto N) __attribute__((always_inline)) {
        constexpr int n = decltype(N)::value;
        const int at = mine + 32 * n + (lane & 31);
        const float to = E::DTYPE == SA2_F16 ? p.scale / f[n] : p.scale;
        if (at < s.len) {
            uint16_t* row = (uint16_t*)p.dq.p + row_offset(p.dq, s, at, h);
            static_for<4 * DT>([&](auto X) __attribute__((always_inline)) {
                constexpr int x = decltype(X)::value;
                const float4 o = L::template get_regs<S0 + n * DT * 16 + 4 * x>();
                const int col = 8 * x + 4 * half;
                if (col < p.D) *(uint2*)(row + col) = make_uint2(pack2<E>(o.x * to, o.y * to), pack2<E>(o.z * to, o.w * to));
            });
        }
    });
}

}  // namespace
}  // namespace sa2
