// The sweep of a workgroup over keys in LDS, bf16 and fp16: logits, weights and outputs of rows of queries that four wavefronts own.
// Causal attention over prompts and large drafted trees run on it.
//
// A wavefront owns NQ blocks of 32 rows of queries: S^T = K Q^T leaves lane l with query l % 32 and 16 of 32 keys, which are, rounded to
// 16 bits, the second operand of O^T = V^T P^T as they are (V through the transposing LDS read).  A unit is one block of queries
// and a piece of 32 keys: D / 8 MFMAs, and 16 weights per lane.  The units run in a pipeline of three: while the vector ALU makes
// the weights of unit u, the matrix pipe has the logits of u+1 and the output of u-1, MFMA by MFMA between them (sa2_mfma_lone.h:
// outputs and queries stay in accumulation registers that the kernel owns; left to the compiler they moved to and fro, 280
// instructions more per 64 MFMAs, and the MFMAs stood in rows: 583 us instead of 302 at B1 N8192 H16/4 D128).
// The weights are e^(s - m) with m the row's maximum over its first 32 keys: no maximum and no scaling of the output in the
// sweep.  Rounding weights to bf16 costs half a step of each, whatever m, to fp16 half a step or 2^-25, which is why there m is lower than
// that (lowered_by).  A unit whose sum passes RefLimit, or first keys whose scores
// are all minus infinity, or so far from zero that s c - m c is not to be had from a rounded m c, have the workgroup sweep its keys a second time,
// with the running maximum; in bf16, whose values reach the end of fp32's range, an output that is no number does so too once weights are above 1.
// K and V come by direct global->LDS loads into three buffers of 64 keys, so that one barrier per 64 keys is enough.
#pragma once

#include "sa2_causal16.h"

namespace sa2 {
namespace {

constexpr int BUFFERS = 3;
template <class SRC, int NQ>
constexpr int SWEEP_BUFFERS = SRC::SLIDING && NQ == 1 ? 4 : BUFFERS;  // (see `sliding`)

template <class E> struct RefLimit;
template <> struct RefLimit<ElemBF16> { static constexpr float value = 1.152921504606847e18f; };   // 2^60
template <> struct RefLimit<ElemF16> { static constexpr float value = 65504.f; };                  // (no weight of a unit is above its sum)
// Many keys far below the first ones add up, and in fp16 all weights under 2^-25 would be lost.  Of `keys` keys rounding takes less than
// 2^-11 of the largest weight, as the result's own rounding does, where weights are 2^lift times as large, that is, the reference point
// lift / c lower (c: |scale| log2(e)).  More would leave less room for scores above the first keys': with a lift of 3 at 8192 keys scores
// of standard deviation 2 send most workgroups through a second sweep (B1 N8192 H16/4 D128 270 -> 880 us; as it is those of 3 do, 960).
template <class E>
__device__ __forceinline__ float lowered_by(int keys, float c) {
    if (E::DTYPE != SA2_F16 || keys <= 16384) return 0.f;
    const int lift = 32 - __clz(keys - 1) - 14;
    const float by = c > 1e-20f ? (float)(lift < 8 ? lift : 8) / c : 0.f;
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(by)));       // (the same in all lanes)
}
constexpr float OUTPUT_CHECK = 64.f;                        // sum of a unit (16 weights of a lane) up to which outputs are not looked at

// Accumulation registers: outputs of block n and columns 32 d .. from O0 + (n * D/32 + d) * 16 on, queries from Q0 + (n * D/16 + kk) * 4
template <int D, int NQ>
struct SweepRegs : Lone<(D * NQ > 128 ? 192 : 96)> {
    static constexpr int O0 = 0, Q0 = NQ * D / 32 * 16;
};

// `src` (of the wavefront, tiles and requests of the workgroup):
//   tiles, request(t, buffer)   tiles of 64 keys, and their K and V rows to LDS (each wavefront its quarter)
//   full                        the leading tiles of which every row of the wavefront sees every key
//   pieces                      pieces of 32 keys that it needs at all
//   sees(n, piece)              what the lane's row of block n sees of a piece, bit by key
//   guarded(piece)              values that some row does not see may be infinite or NaN
//   lower                       lowered_by of the keys
// SLIDING: in the place of full and pieces
//   window, a, b                the leading tiles that hold windows, latest keys first, and those of them that the wavefront's rows see; the
//                               others, which every row sees or does not as sees() says, hold first keys
//   before                      1: the first tile stands before those and is looked at for reference points only
//   clear, clear_end            tiles from clear to clear_end - 1, before b - 1, are seen whole by all rows, and so is the one behind each
//   any(piece)                  some row sees some of a piece
//   begin(base)                 requests of the first two tiles, which the caller makes before it brings the queries (their latencies together)
//   narrow                      some row may see no key of the first piece of tile a
// Queries lie in their registers; outputs are left in theirs, in units of e^(scale m), with the lane's part of their sums in l.
// LDS holds SWEEP_BUFFERS tiles from `base` on (with a fourth, and requests two tiles ahead, times were the same).
// c: |scale| log2(e).  All wavefronts of the workgroup call it.
template <class E, int D, int NQ, class SRC>
__device__ __forceinline__ void sweep16(const SRC& src, uint32_t base, float c, float (&m)[NQ], float (&l)[NQ]) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    using L = SweepRegs<D, NQ>;
    constexpr int KK = D / 16, DT = D / 32, O0 = L::O0, Q0 = L::Q0;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const uint32_t row_lane = T::row_lane(lane), column_lane = T::column_lane(lane);
    constexpr int RING = SWEEP_BUFFERS<SRC, NQ>;
    auto after = [&](uint32_t buf) { return buf == base + (RING - 1) * Buffer<D>::BYTES ? base : buf + Buffer<D>::BYTES; };
    auto buffer_of = [&](int t) { return base + (uint32_t)(t % RING) * Buffer<D>::BYTES; };

    constexpr int UNITS = 2 * NQ;                                          // of a tile: unit v is piece v / NQ, block v % NQ
    floatx16 st[2];                                                        // logits
    X8 w[2][2];                                                            // weights
    constexpr int VB = D * NQ > 128 ? 2 : 1;                               // (a second set spreads the reads over the steps)
    X8 kf[KK], vf[VB][2][DT];                                              // a piece's operands, shared by its blocks
    // (one address per piece, the rest are offsets of the reads)
    auto keys_at = [&](uint32_t buf, int sub) {
        uint32_t at = buf + row_lane + (uint32_t)(Buffer<D>::FIRST + sub * T::BYTES);
        stays(at);
        return at;
    };
    auto values_at = [&](uint32_t buf, int sub) {
        uint32_t at = buf + column_lane + (uint32_t)(Buffer<D>::SECOND + sub * T::BYTES);
        stays(at);
        return at;
    };
    auto load_key = [&](uint32_t at, int kk) { kf[kk] = lds_read_x8<X8>(at + (uint32_t)(kk / 2 * T::BLOCK + kk % 2 * 32)); };
    auto load_value = [&](uint32_t at, int j, int set = 0) { vf[set][j / DT][j % DT] = quad_tile_column<D, X8>(at, 0, j % DT, j / DT); };
    auto load_keys = [&](uint32_t at) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) load_key(at, kk);
    };
    auto load_values = [&](uint32_t at) {
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) load_value(at, j);
    };
    auto logit_mfma = [&](auto N, auto K, floatx16& x) __attribute__((always_inline)) {
        constexpr int kk = decltype(K)::value, at = Q0 + (decltype(N)::value * KK + kk) * 4;
        if constexpr (kk == 0) L::template tile_start<at>(x, kf[0]);
        else L::template tile_more<at>(x, kf[kk]);
    };
    auto output_mfma = [&](auto N, auto J, const X8 (&x)[2], auto SET) __attribute__((always_inline)) {
        constexpr int j = decltype(J)::value;
        L::template sum_more<O0 + (decltype(N)::value * DT + j % DT) * 16>(vf[decltype(SET)::value][j / DT][j % DT], x[j / DT]);
    };
    auto rest = [&]() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); };  // the MFMAs issued so far have ended
    auto logits = [&](auto N, floatx16& x) __attribute__((always_inline)) {
        static_for<KK>([&](auto K) __attribute__((always_inline)) { logit_mfma(N, K, x); });
    };
    auto ready = [&](floatx16& x) { asm volatile("s_nop 15\n\ts_nop 15" : "+v"(x)); };
    auto output = [&](auto N, X8 (&x)[2]) __attribute__((always_inline)) {
        asm volatile("s_nop 3" : "+v"(x[0]), "+v"(x[1]));
        static_for<2 * DT>([&](auto J) __attribute__((always_inline)) { output_mfma(N, J, x, LONE_C(0)); });
    };
    // weights of the logits x; masked: bit k of `seen`: the lane's query sees the piece's key k
    auto weights = [&](const floatx16& x, float at, float& sum, X8 (&y)[2], auto masked, uint32_t seen) {
        const float off = -at * c;
        union { uint32_t u[8]; X8 v[2]; } z;
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float e[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 2 * i + j, key = 8 * (r / 4) + 4 * half + r % 4;
                e[j] = fast_exp2(fmaf(x[r], c, off));
                if constexpr (decltype(masked)::value) e[j] = seen >> key & 1 ? e[j] : 0.f;
                part[j] += e[j];
            }
            z.u[i] = pack2<E>(e[0], e[1]);
        }
        y[0] = z.v[0];
        y[1] = z.v[1];
        sum = part[0] + part[1];
    };
    auto top_of = [&](const floatx16& x, uint32_t seen) {
        float t = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) t = fmaxf(t, seen >> (8 * (r / 4) + 4 * half + r % 4) & 1 ? x[r] : -INFINITY);
        return fmaxf(t, other_half(t));
    };
    float worst = 0.f;                                                     // largest sum of a unit (a NaN is no reason for a second sweep)
    auto weigh = [&](const floatx16& x, int n, X8 (&y)[2]) {
        float sum;
        weights(x, m[n], sum, y, std::false_type{}, 0);
        worst = fmaxf(worst, sum);
        l[n] += sum;
    };
    // One step of the pipeline: logits of unit V + 2, output of unit V, weights of unit V + 1; operands of the units after
    // those, from kat and vat, as soon as the ones before have been read for the last time (two MFMAs later)
    // (MASKED: bit k of `seen` says whether the lane's row sees key k of unit V + 1)
    auto step = [&](auto VV, uint32_t kat, uint32_t vat, auto MASKED, uint32_t seen) __attribute__((always_inline)) {
        constexpr int V = decltype(VV)::value, SLOTS = 4 * DT, LAG = SLOTS - 4;
        const uint32_t own = decltype(MASKED)::value ? seen >> 4 * half : 0u;
        constexpr bool NEXT_K = (V + 3) % NQ == 0, NEXT_V = (V + VB) % NQ == 0;
        constexpr int set = V / NQ % VB, next_set = (V + VB) / NQ % VB;    // of V operands
        constexpr int mid = (V + 1) % NQ;
        const floatx16& x = st[(V + 1) & 1];
        const float off = -m[mid] * c;
        float e[16], sum = 0.f;
        union { uint32_t u[8]; X8 v[2]; } z;
        static_for<SLOTS>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value;
            if constexpr (i % 2 == 0) logit_mfma(LONE_C((V + 2) % NQ), LONE_C(i / 2), st[V & 1]);
            else output_mfma(LONE_C(V % NQ), LONE_C(i / 2), w[V & 1], LONE_C(set));
            deal<16, i - 1, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = fmaf(x[decltype(X)::value], c, off); });
            deal<16, i - 2, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = fast_exp2(e[decltype(X)::value]); });
            deal<16, i - 3, LAG>([&](auto X) __attribute__((always_inline)) {
                constexpr int j = decltype(X)::value;
                if constexpr (decltype(MASKED)::value) e[j] = __uint_as_float(__float_as_uint(e[j]) & (uint32_t)__builtin_amdgcn_sbfe((int)own, 8 * (j / 4) + j % 4, 1));
                sum += e[j];
                if constexpr (j % 2) z.u[j / 2] = pack2<E>(e[j - 1], e[j]);
            });
            if constexpr (NEXT_K && i % 2 == 0 && i >= 2) load_key(kat, i / 2 - 1);
            if constexpr (NEXT_V && VB == 2 && i % 2 == 1) load_value(vat, i / 2, next_set);
            if constexpr (NEXT_V && VB == 1 && i % 2 == 1 && i >= 3) load_value(vat, i / 2 - 1);
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (NEXT_K) load_key(kat, KK - 1);
        w[(V + 1) & 1][0] = z.v[0];
        w[(V + 1) & 1][1] = z.v[1];
        worst = fmaxf(worst, sum);
        l[mid] += sum;
        stays(w[(V + 1) & 1][0]);
        stays(w[(V + 1) & 1][1]);
        stays(worst);
        stays(l[mid]);
        if constexpr (NEXT_V && VB == 1) {
            asm volatile("s_nop 7" ::: "memory");
            load_value(vat, 2 * DT - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    int released;                                                          // tiles 0 .. released are in LDS
    uint32_t arriving;                                                     // the buffer that the next request fills
    auto request = [&](int t) {
        src.request(t, arriving);
        arriving = after(arriving);
    };
    int begun = 0;                                                         // SLIDING: tiles that have been requested
    auto arrive = [&]() {                                                  // the next one too; its successor is on its way
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        ++released;
        if constexpr (SRC::SLIDING) {
            if (begun == released + 1 && begun < src.tiles) request(begun++);
        } else {
            if (released + 1 < src.tiles) request(released + 1);
        }
    };
    // One piece of 32 keys by itself, with masks, and values that a weight of zero would not keep out.  Rows that have no reference point
    // take their maximum here; `safe`: all rows do, as the running one.  The weights of a block stand between the MFMAs of the other.
    auto piece = [&](uint32_t buf, int sub, int which, bool safe) {
        load_keys(keys_at(buf, sub));
        load_values(values_at(buf, sub));
        static_for<NQ>([&](auto N) __attribute__((always_inline)) { logits(N, st[decltype(N)::value]); });
        if constexpr (NQ == 1) ready(st[0]);
        uint32_t bits = 0;
        if (src.guarded(which)) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int d = 0; d < DT; ++d) bits |= odd_bits<E>(vf[0][ks][d]);
        }
        const bool odd = any_odd(bits);
        static_for<NQ>([&](auto N) __attribute__((always_inline)) {
            constexpr int n = decltype(N)::value;
            const uint32_t seen = src.sees(n, which);
            if (safe || __any(m[n] == -INFINITY)) {
                const float top = top_of(st[n], seen) - src.lower;
                if (safe) {
                    const float now = fmaxf(m[n], top), f = m[n] == -INFINITY ? 0.f : exp2f((m[n] - now) * c);
                    l[n] *= f;
                    rest();
                    static_for<4 * DT>([&](auto X) __attribute__((always_inline)) {
                        constexpr int r = O0 + n * DT * 16 + 4 * decltype(X)::value;
                        const float4 o = L::template get_regs<r>();
                        L::template set_regs<r>(__float_as_uint(o.x * f), __float_as_uint(o.y * f), __float_as_uint(o.z * f), __float_as_uint(o.w * f));
                    });
                    m[n] = now;
                } else {
                    m[n] = m[n] == -INFINITY ? top : m[n];                 // (nothing has been added up in its units)
                }
            }
            float at = m[n] == -INFINITY ? 0.f : m[n], sum;
            if (safe && __any(far_from_zero(at, c))) {
#pragma unroll
                for (int r = 0; r < 16; ++r) st[n][r] -= at;
                at = 0.f;
            }
            if (__all(seen == ~0u)) weights(st[n], at, sum, w[n], std::false_type{}, 0);
            else weights(st[n], at, sum, w[n], std::true_type{}, seen);
            if (!safe) worst = fmaxf(worst, sum);
            l[n] += sum;
            if (odd) {
                rest();
                guarded_sum<E, L, O0 + n * DT * 16, D>(buf + (uint32_t)(Buffer<D>::SECOND + sub * T::BYTES), w[n], [&](int key) { return (seen >> key & 1) != 0; });
            } else output(N, w[n]);
        });
        asm volatile("s_nop 7" ::: "memory");                              // (the last MFMA has read its operands)
    };
    constexpr int LOOK = NQ == 1 ? 2 : 1;                                  // tiles ahead that a round of steps reads keys of
    const std::false_type whole{};
    const std::true_type some{};
    // after the first pass: a row's reference point is too far from zero for it
    auto far = [&]() {
        bool any = false;
#pragma unroll
        for (int n = 0; n < NQ; ++n) any = any || (is_finite(m[n]) && far_from_zero(m[n], c));
        return any;
    };
    // SLIDING: the tiles of src.a .. src.b - 1 go through the pipeline to the last, with masks where some row does not see all of
    // a tile or the next; then the first keys' tiles, piece by piece.  Tile `t` is worked on when the one LOOK behind it is there (what
    // the steps read ahead of a wavefront's last tile is not used).  Rows' reference points come from the first of these tiles, the one
    // with their own keys; in fp16, whose weights have less room above it, from the next one and the first keys as well.
    auto sliding = [&](const auto& src, bool safe) {
        auto tops = [&](int t, int sub) {
            load_keys(keys_at(buffer_of(t), sub));
            L::keep_out();
            static_for<NQ>([&](auto N) __attribute__((always_inline)) {
                constexpr int n = decltype(N)::value;
                logits(N, st[n]);
                ready(st[n]);
                m[n] = fmaxf(m[n], top_of(st[n], src.sees(n, 2 * t + sub)) - src.lower);
            });
        };
        auto advance = [&](int t) __attribute__((always_inline)) {
            const int to = t < src.tiles ? t : src.tiles - 1;
#pragma unroll 1
            while (released < to) arrive();
        };
        const bool active = src.a < src.b;
        if (!safe && active) {
            int t = src.a;
            if (E::DTYPE == SA2_F16 && src.before) tops(0, 0);
            advance(t + LOOK);
            if (src.narrow) tops(t, 1);
            if (E::DTYPE == SA2_F16 && t + 1 < src.b) tops(t + 1, 1);
            uint32_t here = buffer_of(t);
            load_keys(keys_at(here, 0));
            L::keep_out();
            static_for<NQ>([&](auto N) __attribute__((always_inline)) {
                constexpr int n = decltype(N)::value;
                logits(N, st[n]);
                ready(st[n]);
                m[n] = fmaxf(m[n], top_of(st[n], src.sees(n, 2 * t)) - src.lower);
                if (m[n] == -INFINITY) {
                    m[n] = 0.f;
                    worst = INFINITY;
                }
            });
            load_keys(keys_at(here, 1));
            L::keep_out();
            if constexpr (NQ == 1) {
                logits(LONE_C(0), st[1]);
                ready(st[1]);
                load_keys(keys_at(after(here), 0));
            }
            load_values(values_at(here, 0));
            L::keep_out();
            float sum;
            weights(st[0], m[0], sum, w[0], some, src.sees(0, 2 * t));
            worst = fmaxf(worst, sum);
            l[0] += sum;
            asm volatile("s_nop 3" : "+v"(w[0][0]), "+v"(w[0][1]));
            // Runs of rounds with and without masks (the last tile is in the first kind); true: that was the last one
            auto rounds = [&](auto MASKED) __attribute__((always_inline)) {
                constexpr bool SOME = decltype(MASKED)::value;
                auto seen = [&](int n, int piece) { return SOME ? src.sees(n, piece) : 0u; };
#pragma unroll 1
                do {
                    advance(t + LOOK);
                    const bool last = t + 1 == src.b;
                    const uint32_t next = after(here);
                    L::keep_out();
                    if constexpr (NQ == 1) {
                        step(LONE_C(0), keys_at(next, 1), values_at(here, 1), MASKED, seen(0, 2 * t + 1));
                        if (SOME && last) return true;
                        step(LONE_C(1), keys_at(after(next), 0), values_at(next, 0), MASKED, seen(0, 2 * t + 2));
                    } else {
                        step(LONE_C(0), 0u, VB == 2 ? values_at(here, 1) : 0u, MASKED, seen(1, 2 * t));
                        step(LONE_C(1), keys_at(next, 0), VB == 2 ? 0u : values_at(here, 1), MASKED, seen(0, 2 * t + 1));
                        step(LONE_C(2), 0u, VB == 2 ? values_at(next, 0) : 0u, MASKED, seen(1, 2 * t + 1));
                        if (SOME && last) return true;
                        step(LONE_C(3), keys_at(next, 1), VB == 2 ? 0u : values_at(next, 0), MASKED, seen(0, 2 * t + 2));
                    }
                    here = next;
                    ++t;
                } while ((t >= src.clear && t < src.clear_end) != SOME);
                return false;
            };
#pragma unroll 1
            while (!rounds(some)) {
                if (t < src.clear_end) rounds(whole);
            }
            L::keep_out();
            rest();
            asm volatile("s_nop 3" : "+v"(w[1][0]), "+v"(w[1][1]));
            static_for<2 * DT>([&](auto J) __attribute__((always_inline)) { output_mfma(LONE_C(NQ - 1), J, w[1], LONE_C(VB - 1)); });
            rest();
        }
        // (up to and with the last tile, which every wavefront waits for)
#pragma unroll 1
        for (int t = safe ? src.before : src.window; t <= src.tiles; ++t) {
            advance(t + LOOK);
            if (!active || t == src.tiles || (t < src.window && (t < src.a || t >= src.b))) continue;
#pragma unroll 1
            for (int sub = 0; sub < 2; ++sub)
                if (src.any(2 * t + sub)) piece(buffer_of(t), sub, 2 * t + sub, safe);
        }
    };
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        released = -1;
        arriving = base;
        if constexpr (SRC::SLIDING) {
            if (pass == 0) {                                               // (the caller has begun with two)
                begun = src.tiles < 2 ? src.tiles : 2;
                arriving = buffer_of(begun);
            } else {
                begun = 1;
                request(0);
            }
        } else {
            request(0);
        }
        arrive();
        rest();
        static_for<NQ * DT * 4>([&](auto X) __attribute__((always_inline)) { L::template set_regs<O0 + 4 * decltype(X)::value>(0u, 0u, 0u, 0u); });
        rest();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            l[n] = 0.f;
            m[n] = -INFINITY;
        }
        if constexpr (SRC::SLIDING) {
            sliding(src, pass != 0);
            // (a weight of zero does not keep an infinity or NaN out: outputs with one are made again, by pieces that do)
            rest();
            float poison = 0.f;
            static_for<NQ * DT * 4>([&](auto X) __attribute__((always_inline)) {
                const float4 o = L::template get_regs<O0 + 4 * decltype(X)::value>();
                poison = fmaf(o.x, 0.f, fmaf(o.y, 0.f, fmaf(o.z, 0.f, fmaf(o.w, 0.f, poison))));
            });
            if (pass != 0 || !__syncthreads_or(worst > RefLimit<E>::value || poison != 0.f || far())) break;
        } else {
            int done = 0;                                                      // pieces of 32 keys
            uint32_t here = base;
            if (pass == 0 && src.full > LOOK) {
                load_keys(keys_at(base, 0));
                static_for<NQ>([&](auto N) __attribute__((always_inline)) {
                    constexpr int n = decltype(N)::value;
                    logits(N, st[n]);
                    ready(st[n]);
                    m[n] = top_of(st[n], ~0u) - src.lower;
                    if (m[n] == -INFINITY) {                                   // (scores of minus infinity say nothing about the others)
                        m[n] = 0.f;
                        worst = INFINITY;
                    }
                });
                if constexpr (NQ == 1) {
                    load_keys(keys_at(base, 1));
                    logits(LONE_C(0), st[1]);
                    ready(st[1]);
                    arrive();
                    load_keys(keys_at(after(base), 0));
                } else {
                    load_keys(keys_at(base, 1));
                }
                load_values(values_at(base, 0));
                weigh(st[0], 0, w[0]);
                asm volatile("s_nop 3" : "+v"(w[0][0]), "+v"(w[0][1]));
                int t = 0;
                for (; t + LOOK < src.full; ++t) {
                    const uint32_t next = after(here);
                    L::keep_out();
                    if constexpr (VB == 2) {
                        step(LONE_C(0), 0u, values_at(here, 1), whole, 0u);
                        arrive();
                        step(LONE_C(1), keys_at(next, 0), 0u, whole, 0u);
                        step(LONE_C(2), 0u, values_at(next, 0), whole, 0u);
                        step(LONE_C(3), keys_at(next, 1), 0u, whole, 0u);
                    } else if constexpr (NQ == 2) {
                        step(LONE_C(0), 0u, 0u, whole, 0u);
                        arrive();
                        step(LONE_C(1), keys_at(next, 0), values_at(here, 1), whole, 0u);
                        step(LONE_C(2), 0u, 0u, whole, 0u);
                        step(LONE_C(3), keys_at(next, 1), values_at(next, 0), whole, 0u);
                    } else {
                        step(LONE_C(0), keys_at(next, 1), values_at(here, 1), whole, 0u);
                        arrive();
                        step(LONE_C(1), keys_at(after(next), 0), values_at(next, 0), whole, 0u);
                    }
                    here = next;
                }
                // the two units that are under way
                rest();
                output(LONE_C(0), w[0]);
                weigh(st[1], NQ - 1, w[1]);
                if constexpr (NQ == 1) load_values(values_at(here, 1));
                output(LONE_C(NQ - 1), w[1]);
                rest();
                done = 2 * t + (NQ == 1 ? 2 : 1);
                if constexpr (NQ == 1) here = after(here);
            }
            // the rest by itself; in the second pass all
            for (int t = done / 2; t < src.tiles; ++t, here = after(here)) {
                if (t > released) arrive();
    #pragma unroll 1
                for (int sub = t == done / 2 ? done % 2 : 0; sub < 2; ++sub)
                    if (2 * t + sub < src.pieces) piece(here, sub, 2 * t + sub, pass != 0);
            }
            bool again = worst > RefLimit<E>::value || (pass == 0 && far());
            if constexpr (E::DTYPE == SA2_BF16) {
                // (with smaller weights a second sweep would come no further; fp16 values times weights up to the limit are far from fp32's end)
                if (pass == 0 && __any(worst > OUTPUT_CHECK)) {
                    rest();
                    uint32_t bits = 0;
                    static_for<NQ * DT * 4>([&](auto X) __attribute__((always_inline)) {
                        const float4 o = L::template get_regs<O0 + 4 * decltype(X)::value>();
                        for (const float y : {o.x, o.y, o.z, o.w}) bits |= (__float_as_uint(y) & 0x7f800000u) + 0x00800000u;
                    });
                    again = again || bits >> 31;
                }
            }
            if (!__syncthreads_or(again)) break;
        }
    }
    rest();
}

}  // namespace
}  // namespace sa2
