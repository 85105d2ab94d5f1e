// Causal attention, forward, bf16 and fp16 on the 16-bit MFMA: head_dim a multiple of 8 up to 128, rows on the 16-byte grid.
//
//   S = scale Q K^T (j <= i), P = softmax(S), O = P V, LSE = log sum e^S
//
// A wavefront owns NQ blocks of 32 queries: S^T = K Q^T leaves lane l with query l % 32 and 16 of 32 keys, which are, rounded to
// 16 bits, the second operand of O^T = V^T P^T as they are (V through the transposing LDS read).  A unit is one block of queries
// and a piece of 32 keys: D / 8 MFMAs, and 16 weights per lane.  The units run in a pipeline of three: while the vector ALU makes
// the weights of unit u, the matrix pipe has the logits of u+1 and the output of u-1, MFMA by MFMA between them (sa2_mfma_lone.h:
// outputs and queries stay in accumulation registers that the kernel owns; left to the compiler they moved to and fro, 280
// instructions more per 64 MFMAs, and the MFMAs stood in rows: 583 us instead of 327 at B1 N8192 H16/4 D128).
// The weights are e^(s - m) with m the row's maximum over its first 32 keys: no maximum and no scaling of the output in the
// sweep.  Rounding weights to 16 bits costs half a step of each, whatever m; a unit whose sum passes REF_LIMIT has the workgroup
// sweep its keys a second time, with the running maximum.
// K and V come by direct global->LDS loads into three buffers of 64 keys, so that one barrier per 64 keys is enough.
#include "sa2_causal16.h"

namespace sa2 {
namespace {

constexpr int BUFFERS = 3;

template <class E> struct RefLimit;
template <> struct RefLimit<ElemBF16> { static constexpr float value = 1.152921504606847e18f; };   // 2^60
template <> struct RefLimit<ElemF16> { static constexpr float value = 32768.f; };                  // below 65504

template <class E, int D, int NQ>
__global__ __launch_bounds__(THREADS, D == 64 ? 2 : 1) void causal_fwd16_kernel(Causal p, bool padded) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    using L = Lone<(D * NQ > 128 ? 192 : 96)>;
    constexpr int KK = D / 16, DT = D / 32, ROWS = 32 * NQ, BLOCK = ROWS * WAVES;
    constexpr int O0 = 0, Q0 = NQ * DT * 16;                               // accumulation registers of outputs and queries
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t base = lds_address(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.H, stream, tile);
    const int b = stream / p.H, h = stream % p.H, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, BLOCK, s)) return;
    float* const lse = p.lse + ((int64_t)s.b * p.H + h) * p.rows.N + s.first;
    typedef typename E::scalar scalar;
    if (s.fill) {
        for (int i = threadIdx.x; i < s.len * p.D; i += THREADS) ((scalar*)p.out.p)[row_offset(p.out, s, i / p.D, h) + i % p.D] = (scalar)0.f;
        for (int i = threadIdx.x; i < s.len; i += THREADS) lse[i] = -INFINITY;
        return;
    }
    const int q0 = ((s.len + BLOCK - 1) / BLOCK - 1 - s.block) * BLOCK, mine = q0 + wave * ROWS;
    const int last = q0 + BLOCK < s.len ? q0 + BLOCK : s.len;              // the workgroup's keys: 0 .. last - 1
    const int tiles = (last + TILE_ROWS - 1) / TILE_ROWS;

    Fetch<D> fetch;
    fetch.init(p.k, p.v, s, hk, p.D);

    // queries, second operand of the logits; a negative scale is taken out of them, so that the largest logit has the largest weight
    const float c = fabsf(p.scale) * LOG2E;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    static_for<NQ>([&](auto N) __attribute__((always_inline)) {
        constexpr int n = decltype(N)::value;
        const int at = mine + 32 * n + (lane & 31);
        const uint16_t* row = (const uint16_t*)p.q.p + row_offset(p.q, s, at < s.len ? at : 0, h);
        uint4 x[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int col = 16 * kk + 8 * half;
            x[kk] = make_uint4(0, 0, 0, 0);
            if (at < s.len && col < p.D) x[kk] = *(const uint4*)(row + col);
        }
        static_for<KK>([&](auto K) __attribute__((always_inline)) {
            constexpr int kk = decltype(K)::value;
            L::template set_regs<Q0 + (n * KK + kk) * 4>(x[kk].x ^ flip, x[kk].y ^ flip, x[kk].z ^ flip, x[kk].w ^ flip);
        });
    });
    float m[NQ], l[NQ];                                                    // outputs and sums are in units of e^(scale m)
    const uint32_t row_lane = T::row_lane(lane), column_lane = T::column_lane(lane);
    auto after = [&](uint32_t buf) { return buf == base + (BUFFERS - 1) * Buffer<D>::BYTES ? base : buf + Buffer<D>::BYTES; };

    constexpr int UNITS = 2 * NQ;                                          // of a tile: unit v is piece v / NQ, block v % NQ
    floatx16 st[2];                                                        // logits
    X8 w[2][2];                                                            // weights
    X8 kf[KK], vf[2][DT];                                                  // a piece's operands, shared by its blocks
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
    auto load_value = [&](uint32_t at, int j) { vf[j / DT][j % DT] = quad_tile_column<D, X8>(at, 0, j % DT, j / DT); };
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
    auto output_mfma = [&](auto N, auto J, const X8 (&x)[2]) __attribute__((always_inline)) {
        constexpr int j = decltype(J)::value;
        L::template sum_more<O0 + (decltype(N)::value * DT + j % DT) * 16>(vf[j / DT][j % DT], x[j / DT]);
    };
    auto rest = [&]() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); };  // the MFMAs issued so far have ended
    auto logits = [&](auto N, floatx16& x) __attribute__((always_inline)) {
        static_for<KK>([&](auto K) __attribute__((always_inline)) { logit_mfma(N, K, x); });
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(x));
    };
    auto output = [&](auto N, X8 (&x)[2]) __attribute__((always_inline)) {
        asm volatile("s_nop 3" : "+v"(x[0]), "+v"(x[1]));
        static_for<2 * DT>([&](auto J) __attribute__((always_inline)) { output_mfma(N, J, x); });
        rest();
    };
    // weights of the logits x; masked: the lane's query sees the piece's keys 0 .. seen
    auto weights = [&](const floatx16& x, float at, float& sum, X8 (&y)[2], auto masked, int seen) {
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
                if constexpr (decltype(masked)::value) e[j] = key <= seen ? e[j] : 0.f;
                part[j] += e[j];
            }
            z.u[i] = pack2<E>(e[0], e[1]);
        }
        y[0] = z.v[0];
        y[1] = z.v[1];
        sum = part[0] + part[1];
    };
    auto top_of = [&](const floatx16& x, int seen) {
        float t = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) t = fmaxf(t, 8 * (r / 4) + 4 * half + r % 4 <= seen ? x[r] : -INFINITY);
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
    auto step = [&](auto VV, uint32_t kat, uint32_t vat) __attribute__((always_inline)) {
        constexpr int V = decltype(VV)::value, SLOTS = 4 * DT, LAG = SLOTS - 4;
        constexpr bool NEXT_K = (V + 3) % NQ == 0, NEXT_V = (V + 1) % NQ == 0;
        constexpr int mid = (V + 1) % NQ;
        const floatx16& x = st[(V + 1) & 1];
        const float off = -m[mid] * c;
        float e[16], sum = 0.f;
        union { uint32_t u[8]; X8 v[2]; } z;
        static_for<SLOTS>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value;
            if constexpr (i % 2 == 0) logit_mfma(LONE_C((V + 2) % NQ), LONE_C(i / 2), st[V & 1]);
            else output_mfma(LONE_C(V % NQ), LONE_C(i / 2), w[V & 1]);
            deal<16, i - 1, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = fmaf(x[decltype(X)::value], c, off); });
            deal<16, i - 2, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = fast_exp2(e[decltype(X)::value]); });
            deal<16, i - 3, LAG>([&](auto X) __attribute__((always_inline)) {
                constexpr int j = decltype(X)::value;
                sum += e[j];
                if constexpr (j % 2) z.u[j / 2] = pack2<E>(e[j - 1], e[j]);
            });
            if constexpr (NEXT_K && i % 2 == 0 && i >= 2) load_key(kat, i / 2 - 1);
            if constexpr (NEXT_V && i % 2 == 1 && i >= 3) load_value(vat, i / 2 - 1);
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
        if constexpr (NEXT_V) {
            asm volatile("s_nop 7" ::: "memory");
            load_value(vat, 2 * DT - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    int released;                                                          // tiles 0 .. released are in LDS
    uint32_t arriving;                                                     // the buffer that the next request fills
    auto request = [&](int t) {
        fetch.request(t * TILE_ROWS, last, arriving, padded);
        arriving = after(arriving);
    };
    auto arrive = [&]() {                                                  // the next one too; its successor is on its way
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        ++released;
        if (released + 1 < tiles) request(released + 1);
    };
    // one piece of 32 keys with the running maximum, masks, and values that a weight of zero would not keep out
    auto piece = [&](uint32_t buf, int sub, int first) {
        load_keys(keys_at(buf, sub));
        load_values(values_at(buf, sub));
        bool odd = false;
        if (first + SUB - 1 > mine) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int d = 0; d < DT; ++d) odd = odd || not_finite<E>(vf[ks][d]);
        }
        odd = __any(odd);
        static_for<NQ>([&](auto N) __attribute__((always_inline)) {
            constexpr int n = decltype(N)::value;
            if (first <= mine + 32 * n + 31) {
                const int seen = mine + 32 * n + (lane & 31) - first;
                logits(N, st[0]);
                const float top = fmaxf(m[n], top_of(st[0], seen)), at = top == -INFINITY ? 0.f : top;
                if (__any(top != m[n])) {
                    const float f = m[n] == -INFINITY ? 0.f : exp2f((m[n] - at) * c);
                    l[n] *= f;
                    static_for<4 * DT>([&](auto X) __attribute__((always_inline)) {
                        constexpr int r = O0 + n * DT * 16 + 4 * decltype(X)::value;
                        const float4 o = L::template get_regs<r>();
                        L::template set_regs<r>(__float_as_uint(o.x * f), __float_as_uint(o.y * f), __float_as_uint(o.z * f), __float_as_uint(o.w * f));
                    });
                    m[n] = top;
                }
                float sum;
                weights(st[0], at, sum, w[0], std::true_type{}, seen);
                l[n] += sum;
                if (odd) guarded_sum<E, L, O0 + n * DT * 16, D>(buf + (uint32_t)(Buffer<D>::SECOND + sub * T::BYTES), w[0], [&](int key) { return key <= seen; });
                else output(N, w[0]);
            }
        });
    };
    const bool active = mine < s.len;
    const int full = active ? mine / TILE_ROWS : 0;                             // tiles that all of the wavefront's queries see
    constexpr int LOOK = NQ == 1 ? 2 : 1;                                  // tiles ahead that a round of steps reads keys of
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        released = -1;
        arriving = base;
        request(0);
        arrive();
        rest();
        static_for<NQ * DT * 4>([&](auto X) __attribute__((always_inline)) { L::template set_regs<O0 + 4 * decltype(X)::value>(0u, 0u, 0u, 0u); });
        rest();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            l[n] = 0.f;
            m[n] = -INFINITY;
        }
        int done = 0;                                                      // pieces of 32 keys
        uint32_t here = base;
        if (pass == 0 && full > LOOK) {
            load_keys(keys_at(base, 0));
            static_for<NQ>([&](auto N) __attribute__((always_inline)) {
                constexpr int n = decltype(N)::value;
                logits(N, st[n]);
                m[n] = top_of(st[n], SUB);
                m[n] = m[n] == -INFINITY ? 0.f : m[n];
            });
            if constexpr (NQ == 1) {
                load_keys(keys_at(base, 1));
                logits(LONE_C(0), st[1]);
                arrive();
                load_keys(keys_at(after(base), 0));
            } else {
                load_keys(keys_at(base, 1));
            }
            load_values(values_at(base, 0));
            weigh(st[0], 0, w[0]);
            asm volatile("s_nop 3" : "+v"(w[0][0]), "+v"(w[0][1]));
            int t = 0;
            for (; t + LOOK < full; ++t) {
                const uint32_t next = after(here);
                L::keep_out();
                if constexpr (NQ == 2) {
                    step(LONE_C(0), 0u, 0u);
                    arrive();
                    step(LONE_C(1), keys_at(next, 0), values_at(here, 1));
                    step(LONE_C(2), 0u, 0u);
                    step(LONE_C(3), keys_at(next, 1), values_at(next, 0));
                } else {
                    step(LONE_C(0), keys_at(next, 1), values_at(here, 1));
                    arrive();
                    step(LONE_C(1), keys_at(after(next), 0), values_at(next, 0));
                }
                here = next;
            }
            // the two units that are under way
            rest();
            output(LONE_C(0), w[0]);
            weigh(st[1], NQ - 1, w[1]);
            if constexpr (NQ == 1) load_values(values_at(here, 1));
            output(LONE_C(NQ - 1), w[1]);
            done = 2 * t + (NQ == 1 ? 2 : 1);
            if constexpr (NQ == 1) here = after(here);
        }
        // the rest up to the wavefront's own keys; in the second pass all of them
        for (int t = done / 2; t < tiles; ++t, here = after(here)) {
            if (t > released) arrive();
            if (active && t <= full) {
#pragma unroll 1
                for (int sub = t == done / 2 ? done % 2 : 0; sub < 2; ++sub) {
                    const int first = t * TILE_ROWS + sub * SUB;
                    if (first < mine + ROWS) piece(here, sub, first);
                }
            }
        }
        if (!__syncthreads_or(worst > RefLimit<E>::value)) break;
    }
    rest();
    static_for<NQ>([&](auto N) __attribute__((always_inline)) {
        constexpr int n = decltype(N)::value;
        const float sum = l[n] + other_half(l[n]), f = 1.f / sum;
        const int at = mine + 32 * n + (lane & 31);
        if (at < s.len) {
            uint16_t* row = (uint16_t*)p.out.p + row_offset(p.out, s, at, h);
            uint16_t* low = p.out_low ? (uint16_t*)p.out_low + row_offset(p.out, s, at, h) : nullptr;
            static_for<4 * DT>([&](auto X) __attribute__((always_inline)) {
                constexpr int x = decltype(X)::value;
                const float4 o = L::template get_regs<O0 + n * DT * 16 + 4 * x>();
                const int col = 8 * x + 4 * half;
                if (col < p.D) {
                    const float4 y = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
                    const uint2 r = make_uint2(pack2<E>(y.x, y.y), pack2<E>(y.z, y.w));
                    *(uint2*)(row + col) = r;
                    if (low) *(uint2*)(low + col) = make_uint2(pack2<E>(y.x - E::lo(r.x), y.y - E::hi(r.x)), pack2<E>(y.z - E::lo(r.y), y.w - E::hi(r.y)));
                }
            });
            if (half == 0) lse[at] = fmaf(m[n], fabsf(p.scale), logf(sum));
        }
    });
}

template <class E, int D, int NQ>
int launch(const Causal& p, hipStream_t st) {
    const auto kernel = causal_fwd16_kernel<E, D, NQ>;
    const int64_t grid = (int64_t)p.rows.B * p.H * count_tiles(p.rows, 32 * NQ * WAVES);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), BUFFERS * Buffer<D>::BYTES, st>>>(p, p.D != D);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

bool causal16_supported(int D, int dtype) { return dtype != SA2_F32 && D % 8 == 0 && D <= 128; }

// 16-byte rows, and a tile's rows within 2^31 bytes of its first
bool causal16_layout(const Causal& p, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->p && (!aligned16(*t, 2, p.rows.B > 1) || (p.rows.N > 1 && t->sn >= 1 << 22))) return false;
    return true;
}

int launch_causal16_fwd(const Causal& p, int dtype, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        // two blocks of queries per wavefront halve what LDS has to deliver; one where the workgroups would leave CUs idle
        const bool two = (int64_t)p.rows.B * p.H * count_tiles(p.rows, 64 * WAVES) >= CUS;
        if (p.D <= 64) return two ? launch<E, 64, 2>(p, st) : launch<E, 64, 1>(p, st);
        return two ? launch<E, 128, 2>(p, st) : launch<E, 128, 1>(p, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace sa2
