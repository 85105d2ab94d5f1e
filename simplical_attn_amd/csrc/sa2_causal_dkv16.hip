// Causal attention, gradients of keys and values, bf16 and fp16 on the 16-bit MFMA; the row terms before, the sums behind.
//
//   P = e^(scale q k - lse), dV_j = sum_i P_ij dO_i, dP = dO V^T, dS = P (dP - delta), dK_j = scale sum_i dS_ij q_i
//
// A wavefront owns 32 keys: S = Q K^T and dP = dO V^T leave lane l with key l % 32 and 16 of 32 queries, which are, rounded to
// 16 bits, the second operands of dV^T += dO^T P and dK^T += Q^T dS as they are.  The first products start from -lse / scale and
// -delta of their rows instead of zero, so that a weight is one product and one exponential, and dS one product more.
// Keys, values and both sums live in accumulation registers (sa2_mfma_lone.h); 32 queries are D / 4 MFMAs.  They run in a pipeline
// of three: the first products of the next 32 queries and the second products of the last between the vector instructions of
// these.  Every operand of an MFMA comes from LDS for it alone (128 bytes per cycle and CU at the full rate of the MFMAs, which is
// what LDS gives), read three or four MFMAs of its kind ahead.
// The queries of the G heads that share the keys are one stream, of which `nsplit` workgroups take shares where the key blocks are
// few or uneven (the first keys are seen by all queries, the last by few); their fp32 sums meet in a last launch, in order.
// fp16: dS is multiplied by a power of two of its key's own (sa2_causal16.h), which comes off the sum; so are the weights in dV, by 2^15
// (they are 1 at most, and in a long or peaked row most are below fp16's smallest normal number): -lse / scale is higher by that.
// Measured: B1 N8192 H16/4 D128 bf16 495 us (1110 TFLOP/s of its four products, MFMAs busy 52 % of the time at 2.0 GHz; LDS reads and the
// exponentials share the rest), row terms 20, sums 14; all gradients of B2 N2048 H8 D64 57, of which one launch for dQ, dK and dV 44; fp16 N16384
// H8/2, all gradients 1760 (bf16 1580).
#include "sa2_causal_dq16.h"

namespace sa2 {
namespace {

constexpr int BUFFERS = 4, BLOCK = SUB * WAVES;            // keys per workgroup
constexpr int STATS = 2 * TILE_ROWS * 4;                    // bytes of the row terms of a tile
constexpr int TERMS_BLOCKS = 1024;
template <class E>
constexpr int LIFT = E::DTYPE == SA2_F16 ? 15 : 0;          // weights in dV are 2^LIFT times as large

// ---- row terms: delta = sum_d dO O, stored as -delta, and -lse / scale ----------------------------------------------
// O with what its rounding left, where the forward wrote that: from the rounded output alone delta carries half a step of every
// value, which in sequences of up to a hundred rows makes dQ and dK 1.5 to 2.3 times as far off as their own rounding does.
template <class E, int LANES>                               // lanes per row, 16 bytes each
__global__ __launch_bounds__(THREADS) void causal_terms_kernel(Causal p, Causal16Terms terms) {
    const int lane = threadIdx.x % LANES, per = THREADS / LANES;
    const int64_t rows = (int64_t)p.rows.B * p.rows.N * p.H;
    const float over = -1.f / p.scale, lift = LIFT<E> / (p.scale * LOG2E);
    int lo = 0, hi = p.rows.N;
    if (p.rows.cu) {
        lo = p.rows.cu[0];
        hi = p.rows.cu[p.rows.sequences];
    }
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < rows; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / LANES;
        float sum = 0.f, square = 0.f;
        int h = 0, n = 0, b = 0;
        if (r < rows) {
            h = (int)(r % p.H);
            const int64_t bn = r / p.H;
            b = (int)(bn / p.rows.N);
            n = (int)(bn % p.rows.N);
            if (lane * 8 < p.D) {
                const uint4 x = *(const uint4*)((const uint16_t*)p.out.p + p.out.off(b, n, h) + lane * 8);
                const uint4 y = *(const uint4*)((const uint16_t*)p.dout.p + p.dout.off(b, n, h) + lane * 8);
                const uint4 z = p.out_low ? *(const uint4*)((const uint16_t*)p.out_low + p.out.off(b, n, h) + lane * 8) : make_uint4(0, 0, 0, 0);
                const uint32_t *xs = &x.x, *ys = &y.x, *zs = &z.x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y0 = E::lo(ys[i]), y1 = E::hi(ys[i]);
                    sum = fmaf(E::lo(xs[i]) + E::lo(zs[i]), y0, fmaf(E::hi(xs[i]) + E::hi(zs[i]), y1, sum));
                    if (E::DTYPE == SA2_F16) square = fmaf(y0, y0, fmaf(y1, y1, square));
                }
            }
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            sum += __shfl_xor(sum, o);
            if (E::DTYPE == SA2_F16) square += __shfl_xor(square, o);
        }
        if (r < rows && n >= lo && n < hi && lane == 0) {
            const int64_t at = ((int64_t)b * p.H + h) * p.rows.N + n;
            p.delta[at] = -sum;
            terms.minus_lse[at] = fmaf(p.lse[at], over, lift);
            if (E::DTYPE == SA2_F16) terms.dout[at] = sqrtf(square);
        }
    }
    if constexpr (E::DTYPE == SA2_F16) {
        const int64_t values = (int64_t)p.rows.B * p.rows.N * p.HK;
        for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < values; r0 += (int64_t)gridDim.x * per) {
            const int64_t r = r0 + threadIdx.x / LANES;
            const int h = (int)(r % p.HK), n = (int)(r / p.HK % p.rows.N), b = (int)(r / p.HK / p.rows.N);
            float square = 0.f;
            if (r < values && lane * 8 < p.D) {
                const uint4 x = *(const uint4*)((const uint16_t*)p.v.p + p.v.off(b, n, h) + lane * 8);
                const uint32_t* xs = &x.x;
#pragma unroll
                for (int i = 0; i < 4; ++i) square = fmaf(E::lo(xs[i]), E::lo(xs[i]), fmaf(E::hi(xs[i]), E::hi(xs[i]), square));
            }
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) square += __shfl_xor(square, o);
            if (r < values && lane == 0) terms.v[((int64_t)b * p.HK + h) * p.rows.N + n] = sqrtf(square);
        }
    }
}

// The factor of the lane's key j0 + 32 * wave + lane % 32 for shares lo .. hi-1 of the stream of tiles (`per` of each head, from row j0 on).
// `lds`: 2 * WAVES + 2 * BLOCK floats.  Every thread calls it
__device__ __forceinline__ float key_factor(const Causal& p, const Causal16Terms& terms, const Span& s, int hk, int j0, int per, int lo, int hi, float* lds) {
    constexpr int OWN = BLOCK / TILE_ROWS, AHEAD = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = ((int64_t)s.b * p.H + hk * p.G) * p.rows.N + s.first + j0;
    // rows behind the block: each wavefront every fourth tile, loads of four under way
    float dout = 0.f, delta = 0.f;
    int g = (lo + wave) / per, i = lo + wave - g * per;
    for (int x = lo + wave; x < hi;) {
        float a[AHEAD], b[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int row = i * TILE_ROWS + lane;
            const bool there = x < hi && i >= OWN && j0 + row < s.len;
            const int64_t at = first + (there ? (int64_t)g * p.rows.N + row : 0);
            a[k] = there ? terms.dout[at] : 0.f;
            b[k] = there ? p.delta[at] : 0.f;
            x += WAVES;
            i += WAVES;
            while (i >= per) {
                i -= per;
                ++g;
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            dout = fmaxf(dout, finite_or_zero(a[k]));
            delta = fmaxf(delta, finite_or_zero(b[k]));
        }
    }
    dout = wave_max(dout);
    delta = wave_max(delta);
    // rows of the block: the largest of a row's heads
    const int t = threadIdx.x;
    if (t < BLOCK) {
        float a = 0.f, b = 0.f;
        if (j0 + t < s.len && lo < hi)
            for (int head = lo / per; head <= (hi - 1) / per; ++head) {
                const int x = head * per + t / TILE_ROWS;
                if (x < lo || x >= hi) continue;
                const int64_t at = first + (int64_t)head * p.rows.N + t;
                a = fmaxf(a, finite_or_zero(terms.dout[at]));
                b = fmaxf(b, finite_or_zero(p.delta[at]));
            }
        lds[2 * WAVES + t] = a;
        lds[2 * WAVES + BLOCK + t] = b;
    }
    if (lane == 0) {
        lds[wave] = dout;
        lds[WAVES + wave] = delta;
    }
    __syncthreads();
    const int key = 32 * wave + (lane & 31);
    float reach[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const float* const own = lds + 2 * WAVES + w * BLOCK;
        float later = 0.f;
#pragma unroll
        for (int k = 0; k < BLOCK / 64; ++k) later = fmaxf(later, 64 * k + lane >= 32 * wave + 32 ? own[64 * k + lane] : 0.f);
#pragma unroll
        for (int k = 0; k < WAVES; ++k) later = fmaxf(later, lds[w * WAVES + k]);
        reach[w] = fmaxf(wave_max(later), largest_from(own[key]));
    }
    const float v = j0 + key < s.len ? terms.v[((int64_t)s.b * p.HK + hk) * p.rows.N + s.first + j0 + key] : 0.f;
    return gradient_factor(fmaf(reach[0], v, reach[1]));
}

// ---- dK, dV ------------------------------------------------------------------------------------------------------------
template <class E, int D>
__device__ __forceinline__ void keys_gradients16(const Causal& p, const Causal16Terms& terms, int nsplit, bool padded, int id, char* lds) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    using L = Lone<(D == 128 ? 192 : 96)>;
    constexpr int KK = D / 16, DT = D / 32;
    constexpr int V0 = 0, K0 = DT * 16, KEY0 = 2 * DT * 16, VALUE0 = KEY0 + KK * 4;      // sums of dV and dK, keys, values
    const uint32_t base = lds_address(lds), stats = base + BUFFERS * Buffer<D>::BYTES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int stream, tile;
    order(id, p.rows.B * p.HK * nsplit, stream, tile);
    const int split = stream % nsplit;
    stream /= nsplit;
    const int b = stream / p.HK, hk = stream % p.HK;
    Span s;
    if (!find_tile(p.rows, b, tile, BLOCK, s)) return;
    typedef typename E::scalar scalar;
    if (s.fill) {
        if (nsplit == 1)
            for (int i = threadIdx.x; i < s.len * p.D; i += THREADS) {
                if (p.dk.p) ((scalar*)p.dk.p)[row_offset(p.dk, s, i / p.D, hk) + i % p.D] = (scalar)0.f;
                if (p.dv.p) ((scalar*)p.dv.p)[row_offset(p.dv, s, i / p.D, hk) + i % p.D] = (scalar)0.f;
            }
        return;
    }
    const int j0 = s.block * BLOCK, mine = j0 + wave * SUB, key = mine + (lane & 31);
    const float c = p.scale * LOG2E;
    // the stream: tiles of 64 queries, from the one with the block's first key on, of one head after the other
    const int t0 = j0 / TILE_ROWS, per = (s.len + TILE_ROWS - 1) / TILE_ROWS - t0;
    const int64_t all = (int64_t)per * p.G;
    const int lo = (int)(all * split / nsplit), hi = (int)(all * (split + 1) / nsplit);
    const float f = E::DTYPE == SA2_F16 ? key_factor(p, terms, s, hk, j0, per, lo, hi, (float*)lds) : 1.f;
    const float fd = f * (1.f / (1 << LIFT<E>));                           // what takes a lifted weight times dP - delta to dS times f

    static_for<2>([&](auto W) __attribute__((always_inline)) {
        const Tensor& t = decltype(W)::value ? p.v : p.k;
        const uint16_t* row = (const uint16_t*)t.p + row_offset(t, s, key < s.len ? key : 0, hk);
        uint4 x[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int col = 16 * kk + 8 * half;
            x[kk] = make_uint4(0, 0, 0, 0);
            if (key < s.len && col < p.D) x[kk] = *(const uint4*)(row + col);
        }
        static_for<KK>([&](auto K) __attribute__((always_inline)) {
            constexpr int kk = decltype(K)::value;
            L::template set_regs<(decltype(W)::value ? VALUE0 : KEY0) + kk * 4>(x[kk].x, x[kk].y, x[kk].z, x[kk].w);
        });
    });
    static_for<8 * DT>([&](auto X) __attribute__((always_inline)) { L::template set_regs<4 * decltype(X)::value>(0u, 0u, 0u, 0u); });

    int rg = lo / per, rt = lo - rg * per;                                 // head and tile of the next request
    Fetch<D> fetch;
    fetch.init(p.q, p.dout, s, hk * p.G + rg, p.D);
    const int64_t stat_row = (int64_t)s.b * p.H * p.rows.N + s.first;
    int sent = lo, released = lo - 1;
    uint32_t arriving = 0, here = 0;                                       // buffers, as numbers
    auto buffer = [&](uint32_t i) { return base + i * Buffer<D>::BYTES; };
    auto after = [&](uint32_t i) { return (i + 1) % BUFFERS; };
    auto request = [&]() {
        const int first = (t0 + rt) * TILE_ROWS;
        fetch.request(first, s.len, buffer(arriving), padded);
        if (wave < 2) {
            const float* src = (wave ? p.delta : terms.minus_lse) + stat_row + (int64_t)(hk * p.G + rg) * p.rows.N + first + lane;
            lds_request4(first + lane < s.len ? (const void*)src : (const void*)zero_chunk, stats + arriving * STATS + wave * TILE_ROWS * 4);
        }
        arriving = after(arriving);
        ++sent;
        if (++rt == per) {
            rt = 0;
            ++rg;
            fetch.next_head(p.q, p.dout);
        }
    };
    auto arrive = [&]() {                                                  // the next tile, with its successor on its way
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        ++released;
        if (sent < hi) request();
    };

    const uint32_t row_lane = T::row_lane(lane), column_lane = T::column_lane(lane);
    floatx16 st[2], dp[2];                                                 // first products of this piece of 32 queries and the next
    X8 pw[2][2], dw[2][2];                                                 // weights and dS of this piece and the last
    X8 rows[2 * KK], cols[4 * DT];                                         // Q then dO; dO then Q
    auto rows_at = [&](uint32_t buf, int sub) {
        uint32_t at = buffer(buf) + row_lane + (uint32_t)(sub * T::BYTES);
        stays(at);
        return at;
    };
    auto cols_at = [&](uint32_t buf, int sub) {
        uint32_t at = buffer(buf) + column_lane + (uint32_t)(sub * T::BYTES);
        stays(at);
        return at;
    };
    auto stats_at = [&](uint32_t buf, int sub) {
        uint32_t at = stats + buf * STATS + (uint32_t)(sub * SUB * 4 + 16 * half);
        stays(at);
        return at;
    };
    auto load_row = [&](auto A, uint32_t at) __attribute__((always_inline)) {
        constexpr int a = decltype(A)::value, kk = a % KK;
        rows[a] = lds_read_x8<X8>(at + (uint32_t)((a < KK ? Buffer<D>::FIRST : Buffer<D>::SECOND) + kk / 2 * T::BLOCK + kk % 2 * 32));
    };
    auto load_col = [&](auto C, uint32_t at) __attribute__((always_inline)) {
        constexpr int x = decltype(C)::value, j = x % (2 * DT);
        cols[x] = quad_tile_column<D, X8>(at + (uint32_t)(x < 2 * DT ? Buffer<D>::SECOND : Buffer<D>::FIRST), 0, j % DT, j / DT);
    };
    // rows 8g + 4 * half + r of the piece: -lse / scale into st, -delta into dp
    auto load_stat = [&](auto X, uint32_t at, floatx16& x, floatx16& y) __attribute__((always_inline)) {
        constexpr int i = decltype(X)::value, g = i % 4;
        typedef float f4 __attribute__((ext_vector_type(4)));
        const f4 v = *(const f4 __attribute__((address_space(3)))*)(uintptr_t)(at + (uint32_t)(i / 4 * TILE_ROWS * 4 + 32 * g));
        floatx16& z = i < 4 ? x : y;
        z[4 * g] = v[0]; z[4 * g + 1] = v[1]; z[4 * g + 2] = v[2]; z[4 * g + 3] = v[3];
    };
    auto first_mfma = [&](auto A, floatx16& x, floatx16& y) __attribute__((always_inline)) {
        constexpr int a = decltype(A)::value;
        if constexpr (a < KK) L::template tile_more<KEY0 + a * 4>(x, rows[a]);
        else L::template tile_more<VALUE0 + (a - KK) * 4>(y, rows[a]);
    };
    auto second_mfma = [&](auto C, const X8 (&x)[2], const X8 (&y)[2]) __attribute__((always_inline)) {
        constexpr int i = decltype(C)::value, j = i % (2 * DT);
        if constexpr (i < 2 * DT) L::template sum_more<V0 + j % DT * 16>(cols[i], x[j / DT]);
        else L::template sum_more<K0 + j % DT * 16>(cols[i], y[j / DT]);
    };
    // One step: first products of piece u + 1 (FIRST), weights of u, second products of u - 1 (SECOND), u of parity PAR; operands of
    // the pieces after those
    // (LEAD: operands ahead; with three the kernel of 64 columns has two wavefronts per SIMD, dK and dV of B1 N8192 H16 285 us, with four one,
    // 306)
    constexpr int SLOTS = 4 * KK, LEAD = D == 64 ? 3 : 4, LAG = SLOTS == 32 ? 20 : 11;
    auto step = [&](auto PP, auto FF, auto SS, uint32_t rat, uint32_t rnext, uint32_t snext, uint32_t cat, uint32_t cnext) __attribute__((always_inline)) {
        constexpr int PAR = decltype(PP)::value;
        constexpr bool FIRST = decltype(FF)::value, SECOND = decltype(SS)::value;
        floatx16 &x = st[PAR], &y = dp[PAR];
        float e[16];
        union { uint32_t u[8]; X8 v[2]; } zp, zd;
        float d0 = 0.f;
        static_for<SLOTS>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = decltype(I)::value, k = i / 2;
            if constexpr (i % 2 == 0 && FIRST) first_mfma(LONE_C(k), st[PAR ^ 1], dp[PAR ^ 1]);
            if constexpr (i % 2 == 1 && SECOND) second_mfma(LONE_C(k), pw[PAR ^ 1], dw[PAR ^ 1]);
            deal<16, i - 1, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = x[decltype(X)::value] * c; });
            deal<16, i - 2, LAG>([&](auto X) __attribute__((always_inline)) { e[decltype(X)::value] = fast_exp2(e[decltype(X)::value]); });
            deal<16, i - 3, LAG>([&](auto X) __attribute__((always_inline)) {
                constexpr int j = decltype(X)::value;
                float ds = e[j] * y[j];
                if constexpr (E::DTYPE == SA2_F16) ds *= fd;
                if constexpr (j % 2) {
                    zp.u[j / 2] = pack2<E>(e[j - 1], e[j]);
                    zd.u[j / 2] = pack2<E>(d0, ds);
                } else d0 = ds;
            });
            if constexpr (i % 2 == 0) {
                if constexpr (FIRST && k + LEAD < 2 * KK) load_row(LONE_C(k + LEAD), rat);
                else if constexpr (FIRST && k + LEAD >= 2 * KK) load_row(LONE_C(k + LEAD - 2 * KK), rnext);
            } else {
                if constexpr (SECOND && k + LEAD < 4 * DT) load_col(LONE_C(k + LEAD), cat);
                else if constexpr (k + LEAD >= 4 * DT) load_col(LONE_C(k + LEAD - 4 * DT), cnext);
            }
            if constexpr (FIRST) deal<8, i - LAG - 3, SLOTS - LAG - 3>([&](auto X) __attribute__((always_inline)) { load_stat(X, snext, x, y); });
            __builtin_amdgcn_sched_barrier(0);
        });
        pw[PAR][0] = zp.v[0];
        pw[PAR][1] = zp.v[1];
        dw[PAR][0] = zd.v[0];
        dw[PAR][1] = zd.v[1];
        stays(pw[PAR][0]);
        stays(pw[PAR][1]);
        stays(dw[PAR][0]);
        stays(dw[PAR][1]);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto rest = [&]() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); };
    // A piece by itself: queries `q0` .. + 31, some of which do not see the wavefront's keys.  dS goes in as two 16-bit parts here: in
    // sequences of a few rows, whose sums cancel, its rounding alone took dK to 1.7 times the error that its own rounding leaves
    auto piece = [&](uint32_t buf, int sub, int q0) {
        const uint32_t sat = stats_at(buf, sub), rat = rows_at(buf, sub), cat = cols_at(buf, sub);
        static_for<8>([&](auto X) __attribute__((always_inline)) { load_stat(X, sat, st[0], dp[0]); });
        static_for<2 * KK>([&](auto A) __attribute__((always_inline)) { load_row(A, rat); });
        asm volatile("s_nop 3" : "+v"(st[0]), "+v"(dp[0]));
        static_for<2 * KK>([&](auto A) __attribute__((always_inline)) { first_mfma(A, st[0], dp[0]); });
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(st[0]));
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(dp[0]));
        const bool masked = q0 < mine + SUB - 1 || q0 == 0;
        union { uint32_t u[8]; X8 v[2]; } zp, zd, zl;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float e[2], ds[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 2 * i + j, query = q0 + 8 * (r / 4) + 4 * half + r % 4;
                e[j] = fast_exp2(st[0][r] * c);
                ds[j] = e[j] * dp[0][r] * fd;
                if (masked) {
                    if (query < key) e[j] = ds[j] = 0.f;
                    if (query == 0) ds[j] = 0.f;             // a first query has one weight, 1, whose gradient is zero
                }
            }
            zp.u[i] = pack2<E>(e[0], e[1]);
            zd.u[i] = pack2<E>(ds[0], ds[1]);
            zl.u[i] = pack2<E>(ds[0] - E::lo(zd.u[i]), ds[1] - E::hi(zd.u[i]));
        }
        static_for<4 * DT>([&](auto C) __attribute__((always_inline)) { load_col(C, cat); });
        uint32_t bits = 0;
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4 * DT; ++i) bits |= odd_bits<E>(cols[i]);
        }
        if (any_odd(bits)) {
            const uint32_t tile = buffer(buf) + (uint32_t)(sub * T::BYTES);
            guarded_sum<E, L, V0, D>(tile + Buffer<D>::SECOND, zp.v, [&](int i) { return q0 + i >= key; });
            guarded_sum<E, L, K0, D>(tile + Buffer<D>::FIRST, zd.v, [&](int i) { return q0 + i >= key && q0 + i > 0; });
            guarded_sum<E, L, K0, D>(tile + Buffer<D>::FIRST, zl.v, [&](int i) { return q0 + i >= key && q0 + i > 0; });
        } else {
            asm volatile("s_nop 3" : "+v"(zp.v[0]), "+v"(zp.v[1]), "+v"(zd.v[0]), "+v"(zd.v[1]), "+v"(zl.v[0]), "+v"(zl.v[1]));
            static_for<4 * DT>([&](auto C) __attribute__((always_inline)) { second_mfma(C, zp.v, zd.v); });
            static_for<2 * DT>([&](auto C) __attribute__((always_inline)) { second_mfma(LONE_C(decltype(C)::value + 2 * DT), zp.v, zl.v); });
            rest();
        }
    };
    if (lo < hi) {
        if (E::DTYPE == SA2_F16) __syncthreads();                          // (the factors have left LDS)
        request();
        arrive();
        constexpr int OWN = BLOCK / TILE_ROWS;                             // a head's first tiles hold the block's own rows
        for (int at = lo; at < hi;) {
            const int g = at / per, i0 = at - g * per, i1 = hi - at < per - i0 ? i0 + hi - at : per;
            int i = i0;
            for (; i < i1 && i < OWN; ++i, here = after(here)) {
                if (at + i - i0 > released) arrive();
#pragma unroll 1
                for (int sub = 0; sub < 2; ++sub) {
                    const int q0 = (t0 + i) * TILE_ROWS + sub * SUB;
                    if (q0 + SUB > mine) piece(here, sub, q0);
                }
            }
            if (i < i1) {
                if (at + i - i0 > released) arrive();
                const std::true_type yes{};
                const std::false_type no{};
                L::keep_out();
                // first products of the first piece
                static_for<8>([&](auto X) __attribute__((always_inline)) { load_stat(X, stats_at(here, 0), st[0], dp[0]); });
                static_for<2 * KK>([&](auto A) __attribute__((always_inline)) { load_row(A, rows_at(here, 0)); });
                asm volatile("s_nop 3" : "+v"(st[0]), "+v"(dp[0]));
                static_for<2 * KK>([&](auto A) __attribute__((always_inline)) { first_mfma(A, st[0], dp[0]); });
                static_for<8>([&](auto X) __attribute__((always_inline)) { load_stat(X, stats_at(here, 1), st[1], dp[1]); });
                static_for<LEAD>([&](auto A) __attribute__((always_inline)) { load_row(A, rows_at(here, 1)); });
                asm volatile("s_nop 15\n\ts_nop 15" : "+v"(st[0]));
                asm volatile("s_nop 15\n\ts_nop 15" : "+v"(dp[0]));
                asm volatile("s_nop 3" : "+v"(st[1]), "+v"(dp[1]));
                if (i + 1 < i1) arrive();
                uint32_t next = after(here);
                // (where no tile follows, `next` is read and its products are not used)
                step(LONE_C(0), yes, no, rows_at(here, 1), rows_at(i + 1 < i1 ? next : here, 0), stats_at(i + 1 < i1 ? next : here, 0), 0u, cols_at(here, 0));
                for (++i; i < i1; ++i) {
                    const uint32_t last = here;
                    here = next;
                    next = after(here);
                    step(LONE_C(1), yes, yes, rows_at(here, 0), rows_at(here, 1), stats_at(here, 1), cols_at(last, 0), cols_at(last, 1));
                    if (i + 1 < i1) arrive();
                    const uint32_t ahead = i + 1 < i1 ? next : here;
                    step(LONE_C(0), yes, yes, rows_at(here, 1), rows_at(ahead, 0), stats_at(ahead, 0), cols_at(last, 1), cols_at(here, 0));
                }
                step(LONE_C(1), no, yes, 0u, 0u, 0u, cols_at(here, 0), cols_at(here, 1));
                static_for<4 * DT - LEAD>([&](auto C) __attribute__((always_inline)) { load_col(LONE_C(decltype(C)::value + LEAD), cols_at(here, 1)); });
                asm volatile("s_nop 3" : "+v"(pw[1][0]), "+v"(pw[1][1]), "+v"(dw[1][0]), "+v"(dw[1][1]));
                static_for<4 * DT>([&](auto C) __attribute__((always_inline)) { second_mfma(C, pw[1], dw[1]); });
                rest();
                here = after(here);
            }
            at += i1 - i0;
        }
    }
    rest();
    if (key < s.len) {
        const int64_t row = ((int64_t)s.b * p.HK + hk) * p.rows.N + s.first + key, total = (int64_t)p.rows.B * p.HK * p.rows.N;
        float* const part = p.part + ((int64_t)split * 2 * total + row) * p.D;
        uint16_t* const dk = p.dk.p ? (uint16_t*)p.dk.p + row_offset(p.dk, s, key, hk) : nullptr;
        uint16_t* const dv = p.dv.p ? (uint16_t*)p.dv.p + row_offset(p.dv, s, key, hk) : nullptr;
        static_for<4 * DT>([&](auto X) __attribute__((always_inline)) {
            constexpr int x = decltype(X)::value;
            const int col = 8 * x + 4 * half;
            float4 v = L::template get_regs<V0 + 4 * x>(), k = L::template get_regs<K0 + 4 * x>();
            const float to = p.scale / f, off = 1.f / (1 << LIFT<E>);
            v.x *= off; v.y *= off; v.z *= off; v.w *= off;
            k.x *= to; k.y *= to; k.z *= to; k.w *= to;
            if (col < p.D) {
                if (nsplit > 1) {
                    *(float4*)(part + col) = k;
                    *(float4*)(part + total * p.D + col) = v;
                } else {
                    if (dk) *(uint2*)(dk + col) = make_uint2(pack2<E>(k.x, k.y), pack2<E>(k.z, k.w));
                    if (dv) *(uint2*)(dv + col) = make_uint2(pack2<E>(v.x, v.y), pack2<E>(v.z, v.w));
                }
            }
        });
    }
}

template <class E, int D>
__global__ __launch_bounds__(THREADS, 1) void causal_dkv16_kernel(Causal p, Causal16Terms terms, int nsplit, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    keys_gradients16<E, D>(p, terms, nsplit, padded, blockIdx.x, lds);
}
// All gradients in one launch where there are few workgroups, so that one's fill the CUs that the other's short ones leave: `queries`
// workgroups for dQ, whose longest chains are the longest of all, then those for dK and dV (B2 N2048 H8 D64 80 us apart, 57 together; B4 N1024
// H16/4 D128 133 and 121; with as many blocks of 256 queries as would give every CU two, B1 N8192 H16/4 D128, 921 and 967: there
// a wavefront with 64 queries saves more).
template <class E, int D>
__global__ __launch_bounds__(THREADS, 1) void causal_bwd16_kernel(Causal p, Causal16Terms terms, int nsplit, int queries, bool padded) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if ((int)blockIdx.x < queries) queries_gradient16<E, D, 1>(p, terms, padded, blockIdx.x, lds);
    else keys_gradients16<E, D>(p, terms, nsplit, padded, blockIdx.x - queries, lds);
}

// Sums of the shares in their order: part[split][dK, dV][row][D]
template <class E>
__global__ __launch_bounds__(THREADS) void causal_sums_kernel(Causal p, int nsplit) {
    const int chunks = p.D / 8;
    const int64_t total = (int64_t)p.rows.B * p.HK * p.rows.N, it = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const int64_t row = it / chunks;
    if (row >= total) return;
    const int col = (int)(it - row * chunks) * 8, n = (int)(row % p.rows.N), hk = (int)(row / p.rows.N % p.HK), b = (int)(row / p.rows.N / p.HK);
    const bool none = p.rows.cu && (n < p.rows.cu[0] || n >= p.rows.cu[p.rows.sequences]);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const Tensor& t = w ? p.dv : p.dk;
        if (!t.p) continue;
        float x[8] = {};
        if (!none)
            for (int i = 0; i < nsplit; ++i) {
                const float* src = p.part + ((int64_t)(2 * i + w) * total + row) * p.D + col;
                const float4 a = *(const float4*)src, c = *(const float4*)(src + 4);
                x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
                x[4] += c.x; x[5] += c.y; x[6] += c.z; x[7] += c.w;
            }
        *(uint4*)((uint16_t*)t.p + t.off(b, n, hk) + col) = make_uint4(pack2<E>(x[0], x[1]), pack2<E>(x[2], x[3]), pack2<E>(x[4], x[5]), pack2<E>(x[6], x[7]));
    }
}

template <class E>
int launch(const Causal& p, const Causal16Terms& terms, hipStream_t st) {
    const int64_t rows = (int64_t)p.rows.B * p.rows.N * p.H;
    const int lanes = p.D > 64 ? 16 : 8;
    const int64_t want = (rows + THREADS / lanes - 1) / (THREADS / lanes);
    const int blocks = (int)(want < TERMS_BLOCKS ? want : TERMS_BLOCKS);
    if (lanes == 16) causal_terms_kernel<E, 16><<<dim3(blocks), dim3(THREADS), 0, st>>>(p, terms);
    else causal_terms_kernel<E, 8><<<dim3(blocks), dim3(THREADS), 0, st>>>(p, terms);
    if (hipGetLastError() != hipSuccess) return SA2_ERR_LAUNCH_FAILED;
    const bool together = p.dq.p && (p.dk.p || p.dv.p) && !causal16_two(p);
    if (p.dk.p || p.dv.p) {
        const int nsplit = causal16_splits(p.rows.B, p.rows.N, p.HK, p.G);
        auto of = [&](auto w) {
            constexpr int D = decltype(w)::value;
            const int64_t keys = (int64_t)p.rows.B * p.HK * nsplit * count_tiles(p.rows, BLOCK), queries = together ? (int64_t)p.rows.B * p.H * count_tiles(p.rows, BLOCK) : 0;
            constexpr int LDS = BUFFERS * (Buffer<D>::BYTES + STATS);
            static_assert(LDS >= DQ_BUFFERS * Buffer<D>::BYTES, "");
            if (keys + queries > 0x7fffffff) return (int)SA2_ERR_TOO_LARGE;
            const dim3 grid((unsigned)(keys + queries)), block(THREADS);
            if (!allow_full_lds(together ? (const void*)causal_bwd16_kernel<E, D> : (const void*)causal_dkv16_kernel<E, D>)) return (int)SA2_ERR_LAUNCH_FAILED;
            if (together) causal_bwd16_kernel<E, D><<<grid, block, LDS, st>>>(p, terms, nsplit, (int)queries, p.D != D);
            else causal_dkv16_kernel<E, D><<<grid, block, LDS, st>>>(p, terms, nsplit, p.D != D);
            return (int)(hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED);
        };
        const int rc = p.D <= 64 ? of(std::integral_constant<int, 64>{}) : of(std::integral_constant<int, 128>{});
        if (rc != SA2_OK) return rc;
        if (nsplit > 1) {
            const int64_t items = (int64_t)p.rows.B * p.HK * p.rows.N * (p.D / 8);
            causal_sums_kernel<E><<<dim3((unsigned)((items + THREADS - 1) / THREADS)), dim3(THREADS), 0, st>>>(p, nsplit);
            if (hipGetLastError() != hipSuccess) return SA2_ERR_LAUNCH_FAILED;
        }
    }
    return p.dq.p && !together ? launch_causal16_dq(p, E::DTYPE, terms, st) : SA2_OK;
}

}  // namespace

// Shares of a key block's stream: two workgroups per CU over the chip, where the stream is that long (packed sequences: as if
// they were one, the bound that the host knows)
int causal16_splits(int B, int N, int HK, int G) {
    const int64_t blocks = (int64_t)B * HK * ((N + BLOCK - 1) / BLOCK), tiles = (int64_t)G * ((N + TILE_ROWS - 1) / TILE_ROWS);
    int64_t n = (2 * CUS + blocks - 1) / blocks;
    if (n > tiles / 8) n = tiles / 8;
    return n < 1 ? 1 : n > 16 ? 16 : (int)n;
}
size_t causal16_part_bytes(int B, int N, int HK, int G, int D) {
    const int n = causal16_splits(B, N, HK, G);
    return n > 1 ? (size_t)n * 2 * B * HK * N * D * sizeof(float) : 0;
}

int launch_causal16_bwd(const Causal& p, int dtype, const Causal16Terms& terms, hipStream_t st) {
    return dtype == SA2_F16 ? launch<ElemF16>(p, terms, st) : launch<ElemBF16>(p, terms, st);
}

}  // namespace sa2
