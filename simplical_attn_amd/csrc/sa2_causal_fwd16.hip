// Causal attention, forward, bf16 and fp16 on the 16-bit MFMA: head_dim a multiple of 8 up to 128, rows on the 16-byte grid.
//
//   S = scale Q K^T (j <= i), P = softmax(S), O = P V, LSE = log sum e^S
//
// A wavefront owns NQ blocks of 32 queries and sweeps the keys that they see (sa2_sweep16.h); four wavefronts are a workgroup.
// Measured (bf16): B1 N8192 H16/4 D128 260 us (1060 TFLOP/s), N16384 H8/2 fp16 510 (1080), N8192 H16 D64 172 (800), B2 N2048 H8 D64
// 31 (280).  Large calls are bound by the MFMAs at the clock that this load leaves (busy 48 % of the time at 2.05 GHz) and the
// exponentials between them, small ones by the longest block's chain of tiles: 2200 cycles per 64 keys with 32 queries of 128.
#include "sa2_sweep16.h"

namespace sa2 {
namespace {

// The keys of a workgroup's block of queries, as the sweep takes them (sa2_sweep16.h)
template <int D>
struct CausalKeys {
    static constexpr bool SLIDING = false;
    Fetch<D> fetch;
    bool padded, active;
    int last, mine, tiles, full, pieces;
    float lower;
    __device__ __forceinline__ void request(int t, uint32_t buffer) const { fetch.request(t * TILE_ROWS, last, buffer, padded); }
    __device__ __forceinline__ bool guarded(int piece) const { return piece * SUB + SUB - 1 > mine; }
    __device__ __forceinline__ uint32_t sees(int n, int piece) const {
        const int up_to = mine + 32 * n + (int)(threadIdx.x & 31) - piece * SUB;
        return up_to >= 31 ? ~0u : up_to < 0 ? 0u : (2u << up_to) - 1;
    }
};

template <class E, int D, int NQ>
__global__ __launch_bounds__(THREADS, D == 64 ? 2 : 1) void causal_fwd16_kernel(Causal p, bool padded) {
    using T = QuadTile<D>;
    using X8 = typename E::x8;
    using L = SweepRegs<D, NQ>;
    constexpr int KK = D / 16, DT = D / 32, ROWS = 32 * NQ, BLOCK = ROWS * WAVES;
    constexpr int O0 = L::O0, Q0 = L::Q0;
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
    float m[NQ], l[NQ];
    CausalKeys<D> keys{fetch, padded, mine < s.len, last, mine, tiles, 0, 0, lowered_by<E>(last, c)};
    keys.full = keys.active ? mine / TILE_ROWS : 0;
    keys.pieces = keys.active ? (mine + ROWS) / SUB : 0;
    sweep16<E, D, NQ>(keys, base, c, m, l);
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
        const bool two = causal16_two(p);
        if (p.D <= 64) return two ? launch<E, 64, 2>(p, st) : launch<E, 64, 1>(p, st);
        return two ? launch<E, 128, 2>(p, st) : launch<E, 128, 1>(p, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace sa2
