// Windowed attention, forward, bf16 and fp16 on the 16-bit MFMA: head_dim a multiple of 8 up to 128, rows on the 16-byte grid.
//
//   S = scale Q K^T (j <= i and (i - j < window or j < sinks)), P = softmax(S), O = P V, LSE = log sum e^S
//
// The sweep of sa2_sweep16.h over the tiles in reach, latest first, masks in the pipeline.  A workgroup's four wavefronts own blocks of
// 32 NQ queries; where heads share keys, they are the same queries of two or four of these heads, so that all wavefronts need the same
// tiles: with the blocks of one head one behind the other, as without a window, a workgroup of 256 queries fetches 768 keys for a window
// of 512 of which a wavefront needs 576.
// 16 heads over 4 key heads, 8192 queries, head_dim 128, bf16, window 512 with 4 first keys: 105 us (0.32 PFLOP/s); 8 heads over 2, 32768 queries,
// window 4096, fp16: 540 us (0.96, 78 % of a large product's rate).  A tile of 64 keys takes 1.35 us, a workgroup's start and end 17: first
// loads, queries to accumulation registers, masks, the join of the first keys, the output.
#include "sa2_sweep16.h"

namespace sa2 {
namespace {

template <int D, int NQ>
struct WindowKeys {
    static constexpr bool SLIDING = true;
    Fetch<D> fetch;
    Band band;
    bool padded, narrow;
    int mine, len, top, head;                               // top: the last window tile; head: tiles of first keys before the first
    int tiles, window, a, b, clear, clear_end, before;
    float lower;
    // the first key of tile t
    __device__ __forceinline__ int key(int t) const { return (t < before ? 0 : t < window ? top - (t - before) : head - 1 - (t - window)) * TILE_ROWS; }
    __device__ __forceinline__ void request(int t, uint32_t buffer) const { fetch.request(key(t), len, buffer, padded); }
    __device__ __forceinline__ void begin(uint32_t base) const {
        request(0, base);
        if (tiles > 1) request(1, base + Buffer<D>::BYTES);
    }
    __device__ __forceinline__ bool any(int piece) const {
        const int k0 = key(piece / 2) + piece % 2 * SUB;
        return k0 < mine + 32 * NQ && (mine - (k0 + SUB - 1) < band.window || k0 < band.sinks);
    }
    __device__ __forceinline__ bool guarded(int piece) const {
        const int k0 = key(piece / 2) + piece % 2 * SUB;
        return !band_full(band, mine, mine + 32 * NQ - 1, k0, k0 + SUB - 1);
    }
    __device__ __forceinline__ uint32_t sees(int n, int piece) const {
        int row = mine + 32 * n + (int)(threadIdx.x & 31);
        stays(row);                                         // (what can be had from it before the sweep took 45 registers of the sweep's)
        return band_keys(band, row, key(piece / 2) + piece % 2 * SUB);
    }
};

template <class E, int D, int NQ>
__global__ __launch_bounds__(THREADS, D == 64 && NQ == 2 ? 2 : 1) void window_fwd16_kernel(Causal p, bool padded, int heads) {
    using L = SweepRegs<D, NQ>;
    constexpr int KK = D / 16, DT = D / 32, ROWS = 32 * NQ;
    constexpr int O0 = L::O0, Q0 = L::Q0;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t base = lds_address(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int block = ROWS * WAVES / heads;
    int stream, tile;
    order(blockIdx.x, p.rows.B * p.H / heads, stream, tile);
    const int b = stream / (p.H / heads), h0 = stream % (p.H / heads) * heads, h = h0 + wave % heads, hk = h / p.G;
    Span s;
    if (!find_tile(p.rows, b, tile, block, s)) return;
    float* const lse = p.lse + ((int64_t)s.b * p.H + h) * p.rows.N + s.first;
    typedef typename E::scalar scalar;
    if (s.fill) {
        for (int i = threadIdx.x; i < heads * s.len * p.D; i += THREADS) {
            const int at = i / p.D;
            ((scalar*)p.out.p)[row_offset(p.out, s, at % s.len, h0 + at / s.len) + i % p.D] = (scalar)0.f;
        }
        for (int i = threadIdx.x; i < heads * s.len; i += THREADS) p.lse[((int64_t)s.b * p.H + h0 + i / s.len) * p.rows.N + s.first + i % s.len] = -INFINITY;
        return;
    }
    const int q0 = s.block * block, mine = q0 + wave / heads * ROWS, last = q0 + block < s.len ? q0 + block : s.len;
    const float c = fabsf(p.scale) * LOG2E;
    const KeyTiles<true, TILE_ROWS> reach(p.band, q0, last - 1);
    WindowKeys<D, NQ> keys;
    keys.fetch.init(p.k, p.v, s, hk, p.D);
    keys.band = p.band;
    keys.padded = padded;
    keys.narrow = p.band.window < TILE_ROWS;
    keys.mine = mine;
    keys.len = last;
    keys.head = reach.head;
    keys.top = (last - 1) / TILE_ROWS;
    keys.before = E::DTYPE == SA2_F16 && reach.head > 0 ? 1 : 0;
    keys.tiles = keys.before + reach.count;
    keys.window = keys.tiles - reach.head;
    keys.a = keys.b = keys.clear = keys.clear_end = 0;
    if (mine < s.len) {
        const int end = mine + ROWS < s.len ? mine + ROWS : s.len, low = mine < p.band.window ? 0 : mine - p.band.window + 1;
        keys.a = keys.before + keys.top - (end - 1) / TILE_ROWS;
        // (first keys that the workgroup's windows reach into)
        const bool joined = (p.band.sinks + TILE_ROWS - 1) / TILE_ROWS > reach.start;
        keys.b = keys.before + keys.top - (joined ? reach.start : low / TILE_ROWS) + 1;
        // seen whole: tiles behind (in the list) the one of the first own key, as far as the last row's window reaches
        const int first = keys.before + keys.top - mine / TILE_ROWS + 1, edge = mine + ROWS - p.band.window;
        keys.clear = first;
        keys.clear_end = keys.before + keys.top - (edge > 0 ? (edge + TILE_ROWS - 1) / TILE_ROWS : 0);   // (all but the last of them: the one behind it counts too)
    }
    // (weights that are lost below 2^-25 of a row's largest: of the keys that it sees)
    const int64_t most = (int64_t)p.band.window + p.band.sinks;
    keys.lower = lowered_by<E>(most < last ? (int)most : last, c);
    keys.begin(base);
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
int launch(const Causal& p, int heads, hipStream_t st) {
    const auto kernel = window_fwd16_kernel<E, D, NQ>;
    const int64_t grid = (int64_t)p.rows.B * (p.H / heads) * count_tiles(p.rows, 32 * NQ * WAVES / heads);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    if (!allow_full_lds((const void*)kernel)) return SA2_ERR_LAUNCH_FAILED;
    kernel<<<dim3((unsigned)grid), dim3(THREADS), SWEEP_BUFFERS<WindowKeys<D, NQ>, NQ> * Buffer<D>::BYTES, st>>>(p, p.D != D, heads);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

int launch_window16_fwd(const Causal& p, int dtype, hipStream_t st) {
    auto of = [&](auto e) {
        using E = decltype(e);
        const int heads = window_heads(p);
        const bool two = window_two(p, heads);
        if (p.D <= 64) return two ? launch<E, 64, 2>(p, heads, st) : launch<E, 64, 1>(p, heads, st);
        return two ? launch<E, 128, 2>(p, heads, st) : launch<E, 128, 1>(p, heads, st);
    };
    return dtype == SA2_F16 ? of(ElemF16{}) : of(ElemBF16{});
}

}  // namespace sa2
