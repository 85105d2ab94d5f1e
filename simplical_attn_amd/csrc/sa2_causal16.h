// What the 16-bit causal attention kernels share: tiles of rows in LDS and sums that hidden rows stay out of.
#pragma once

#include "sa2_causal_common.h"
#include "sa2_mfma_lone.h"

namespace sa2 {
namespace {

constexpr int THREADS = 256, WAVES = 4, SUB = 32, TILE_ROWS = 2 * SUB;

template <int D>
struct Buffer {                                             // TILE_ROWS rows of two tensors: two QuadTiles each
    static constexpr int FIRST = 0, SECOND = 2 * QuadTile<D>::BYTES, BYTES = 4 * QuadTile<D>::BYTES;
};

// TILE_ROWS rows of two tensors (K and V, or Q and dO) to LDS; each wavefront brings a quarter.  Rows from `len` on and columns
// from `width` on: zeros.
template <int D>
struct Fetch {
    using T = QuadTile<D>;
    static constexpr int INSTR = TILE_ROWS / T::RPW / WAVES;   // per tensor and wavefront
    const char *a, *b;                                      // row 0 of the sequence
    int64_t as, bs;                                         // bytes from row to row
    uint32_t aoff[INSTR], boff[INSTR];                      // of the lane's rows in a tile
    int row[INSTR];
    bool pad;                                               // the lane's columns lie behind the row
    __device__ __forceinline__ void init(const Tensor& x, const Tensor& y, const Span& s, int h, int width) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        a = (const char*)x.p + row_offset(x, s, 0, h) * 2;
        b = (const char*)y.p + row_offset(y, s, 0, h) * 2;
        as = x.sn * 2;
        bs = y.sn * 2;
        const int chunk = T::dma_chunk(lane);
        pad = chunk * 8 >= width;
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
            row[i] = (wave * INSTR + i) * T::RPW + T::dma_row(lane);
            aoff[i] = (uint32_t)(row[i] * as) + chunk * 16;
            boff[i] = (uint32_t)(row[i] * bs) + chunk * 16;
        }
    }
    // the next head of both
    __device__ __forceinline__ void next_head(const Tensor& x, const Tensor& y) {
        a += x.sh * 2;
        b += y.sh * 2;
    }
    __device__ __forceinline__ void request(int first, int len, uint32_t buffer, bool padded) const {
        const int wave = threadIdx.x >> 6;
        const char *ab = a + first * as, *bb = b + first * bs;
        if (first + TILE_ROWS <= len && !padded) {
#pragma unroll
            for (int i = 0; i < INSTR; ++i) {
                const int g = wave * INSTR + i;             // group of RPW rows
                lds_request(ab, aoff[i], buffer + Buffer<D>::FIRST + g * T::GROUP);
                lds_request(bb, boff[i], buffer + Buffer<D>::SECOND + g * T::GROUP);
            }
        } else {
#pragma unroll
            for (int i = 0; i < INSTR; ++i) {
                const int g = wave * INSTR + i;
                const bool there = first + row[i] < len && !pad;
                lds_request(there ? ab + aoff[i] : (const char*)zero_chunk, buffer + Buffer<D>::FIRST + g * T::GROUP);
                lds_request(there ? bb + boff[i] : (const char*)zero_chunk, buffer + Buffer<D>::SECOND + g * T::GROUP);
            }
        }
    }
};
// (groups of the two QuadTiles of a buffer follow one another)
static_assert(QuadTile<64>::BYTES == QuadTile<64>::NGROUP * QuadTile<64>::GROUP && QuadTile<128>::BYTES == QuadTile<128>::NGROUP * QuadTile<128>::GROUP, "");

// Eight 16-bit values each of whose exponents of ones carries into the top bit of its half: `any_odd` of these ORed together tells
// whether one was an infinity or NaN
template <class E>
__device__ __forceinline__ uint32_t odd_bits(const typename E::x8& x) {
    constexpr uint32_t EXP = E::DTYPE == SA2_BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = E::DTYPE == SA2_BF16 ? 0x00800080u : 0x04000400u;
    union { typename E::x8 v; uint32_t u[4]; } w;
    w.v = x;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= (w.u[i] & EXP) + ONE;
    return bits;
}
__device__ __forceinline__ bool any_odd(uint32_t bits) { return __any((bits & 0x80008000u) != 0); }
// Sums S0 .. += tile^T w one row of the tile (in LDS) at a time and on the vector ALU, for the lanes that see the row: a weight of
// zero would not keep an infinity or NaN out
template <class E, class L, int S0, int D, class F>
__device__ __forceinline__ void guarded_sum(uint32_t tile, const typename E::x8 (&w)[2], F&& visible) {
    using T = QuadTile<D>;
    const int half = (threadIdx.x & 63) >> 5;
    union { typename E::x8 v[2]; uint32_t u[8]; } x;
    x.v[0] = w[0];
    x.v[1] = w[1];
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
        const int at = 8 * (key / 16) + 4 * (key % 16 / 8) + key % 4;      // of the half that holds the key's weight
        uint32_t pair = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) pair = at / 2 == i ? x.u[i] : pair;
        const float held = at & 1 ? E::hi(pair) : E::lo(pair), other = other_half(held), weight = (key / 4 & 1) == half ? held : other;
        const bool sees = visible(key);
        const uint32_t row = tile + (uint32_t)((key / T::RPW) * T::GROUP + key % T::RPW * 64), flip = (uint32_t)T::flip(key);
        static_for<D / 8>([&](auto C) __attribute__((always_inline)) {
            constexpr int ch = decltype(C)::value, r = S0 + 4 * ch;
            typedef uint32_t u2 __attribute__((ext_vector_type(2)));
            const u2 v = *(const u2 __attribute__((address_space(3)))*)(uintptr_t)(row + ch / 4 * T::BLOCK + ((ch % 4) ^ flip) * 16 + half * 8);
            const float4 o = L::template get_regs<r>();
            auto plus = [&](float o, float v) { return __float_as_uint(sees ? fmaf(weight, v, o) : o); };
            L::template set_regs<r>(plus(o.x, E::lo(v.x)), plus(o.y, E::hi(v.x)), plus(o.z, E::lo(v.y)), plus(o.w, E::hi(v.y)));
        });
    }
    asm volatile("s_nop 7" ::: "memory");
}

// 4 bytes per lane from global memory straight to LDS, lane L to `to` + 4 * L (see lds_request)
__device__ __forceinline__ void lds_request4(const void* src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(src) : "memory");
}

// ---- factors of fp16's dS -------------------------------------------------------------------------------------------
// dS_ij = P_ij (dO_i v_j - delta_i) is at most |dO_i| |v_j| + |delta_i|.  Before it is rounded to fp16 it is multiplied by the power of
// two that takes such a bound to 2^13 .. 2^14: it cannot leave fp16's range, and N(0,1) rows' dS, 2^18 below their bound in 16384 rows of
// 128, stay above its smallest normal number by 2^10.  A row of dQ has its own factor, from the keys that it sees; a key its own, from
// the rows of all heads that see it (a workgroup's shares of them): what rows it does not see hold changes neither.  Norms that are no
// numbers are left out: where one is seen, the sums are none either.  With the norms and their largest found before the sweeps, fp16 gradients take
// 2 to 3 % longer than with one factor for the whole call (B1 N8192 H16/4 D128 901 -> 924 us).
__device__ __forceinline__ float gradient_factor(float bound) {
    return bound > 0.f && is_finite(bound) ? __builtin_amdgcn_ldexpf(1.f, 14 - __builtin_amdgcn_frexp_expf(bound)) : 1.f;
}
__device__ __forceinline__ float finite_or_zero(float x) { return is_finite(x) ? fabsf(x) : 0.f; }
// The largest over lanes 0 .. l % 32 of x (of the lane's half), or from l % 32 on
__device__ __forceinline__ float largest_up_to(float x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float y = __shfl_up(x, o, 32);
        if ((threadIdx.x & 31) >= o) x = fmaxf(x, y);
    }
    return x;
}
__device__ __forceinline__ float largest_from(float x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float y = __shfl_down(x, o, 32);
        if ((int)(threadIdx.x & 31) + o < 32) x = fmaxf(x, y);
    }
    return x;
}

}  // namespace
}  // namespace sa2
