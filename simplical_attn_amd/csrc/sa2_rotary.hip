// Rotation of q and k by the angles of their positions, forward and backward.
//
// Pair j of a row at position p turns by p * f_j: y0 = a (x0 cos - x1 sin), y1 = a (x1 cos + x0 sin), a the amplitude; the
// pair is (2j, 2j+1) of the rotated part (interleaved) or (j, j + rot/2).  The gradient is the same rotation by the
// opposite angle.  Columns from rot on are copied.
//
// Bound by memory: every element is read once and written once.  A thread keeps the cosines and sines of the pairs of one
// 16-byte chunk of a row (interleaved) or of two, half a rotated part apart, and goes through heads of q and of k with them, so
// that the angles, which cost about 40 instructions each, are shared by the heads and never lie in memory.  Angles: the product and its reduction to an eighth
// of a turn in 64 bits (a position of 10^6 leaves 10^-10 of a radian), the series of sine and cosine in 32.
// Measured: 16384 rows of 16 + 4 heads of 128 bf16, forward 37 us (4500 GB/s of the 4830 that a copy reaches), with the gradient 82;
// four single rows 5.5 us, the launch.
#include "sa2_layer_common.h"

namespace sa2 {
namespace {

constexpr int THREADS = 256;

// cos and sin of p * f radians, times a
__device__ __forceinline__ void turn(double p, double f, float a, float& c, float& s) {
    const double r = p * f * 0.15915494309189533577;                    // turns
    const double q = rint(4.0 * r);
    const float x = (float)((r - 0.25 * q) * 6.28318530717958647693);   // within pi/4: the series end below 2^-28
    const float z = x * x;
    const float sn = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 1.f);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
    const int k = (int)((long long)q & 3);
    const float u = (k & 1) ? sn : cs, v = (k & 1) ? cs : sn;
    c = (k == 1 || k == 2) ? -a * u : a * u;
    s = k >= 2 ? -a * v : a * v;
}

// A block takes `rows` rows; `share` threads of a row take every share-th of the H + HK heads, `units` the row's chunks.
struct Split {
    int rows, share, units;
};

// Elements of a chunk V, pairs of a thread: an interleaved chunk holds V / 2 whole pairs
template <int V, bool INTERLEAVED>
constexpr int pairs_of() { return INTERLEAVED && V > 1 ? V / 2 : V; }

template <class T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(THREADS) void rotary_kernel(Rotary p, Split sp) {
    constexpr bool ONE = INTERLEAVED && V > 1;                              // one chunk, not two
    constexpr int NP = pairs_of<V, INTERLEAVED>();
    const int64_t total = (int64_t)p.rows.B * p.rows.N;
    const int per_row = sp.share * sp.units, turning = p.rot / 2 / NP;
    for (int it = threadIdx.x; it < sp.rows * per_row; it += THREADS) {
        const int rl = it / per_row, rest = it - rl * per_row, first = rest / sp.units, unit = rest - first * sp.units;
        const int64_t row = (int64_t)blockIdx.x * sp.rows + rl;
        if (row >= total) break;
        const int b = p.rows.B == 1 ? 0 : (int)(row / p.rows.N), n = (int)(row - (int64_t)b * p.rows.N);
        const bool turns = unit < turning;
        float c[NP], s[NP];
        int d0, d1;
        if (turns) {
            double pos;
            if (p.positions) pos = p.position_bytes == 8 ? (double)((const int64_t*)p.positions)[row] : (double)((const int32_t*)p.positions)[row];
            else if (p.rows.cu) {
                const int sq = sequence_of(p.rows, n);
                pos = sq < 0 ? 0.0 : (double)place_of(p.rows, sq, n);
            } else pos = (double)n;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                turn(pos, p.frequencies[unit * NP + i], p.amplitude, c[i], s[i]);
                if (p.inverse) s[i] = -s[i];
            }
            d0 = INTERLEAVED ? 2 * NP * unit : V * unit;
            d1 = INTERLEAVED ? d0 + 1 : d0 + p.rot / 2;
        } else {
            d0 = d1 = p.rot + (unit - turning) * V;
        }
        constexpr int AHEAD = 4;                                            // heads with their loads under way together
        const int heads = p.H + p.HK;
        for (int h0 = first; h0 < heads; h0 += AHEAD * sp.share) {
            float x[AHEAD][V], y[ONE ? 1 : AHEAD][V];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int h = h0 + i * sp.share;
                if (h < heads) {
                    const T* src = h < p.H ? (const T*)p.q.p + p.q.off(b, n, h) : (const T*)p.k.p + p.k.off(b, n, h - p.H);
                    load_floats<T, V>(src + d0, x[i]);
                    if constexpr (!ONE)
                        if (turns) load_floats<T, V>(src + d1, y[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int h = h0 + i * sp.share;
                if (h < heads) {
                    T* dst = h < p.H ? (T*)p.q_out.p + p.q_out.off(b, n, h) : (T*)p.k_out.p + p.k_out.off(b, n, h - p.H);
                    if (turns) {
#pragma unroll
                        for (int j = 0; j < NP; ++j) {
                            float& a0 = ONE ? x[i][2 * j % V] : x[i][j];
                            float& a1 = ONE ? x[i][(2 * j + 1) % V] : y[ONE ? 0 : i][j];
                            const float r0 = fmaf(-a1, s[j], a0 * c[j]), r1 = fmaf(a0, s[j], a1 * c[j]);
                            a0 = r0;
                            a1 = r1;
                        }
                    }
                    store_floats<T, V>(dst + d0, x[i]);
                    if constexpr (!ONE)
                        if (turns) store_floats<T, V>(dst + d1, y[i]);
                }
            }
        }
    }
}

template <class T, int V, bool INTERLEAVED>
int launch(const Rotary& p, hipStream_t st) {
    Split sp;
    sp.units = p.rot / 2 / pairs_of<V, INTERLEAVED>() + (p.D - p.rot) / V;
    const int64_t rows = (int64_t)p.rows.B * p.rows.N;
    const int heads = p.H + p.HK;
    // Eight heads per thread where that leaves the chip eight wavefronts per SIMD (16384 rows of 20 heads, half of head_dim 128, interleaved:
    // 37 us, 44 with four), four where it leaves two, one elsewhere
    sp.share = rows * sp.units * ((heads + 7) / 8) >= 8 * 4 * 64 * CUS ? (heads + 7) / 8 : rows * sp.units * ((heads + 3) / 4) >= 2 * 4 * 64 * CUS ? (heads + 3) / 4 : heads;
    const int per_row = sp.units * sp.share;
    sp.rows = per_row >= THREADS ? 1 : THREADS / per_row;
    const int64_t blocks = (rows + sp.rows - 1) / sp.rows;
    if (blocks > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    rotary_kernel<T, V, INTERLEAVED><<<dim3((unsigned)blocks), dim3(THREADS), 0, st>>>(p, sp);
    return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
}

}  // namespace

int launch_rotary(const Rotary& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        constexpr int V = 16 / sizeof(T), S = sizeof(T);
        const bool batched = p.rows.B > 1, k = p.HK > 0;
        // 16-byte chunks where no pair and no copied column straddles one, single elements elsewhere
        const bool wide = p.rot % (p.interleaved ? V : 2 * V) == 0 && p.D % V == 0 && aligned16(p.q, S, batched) && aligned16(p.q_out, S, batched) &&
                          (!k || (aligned16(p.k, S, batched) && aligned16(p.k_out, S, batched)));
        if (p.interleaved) return wide ? launch<T, V, true>(p, st) : launch<T, 1, true>(p, st);
        return wide ? launch<T, V, false>(p, st) : launch<T, 1, false>(p, st);
    });
}

}  // namespace sa2
