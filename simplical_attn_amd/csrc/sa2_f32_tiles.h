// Tiles of 32 rows in LDS as fp32, and their products with what a wavefront owns (v_mfma_f32_32x32x2_f32).
#pragma once

#include "sa2_causal_common.h"

namespace sa2 {
namespace {

constexpr int TILE = 32;

__device__ __forceinline__ floatx16 mfma(float a, float b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 zero16() {
    floatx16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// Columns d .. d+3 of a row of D, zeros behind it and where the row is not `there` (`row` can be read all the same: as a branch around
// every load this cost twice the time of the products).  `wide`: rows on the 16-byte grid (fp32) or 8-byte grid, D a multiple of 4
template <class T>
__device__ __forceinline__ float4 load4(const T* row, int d, int D, bool wide, bool there) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (wide) {
        const bool ok = there && d < D;
        const T* from = row + (d < D ? d : 0);
        if constexpr (sizeof(T) == 4) x = *(const float4*)from;
        else {
            union { uint2 u; T e[4]; } w;
            w.u = *(const uint2*)from;
            x = make_float4(to_float(w.e[0]), to_float(w.e[1]), to_float(w.e[2]), to_float(w.e[3]));
        }
        x.x = ok ? x.x : 0.f;
        x.y = ok ? x.y : 0.f;
        x.z = ok ? x.z : 0.f;
        x.w = ok ? x.w : 0.f;
    } else if (there) {
        float* y = &x.x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < D) y[i] = to_float(row[d + i]);
    }
    return x;
}
template <class T>
__device__ __forceinline__ void store4(T* row, int d, int D, bool wide, float4 x) {
    if (wide) {
        if (d < D) {
            if constexpr (sizeof(T) == 4) *(float4*)(row + d) = x;
            else *(uint2*)(row + d) = make_uint2(pack_pair(x.x, x.y, row), pack_pair(x.z, x.w, row));
        }
    } else {
        const float* y = &x.x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < D) from_float(y[i], row + d + i);
    }
}

// LDS rows are four floats longer than the tile's columns: neighbours start in other banks
template <int DP>
struct Pitch { static constexpr int value = DP + 4; };

// The wavefront's own 32 rows as second operand: slot (4c + i, half) holds column 8c + 4 * half + i of row lane % 32
template <class T, int DP>
__device__ __forceinline__ void own_rows(float (&x)[DP / 2], const Tensor& t, const Span& s, int first, int h, int D, bool wide, float factor) {
    const int lane = threadIdx.x & 63, r = first + (lane & 31), half = lane >> 5;
    const T* row = (const T*)t.p + row_offset(t, s, r < s.len ? r : 0, h);
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
        const float4 v = load4(row, 8 * c + 4 * half, D, wide, r < s.len);
        x[4 * c] = v.x * factor; x[4 * c + 1] = v.y * factor; x[4 * c + 2] = v.z * factor; x[4 * c + 3] = v.w * factor;
    }
}
// [tile rows] x [own rows]: rows of the tile in the registers, own ones in the lanes
template <int DP>
__device__ __forceinline__ floatx16 tile_product(const float* lds, const float (&own)[DP / 2]) {
    const int lane = threadIdx.x & 63;
    const float* row = lds + (lane & 31) * Pitch<DP>::value + 4 * (lane >> 5);
    floatx16 s = zero16();
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
        const float4 a = *(const float4*)(row + 8 * c);
        s = mfma(a.x, own[4 * c], s);
        s = mfma(a.y, own[4 * c + 1], s);
        s = mfma(a.z, own[4 * c + 2], s);
        s = mfma(a.w, own[4 * c + 3], s);
    }
    return s;
}
// acc[columns] += (tile columns first .. first + DO)^T x w, w the weights of (tile row, own row).  visible(row): whether the
// lane's own row sees that row of the tile.  With GUARD, tile rows that hold an infinity or NaN are added one by one to the
// rows that see them only: a weight of zero would not keep them out.
template <int DP, int DO, bool GUARD, class F>
__device__ __forceinline__ void weighted_rows(const float* lds, int first, const floatx16& w, floatx16 (&acc)[DO / 32], F&& visible) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float* row = lds + (8 * g + 4 * half + r) * Pitch<DP>::value + first + (lane & 31);
            float a[DO / 32];
            bool odd = false;
#pragma unroll
            for (int b = 0; b < DO / 32; ++b) {
                a[b] = row[32 * b];
                if (GUARD) odd = odd || !is_finite(a[b]);
            }
            const float p = w[4 * g + r];
            if (GUARD && __any(odd)) {
#pragma unroll 1
                for (int hh = 0; hh < 2; ++hh) {
                    const bool sees = visible(8 * g + 4 * hh + r);
#pragma unroll
                    for (int b = 0; b < DO / 32; ++b) {
                        const floatx16 one = mfma(half == hh ? a[b] : 0.f, half == hh ? p : 0.f, zero16());
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[b][i] = sees ? acc[b][i] + one[i] : acc[b][i];
                    }
                }
            } else {
#pragma unroll
                for (int b = 0; b < DO / 32; ++b) acc[b] = mfma(a[b], p, acc[b]);
            }
        }
}
template <class F>
int for_width(int D, F&& f) {
    if (D <= 32) return f(std::integral_constant<int, 32>{});
    if (D <= 64) return f(std::integral_constant<int, 64>{});
    if (D <= 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

}  // namespace
}  // namespace sa2
