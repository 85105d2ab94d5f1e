// The join of the shares of a tree's attention.
#pragma once

#include "sa2_tree_common.h"

namespace sa2 {
namespace {

// Partial results of the splits.  A workgroup of 256 threads has one row: W / 4 threads its columns, 1024 / W groups of them the splits in turn, all
// of whose values are under way together (one after the other, by the thread that adds them, 64 splits took 45 us); the groups
// are added in order.
template <class T, int W>
__device__ __forceinline__ void tree_join_row(const Tree& p, bool wide, int64_t row) {
    constexpr int GROUPS = 1024 / W, EACH = 64 / GROUPS;      // at most 64 splits
    __shared__ float4 sums[GROUPS][W / 4];
    const int64_t R = p.T * p.G, stream = row / R;
    const int hk = (int)(stream % p.HK), b = (int)(stream / p.HK);
    TreeShare share;
    tree_shares_of(p, b, share);
    const int r = (int)(row - stream * R), lane = threadIdx.x & 63, group = threadIdx.x / (W / 4), d = threadIdx.x % (W / 4) * 4;
    const float c = fabsf(p.scale) * LOG2E;
    float4 y[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int split = i * GROUPS + group;
        y[i] = split < share.count ? *(const float4*)(tree_values(p, share.first + split, hk, r, W) + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const TreePart s = lane < share.count ? *tree_stat(p, share.first + lane, hk, r) : TreePart{-INFINITY, 0.f};
    const float top = wave_max(s.top), f = s.sum == 0.f ? 0.f : s.top == -INFINITY ? 1.f : exp2f((s.top - top) * c), sum = wave_sum(f * s.sum);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const float g = __shfl(f, i * GROUPS + group);
        o.x += g * y[i].x; o.y += g * y[i].y; o.z += g * y[i].z; o.w += g * y[i].w;
    }
    sums[group][d / 4] = o;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
        const float4 z = sums[i][d / 4];
        o.x += z.x; o.y += z.y; o.z += z.z; o.w += z.w;
    }
    const float g = sum == 0.f ? 0.f : 1.f / sum;
    store4((T*)p.out.p + p.out.off(b, r / p.G, hk * p.G + r % p.G), d, p.D, wide, make_float4(o.x * g, o.y * g, o.z * g, o.w * g));
}

}  // namespace
}  // namespace sa2
