// Launches of attention of drafted tokens with a window, or with the cached rows' weights, with fp32 products; and the kernel that adds
// up weights.  Sixteen caches of up to 4096 rows, 16 heads over 4 key heads, head_dim 128, bf16: the sweep that leaves its scores 34 us (2.7 TB/s of
// keys and values), weights and join 8.
#include "sa2_tree_f32.h"
#include "sa2_tree_join.h"

namespace sa2 {
namespace {

// weights[b, hk, place of row] += sum over the G query heads of e^(score - lse), from the scores that the sweep left and the reference
// points and sums of its shares.  A workgroup has 1024 rows; every wavefront joins the shares for itself.  The first `joins` workgroups join the
// outputs' rows (in a launch of its own before this one: 5 us more)
// `lift`: sums are 2^lift times as large as their reference points say
template <class T, int W>
__global__ __launch_bounds__(256) void tree_weights_kernel(Tree p, float lift, bool wide, int joins) {
    if ((int)blockIdx.x < joins) {
        tree_join_row<T, W>(p, wide, blockIdx.x);
        return;
    }
    constexpr int EACH = 4;
    const int64_t per = (p.span + 256 * EACH - 1) / (256 * EACH), at = blockIdx.x - joins, stream = at / per;
    const int hk = (int)(stream % p.HK), b = (int)(stream / p.HK), lane = threadIdx.x & 63;
    const TreeRows<true, 32> cache(p, b);
    const int64_t first = (at - stream * per) * 256 * EACH, number = first + threadIdx.x * EACH;
    const int tile = (int)(number / 32), rows = cache.cached * 32;
    if (first > rows) return;                               // (the tile behind the cached ones has the node itself)
    TreeShare share;
    tree_shares_of(p, b, share);
    const float c = fabsf(p.scale) * LOG2E;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < p.G; ++r) {
        const TreePart s = lane < share.count ? *tree_stat(p, share.first + lane, hk, r) : TreePart{-INFINITY, 0.f};
        const float top = wave_max(s.top), f = s.sum == 0.f ? 0.f : s.top == -INFINITY ? 1.f : exp2f((s.top - top) * c), total = wave_sum(f * s.sum);
        if (total == 0.f || number > rows) continue;
        const float4 x = *(const float4*)(p.scores + (stream * p.G + r) * p.span + number);
        const float over = 1.f / total, from = top == -INFINITY ? 0.f : top;
        // (hidden rows and those that are not there have -infinity)
        auto weight = [&](float y) { return y == -INFINITY ? 0.f : exp2f(fmaf(y - from, c, lift)) * over; };
        sum.x += weight(x.x); sum.y += weight(x.y); sum.z += weight(x.z); sum.w += weight(x.w);
    }
    if (number > rows) return;
    const int64_t room = p.cache.table ? (int64_t)p.cache.width * p.cache.page_size : p.cache.page_size;
    const int64_t place = number == rows ? cache.held : cache.row(tile) + number % 32;
    float* const to = p.weights + b * p.weights_sb + hk * p.weights_sh + place;
    const float* const add = &sum.x;
    for (int i = 0; i < EACH; ++i) {
        if (number == rows ? i > 0 || place >= room : place + i >= cache.held) break;
        to[i] += add[i];
    }
}

}  // namespace

int launch_tree_weights(const Tree& p, int dtype, float lift, hipStream_t st) {
    const int64_t joins = (int64_t)p.B * p.HK * p.T * p.G, grid = joins + (int64_t)p.B * p.HK * ((p.span + 1023) / 1024);
    if (grid > 0x7fffffff) return SA2_ERR_TOO_LARGE;
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        const dim3 blocks((unsigned)grid), block(256);
        const bool wide = wide_tree<T>(p);
        if (tree_width(p.D) == 64) tree_weights_kernel<T, 64><<<blocks, block, 0, st>>>(p, lift, wide, (int)joins);
        else if (tree_width(p.D) == 128) tree_weights_kernel<T, 128><<<blocks, block, 0, st>>>(p, lift, wide, (int)joins);
        else tree_weights_kernel<T, 256><<<blocks, block, 0, st>>>(p, lift, wide, (int)joins);
        return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
    });
}

int launch_window_tree_f32(const Tree& p, int dtype, hipStream_t st) {
    const int rc = launch_tree_f32_of<true>(p, dtype, st);
    if (rc != SA2_OK || (p.nsplit == 1 && !p.scores)) return rc;
    return p.scores ? launch_tree_weights(p, dtype, 0.f, st) : launch_tree_join(p, dtype, st);
}

}  // namespace sa2
