// Launches of attention of drafted tokens with fp32 products (sa2_tree_f32.h), and the kernel that joins partial results.
#include "sa2_tree_f32.h"
#include "sa2_tree_join.h"

namespace sa2 {
namespace {

template <class T, int W>
__global__ __launch_bounds__(256) void tree_join_kernel(Tree p, bool wide) {
    tree_join_row<T, W>(p, wide, blockIdx.x);
}

}  // namespace

int launch_tree_join(const Tree& p, int dtype, hipStream_t st) {
    return for_type(dtype, [&](auto* e) {
        using T = std::remove_pointer_t<decltype(e)>;
        const dim3 grid((unsigned)((int64_t)p.B * p.HK * p.T * p.G));
        const bool wide = wide_tree<T>(p);
        if (tree_width(p.D) == 64) tree_join_kernel<T, 64><<<grid, dim3(256), 0, st>>>(p, wide);
        else if (tree_width(p.D) == 128) tree_join_kernel<T, 128><<<grid, dim3(256), 0, st>>>(p, wide);
        else tree_join_kernel<T, 256><<<grid, dim3(256), 0, st>>>(p, wide);
        return hipGetLastError() == hipSuccess ? SA2_OK : SA2_ERR_LAUNCH_FAILED;
    });
}

int launch_tree_f32(const Tree& p, int dtype, hipStream_t st) {
    const int rc = launch_tree_f32_of<false>(p, dtype, st);
    return rc == SA2_OK && p.nsplit > 1 ? launch_tree_join(p, dtype, st) : rc;
}

}  // namespace sa2
