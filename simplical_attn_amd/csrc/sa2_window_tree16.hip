// Launches of attention of drafted tokens with a window, or with the cached rows' weights, on the 16-bit MFMA.  Eight caches of up to
// 32768 rows, window 1024 with 4 first keys, 16 heads over 4, head_dim 128, bf16: 16.5 us with the join, of which the rows take 3 at a copy's rate; the
// rest is the start of a workgroup (length, pages, rows, one after the other) and the second launch.
#include "sa2_tree16.h"

namespace sa2 {

int launch_window_tree16(const Tree& p, int dtype, hipStream_t st) {
    // (the kernel for large trees leaves no scores; a tree of one node is large from 65 query heads per key head on)
    const int rc = tree16_rows(p) > 64 && !p.scores ? launch_window_tree_rows16(p, dtype, st) : launch_tree16_of<true>(p, dtype, st);
    if (rc != SA2_OK || (p.nsplit == 1 && !p.scores)) return rc;
    return p.scores ? launch_tree_weights(p, dtype, dtype == SA2_F16 ? 15.f : 0.f, st) : launch_tree_join(p, dtype, st);
}

}  // namespace sa2
