// Launches of attention of drafted tokens on the 16-bit MFMA (sa2_tree16.h, large trees: sa2_tree_rows16.h).
#include "sa2_tree16.h"

namespace sa2 {

// 16-byte rows
bool tree16_layout(const Tree& p, int dtype) {
    if (dtype == SA2_F32 || p.D % 8 || p.D > 128) return false;
    for (const Tensor* t : {&p.q, &p.k, &p.v, &p.cache.k, &p.cache.v, &p.out})
        if (!aligned16(*t, 2, true) || t->sn >= 1 << 22) return false;     // (a group's rows within 2^31 bytes of its first)
    return true;
}
// and a share of the page table that fits LDS
bool tree16_supported(const Tree& p, int dtype) {
    if (!tree16_layout(p, dtype)) return false;
    // (of nsplit shares for each, a sequence has at least nsplit - 1 where they are dealt and its cache is full)
    const int shares = p.nsplit > 1 ? p.nsplit - 1 : 1;
    return !p.cache.table || (p.cache.width + shares - 1) / shares + 256 / p.cache.page_size + 3 <= TREE16_ENTRIES;
}

int launch_tree16(const Tree& p, int dtype, hipStream_t st) {
    const int rc = tree16_rows(p) > 64 ? launch_tree_rows16(p, dtype, st) : launch_tree16_of<false>(p, dtype, st);
    return rc == SA2_OK && p.nsplit > 1 ? launch_tree_join(p, dtype, st) : rc;
}

}  // namespace sa2
