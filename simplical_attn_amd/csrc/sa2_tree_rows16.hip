// Launches of large drafted trees on the 16-bit MFMA (sa2_tree_rows16.h).
#include "sa2_tree_rows16.h"

namespace sa2 {

int launch_tree_rows16(const Tree& p, int dtype, hipStream_t st) { return launch_tree_rows16_of<false>(p, dtype, st); }

}  // namespace sa2
