// Launches of large drafted trees with a window on the 16-bit MFMA (sa2_tree_rows16.h): work and bounds are those of the kernel without a window, over the tiles in reach.
#include "sa2_tree_rows16.h"

namespace sa2 {

int launch_window_tree_rows16(const Tree& p, int dtype, hipStream_t st) { return launch_tree_rows16_of<true>(p, dtype, st); }

}  // namespace sa2
