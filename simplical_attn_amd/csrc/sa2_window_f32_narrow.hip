// Launches of windowed attention with fp32 products, head_dim up to 128 (sa2_causal_f32_narrow.h).
#include "sa2_causal_f32_narrow.h"

namespace sa2 {

int launch_window_f32_narrow_fwd(const Causal& p, int dtype, bool wide, hipStream_t st) { return narrow_forward<true>(p, dtype, wide, st); }
int launch_window_f32_narrow_bwd(const Causal& p, int dtype, bool wide, hipStream_t st) { return narrow_backward<true>(p, dtype, wide, st); }

}  // namespace sa2
