// Launches of causal attention with fp32 products, head_dim up to 128 (sa2_causal_f32_narrow.h).
#include "sa2_causal_f32_narrow.h"

namespace sa2 {

int launch_causal_f32_narrow_fwd(const Causal& p, int dtype, bool wide, hipStream_t st) { return narrow_forward<false>(p, dtype, wide, st); }
int launch_causal_f32_narrow_bwd(const Causal& p, int dtype, bool wide, hipStream_t st) { return narrow_backward<false>(p, dtype, wide, st); }

}  // namespace sa2
