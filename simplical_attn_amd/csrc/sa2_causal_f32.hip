// Launches of causal attention with fp32 products (sa2_causal_f32.h).
#include "sa2_causal_f32.h"

namespace sa2 {

int launch_causal_f32_fwd(const Causal& p, int dtype, hipStream_t st) { return f32_forward<false>(p, dtype, st); }
int launch_causal_f32_bwd(const Causal& p, int dtype, hipStream_t st) { return f32_backward<false>(p, dtype, st); }

}  // namespace sa2
