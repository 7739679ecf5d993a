// Panels of the expert layers over 4-bit weights: f16 activations, groups of 64 weights, without zero points.
#include "mlk_w4_moe_panel.cuh"

namespace mlk {
template int w4_launch_moe_panel<F16, 2, false>(const W4MoeArgs &, const W4MoePlan &, hipStream_t);
}  // namespace mlk
