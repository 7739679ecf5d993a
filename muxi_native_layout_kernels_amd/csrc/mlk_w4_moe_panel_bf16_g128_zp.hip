// Panels of the expert layers over 4-bit weights: bf16 activations, groups of 128 weights and more, with zero points.
#include "mlk_w4_moe_panel.cuh"

namespace mlk {
template int w4_launch_moe_panel<BF16, 4, true>(const W4MoeArgs &, const W4MoePlan &, hipStream_t);
}  // namespace mlk
