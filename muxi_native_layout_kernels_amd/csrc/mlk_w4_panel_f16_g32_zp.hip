// Panels of the 4-bit linear layers: f16 activations, groups of 32 weights, with zero points.
#include "mlk_w4_panel_gemm.cuh"

namespace mlk {
template int w4_launch_panel<F16, 1, true>(const W4PanelArgs &, int, hipStream_t);
}  // namespace mlk
