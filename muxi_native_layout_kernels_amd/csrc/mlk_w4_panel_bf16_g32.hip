// Panels of the 4-bit linear layers: bf16 activations, groups of 32 weights, without zero points.
#include "mlk_w4_panel_gemm.cuh"

namespace mlk {
template int w4_launch_panel<BF16, 1, false>(const W4PanelArgs &, int, hipStream_t);
}  // namespace mlk
