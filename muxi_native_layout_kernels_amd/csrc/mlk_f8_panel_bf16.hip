// The e4m3 panels with bf16 outputs.
#include "mlk_f8_panel.cuh"

namespace mlk {
template int f8_launch_panel<BF16>(const F8PanelArgs &, int, int, hipStream_t);
}
