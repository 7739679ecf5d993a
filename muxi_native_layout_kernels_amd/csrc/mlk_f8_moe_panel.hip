// The expert layers' panels in e4m3, with fp16 and bf16 outputs.
#include "mlk_f8_moe_panel.cuh"

namespace mlk {
template int f8_launch_moe_panels<F16>(const F8MoeArgs &, int, hipStream_t);
template int f8_launch_moe_panels<BF16>(const F8MoeArgs &, int, hipStream_t);
}
