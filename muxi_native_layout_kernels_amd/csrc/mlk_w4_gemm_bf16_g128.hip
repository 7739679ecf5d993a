// Streaming kernels of the 4-bit linear layers: bf16 activations, groups of 128 weights and more, without zero points.
#include "mlk_w4_gemm.cuh"

namespace mlk {
template int w4_launch_stream<BF16, 4, false>(const W4GemmArgs &, int, int, int, int, hipStream_t);
}  // namespace mlk
