// Streaming kernels of the 4-bit linear layers: f16 activations, groups of 64 weights, with zero points.
#include "mlk_w4_gemm.cuh"

namespace mlk {
template int w4_launch_stream<F16, 2, true>(const W4GemmArgs &, int, int, int, int, hipStream_t);
}  // namespace mlk
