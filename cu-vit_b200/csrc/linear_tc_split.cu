// FP32-faithful linear layers: float operands split into a TF32 head and a TF32 remainder
// (3xTF32, as the GEMM's FP32 mode).
#include "linear_tc_instances.cuh"

namespace cuvit::linear {

int launch_tc_split(const TcPlan& plan, cudaStream_t stream) {
    return plan.block_n == 64 ? launch_instance<4, 64, true>(plan, stream)
                              : launch_instance<4, 128, true>(plan, stream);
}

} // namespace cuvit::linear
