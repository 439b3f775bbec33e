// Linear layers with float operands read as TF32 (one pass).
#include "linear_tc_instances.cuh"

namespace cuvit::linear {

int launch_tc_tf32(const TcPlan& plan, cudaStream_t stream) {
    switch (plan.block_n) {
    case 64:
        return launch_instance<4, 64>(plan, stream);
    case 128:
        return launch_instance<4, 128>(plan, stream);
    default:
        return launch_instance<4, 256>(plan, stream);
    }
}

} // namespace cuvit::linear
