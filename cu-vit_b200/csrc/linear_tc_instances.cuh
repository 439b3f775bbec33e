// Shared body of the per-type launchers of linear layers: raises the instance's dynamic shared
// memory limit (once per device) and launches it.
#pragma once

#include "linear.hpp"

namespace cuvit::linear {

template <int ElemBytes, int BN>
int launch_instance(const TcPlan& plan, cudaStream_t stream) {
    using Shape = gemm::TcShape<ElemBytes, BN, false>;
    auto* kernel = &gemm::tc_gemm_kernel<ElemBytes, BN, false, false, gemm::LinearParams>;
    CUVIT_TRY_CUDA(host::allow_dynamic_smem(reinterpret_cast<const void*>(kernel),
                                            Shape::kSmemBytes));
    host::pdl_launch(kernel, dim3(static_cast<unsigned>(plan.grid)), dim3(Shape::kThreads),
                     Shape::kSmemBytes, stream, plan.map_x, plan.map_w, plan.map_out, plan.params);
    return host::after_launch("linear tc_gemm_kernel");
}

} // namespace cuvit::linear
