// Linear layers with bfloat16 operands: the one-CTA kernel, and CTA pairs for large ones.
#include "gemm_tc_pair.cuh"
#include "linear_tc_instances.cuh"

namespace cuvit::linear {
namespace {

constexpr int kMaxDevices = 64;

int launch_pair(const TcPlan& plan, cudaStream_t stream) {
    using Shape = gemm::PairShape<256>;
    auto* kernel = &gemm::tc_gemm_pair_kernel<256, gemm::LinearParams>;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(plan.grid));
    config.blockDim = dim3(Shape::kThreads);
    config.dynamicSmemBytes = Shape::kSmemBytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = 2;
    attributes[0].val.clusterDim.y = 1;
    attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attributes;
    config.numAttrs = host::pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&config, kernel, plan.map_x, plan.map_w, plan.map_out, plan.params);
    return host::after_launch("linear tc_gemm_pair_kernel");
}

} // namespace

int pair_resident(int* pairs) {
    static int resident[kMaxDevices] = {};
    using Shape = gemm::PairShape<256>;
    auto* kernel = &gemm::tc_gemm_pair_kernel<256, gemm::LinearParams>;
    int device = 0;
    CUVIT_TRY_CUDA(cudaGetDevice(&device));
    if (device < 0 || device >= kMaxDevices) {
        return host::fail(CUVIT_UNSUPPORTED, "device ordinal out of range");
    }
    CUVIT_TRY_CUDA(host::once_per_device(
        reinterpret_cast<const void*>(kernel), [&](int current) {
            const cudaError_t error = cudaFuncSetAttribute(
                kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmemBytes);
            if (error != cudaSuccess) {
                return error;
            }
            cudaLaunchAttribute attribute{};
            attribute.id = cudaLaunchAttributeClusterDimension;
            attribute.val.clusterDim.x = 2;
            attribute.val.clusterDim.y = 1;
            attribute.val.clusterDim.z = 1;
            cudaLaunchConfig_t probe{};
            probe.gridDim = dim3(2, 1, 1);
            probe.blockDim = dim3(Shape::kThreads, 1, 1);
            probe.dynamicSmemBytes = Shape::kSmemBytes;
            probe.attrs = &attribute;
            probe.numAttrs = 1;
            return cudaOccupancyMaxActiveClusters(&resident[current], kernel, &probe);
        }));
    if (resident[device] < 1) {
        return host::fail(CUVIT_RUNTIME_ERROR,
                          "no CTA pair of the linear kernel fits on this device");
    }
    *pairs = resident[device];
    return CUVIT_OK;
}

int launch_tc_bf16(const TcPlan& plan, cudaStream_t stream) {
    if (plan.pair) {
        return launch_pair(plan, stream);
    }
    switch (plan.block_n) {
    case 64:
        return launch_instance<2, 64>(plan, stream);
    case 128:
        return launch_instance<2, 128>(plan, stream);
    default:
        return launch_instance<2, 256>(plan, stream);
    }
}

} // namespace cuvit::linear
