// launch.cuh -- kernel launches that may begin while the kernel before them in the stream still runs.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace nfx {

// A launch in clusters of `cluster` blocks that may begin while the kernel before it in the stream still runs: up to
// grid_dep_wait() the kernel touches nothing that another one writes.
template <typename... P, typename... A>
cudaError_t launch_early(void (*kern)(P...), int64_t grid, int threads, int smem, int cluster, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

}  // namespace nfx
