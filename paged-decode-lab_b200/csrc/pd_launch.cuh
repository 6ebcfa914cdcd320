// pd_launch.cuh — launches that may start before the kernel ahead of them in the stream has finished.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace pd {

// The kernel waits for its predecessor itself (griddepcontrol.wait).
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), int64_t grid, unsigned threads, size_t smem,
                             cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(grid));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace pd
