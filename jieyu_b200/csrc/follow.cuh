// follow.cuh — launches that start as the stream's last kernel ends (programmatic stream serialization).
#pragma once
#include "common.cuh"

namespace jyc {

// A launch that may start before the last one has ended, for which it waits by itself (griddep_wait, in every thread).
template <class... Params, class... Args>
int launch_follow(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    JYC_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    JYC_LAUNCHED();
    return JYC_OK;
}

}  // namespace jyc
