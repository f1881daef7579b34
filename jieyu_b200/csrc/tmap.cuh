// tmap.cuh — the driver's encoder of tensor maps, found once.
#pragma once
#include "common.cuh"

#include <cuda.h>

#include <atomic>

namespace jyc {

// *fn: cuTensorMapEncodeTiled.
inline int tensor_map_encoder(void** fn) {
    static std::atomic<void*> entry;
    *fn = entry.load(std::memory_order_acquire);
    if (*fn) return JYC_OK;
    cudaDriverEntryPointQueryResult found;
    JYC_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", fn, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !*fn) return cuda_fail(cudaErrorNotSupported, "cuTensorMapEncodeTiled");
    entry.store(*fn, std::memory_order_release);
    return JYC_OK;
}

}  // namespace jyc
