// What the paged-cache kernels share.
#pragma once

#include "nz_b200.h"
#include "nz_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

namespace nz {

inline int cuda_status(cudaError_t err, const char* what) {
    if (err == cudaSuccess) return NZ_OK;
    NZ_GUARD(throw Error(NZ_ECUDA, std::string(what) + ": " + cudaGetErrorString(err)))
}

// Message failures of the paged entry points, which must not throw.
inline int paged_fail(const char* message) { NZ_GUARD(throw Error(NZ_EVALUE, message)) }

template <typename T>
__host__ __device__ __forceinline__ T* device_ptr(uint64_t address) {
    return reinterpret_cast<T*>(address);
}

// Page ids, slots and positions are 32-bit; pages are at most 2^20 tokens.
inline bool paged_sizes_fit(uint32_t pages, uint32_t width, uint32_t page_shift) {
    return page_shift <= 20 && pages < (1U << 30) && width < (1U << 30) &&
           (static_cast<uint64_t>(pages) << page_shift) <= INT32_MAX &&
           (static_cast<uint64_t>(width) << page_shift) <= INT32_MAX;
}

// The paged kernels are launched as programmatic dependents of what the
// stream holds before them: their CTAs may come onto the GPU while the kernel
// before ends, and wait here, all of them and before any access to memory,
// until it has and its results are there; then the next kernel's may come
// (let_next; else when this one ends).
// Saves 0.3 us a kernel (a step's rotary and attention on 8 requests of 384
// tokens, with the product behind them: 18.2 us a layer, 18.8 without).
__device__ __forceinline__ void after_predecessor(bool let_next = true) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (let_next) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// A launch configuration with that attribute and, from 2 on, a cluster size.
struct PagedLaunch {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attributes[2] = {};

    PagedLaunch(uint32_t grid_x, uint32_t grid_y, uint32_t threads, size_t shared, cudaStream_t stream, uint32_t cluster) {
        config.gridDim = dim3(grid_x, grid_y);
        config.blockDim = dim3(threads);
        config.dynamicSmemBytes = shared;
        config.stream = stream;
        attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[0].val.programmaticStreamSerializationAllowed = 1;
        attributes[1].id = cudaLaunchAttributeClusterDimension;
        attributes[1].val.clusterDim.x = cluster;
        attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
        config.attrs = attributes;
        config.numAttrs = cluster > 1 ? 2 : 1;
    }
    PagedLaunch(const PagedLaunch&) = delete;
};

}  // namespace nz
