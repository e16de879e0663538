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

}  // namespace nz
