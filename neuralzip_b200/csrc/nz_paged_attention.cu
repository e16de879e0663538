// Attention of one new token a request over its pages of the cache.
//
// For request b with n tokens, key/value head k and a query head h of its
// group: s_j = scale * q_h . K_j over the live positions j, out = sum_j
// exp(s_j - max s) V_j / sum_j exp(s_j - max s), the maximum and the sum
// kept running in 32 bits so that keys and values are read once.

#include "nz_paged.h"

namespace {

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_float(float x) { return x; }

constexpr int kWarps = 8;
constexpr int kPerLane = NZ_PAGED_MAX_DIM / 32;

// One CTA a (request, query head); a warp takes every eighth position, a
// lane the elements lane, lane + 32, ... of the head.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) nz_paged_attention_kernel(const nz_attention a) {
    __shared__ float sums[kWarps][NZ_PAGED_MAX_DIM];
    __shared__ float most[kWarps], total[kWarps];
    const uint32_t b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, k = h / (a.heads / a.kv_heads);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31U;
    const uint32_t mask = (1U << a.page_shift) - 1U;
    const int32_t length = max(0, min(nz::device_ptr<const int32_t>(a.lengths)[b],
                                      static_cast<int32_t>(a.width << a.page_shift)));
    const int32_t start = a.window && length > static_cast<int64_t>(a.window) ? length - static_cast<int32_t>(a.window) : 0;
    const int32_t* table = nz::device_ptr<const int32_t>(a.block_table) + b * a.table_stride;
    const T* query = nz::device_ptr<const T>(a.query) + b * a.query_stride[0] + h * a.query_stride[1];
    float q[kPerLane], o[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        q[i] = i * 32 + lane < a.dim ? to_float(query[i * 32 + lane]) * a.scale : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int32_t j = start + static_cast<int32_t>(warp); j < length; j += kWarps) {
        const int32_t page = table[j >> a.page_shift];
        if (page < 0 || static_cast<uint32_t>(page) >= a.pages) continue;
        const int64_t line = j & mask;
        const T* key = nz::device_ptr<const T>(a.key_pages) + page * a.key_stride[0] + line * a.key_stride[1] + k * a.key_stride[2];
        const T* value = nz::device_ptr<const T>(a.value_pages) + page * a.value_stride[0] + line * a.value_stride[1] + k * a.value_stride[2];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (i * 32 + lane < a.dim) s += q[i] * to_float(key[i * 32 + lane]);
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFU, s, d);
        const float next = fmaxf(m, s);
        const float old = m == -INFINITY ? 0.0f : expf(m - next), p = expf(s - next);
        m = next;
        l = l * old + p;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (i * 32 + lane < a.dim) o[i] = o[i] * old + p * to_float(value[i * 32 + lane]);
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) sums[warp][i * 32 + lane] = o[i];
    if (lane == 0) {
        most[warp] = m;
        total[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY, all = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, most[w]);
    for (int w = 0; w < kWarps; ++w)
        if (most[w] != -INFINITY) all += total[w] * expf(most[w] - top);
    T* out = nz::device_ptr<T>(a.out) + b * a.out_stride[0] + h * a.out_stride[1];
    for (uint32_t d = threadIdx.x; d < a.dim; d += blockDim.x) {
        float sum = 0.0f;
        for (int w = 0; w < kWarps; ++w)
            if (most[w] != -INFINITY) sum += sums[w][d] * expf(most[w] - top);
        out[d] = from_float<T>(all > 0.0f ? sum / all : 0.0f);
    }
    if (a.lse && threadIdx.x == 0)
        nz::device_ptr<float>(a.lse)[static_cast<uint64_t>(b) * a.heads + h] = all > 0.0f ? top + logf(all) : -INFINITY;
}

}  // namespace

extern "C" {

int nz_paged_attention_workspace(uint32_t requests, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t dtype,
                                 uint64_t* bytes) {
    (void)requests, (void)heads, (void)kv_heads, (void)dim, (void)dtype;
    if (!bytes) return nz::paged_fail("Null output.");
    *bytes = 0;
    return NZ_OK;
}

int nz_paged_attention(const nz_attention* args, void* cuda_stream) {
    if (!args) return nz::paged_fail("Null arguments.");
    const nz_attention& a = *args;
    if (a.dim == 0 || a.dim > NZ_PAGED_MAX_DIM || a.dim % 8)
        return nz::paged_fail("The head width must be a multiple of 8 up to 256.");
    if (a.kv_heads == 0 || a.heads == 0 || a.heads % a.kv_heads || a.heads > 65536)
        return nz::paged_fail("The query heads must be a multiple of the key/value heads.");
    if (a.requests > NZ_PAGED_MAX_REQUESTS) return nz::paged_fail("At most 4096 requests.");
    if (!nz::paged_sizes_fit(a.pages, a.width, a.page_shift))
        return nz::paged_fail("A cache and a block-table row hold fewer than 2^30 pages and 2^31 tokens.");
    if (a.requests == 0) return NZ_OK;
    if (!a.query || !a.out || !a.lengths || (a.width && !a.block_table) || (a.pages && (!a.key_pages || !a.value_pages)))
        return nz::paged_fail("Null device array.");
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(cuda_stream);
    const uint32_t grid = a.requests * a.heads;
    switch (a.dtype) {
        case NZ_PAGED_BF16: nz_paged_attention_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, stream>>>(a); break;
        case NZ_PAGED_FP16: nz_paged_attention_kernel<__half><<<grid, kWarps * 32, 0, stream>>>(a); break;
        case NZ_PAGED_FP32: nz_paged_attention_kernel<float><<<grid, kWarps * 32, 0, stream>>>(a); break;
        default: return nz::paged_fail("The type must be bf16, fp16 or fp32.");
    }
    return nz::cuda_status(cudaGetLastError(), "nz_paged_attention");
}

}  // extern "C"
