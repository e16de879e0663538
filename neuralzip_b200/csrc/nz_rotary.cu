// Rotary positions (after an optional norm of each head) and the write into
// the paged cache, in one pass over the projections' outputs.
//
//   x' = x * w / sqrt(mean(x^2) + eps)                      (with a norm)
//   (a, b) -> (a cos - b sin, b cos + a sin)                (each rotated pair)
// in 32 bits, rounded once to the stored type. Every element is read once
// and written once (queries to query_out, keys and values to their slots),
// so prompts are bound by HBM and a step's few rows by the launch and one
// load latency.
//
// A row of one head is held by a group of 1 to 32 lanes; a lane owns the
// same VEC elements of both halves of a pair range, so that a rotation
// needs no exchange and the norm's sum is a shuffle inside the group.

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

template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Vec {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load(const T* p) {
    return *reinterpret_cast<const Vec<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const Vec<T, VEC>& x) {
    *reinterpret_cast<Vec<T, VEC>*>(p) = x;
}

__device__ __forceinline__ void turn(float& a, float& b, float cosine, float sine) {
    const float u = a * cosine - b * sine;
    b = b * cosine + a * sine;
    a = u;
}

constexpr uint32_t kThreads = 256;

// CHUNKS: pair chunks of VEC a lane owns; group_log: lanes of a group.
template <typename T, int VEC, int CHUNKS>
__global__ void __launch_bounds__(kThreads) nz_rotary_kernel(const nz_rotary a, uint32_t group_log) {
    const uint32_t group = 1U << group_log, lane = threadIdx.x & (group - 1U);
    const uint32_t all = a.heads + 2U * a.kv_heads;
    const uint32_t unit = (blockIdx.x << (8U - group_log)) + (threadIdx.x >> group_log);
    const bool live = unit < a.tokens * all;
    const uint32_t token = live ? unit / all : 0U;
    const uint32_t row = live ? unit - token * all : 0U;
    const bool is_query = row < a.heads, is_key = !is_query && row < a.heads + a.kv_heads;
    const uint32_t head = is_query ? row : is_key ? row - a.heads : row - a.heads - a.kv_heads;
    const uint32_t half = a.dim / 2, turned = a.rot / 2;

    const T* source = is_query ? nz::device_ptr<const T>(a.query) + token * a.query_stride[0] + head * a.query_stride[1]
                      : is_key ? nz::device_ptr<const T>(a.key) + token * a.key_stride[0] + head * a.key_stride[1]
                               : nz::device_ptr<const T>(a.value) + token * a.value_stride[0] + head * a.value_stride[1];
    // Where the two vectors of each chunk lie in the row.
    uint32_t at[CHUNKS][2];
    bool have[CHUNKS];
    Vec<T, VEC> x[CHUNKS][2];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t pair = (c * group + lane) * VEC;
        have[c] = live && pair < half;
        if (pair >= turned) {
            at[c][0] = turned + pair;
            at[c][1] = half + pair;
        } else if (a.interleaved) {
            at[c][0] = 2U * pair;
            at[c][1] = 2U * pair + VEC;
        } else {
            at[c][0] = pair;
            at[c][1] = turned + pair;
        }
        if (have[c]) {
            x[c][0] = load<T, VEC>(source + at[c][0]);
            x[c][1] = load<T, VEC>(source + at[c][1]);
        }
    }
    int32_t slot = -1;
    if (live && !is_query) slot = nz::device_ptr<const int32_t>(a.slots)[token];
    const int32_t page = slot >> a.page_shift;
    const bool cached = slot >= 0 && static_cast<uint32_t>(page) < a.pages;
    const uint32_t line = static_cast<uint32_t>(slot) & ((1U << a.page_shift) - 1U);

    if (is_query || is_key) {
        const T* weight = nz::device_ptr<const T>(is_query ? a.query_norm : a.key_norm);
        float f[CHUNKS][2 * VEC];
        float squares = 0.0f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int i = 0; i < 2 * VEC; ++i) {
                f[c][i] = have[c] ? to_float(x[c][i / VEC].v[i % VEC]) : 0.0f;
                squares += f[c][i] * f[c][i];
            }
        if (a.query_norm || a.key_norm) {
            // A group's lanes hold one row, so they are all here.
            const uint32_t mask = (0xFFFFFFFFU >> (32U - group)) << (threadIdx.x & 31U & ~(group - 1U));
            for (uint32_t d = 1; d < group; d <<= 1) squares += __shfl_xor_sync(mask, squares, d);
        }
        if (weight) {
            const float scale = 1.0f / sqrtf(squares / static_cast<float>(a.dim) + a.eps);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                if (!have[c]) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Vec<T, VEC> w = load<T, VEC>(weight + at[c][h]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[c][h * VEC + i] *= scale * to_float(w.v[i]);
                }
            }
        }
        const int32_t position = live ? nz::device_ptr<const int32_t>(a.positions)[token] : 0;
        const bool known = position >= 0 && static_cast<uint32_t>(position) < a.table_rows;
        const float* angles = nz::device_ptr<const float>(a.table) + (known ? position : 0) * a.table_stride;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t pair = (c * group + lane) * VEC;
            if (have[c] && pair < turned) {
                Vec<float, VEC> cosine, sine;
                if (known) {
                    cosine = load<float, VEC>(angles + pair);
                    sine = load<float, VEC>(angles + turned + pair);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) cosine.v[i] = sine.v[i] = __int_as_float(0x7FFFFFFF);
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    if (a.interleaved)
                        turn(f[c][2 * i], f[c][2 * i + 1], cosine.v[i], sine.v[i]);
                    else
                        turn(f[c][i], f[c][VEC + i], cosine.v[i], sine.v[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * VEC; ++i) x[c][i / VEC].v[i % VEC] = from_float<T>(f[c][i]);
        }
    }

    T* targets[2] = {nullptr, nullptr};
    if (is_query) {
        targets[0] = nz::device_ptr<T>(a.query_out) + token * a.query_out_stride[0] + head * a.query_out_stride[1];
    } else if (is_key) {
        if (a.key_out) targets[0] = nz::device_ptr<T>(a.key_out) + token * a.key_out_stride[0] + head * a.key_out_stride[1];
        if (cached)
            targets[1] = nz::device_ptr<T>(a.key_pages) + page * a.key_pages_stride[0] + line * a.key_pages_stride[1] +
                         head * a.key_pages_stride[2];
    } else if (cached) {
        targets[1] = nz::device_ptr<T>(a.value_pages) + page * a.value_pages_stride[0] +
                     line * a.value_pages_stride[1] + head * a.value_pages_stride[2];
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if (!targets[t]) continue;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            if (!have[c]) continue;
            store<T, VEC>(targets[t] + at[c][0], x[c][0]);
            store<T, VEC>(targets[t] + at[c][1], x[c][1]);
        }
    }
}

template <typename T, int VEC, int CHUNKS>
cudaError_t launch(const nz_rotary& a, cudaStream_t stream) {
    const uint32_t chunks = (a.dim / 2 + VEC - 1) / VEC;
    uint32_t group_log = 0;
    while ((1U << group_log) * CHUNKS < chunks) ++group_log;
    const uint64_t threads = (static_cast<uint64_t>(a.tokens) * (a.heads + 2U * a.kv_heads)) << group_log;
    const uint32_t blocks = static_cast<uint32_t>((threads + kThreads - 1) / kThreads);
    nz_rotary_kernel<T, VEC, CHUNKS><<<blocks, kThreads, 0, stream>>>(a, group_log);
    return cudaGetLastError();
}

// The widest vector that divides both kinds of pair chunks and every
// address: 8 elements (16 bytes of 16-bit types) for the usual head widths,
// less for odd rotations or strides.
bool vector_fits(const nz_rotary& a, uint32_t vec, uint32_t size) {
    if ((a.rot / 2) % vec || ((a.dim - a.rot) / 2) % vec) return false;
    const uint32_t bytes = vec * size < 16 ? vec * size : 16;
    uint64_t bits = a.query | a.key | a.value | a.query_out | a.key_out | a.key_pages | a.value_pages | a.query_norm |
                    a.key_norm;
    int64_t strides = 0;
    for (int i = 0; i < 2; ++i)
        strides |= a.query_stride[i] | a.key_stride[i] | a.value_stride[i] | a.query_out_stride[i] |
                   (a.key_out ? a.key_out_stride[i] : 0);
    for (int i = 0; i < 3; ++i) strides |= a.key_pages_stride[i] | a.value_pages_stride[i];
    bits |= static_cast<uint64_t>(strides) * size;
    const uint32_t float_bytes = vec * 4 < 16 ? vec * 4 : 16;
    const uint64_t table = a.table | static_cast<uint64_t>(a.table_stride) * 4 | static_cast<uint64_t>(a.rot / 2) * 4;
    return bits % bytes == 0 && table % float_bytes == 0;
}

template <typename T>
cudaError_t launch_type(const nz_rotary& a, cudaStream_t stream) {
    if (vector_fits(a, 8, sizeof(T))) return launch<T, 8, 1>(a, stream);
    if (vector_fits(a, 4, sizeof(T))) return launch<T, 4, 1>(a, stream);
    if (vector_fits(a, 2, sizeof(T))) return launch<T, 2, 2>(a, stream);
    return launch<T, 1, 4>(a, stream);
}

}  // namespace

extern "C" int nz_rotary_store(const nz_rotary* args, void* cuda_stream) {
    if (!args) return nz::paged_fail("Null arguments.");
    const nz_rotary& a = *args;
    if (a.dim == 0 || a.dim > NZ_PAGED_MAX_DIM || a.dim % 2 || a.rot > a.dim || a.rot % 2)
        return nz::paged_fail("The head width must be even and at most 256, the rotated part even and no wider.");
    if (!nz::paged_sizes_fit(a.pages, 0, a.page_shift))
        return nz::paged_fail("A cache holds fewer than 2^30 pages and 2^31 tokens.");
    if (a.heads > 65536 || a.kv_heads > 65536 ||
        static_cast<uint64_t>(a.tokens) * (a.heads + 2ULL * a.kv_heads) > INT32_MAX)
        return nz::paged_fail("At most 65536 heads and 2^31 - 1 rows of a head.");
    if (a.tokens == 0 || a.heads + a.kv_heads == 0) return NZ_OK;
    if ((a.heads && (!a.query || !a.query_out)) || (a.kv_heads && (!a.key || !a.value)) || !a.positions || !a.slots ||
        (a.rot && a.table_rows && !a.table) || (a.pages && a.kv_heads && (!a.key_pages || !a.value_pages)))
        return nz::paged_fail("Null device array.");
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(cuda_stream);
    cudaError_t err;
    switch (a.dtype) {
        case NZ_PAGED_BF16: err = launch_type<__nv_bfloat16>(a, stream); break;
        case NZ_PAGED_FP16: err = launch_type<__half>(a, stream); break;
        case NZ_PAGED_FP32: err = launch_type<float>(a, stream); break;
        default: return nz::paged_fail("The type must be bf16, fp16 or fp32.");
    }
    return nz::cuda_status(err, "nz_rotary_store");
}
