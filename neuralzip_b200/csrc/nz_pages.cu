// Page bookkeeping of the paged key-value cache: block tables, positions and
// slots from request lengths, on the GPU, so that a captured generation step
// can cross page borders without the host.
//
// For request b with n_b cached and m_b new tokens and pages of P tokens:
//   need_b = ceil((n_b + m_b) / P) - ceil(n_b / P)
//   page j of the request (j >= ceil(n_b / P)) = free[used + sum_{a<b} need_a + j - ceil(n_b / P)]
//   token i of the request: position n_b + i, slot page(position / P) * P + position % P
// A few integers a request and 8 bytes a row: the call is bound by its
// launch and by the latency of a load, two block scans and a store (a step
// of 64 requests), or by the stores of 8 bytes a row (prompts).
//
// One cluster does all of it: every CTA scans all requests for itself (at
// most 4096, 16 KB of loads that hit L2) and then writes its share of the
// rows; a cluster barrier separates the last read of lengths and of the
// stack's top from their update, so both may be updated in place without a
// second launch or a scratch counter.

#include "nz_paged.h"

namespace {

constexpr uint32_t kMostCtas = 8;           // portable cluster size
constexpr uint32_t kSaturated = 1U << 30;   // sums stop here: above every legal row and page count

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kSaturated); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// Every thread of every CTA of the cluster calls this once.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Inclusive saturating scan over the block's threads plus `carry` (the sum
// before them), which becomes the sum behind them. Saturating addition of
// values in [0, kSaturated] is associative.
__device__ __forceinline__ uint32_t block_scan(uint32_t value, uint32_t* warp_sums, uint32_t& carry) {
    const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint32_t sum = value;
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t below = __shfl_up_sync(0xFFFFFFFFU, sum, d);
        if (lane >= d) sum = add_sat(sum, below);
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    uint32_t base = lane < warps ? warp_sums[lane] : 0U;
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t below = __shfl_up_sync(0xFFFFFFFFU, base, d);
        if (lane >= d) base = add_sat(base, below);
    }
    const uint32_t total = __shfl_sync(0xFFFFFFFFU, base, 31);
    const uint32_t before = __shfl_sync(0xFFFFFFFFU, base, (warp + 31U) & 31U);
    __syncthreads();  // warp_sums is free again
    const uint32_t result = add_sat(add_sat(carry, warp ? before : 0U), sum);
    carry = add_sat(carry, total);
    return result;
}

// What phase 2 needs of a request: its first row, its cached length (-1:
// refused, no rows), the free-stack index of its page 0 if all its pages
// came from there, and its new tokens.
struct Request {
    uint32_t start;
    int32_t length;
    int32_t stack;
    uint32_t count;
};

__global__ void nz_pages_reserve_kernel(const nz_reserve a) {
    extern __shared__ Request requests[];
    __shared__ uint32_t warp_sums[32];
    const int32_t* lengths = nz::device_ptr<const int32_t>(a.lengths);
    const int32_t* new_tokens = nz::device_ptr<const int32_t>(a.new_tokens);
    const int32_t* free_pages = nz::device_ptr<const int32_t>(a.free_pages);
    int32_t* table = nz::device_ptr<int32_t>(a.block_table);
    int32_t* row_offsets = nz::device_ptr<int32_t>(a.row_offsets);
    const uint32_t shift = a.page_shift, page_mask = (1U << shift) - 1U;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const uint64_t capacity = static_cast<uint64_t>(a.width) << shift;

    const int32_t used = *nz::device_ptr<const int32_t>(a.used);
    const bool sound = used >= 0 && static_cast<uint32_t>(used) <= a.pages;
    const uint32_t available = sound ? a.pages - static_cast<uint32_t>(used) : 0U;
    uint32_t row_carry = 0, page_carry = 0, taken = 0, refused = 0;
    for (uint32_t first = 0; first < a.requests; first += blockDim.x) {
        const uint32_t b = first + threadIdx.x;
        const bool live = b < a.requests;
        const int32_t length = live ? lengths[b] : 0;
        const int32_t count = live ? new_tokens[b] : 0;
        const uint32_t rows = count > 0 ? min(static_cast<uint32_t>(count), kSaturated) : 0U;
        const uint32_t ends = block_scan(rows, warp_sums, row_carry);
        const uint64_t row = a.row_stride ? static_cast<uint64_t>(b) * a.row_stride : ends - rows;
        bool fits = live && length >= 0 && count >= 0 &&
                    static_cast<uint64_t>(length) + static_cast<uint64_t>(rows) <= capacity;
        if (rows) fits = fits && row + rows <= a.rows && (a.row_stride ? rows <= a.row_stride : ends < kSaturated);
        const uint32_t held = fits ? (static_cast<uint32_t>(length) + page_mask) >> shift : 0U;
        const uint32_t need = fits ? ((static_cast<uint32_t>(length) + rows + page_mask) >> shift) - held : 0U;
        const uint32_t upto = block_scan(need, warp_sums, page_carry);
        const bool served = fits && (need == 0U || upto <= available);
        if (live) {
            Request r;
            r.start = static_cast<uint32_t>(min(row, static_cast<uint64_t>(kSaturated)));
            r.length = served ? length : -1;
            r.stack = used + static_cast<int32_t>(upto - need) - static_cast<int32_t>(held);
            r.count = rows;
            requests[b] = r;
            if (rank == 0) {
                row_offsets[b] = static_cast<int32_t>(r.start);
                if (b + 1 == a.requests)
                    row_offsets[a.requests] = static_cast<int32_t>(
                        a.row_stride ? min(row + a.row_stride, static_cast<uint64_t>(kSaturated)) : ends);
                refused += served ? 0U : 1U;
                if (served && need) taken = max(taken, upto);
            }
        }
    }
    // The number of pages taken (sums that fit only grow) and of refusals.
    __shared__ uint32_t totals[2];
    if (threadIdx.x < 2) totals[threadIdx.x] = 0U;
    __syncthreads();
    if (taken) atomicMax(&totals[0], taken);
    if (refused) atomicAdd(&totals[1], refused);

    const uint32_t threads = blockDim.x * ctas;
    int32_t* positions = nz::device_ptr<int32_t>(a.positions);
    int32_t* slots = nz::device_ptr<int32_t>(a.slots);
    for (uint32_t row = rank * blockDim.x + threadIdx.x; row < a.rows; row += threads) {
        uint32_t b = 0;
        if (a.row_stride) {
            b = row / a.row_stride;
        } else {  // the last request that starts at or before the row
            uint32_t high = a.requests;
            while (high - b > 1U) {
                const uint32_t middle = (b + high) >> 1;
                if (requests[middle].start <= row) b = middle; else high = middle;
            }
        }
        int32_t position = 0, slot = -1;
        if (b < a.requests) {
            const Request r = requests[b];
            const uint32_t step = row - r.start;
            if (r.length >= 0 && row >= r.start && step < r.count) {
                const uint32_t at = static_cast<uint32_t>(r.length) + step, column = at >> shift;
                const uint32_t held = (static_cast<uint32_t>(r.length) + page_mask) >> shift;
                int32_t* entry = table + static_cast<uint64_t>(b) * a.table_stride + column;
                int32_t page;
                if (column < held) {
                    page = *entry;
                } else {
                    page = free_pages[r.stack + static_cast<int32_t>(column)];
                    if ((at & page_mask) == 0U) *entry = page;  // the row that starts the page
                }
                position = static_cast<int32_t>(at);
                if (page >= 0 && static_cast<uint32_t>(page) < a.pages)
                    slot = (page << shift) | static_cast<int32_t>(at & page_mask);
            }
        }
        positions[row] = position;
        slots[row] = slot;
    }

    // Every CTA has read the lengths and the stack's top.
    if (ctas > 1) cluster_barrier(); else __syncthreads();
    if (rank == 0) {
        int32_t* lengths_out = nz::device_ptr<int32_t>(a.lengths_out);
        for (uint32_t b = threadIdx.x; b < a.requests; b += blockDim.x) {
            const Request r = requests[b];
            if (r.length >= 0)
                lengths_out[b] = r.length + static_cast<int32_t>(r.count);
            else if (lengths_out != lengths)
                lengths_out[b] = lengths[b];
        }
        if (threadIdx.x == 0) {
            *nz::device_ptr<int32_t>(a.used_out) = used + static_cast<int32_t>(totals[0]);
            *nz::device_ptr<int32_t>(a.refused) = static_cast<int32_t>(totals[1]);
        }
    }
}

struct Released {
    uint32_t ends;   // pages released up to and including the request
    uint32_t count;  // its own
};

__global__ void nz_pages_release_kernel(const nz_release a) {
    extern __shared__ Released released[];
    __shared__ uint32_t warp_sums[32];
    const int32_t* lengths = nz::device_ptr<const int32_t>(a.lengths);
    const uint8_t* done = nz::device_ptr<const uint8_t>(a.done);
    const int32_t* table = nz::device_ptr<const int32_t>(a.block_table);
    int32_t* free_pages = nz::device_ptr<int32_t>(a.free_pages);
    const uint32_t shift = a.page_shift, page_mask = (1U << shift) - 1U;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int32_t used = *nz::device_ptr<const int32_t>(a.used);

    uint32_t total = 0;
    for (uint32_t first = 0; first < a.requests; first += blockDim.x) {
        const uint32_t b = first + threadIdx.x;
        uint32_t count = 0;
        if (b < a.requests && done[b]) {
            const int32_t length = lengths[b];
            if (length > 0) count = min((static_cast<uint32_t>(length) + page_mask) >> shift, a.width);
        }
        const uint32_t ends = block_scan(count, warp_sums, total);
        if (b < a.requests) released[b] = {ends, count};
    }
    __syncthreads();
    const int64_t base = static_cast<int64_t>(used) - total;
    for (uint32_t e = rank * blockDim.x + threadIdx.x; e < total; e += blockDim.x * ctas) {
        uint32_t b = 0, high = a.requests;  // the first request that ends behind e
        while (b < high) {
            const uint32_t middle = (b + high) >> 1;
            if (released[middle].ends > e) high = middle; else b = middle + 1U;
        }
        const int64_t place = base + e;
        if (b >= a.requests || place < 0 || place >= a.pages) continue;  // more pages than the stack gave out
        const uint32_t column = e + released[b].count - released[b].ends;
        free_pages[place] = table[static_cast<uint64_t>(b) * a.table_stride + column];
    }

    if (ctas > 1) cluster_barrier(); else __syncthreads();
    if (rank == 0) {
        int32_t* lengths_out = nz::device_ptr<int32_t>(a.lengths_out);
        for (uint32_t b = threadIdx.x; b < a.requests; b += blockDim.x) {
            const int32_t length = lengths[b];
            lengths_out[b] = done[b] ? 0 : length;
        }
        if (threadIdx.x == 0) *nz::device_ptr<int32_t>(a.used_out) = static_cast<int32_t>(base < 0 ? 0 : base);
    }
}

// One CTA while `items` fit a few passes of it, else up to a cluster of 8;
// 256 threads for small calls, whose block scans are shorter.
template <typename Args>
int launch(void (*kernel)(const Args), const Args& args, uint64_t items, size_t smem, void* cuda_stream,
           const char* what) {
    const bool small = items <= 256 && args.requests <= 256;
    cudaLaunchConfig_t config = {};
    config.blockDim = dim3(small ? 256 : 1024);
    const uint64_t wanted = (items + 2047) / 2048;
    const uint32_t ctas = wanted <= 1 ? 1U : wanted <= 2 ? 2U : wanted <= 4 ? 4U : kMostCtas;
    config.gridDim = dim3(ctas);
    config.dynamicSmemBytes = smem;
    config.stream = reinterpret_cast<cudaStream_t>(cuda_stream);
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = ctas;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    if (smem > 47 * 1024) {
        const cudaError_t err =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (err != cudaSuccess) return nz::cuda_status(err, what);
    }
    return nz::cuda_status(cudaLaunchKernelEx(&config, kernel, args), what);
}

}  // namespace

extern "C" {

int nz_pages_reserve(const nz_reserve* args, void* cuda_stream) {
    if (!args) return nz::paged_fail("Null arguments.");
    const nz_reserve& a = *args;
    if (a.requests == 0 || a.requests > NZ_PAGED_MAX_REQUESTS)
        return nz::paged_fail("The number of requests must be 1 to 4096.");
    if (a.rows > NZ_PAGED_MAX_ROWS || a.row_stride > NZ_PAGED_MAX_ROWS)
        return nz::paged_fail("At most 2^30 rows.");
    if (!nz::paged_sizes_fit(a.pages, a.width, a.page_shift))
        return nz::paged_fail("A cache and a block-table row hold fewer than 2^30 pages and 2^31 tokens.");
    if (!a.lengths || !a.new_tokens || !a.used || !a.row_offsets || !a.lengths_out || !a.used_out || !a.refused ||
        (a.width && !a.block_table) || (a.pages && !a.free_pages) || (a.rows && (!a.positions || !a.slots)))
        return nz::paged_fail("Null device array.");
    return launch(nz_pages_reserve_kernel, a, a.rows, a.requests * sizeof(Request), cuda_stream, "nz_pages_reserve");
}

int nz_pages_release(const nz_release* args, void* cuda_stream) {
    if (!args) return nz::paged_fail("Null arguments.");
    const nz_release& a = *args;
    if (a.requests == 0 || a.requests > NZ_PAGED_MAX_REQUESTS)
        return nz::paged_fail("The number of requests must be 1 to 4096.");
    if (!nz::paged_sizes_fit(a.pages, a.width, a.page_shift))
        return nz::paged_fail("A cache and a block-table row hold fewer than 2^30 pages and 2^31 tokens.");
    if (!a.lengths || !a.done || !a.used || !a.lengths_out || !a.used_out || (a.width && !a.block_table) ||
        (a.pages && !a.free_pages))
        return nz::paged_fail("Null device array.");
    const uint64_t most = static_cast<uint64_t>(a.requests) * a.width;
    return launch(nz_pages_release_kernel, a, most < a.pages ? most : a.pages, a.requests * sizeof(Released),
                  cuda_stream, "nz_pages_release");
}

}  // extern "C"
