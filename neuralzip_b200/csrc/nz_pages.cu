// Page bookkeeping of the paged key-value cache: block tables, positions and
// slots from request lengths, on the GPU, so that a captured generation step
// can cross page borders without the host.
//
// For request b with n_b cached and m_b new tokens and pages of P tokens:
//   need_b = ceil((n_b + m_b) / P) - ceil(n_b / P)
//   page j of the request (j >= ceil(n_b / P)) = free[used + sum_{a<b} need_a + j - ceil(n_b / P)]
//   token i of the request: position n_b + i, slot page(position / P) * P + position % P
// A few integers a request and 8 bytes a row: the call is bound by its
// launch and by the latency of a load, two block scans, a load and a store:
// 2.5 us for a step of 64 requests, 3.0 us for 66k rows of 129 prompts.
//
// One launch does all of it: every CTA scans all requests for itself (at
// most 4096, 16 KB of loads that hit L2) and then writes its share of the
// rows, and the first CTA the new lengths and the stack's top. Where these
// are updated in place, as a captured step does, the CTAs are one cluster
// whose barrier separates the last read from the update, so that no second
// launch and no counter that calls would share is needed.

#include "nz_paged.h"

namespace {

constexpr uint32_t kMostCtas = 8;           // portable cluster size
// Where sums stop: above every legal row and page count, and above every
// value of the stack's top.
constexpr uint32_t kSaturated = 1U << 30, kMostReleased = 0x7FFFFFFFU;

template <uint32_t MOST>
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, MOST); }

// Every thread calls this once, where all CTAs are one cluster.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Exclusive saturating scan: the sum of the values of the block's threads
// before this one and of `carry` (the sum before the block's), which becomes
// the sum behind them. Saturating addition of values in [0, MOST] is
// associative, so sums never fall from one thread to the next, and are exact
// below MOST; the sum before a value is not the sum up to it less it.
template <uint32_t MOST>
__device__ __forceinline__ uint32_t block_scan(uint32_t value, uint32_t* warp_sums, uint32_t& carry) {
    const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint32_t sum = value;
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t below = __shfl_up_sync(0xFFFFFFFFU, sum, d);
        if (lane >= d) sum = add_sat<MOST>(sum, below);
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    uint32_t base = lane < warps ? warp_sums[lane] : 0U;
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t below = __shfl_up_sync(0xFFFFFFFFU, base, d);
        if (lane >= d) base = add_sat<MOST>(base, below);
    }
    const uint32_t total = __shfl_sync(0xFFFFFFFFU, base, 31);
    const uint32_t before = __shfl_sync(0xFFFFFFFFU, base, (warp + 31U) & 31U);
    const uint32_t below = __shfl_up_sync(0xFFFFFFFFU, sum, 1);
    __syncthreads();  // warp_sums is free again
    const uint32_t result = add_sat<MOST>(add_sat<MOST>(carry, warp ? before : 0U), lane ? below : 0U);
    carry = add_sat<MOST>(carry, total);
    return result;
}

// What phase 2 needs of a request: its first row, its cached length (-1:
// refused, no rows), the free-stack index of its page 0 if all its pages
// came from there, and its new tokens (a refused request's may be any number).
struct Request {
    uint32_t start;
    int32_t length;
    int32_t stack;
    uint32_t count;
};

__global__ void __launch_bounds__(1024) nz_pages_reserve_kernel(const nz_reserve a, const bool in_place) {
    nz::after_predecessor();
    extern __shared__ Request requests[];
    __shared__ uint32_t warp_sums[32];
    const int32_t* lengths = nz::device_ptr<const int32_t>(a.lengths);
    const int32_t* new_tokens = nz::device_ptr<const int32_t>(a.new_tokens);
    int32_t* free_pages = nz::device_ptr<int32_t>(a.free_pages);  // only read
    int32_t* table = nz::device_ptr<int32_t>(a.block_table);
    int32_t* row_offsets = nz::device_ptr<int32_t>(a.row_offsets);
    const uint32_t shift = a.page_shift, page_mask = (1U << shift) - 1U;
    const uint32_t rank = blockIdx.x, ctas = gridDim.x;
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
        const uint32_t rows = count > 0 ? static_cast<uint32_t>(count) : 0U;
        const uint32_t packed = block_scan<kSaturated>(min(rows, kSaturated), warp_sums, row_carry);
        const uint64_t row = a.row_stride ? static_cast<uint64_t>(b) * a.row_stride : packed;
        bool fits = live && length >= 0 && count >= 0 &&
                    static_cast<uint64_t>(length) + static_cast<uint64_t>(rows) <= capacity;
        // A saturated row is above every row there may be.
        if (rows) fits = fits && row + rows <= a.rows && (!a.row_stride || rows <= a.row_stride);
        const uint32_t held = fits ? (static_cast<uint32_t>(length) + page_mask) >> shift : 0U;
        const uint32_t need = fits ? ((static_cast<uint32_t>(length) + rows + page_mask) >> shift) - held : 0U;
        const uint32_t asked = block_scan<kSaturated>(need, warp_sums, page_carry), upto = add_sat<kSaturated>(asked, need);
        const bool served = fits && (need == 0U || upto <= available);
        if (live) {
            Request r;
            r.start = static_cast<uint32_t>(min(row, static_cast<uint64_t>(kSaturated)));
            r.length = served ? length : -1;
            r.stack = used + static_cast<int32_t>(asked) - static_cast<int32_t>(held);
            r.count = rows;
            requests[b] = r;
            if (rank == 0) {
                row_offsets[b] = static_cast<int32_t>(r.start);
                if (b + 1 == a.requests)
                    row_offsets[a.requests] = static_cast<int32_t>(
                        min(row + (a.row_stride ? a.row_stride : rows), static_cast<uint64_t>(kSaturated)));
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
    // With more rows than threads, a thread takes four neighbours at a time:
    // one search, and their page ids are loaded together.
    const uint32_t run = a.rows > threads ? 4U : 1U;
    for (uint32_t row = run * (rank * blockDim.x + threadIdx.x); row < a.rows; row += run * threads) {
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
        Request r = b < a.requests ? requests[b] : Request{0U, -1, 0, 0U};
        int32_t position[4], page[4];
        int32_t* entry[4];  // of the block table, where the row starts a page
#pragma unroll
        for (uint32_t i = 0; i < 4U; ++i) {
            position[i] = page[i] = -1;
            entry[i] = nullptr;
            if (i >= run || row + i >= a.rows) continue;
            while (b + 1U < a.requests && requests[b + 1U].start <= row + i) r = requests[++b];
            const uint32_t step = row + i - r.start;
            if (r.length < 0 || row + i < r.start || step >= r.count) continue;
            const uint32_t at = static_cast<uint32_t>(r.length) + step, column = at >> shift;
            const uint32_t held = (static_cast<uint32_t>(r.length) + page_mask) >> shift;
            int32_t* own = table + static_cast<uint64_t>(b) * a.table_stride + column;
            page[i] = *(column < held ? own : free_pages + (r.stack + static_cast<int32_t>(column)));
            if (column >= held && (at & page_mask) == 0U) entry[i] = own;
            position[i] = static_cast<int32_t>(at);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4U; ++i) {
            if (i >= run || row + i >= a.rows) continue;
            if (entry[i]) *entry[i] = page[i];
            const bool cached = page[i] >= 0 && static_cast<uint32_t>(page[i]) < a.pages;
            positions[row + i] = max(position[i], 0);
            slots[row + i] = cached ? (page[i] << shift) | (position[i] & static_cast<int32_t>(page_mask)) : -1;
        }
    }

    // Every CTA has read the lengths and the stack's top.
    if (in_place && ctas > 1) cluster_barrier(); else __syncthreads();
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

// Of the i-th request from the last one. Counted from there, an entry's
// place under the stack's top depends on nothing that may have saturated:
// entry e of all that are released goes to free_pages[used - 1 - e].
struct Released {
    uint32_t before;  // pages released of the requests behind it
    uint32_t count;   // its own
};

__global__ void __launch_bounds__(1024) nz_pages_release_kernel(const nz_release a, const bool in_place) {
    nz::after_predecessor();
    extern __shared__ Released released[];
    __shared__ uint32_t warp_sums[32];
    const int32_t* lengths = nz::device_ptr<const int32_t>(a.lengths);
    const uint8_t* done = nz::device_ptr<const uint8_t>(a.done);
    const int32_t* table = nz::device_ptr<const int32_t>(a.block_table);
    int32_t* free_pages = nz::device_ptr<int32_t>(a.free_pages);
    const uint32_t shift = a.page_shift, page_mask = (1U << shift) - 1U;
    const uint32_t rank = blockIdx.x, ctas = gridDim.x;
    const int32_t used = *nz::device_ptr<const int32_t>(a.used);

    uint32_t total = 0;
    for (uint32_t first = 0; first < a.requests; first += blockDim.x) {
        const uint32_t i = first + threadIdx.x, b = a.requests - 1U - i;
        uint32_t count = 0;
        if (i < a.requests && done[b]) {
            const int32_t length = lengths[b];
            if (length > 0) count = min((static_cast<uint32_t>(length) + page_mask) >> shift, a.width);
        }
        const uint32_t before = block_scan<kMostReleased>(count, warp_sums, total);
        if (i < a.requests) released[i] = {before, count};
    }
    __syncthreads();
    // The entries that lie in the stack: no more than it gave out.
    const uint32_t top = static_cast<uint32_t>(max(used, 0));
    const uint32_t begin = top > a.pages ? top - a.pages : 0U, end = min(total, top), entries = end > begin ? end - begin : 0U;
    // With more entries than threads, a thread takes four neighbours at a
    // time: one search, and their ids are loaded together.
    const uint32_t run = entries > blockDim.x * ctas ? 4U : 1U;
    for (uint32_t first = run * (rank * blockDim.x + threadIdx.x); first < entries; first += run * blockDim.x * ctas) {
        uint32_t i = 0, high = a.requests;  // the last one that starts at or before the entry
        while (high - i > 1U) {
            const uint32_t middle = (i + high) >> 1;
            if (released[middle].before <= begin + first) i = middle; else high = middle;
        }
        int32_t page[4];
#pragma unroll
        for (uint32_t j = 0; j < 4U; ++j) {
            const uint32_t e = begin + first + j;
            if (j >= run || first + j >= entries) continue;
            while (i + 1U < a.requests && released[i + 1U].before <= e) ++i;
            const uint32_t column = released[i].count - 1U - (e - released[i].before);
            page[j] = table[static_cast<uint64_t>(a.requests - 1U - i) * a.table_stride + column];
        }
#pragma unroll
        for (uint32_t j = 0; j < 4U; ++j)
            if (j < run && first + j < entries) free_pages[top - 1U - (begin + first + j)] = page[j];
    }

    if (in_place && ctas > 1) cluster_barrier(); else __syncthreads();
    if (rank == 0) {
        int32_t* lengths_out = nz::device_ptr<int32_t>(a.lengths_out);
        for (uint32_t b = threadIdx.x; b < a.requests; b += blockDim.x) {
            const int32_t length = lengths[b];
            lengths_out[b] = done[b] ? 0 : length;
        }
        if (threadIdx.x == 0) *nz::device_ptr<int32_t>(a.used_out) = static_cast<int32_t>(top > total ? top - total : 0U);
    }
}

// 256 threads a CTA where they cover the requests (block scans are shorter),
// else 1024, and CTAs for all items up to a GPU full. Updating in place
// takes one cluster, so at most 8 CTAs: 66k rows of 129 requests take 11 us
// that way, the release of 65k pages of 512 requests 7.3 (3.1 apart).
// Item: what a CTA keeps of each request in shared memory.
template <typename Item, typename Args>
int launch(void (*kernel)(const Args, const bool), const Args& args, uint64_t items, void* cuda_stream, const char* what) {
    const size_t smem = args.requests * sizeof(Item);
    const bool in_place = args.lengths == args.lengths_out || args.used == args.used_out;
    const uint32_t threads = args.requests <= 256 && (!in_place || items <= 256) ? 256U : 1024U;
    const uint64_t wanted = (items + threads - 1) / threads, most = in_place ? kMostCtas : 148U * 1024U / threads;
    uint32_t ctas = static_cast<uint32_t>(wanted < 1 ? 1 : wanted < most ? wanted : most);
    if (in_place) ctas = ctas > 4 ? 8U : ctas > 2 ? 4U : ctas;
    if (smem > 47 * 1024) {
        // The most that any call takes, not this one's: another thread's launch may be on its way.
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     static_cast<int>(NZ_PAGED_MAX_REQUESTS * sizeof(Item)));
        if (err != cudaSuccess) return nz::cuda_status(err, what);
    }
    const nz::PagedLaunch l(ctas, 1, threads, smem, reinterpret_cast<cudaStream_t>(cuda_stream), in_place ? ctas : 1U);
    return nz::cuda_status(cudaLaunchKernelEx(&l.config, kernel, args, in_place), what);
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
    return launch<Request>(nz_pages_reserve_kernel, a, a.rows, cuda_stream, "nz_pages_reserve");
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
    return launch<Released>(nz_pages_release_kernel, a, most < a.pages ? most : a.pages, cuda_stream, "nz_pages_release");
}

}  // extern "C"
