// Attention of one new token a request over its pages of the cache.
//
// For request b with n tokens, key/value head k and the query heads h that
// share it: s_j = scale * q_h . K_j over the live positions j,
//   out_h = sum_j exp(s_j - max s) V_j / sum_j exp(s_j - max s),
// with the maximum and the sum kept running in 32 bits, so that every key
// and value is read once. Keys and values are all there is to read: the
// kernel is bound by HBM, and by latency where they are few.
//
// The way in. A warp takes tiles of 32 positions of one key/value head,
// whose pages each lane looks up for one position. 128 bytes of each
// position's row are a unit of 4 KB; units are copied ahead into a ring in
// shared memory that only this warp reads, so nothing waits for other warps,
// and positions that are masked are not read but filled with zeros. (Copies
// straight into the registers of the products were as fast at best, and a
// third slower whenever the compiler ordered them differently.)
//
// Products, 16-bit types. Keys and values are the left operand of mma.sync
// (16 positions, or 16 elements of the head, by 16) and up to 8 query heads
// that share them the right one, so that no half-empty tile is multiplied:
//   S^T = K Q^T (positions x heads),  O^T += V^T P^T (elements x heads).
// ldmatrix reads both, V^T transposed; movmatrix turns P^T. tcgen05.mma would
// multiply 128 rows at a time, of which a tile has 32, and the products are
// not what bounds the kernel.
// The products are exact and the sums 32-bit; P is split into two 16-bit
// parts (16 or more bits of each weight), because one rounding of P would
// cost as much as the rounding of the result. fp32: see Arithmetic<float>.
//
// The work is shared out in three ways, see launch(): a CTA an item
// (request, key/value head, group of query heads), a cluster an item, whose
// CTAs add up through each other's shared memory, or equal runs of all
// items' tiles, whose parts a second kernel joins. Each adds in an order
// that sizes alone fix.
//
// Measured, of the rate of a plain copy (6.53 TB/s): 32 requests of 2047 to
// 32768 tokens, 32 heads over 8 of 128 in bf16, 2.28 GB, 353-365 us (96-99%); one
// request of 65537, 64 heads, 268 MB, 49 us (84%: the ends of the two
// launches); 8 requests of 129 to 384, 6.1 us, and one of 160, 14 heads over
// 2 of 64, 3.9 us, bound by the latency of a launch, four dependent loads
// and a tile's arithmetic.

#include "nz_paged.h"

#include <mutex>
#include <type_traits>

namespace {

// Units that a warp's ring holds: one in use, the others on their way.
constexpr int kRing = 3;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kSplitWarps = 4;
constexpr uint32_t kMostCtas = 8;     // of a cluster
constexpr uint32_t kLeastChunks = 2;  // of a CTA where the work is split

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_float(float x) { return x; }

__device__ __forceinline__ float exp2_approx(float x) {  // within 2 ulp; -inf gives 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes into shared memory, zeros (and no access) where `live` is not set.
__device__ __forceinline__ void copy_async(uint32_t shared, const void* global, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(global), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8x8 matrices of 16-bit values, whose rows of 16 bytes the lanes name
// in turn: a left operand; or their transposes.
__device__ __forceinline__ void load_matrices(uint32_t (&x)[4], uint32_t shared) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(shared)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&x)[4], uint32_t shared) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(shared)
                 : "memory");
}
__device__ __forceinline__ float4 load_shared(uint32_t shared) {
    float4 x;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(shared)
                 : "memory");
    return x;
}

// Another CTA's shared memory, in a cluster.
__device__ __forceinline__ float load_peer(const float* mine, uint32_t rank) {
    uint32_t at;
    float x;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ void cluster_barrier() {  // every thread of every CTA of the cluster
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Two products and sums in one instruction.
__device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // of an 8x8 matrix of 16-bit values over the warp
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
    const __half2 x = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ float2 unpack(uint32_t x, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}
__device__ __forceinline__ float2 unpack(uint32_t x, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// Sizes of an instantiation: head width padded to kDim, kHeadTiles tiles of
// 8 query heads. A warp's tile is 32 positions; it is read in units of 128
// bytes of each position's row, 4 KB, first of the keys, then of the values.
constexpr uint32_t kTile = 32;
constexpr uint32_t kUnitBytes = 4096;

template <typename T, int kDim, int kHeadTiles, int kWarps_>
struct Shape {
    static constexpr int kWarps = kWarps_;
    static constexpr uint32_t kThreads = kWarps * 32;
    static constexpr int kSize = sizeof(T);
    static constexpr int kUnit = 128 / kSize;                     // elements of a unit
    static constexpr int kUnits = kDim / kUnit;                   // of a tile's keys, and of its values
    static constexpr uint32_t kChunk = kTile * kWarps;            // positions of a CTA's pass
    static constexpr int kLaneElems = 16 / kSize;                 // elements of 16 bytes
    static constexpr bool kWide = kSize == 4;
    static constexpr int kHeads = kWide ? (kHeadTiles == 1 ? 1 : 4) : 8 * kHeadTiles;  // of an item
    static constexpr int kQueryBlocks = kDim * kSize / 64;        // of 64 bytes of a query
    static constexpr int kRowTiles = kDim / 16;                   // 16-element tiles of O^T
    static constexpr int kUnitRows = kUnit / 16;                  // of them in a unit
    static constexpr int kSumStride = kDim + 4;
    static constexpr int kAhead = (kRing - 2) / (2 * kUnits) + 2; // tiles whose pages are known ahead
    static constexpr size_t kQueryBytes =  // fp32: also a tile's weights, [warp][head][position]
        kWide ? static_cast<size_t>(kHeads) * (kDim + kWarps * kTile) * 4 : static_cast<size_t>(kHeadTiles) * kQueryBlocks * 512;
    static constexpr size_t kSumBytes = static_cast<size_t>(kWarps) * kHeads * kSumStride * 4;
    static constexpr size_t kStatBytes = 2 * kWarps * kHeads * 4;
    static constexpr size_t kRingBytes = static_cast<size_t>(kWarps) * kRing * kUnitBytes;
    // Each part a multiple of 128 bytes before the rings, whose swizzle counts on it.
    static constexpr size_t kHeadBytes = (kQueryBytes + kStatBytes + 127) / 128 * 128;
    static constexpr size_t kSharedBytes = kHeadBytes + (kRingBytes > kSumBytes ? kRingBytes : kSumBytes);
    static constexpr size_t kPartFloats = (static_cast<size_t>(kHeads) * (kDim + 2) + 3) / 4 * 4;  // a partial result
};

// What a split launch adds: its workspace holds two partial results a CTA
// ("worker"), then one Join a worker or an item.
struct Join {
    uint32_t request, item;  // item: (key/value head, group of kHeads query heads)
    uint32_t parts;          // of workers `worker`, `worker` + 1, ...; 0: not split
    uint32_t worker;
    uint32_t slot;           // of the first worker's part (the others' is 0)
};

struct Plan {
    uint32_t workers;   // CTAs of a split launch
    uint32_t groups;    // of kHeads query heads that share a key/value head
    uint32_t by_item;   // one Join an item, else one a worker (of the item that starts, split, in its run)
    uint32_t shares;    // warps of the join that add up one head
    uint32_t cluster;   // CTAs an item, where nothing is split
    uint32_t let_next;  // the next kernel may come onto the GPU before this one ends
};

__device__ __forceinline__ int32_t held_length(const nz_attention& a, uint32_t b) {
    const int32_t n = nz::device_ptr<const int32_t>(a.lengths)[b];
    return max(0, min(n, static_cast<int32_t>(a.width << a.page_shift)));
}
__device__ __forceinline__ int32_t first_position(const nz_attention& a, int32_t length) {
    return a.window && static_cast<uint32_t>(length) > a.window ? length - static_cast<int32_t>(a.window) : 0;
}

// What both kinds of arithmetic share: a CTA's shared memory, and the way of
// keys and values into it.
template <typename T, int kDim, int kHeadTiles, int kWarps_>
struct Reader {
    using S = Shape<T, kDim, kHeadTiles, kWarps_>;
    static constexpr int kWarps = S::kWarps;
    static constexpr uint32_t kThreads = S::kThreads;
    static constexpr bool kWide = S::kWide;

    const nz_attention& a;
    unsigned char* query;  // shared: queries, as the arithmetic wants them
    float* stats;          // shared: [2][warp][head]
    float* sums;           // shared: [warp][head][kSumStride], where the rings are while tiles are read
    uint32_t ring;         // shared address of the warp's ring
    uint32_t warp, lane;

    __device__ Reader(const nz_attention& args, unsigned char* shared) : a(args) {
        query = shared;
        stats = reinterpret_cast<float*>(shared + S::kQueryBytes);
        sums = reinterpret_cast<float*>(shared + S::kHeadBytes);
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31U;
        ring = static_cast<uint32_t>(__cvta_generic_to_shared(sums)) + warp * (kRing * kUnitBytes);
    }

    // Page of the lane's position of a tile, -1 where nothing is to be read.
    __device__ int32_t page_of(const int32_t* table, uint32_t tile, uint32_t tiles, int32_t start, int32_t length) const {
        const int32_t position = static_cast<int32_t>(tile * kTile + lane);
        int32_t page = -1;
        if (tile < tiles && position >= start && position < length) {
            page = table[position >> a.page_shift];
            if (page < 0 || static_cast<uint32_t>(page) >= a.pages) page = -1;
        }
        return page;
    }

    // The 16-byte chunks of a unit's rows are permuted so that one chunk of 8
    // positions touches every bank once.
    __device__ static uint32_t swizzle(uint32_t position) { return position & 7U; }

    // What the copies of a tile need: byte offsets of the rows that the lane
    // copies (position 4 * i + lane / 8), and which of the 32 are live.
    struct Rows {
        int64_t offset[8];
        uint32_t live;
    };
    __device__ void find_rows(Rows& rows, uint32_t tile, int32_t page, const int64_t (&stride)[3]) const {
        const uint32_t line = (tile * kTile + lane) & ((1U << a.page_shift) - 1U);
        const int64_t mine = page < 0 ? 0 : (page * stride[0] + line * stride[1]) * S::kSize;
        rows.live = __ballot_sync(0xFFFFFFFFU, page >= 0) >> (lane >> 3);
#pragma unroll
        for (int i = 0; i < 8; ++i) rows.offset[i] = __shfl_sync(0xFFFFFFFFU, mine, 4 * i + (lane >> 3));
    }
    // Unit u of a tile's rows into the ring; `base` is the key/value head's first element.
    __device__ void copy_rows(uint32_t to, const T* base, const Rows& rows, int u) const {
        const uint32_t chunk = lane & 7U, first = lane >> 3;
        const char* from = reinterpret_cast<const char*>(base) + u * 128 + chunk * 16U;
        const bool inside = u * S::kUnit + chunk * S::kLaneElems < a.dim;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t position = 4U * i + first;
            copy_async(to + position * 128U + ((chunk ^ swizzle(position)) << 4),
                       inside ? from + rows.offset[i] : reinterpret_cast<const char*>(base),
                       inside && ((rows.live >> (4 * i)) & 1U));
        }
    }
};

// 16-bit types: products on the tensor cores.
template <typename T, int kDim, int kHeadTiles, int kWarps_>
struct Arithmetic : Reader<T, kDim, kHeadTiles, kWarps_> {
    using R = Reader<T, kDim, kHeadTiles, kWarps_>;
    using S = typename R::S;
    using R::a, R::query, R::stats, R::sums, R::lane, R::warp, R::swizzle;
    static constexpr int kSteps = 2;  // of 16 positions of a tile
    // Weights are relative to 2^-kRaise of the largest: fp16, which ends at
    // 2^-24, would lose those that a hundred thousand positions add up to
    // next to one that stands out. `most` is the maximum less kRaise.
    static constexpr float kRaise = std::is_same_v<T, __half> ? 14.0f : 0.0f;

    uint32_t row, col;  // the lane's place in an mma's operands
    float o[S::kRowTiles][kHeadTiles][4], most[kHeadTiles][2], total[kHeadTiles][2];
    float s[kSteps][kHeadTiles][4];
    uint32_t w[kSteps][kHeadTiles][2][2];  // weights as right operands: [step][head tile][high and low part]

    __device__ Arithmetic(const nz_attention& args, unsigned char* shared) : R(args, shared) {
        row = lane >> 2;
        col = lane & 3U;
    }

    __device__ void clear() {
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t) {
#pragma unroll
            for (int i = 0; i < S::kRowTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][t][e] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                most[t][e] = -INFINITY;
                total[t][e] = 0.0f;
            }
        }
    }

    // Query heads [head, head + heads) of request b as right operands, zeros
    // behind the last head and the head's width: [head tile][64 bytes][lane],
    // where lane (row, col) holds, of head `row`, what its column takes of
    // two mma steps.
    __device__ void load_query(uint32_t b, uint32_t head, uint32_t heads) {
        const T* source = nz::device_ptr<const T>(a.query) + b * a.query_stride[0];
        for (uint32_t i = threadIdx.x; i < kHeadTiles * S::kQueryBlocks * 32U; i += S::kThreads) {
            const uint32_t at = i & 31U, block = (i >> 5) % S::kQueryBlocks, tile = (i >> 5) / S::kQueryBlocks;
            const uint32_t h = tile * 8U + (at >> 2), first = block * 32U + 2U * (at & 3U);
            alignas(16) T x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t d = first + 8U * (e >> 1) + (e & 1);
                x[e] = h < heads && d < a.dim ? source[(head + h) * a.query_stride[1] + d] : T(0.0f);
            }
            reinterpret_cast<uint4*>(query)[i] = *reinterpret_cast<const uint4*>(x);
        }
    }

    __device__ void begin_tile() {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][t][e] = 0.0f;
    }

    // S^T += K Q^T over unit u, in the ring at `from`.
    __device__ void scores(uint32_t from, int u) {
        // The lane's row of the four 8x8 matrices of a left operand.
        const uint32_t position = (lane & 7U) + (lane & 8U), half = lane >> 4;
        const uint32_t rows = from + position * 128U, mix = swizzle(position);
#pragma unroll
        for (int block = 0; block < 2; ++block) {  // of 64 bytes, two mma steps
            uint4 q[kHeadTiles];
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t)
                q[t] = reinterpret_cast<const uint4*>(query)[(t * S::kQueryBlocks + u * 2 + block) * 32U + lane];
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                uint32_t k0[4], k1[4];
                load_matrices(k0, rows + step * 2048U + (((4U * block + half) ^ mix) << 4));
                load_matrices(k1, rows + step * 2048U + (((4U * block + 2U + half) ^ mix) << 4));
#pragma unroll
                for (int t = 0; t < kHeadTiles; ++t) {
                    mma(s[step][t], k0, q[t].x, q[t].y, T());
                    mma(s[step][t], k1, q[t].z, q[t].w, T());
                }
            }
        }
    }

    // O^T += V^T P^T for the elements of unit u, in the ring at `from`.
    __device__ void products(uint32_t from, int u) {
        const uint32_t position = (lane & 7U) + ((lane >> 4) << 3), half = (lane >> 3) & 1U;
        const uint32_t rows = from + position * 128U, mix = swizzle(position);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int j = 0; j < S::kUnitRows; ++j) {
                uint32_t v[4];
                load_matrices_transposed(v, rows + i * 2048U + (((2U * j + half) ^ mix) << 4));
#pragma unroll
                for (int t = 0; t < kHeadTiles; ++t) {
                    mma(o[u * S::kUnitRows + j][t], v, w[i][t][1][0], w[i][t][1][1], T());
                    mma(o[u * S::kUnitRows + j][t], v, w[i][t][0][0], w[i][t][0][1], T());
                }
            }
    }

    // Masks and weighs a tile's scores; rescales the sums when a maximum rose.
    __device__ void softmax(int32_t page, float scale) {
        const uint32_t live = __ballot_sync(0xFFFFFFFFU, page >= 0);
        float top[kHeadTiles][2];
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[t][e] = most[t][e] + kRaise;
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) s[i][t][2 * half + e] *= scale;
            }
        if (live != 0xFFFFFFFFU) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    if (!((live >> (i * 16 + half * 8 + row)) & 1U))
#pragma unroll
                        for (int t = 0; t < kHeadTiles; ++t) s[i][t][2 * half] = s[i][t][2 * half + 1] = -INFINITY;
        }
        bool rose = false;
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) top[t][e] = fmaxf(top[t][e], fmaxf(s[i][t][e], s[i][t][2 + e]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[t][e] = fmaxf(top[t][e], __shfl_xor_sync(0xFFFFFFFFU, top[t][e], d));
                top[t][e] -= kRaise;
                rose |= top[t][e] > most[t][e];
            }
        if (__any_sync(0xFFFFFFFFU, rose)) {
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float down = most[t][e] == -INFINITY ? 0.0f : exp2_approx(most[t][e] - top[t][e]);
                    most[t][e] = top[t][e];
                    total[t][e] *= down;
#pragma unroll
                    for (int i = 0; i < S::kRowTiles; ++i) {
                        o[i][t][e] *= down;
                        o[i][t][2 + e] *= down;
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = most[t][e] == -INFINITY ? 0.0f : most[t][e];
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float& x = s[i][t][2 * half + e];
                        x = exp2_approx(x - base);
                        total[t][e] += x;
                    }
            }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float* x = &s[i][t][2 * half];
                    const uint32_t high = pack(x[0], x[1], T());
                    const float2 back = unpack(high, T());
                    w[i][t][0][half] = transposed(high);
                    w[i][t][1][half] = transposed(pack(x[0] - back.x, x[1] - back.y, T()));
                }
    }

    // The warp's statistics, then (when all warps' are there) its sums relative to the CTA's maximum.
    __device__ void leave_stats() {
        float *tops = stats, *totals = stats + S::kWarps * S::kHeads;
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) total[t][e] += __shfl_xor_sync(0xFFFFFFFFU, total[t][e], d);
                if (row == 0) {
                    tops[warp * S::kHeads + t * 8 + 2 * col + e] = most[t][e];
                    totals[warp * S::kHeads + t * 8 + 2 * col + e] = total[t][e];
                }
            }
    }
    __device__ void leave_sums() {
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t h = t * 8 + 2 * col + e;
                float top = -INFINITY;
#pragma unroll
                for (int v = 0; v < S::kWarps; ++v) top = fmaxf(top, stats[v * S::kHeads + h]);
                const float down = most[t][e] == -INFINITY ? 0.0f : exp2_approx(most[t][e] - top);
                float* to = sums + (warp * S::kHeads + h) * S::kSumStride + row;
#pragma unroll
                for (int i = 0; i < S::kRowTiles; ++i) {
                    to[i * 16] = o[i][t][e] * down;
                    to[i * 16 + 8] = o[i][t][2 + e] * down;
                }
            }
    }
};

// fp32: ordinary arithmetic, two products an instruction. The tensor cores
// hold 11 bits of a factor, so they would need three products of split
// factors, 8 query heads at a time whether there are as many or not.
// A lane takes one position's scores, and of the sums 4 elements of each
// unit over a quarter of the positions.
template <int kDim, int kHeadTiles, int kWarps_>
struct Arithmetic<float, kDim, kHeadTiles, kWarps_> : Reader<float, kDim, kHeadTiles, kWarps_> {
    using R = Reader<float, kDim, kHeadTiles, kWarps_>;
    using S = typename R::S;
    using R::a, R::query, R::stats, R::sums, R::lane, R::warp, R::swizzle;

    float2 o[S::kHeads][S::kUnits][2], s[S::kHeads][2];
    float most[S::kHeads], total[S::kHeads];
    float* weights;  // shared: [head][position] of the warp

    __device__ Arithmetic(const nz_attention& args, unsigned char* shared) : R(args, shared) {
        weights = reinterpret_cast<float*>(query) + S::kHeads * (kDim + warp * kTile);
    }

    __device__ void clear() {
#pragma unroll
        for (int h = 0; h < S::kHeads; ++h) {
#pragma unroll
            for (int u = 0; u < S::kUnits; ++u) o[h][u][0] = o[h][u][1] = make_float2(0.0f, 0.0f);
            most[h] = -INFINITY;
            total[h] = 0.0f;
        }
    }

    __device__ void load_query(uint32_t b, uint32_t head, uint32_t heads) {  // [head][element]
        const float* source = nz::device_ptr<const float>(a.query) + b * a.query_stride[0];
        for (uint32_t i = threadIdx.x; i < S::kHeads * kDim; i += S::kThreads) {
            const uint32_t h = i / kDim, d = i % kDim;
            reinterpret_cast<float*>(query)[i] = h < heads && d < a.dim ? source[(head + h) * a.query_stride[1] + d] : 0.0f;
        }
    }

    __device__ void begin_tile() {
#pragma unroll
        for (int h = 0; h < S::kHeads; ++h) s[h][0] = s[h][1] = make_float2(0.0f, 0.0f);
    }

    __device__ void scores(uint32_t from, int u) {
        if (u * S::kUnit >= a.dim) return;
        const uint32_t mine = from + lane * 128U, mix = swizzle(lane);
#pragma unroll
        for (uint32_t chunk = 0; chunk < 8; ++chunk) {
            const float4 x = load_shared(mine + ((chunk ^ mix) << 4));
#pragma unroll
            for (int h = 0; h < S::kHeads; ++h) {
                const float4 q = reinterpret_cast<const float4*>(query)[(h * kDim + u * S::kUnit) / 4 + chunk];
                s[h][0] = fma(make_float2(x.x, x.y), make_float2(q.x, q.y), s[h][0]);
                s[h][1] = fma(make_float2(x.z, x.w), make_float2(q.z, q.w), s[h][1]);
            }
        }
    }

    __device__ void softmax(int32_t page, float scale) {
#pragma unroll
        for (int h = 0; h < S::kHeads; ++h) {
            const float x = page >= 0 ? ((s[h][0].x + s[h][0].y) + (s[h][1].x + s[h][1].y)) * scale : -INFINITY;
            float top = fmaxf(most[h], x);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFU, top, d));
            if (top > most[h]) {  // the whole warp
                const float down = most[h] == -INFINITY ? 0.0f : exp2_approx(most[h] - top);
                most[h] = top;
                total[h] *= down;
#pragma unroll
                for (int u = 0; u < S::kUnits; ++u)
#pragma unroll
                    for (int e = 0; e < 2; ++e) o[h][u][e] = make_float2(o[h][u][e].x * down, o[h][u][e].y * down);
            }
            const float p = exp2_approx(x - (top == -INFINITY ? 0.0f : top));
            total[h] += p;
            weights[h * kTile + lane] = p;
        }
        __syncwarp();
    }

    __device__ void products(uint32_t from, int u) {
        if (u * S::kUnit >= a.dim) return;
        const uint32_t chunk = lane & 7U, first = (lane >> 3) * 8U;  // positions first .. first + 7
        float4 p[S::kHeads];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (i % 4 == 0)
#pragma unroll
                for (int h = 0; h < S::kHeads; ++h) p[h] = reinterpret_cast<const float4*>(weights)[(h * kTile + first + i) / 4];
            const float4 x = load_shared(from + (first + i) * 128U + ((chunk ^ swizzle(i)) << 4));
#pragma unroll
            for (int h = 0; h < S::kHeads; ++h) {
                const float y = i % 4 == 0 ? p[h].x : i % 4 == 1 ? p[h].y : i % 4 == 2 ? p[h].z : p[h].w;
                o[h][u][0] = fma(make_float2(x.x, x.y), make_float2(y, y), o[h][u][0]);
                o[h][u][1] = fma(make_float2(x.z, x.w), make_float2(y, y), o[h][u][1]);
            }
        }
    }

    __device__ void leave_stats() {
#pragma unroll
        for (int h = 0; h < S::kHeads; ++h) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) total[h] += __shfl_xor_sync(0xFFFFFFFFU, total[h], d);
            if (lane == 0) {
                stats[warp * S::kHeads + h] = most[h];
                stats[(S::kWarps + warp) * S::kHeads + h] = total[h];
            }
        }
    }
    __device__ void leave_sums() {
#pragma unroll
        for (int h = 0; h < S::kHeads; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int v = 0; v < S::kWarps; ++v) top = fmaxf(top, stats[v * S::kHeads + h]);
            const float down = most[h] == -INFINITY ? 0.0f : exp2_approx(most[h] - top);
            float* to = sums + (warp * S::kHeads + h) * S::kSumStride + (lane & 7U) * 4U;
#pragma unroll
            for (int u = 0; u < S::kUnits; ++u) {
                float4 x = make_float4(o[h][u][0].x, o[h][u][0].y, o[h][u][1].x, o[h][u][1].y);
#pragma unroll
                for (int d = 8; d < 32; d <<= 1) {
                    x.x += __shfl_xor_sync(0xFFFFFFFFU, x.x, d);
                    x.y += __shfl_xor_sync(0xFFFFFFFFU, x.y, d);
                    x.z += __shfl_xor_sync(0xFFFFFFFFU, x.z, d);
                    x.w += __shfl_xor_sync(0xFFFFFFFFU, x.w, d);
                }
                if (lane < 8U) *reinterpret_cast<float4*>(to + u * 32) = make_float4(x.x * down, x.y * down, x.z * down, x.w * down);
            }
        }
    }
};

template <typename T, int kDim, int kHeadTiles, int kWarps_>
struct Attention : Arithmetic<T, kDim, kHeadTiles, kWarps_> {
    using A = Arithmetic<T, kDim, kHeadTiles, kWarps_>;
    using R = Reader<T, kDim, kHeadTiles, kWarps_>;
    using S = typename R::S;
    using R::a, R::stats, R::sums, R::ring, R::lane, R::warp;
    static constexpr int kWarps = S::kWarps;
    static constexpr uint32_t kThreads = S::kThreads;

    __device__ Attention(const nz_attention& args, unsigned char* shared) : A(args, shared) {}

    // Chunks [chunk, chunk_end) of request b for query heads [head, head +
    // heads) of key/value head k: the joined sums of the CTA's warps end in
    // sums[0] (relative to the maximum), the maximum (of scores times
    // log2 e) and the denominator in stats[0][0] and stats[1][0].
    __device__ void segment(uint32_t b, uint32_t k, uint32_t head, uint32_t heads, uint32_t chunk, uint32_t chunk_end,
                            int32_t start, int32_t length) {
        constexpr int kTileUnits = 2 * S::kUnits;
        const int32_t* table = nz::device_ptr<const int32_t>(a.block_table) + b * a.table_stride;
        const T* keys = nz::device_ptr<const T>(a.key_pages) + k * a.key_stride[2];
        const T* values = nz::device_ptr<const T>(a.value_pages) + k * a.value_stride[2];
        const bool alike = a.key_stride[0] == a.value_stride[0] && a.key_stride[1] == a.value_stride[1];
        const uint32_t tiles = min(chunk_end * kWarps, (static_cast<uint32_t>(length) + kTile - 1U) / kTile);
        const float scale = a.scale * kLog2e;

        this->clear();

        // pages[i]: of the lane's position of the warp's i-th tile from the current one on.
        uint32_t tile = chunk * kWarps + warp, slot = 0;
        int32_t pages[S::kAhead + 1];
        typename R::Rows rows;
        // Starts the copy of a tile's unit into the ring's place `to`.
        auto copy = [&](uint32_t to, int ahead, int u) {
            const uint32_t at = tile + ahead * kWarps;
            if (at < tiles) {
                if (u == 0) this->find_rows(rows, at, pages[ahead], a.key_stride);
                if (u == S::kUnits && !alike) this->find_rows(rows, at, pages[ahead], a.value_stride);
                this->copy_rows(ring + to * kUnitBytes, u < S::kUnits ? keys : values, rows, u % S::kUnits);
            }
            copies_end();
        };
#pragma unroll
        for (int i = 0; i <= S::kAhead; ++i) pages[i] = this->page_of(table, tile + i * kWarps, tiles, start, length);
        __syncthreads();  // the previous segment's shared memory is free
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) copy(i, i / kTileUnits, i % kTileUnits);
        this->load_query(b, head, heads);
        __syncthreads();
        for (; tile < tiles; tile += kWarps) {
            this->begin_tile();
#pragma unroll
            for (int u = 0; u < kTileUnits; ++u) {
                copies_wait<kRing - 2>();
                __syncwarp();  // the unit is there for all lanes, and the one before it is read
                copy(slot == 0 ? kRing - 1 : slot - 1, (u + kRing - 1) / kTileUnits, (u + kRing - 1) % kTileUnits);
                const uint32_t from = ring + slot * kUnitBytes;
                if (u < S::kUnits) this->scores(from, u);
                else this->products(from, u - S::kUnits);
                if (u == S::kUnits - 1) this->softmax(pages[0], scale);
                slot = slot == kRing - 1 ? 0 : slot + 1;
            }
#pragma unroll
            for (int i = 0; i < S::kAhead; ++i) pages[i] = pages[i + 1];
            pages[S::kAhead] = this->page_of(table, tile + (S::kAhead + 1) * kWarps, tiles, start, length);
        }
        copies_wait<0>();
        join_warps();
    }

    __device__ void join_warps() {
        float* tops = stats;
        float* totals = stats + kWarps * S::kHeads;
        this->leave_stats();
        __syncthreads();  // also: every warp is done with its ring
        this->leave_sums();
        __syncthreads();
        // The CTA's sums, in warp order.
        for (uint32_t i = threadIdx.x; i < S::kHeads * kDim / 4U; i += kThreads) {
            float4* at = reinterpret_cast<float4*>(sums + (i / (kDim / 4U)) * S::kSumStride + (i % (kDim / 4U)) * 4U);
            float4 x = *at;
#pragma unroll
            for (int v = 1; v < kWarps; ++v) {
                const float4 y = at[v * S::kHeads * S::kSumStride / 4];
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            *at = x;
        }
        float top = -INFINITY, sum = 0.0f;
        if (threadIdx.x < S::kHeads) {
#pragma unroll
            for (int v = 0; v < kWarps; ++v) top = fmaxf(top, tops[v * S::kHeads + threadIdx.x]);
#pragma unroll
            for (int v = 0; v < kWarps; ++v) {
                const float m = tops[v * S::kHeads + threadIdx.x];
                if (m != -INFINITY) sum += totals[v * S::kHeads + threadIdx.x] * exp2_approx(m - top);
            }
            tops[threadIdx.x] = top;
            totals[threadIdx.x] = sum;
        }
        __syncthreads();
    }

    __device__ void write(uint32_t b, uint32_t head, uint32_t heads) const {
        const float* totals = stats + kWarps * S::kHeads;
        T* out = nz::device_ptr<T>(a.out) + b * a.out_stride[0];
        for (uint32_t i = threadIdx.x; i < heads * kDim; i += kThreads) {
            const uint32_t h = i / kDim, d = i % kDim;
            if (d >= a.dim) continue;
            const float total = totals[h];
            out[(head + h) * a.out_stride[1] + d] = from_float<T>(total == 0.0f ? 0.0f : sums[h * S::kSumStride + d] / total);
        }
        if (a.lse && threadIdx.x < heads) {
            const float total = totals[threadIdx.x];
            nz::device_ptr<float>(a.lse)[static_cast<uint64_t>(b) * a.heads + head + threadIdx.x] =
                total == 0.0f ? -INFINITY : (stats[threadIdx.x] + log2f(total)) * kLn2;
        }
    }

    // The same from the sums that the CTAs of a cluster hold, each CTA its
    // share of the elements, the CTAs added in order.
    __device__ void write_cluster(uint32_t b, uint32_t head, uint32_t heads, uint32_t rank, uint32_t ctas) const {
        __shared__ float peers[2][kMostCtas][S::kHeads];
        cluster_barrier();
        if (threadIdx.x < ctas * S::kHeads) {
            const uint32_t c = threadIdx.x / S::kHeads, h = threadIdx.x % S::kHeads;
            peers[0][c][h] = load_peer(stats + h, c);
            peers[1][c][h] = load_peer(stats + kWarps * S::kHeads + h, c);
        }
        __syncthreads();
        T* out = nz::device_ptr<T>(a.out) + b * a.out_stride[0];
        for (uint32_t i = rank * kThreads + threadIdx.x; i < heads * kDim; i += ctas * kThreads) {
            const uint32_t h = i / kDim, d = i % kDim;
            if (d >= a.dim) continue;
            float top = -INFINITY, x = 0.0f, total = 0.0f;
            for (uint32_t c = 0; c < ctas; ++c) top = fmaxf(top, peers[0][c][h]);
#pragma unroll 4
            for (uint32_t c = 0; c < ctas; ++c) {
                const float down = peers[0][c][h] == -INFINITY ? 0.0f : exp2_approx(peers[0][c][h] - top);
                x += load_peer(sums + h * S::kSumStride + d, c) * down;
                total += peers[1][c][h] * down;
            }
            out[(head + h) * a.out_stride[1] + d] = from_float<T>(total == 0.0f ? 0.0f : x / total);
            if (d == 0 && a.lse)
                nz::device_ptr<float>(a.lse)[static_cast<uint64_t>(b) * a.heads + head + h] =
                    total == 0.0f ? -INFINITY : (top + log2f(total)) * kLn2;
        }
        cluster_barrier();  // the others are done with this CTA's sums
    }

    __device__ void write_part(float* part) const {
        const float* totals = stats + kWarps * S::kHeads;
        for (uint32_t i = threadIdx.x; i < S::kHeads * kDim / 4U; i += kThreads)
            reinterpret_cast<float4*>(part)[i] =
                *reinterpret_cast<const float4*>(sums + (i / (kDim / 4U)) * S::kSumStride + (i % (kDim / 4U)) * 4U);
        if (threadIdx.x < S::kHeads) {
            part[S::kHeads * kDim + threadIdx.x] = stats[threadIdx.x];
            part[S::kHeads * (kDim + 1) + threadIdx.x] = totals[threadIdx.x];
        }
    }
};

__device__ __forceinline__ uint32_t chunk_count(const nz_attention& a, uint32_t b, uint32_t chunk) {
    const int32_t length = held_length(a, b);
    if (length == 0) return 0U;
    const uint32_t first = static_cast<uint32_t>(first_position(a, length)) / chunk;
    return (static_cast<uint32_t>(length) + chunk - 1U) / chunk - first;
}

// One CTA, or a cluster of up to kMostCtas, an item: (request, key/value
// head, group of query heads). A cluster's CTAs take runs of its chunks.
template <typename T, int kDim, int kHeadTiles, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) nz_paged_attention_direct(const nz_attention a, const Plan plan) {
    using S = Shape<T, kDim, kHeadTiles, kWarps>;
    extern __shared__ __align__(128) unsigned char shared[];
    nz::after_predecessor(plan.let_next);
    Attention<T, kDim, kHeadTiles, kWarps> run(a, shared);
    const uint32_t group = a.heads / a.kv_heads, items = a.kv_heads * plan.groups;
    const uint32_t rank = blockIdx.x % plan.cluster, unit = blockIdx.x / plan.cluster;
    const uint32_t b = unit / items, item = unit % items, k = item / plan.groups;
    const uint32_t first = (item % plan.groups) * S::kHeads, heads = min(group - first, static_cast<uint32_t>(S::kHeads));
    const int32_t length = held_length(a, b), start = first_position(a, length);
    const uint32_t count = chunk_count(a, b, S::kChunk), share = (count + plan.cluster - 1U) / plan.cluster;
    const uint32_t base = static_cast<uint32_t>(start) / S::kChunk;
    run.segment(b, k, k * group + first, heads, base + min(count, rank * share), base + min(count, (rank + 1U) * share),
                start, length);
    if (plan.cluster > 1)
        run.write_cluster(b, k * group + first, heads, rank, plan.cluster);
    else
        run.write(b, k * group + first, heads);
}

// The chunks of all items, request by request and item by item, in equal
// runs, one a CTA, whatever the lengths. A run may end inside an item; then
// its CTAs leave partial results to the join.
template <typename T, int kDim, int kHeadTiles>
__global__ void __launch_bounds__(kSplitWarps * 32, kDim <= 128 && kHeadTiles == 1 ? 3 : 1) nz_paged_attention_split(const nz_attention a, const Plan plan) {
    using S = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    constexpr int kWarps = kSplitWarps;
    constexpr uint32_t kThreads = S::kThreads;
    extern __shared__ __align__(128) unsigned char shared[];
    nz::after_predecessor(false);  // the join has nothing to do before
    Attention<T, kDim, kHeadTiles, kSplitWarps> run(a, shared);
    const uint32_t group = a.heads / a.kv_heads, items = a.kv_heads * plan.groups;

    // ends[b]: chunks of one item of requests 0 .. b.
    uint32_t* ends = reinterpret_cast<uint32_t*>(shared + S::kSharedBytes);
    __shared__ uint32_t warp_sums[kWarps];
    uint32_t carry = 0;
    for (uint32_t base = 0; base < a.requests; base += kThreads) {
        const uint32_t b = base + threadIdx.x;
        uint32_t sum = b < a.requests ? chunk_count(a, b, S::kChunk) : 0U;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t below = __shfl_up_sync(0xFFFFFFFFU, sum, d);
            if (run.lane >= d) sum += below;
        }
        if (run.lane == 31) warp_sums[run.warp] = sum;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
            if (v < static_cast<int>(run.warp)) sum += warp_sums[v];
            all += warp_sums[v];
        }
        if (b < a.requests) ends[b] = carry + sum;
        carry += all;
        __syncthreads();
    }
    const uint32_t total = carry * items;
    const uint32_t each = max(kLeastChunks, (total + plan.workers - 1U) / plan.workers);
    const uint32_t worker = blockIdx.x;
    const uint32_t begin = min(total, worker * each), end = min(total, begin + each);
    float* parts = nz::device_ptr<float>(a.workspace);
    Join* joins = reinterpret_cast<Join*>(parts + 2 * S::kPartFloats * plan.workers);
    Join join = {0U, 0U, 0U, 0U, 0U};

    // Requests with nothing to attend to, shared out among the CTAs.
    for (uint32_t b = worker; b < a.requests; b += plan.workers) {
        if (ends[b] != (b ? ends[b - 1] : 0U)) continue;
        if (plan.by_item)
            for (uint32_t i = threadIdx.x; i < items; i += kThreads) joins[b * items + i].parts = 0U;
        T* out = nz::device_ptr<T>(a.out) + b * a.out_stride[0];
        for (uint32_t i = threadIdx.x; i < a.heads * a.dim; i += kThreads)
            out[(i / a.dim) * a.out_stride[1] + i % a.dim] = from_float<T>(0.0f);
        if (a.lse)
            for (uint32_t h = threadIdx.x; h < a.heads; h += kThreads)
                nz::device_ptr<float>(a.lse)[static_cast<uint64_t>(b) * a.heads + h] = -INFINITY;
    }

    uint32_t b = 0, high = a.requests;  // the request of chunk `begin`
    while (b < high) {
        const uint32_t middle = (b + high) >> 1;
        if (ends[middle] * items > begin) high = middle; else b = middle + 1U;
    }
    for (uint32_t at = begin; at < end;) {
        while (ends[b] * items <= at) ++b;
        const uint32_t before = b ? ends[b - 1] : 0U, count = ends[b] - before;
        const uint32_t in = at - before * items, item = in / count, chunk = in % count;
        const uint32_t taken = min(count - chunk, end - at);
        const uint32_t k = item / plan.groups, first = (item % plan.groups) * S::kHeads;
        const uint32_t heads = min(group - first, static_cast<uint32_t>(S::kHeads));
        const int32_t length = held_length(a, b), start = first_position(a, length);
        const uint32_t base = static_cast<uint32_t>(start) / S::kChunk + chunk;
        run.segment(b, k, k * group + first, heads, base, base + taken, start, length);
        if (taken == count) {
            run.write(b, k * group + first, heads);
        } else {
            const uint32_t slot = at == begin ? 0U : 1U;
            run.write_part(parts + (2ULL * worker + slot) * S::kPartFloats);
            if (chunk == 0) {
                const uint32_t last = (at + count - 1U) / each;  // the worker of the item's last chunk
                join = {b, item, last - worker + 1U, worker, slot};
            }
        }
        if (plan.by_item && chunk == 0 && threadIdx.x == 0) {
            joins[b * items + item] = join;
            join.parts = 0U;
        }
        at += taken;
    }
    if (!plan.by_item && threadIdx.x == 0) joins[worker] = join;
}

// Adds up the partial results of a split item: 16 warps for 16 / shares
// query heads, the parts of a head dealt to `shares` warps. Parts are added
// in an order that the sizes alone fix, so results do not depend on timing.
constexpr uint32_t kJoinWarps = 16;

template <typename T, int kDim, int kHeadTiles>
__global__ void __launch_bounds__(kJoinWarps * 32) nz_paged_attention_join(const nz_attention a, const Plan plan) {
    using S = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    constexpr int kRun = kDim / 64;  // float2s of a lane
    constexpr uint32_t kBatch = 16 / kRun;
    __shared__ float sums[kJoinWarps][kDim];
    __shared__ float tops[kJoinWarps], totals[kJoinWarps];
    nz::after_predecessor();
    const float* parts = nz::device_ptr<const float>(a.workspace);
    const Join join = reinterpret_cast<const Join*>(parts + 2 * S::kPartFloats * plan.workers)[blockIdx.x];
    if (join.parts == 0) return;
    const uint32_t group = a.heads / a.kv_heads, k = join.item / plan.groups;
    const uint32_t from = (join.item % plan.groups) * S::kHeads, heads = min(group - from, static_cast<uint32_t>(S::kHeads));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31U, shares = plan.shares, each = kJoinWarps / shares;
    const uint32_t base = blockIdx.y * each;  // the CTA's first head
    if (base >= heads) return;
    const uint32_t h = base + warp / shares, share = warp % shares;
    const float* first = parts + (2ULL * join.worker + join.slot) * S::kPartFloats;
    auto part = [&](uint32_t i) { return i ? parts + 2ULL * (join.worker + i) * S::kPartFloats : first; };

    float top = -INFINITY, total = 0.0f;
    float2 sum[kRun];
#pragma unroll
    for (int r = 0; r < kRun; ++r) sum[r] = make_float2(0.0f, 0.0f);
    if (h < heads)
        for (uint32_t block = share; block < join.parts; block += 32U * shares) {  // up to 32 parts, a lane each
            const uint32_t mine = block + lane * shares, count = min(32U, (join.parts - block + shares - 1U) / shares);
            float m = -INFINITY, l = 0.0f;
            if (mine < join.parts) {
                m = part(mine)[S::kHeads * kDim + h];
                l = part(mine)[S::kHeads * (kDim + 1) + h];
            }
            float next = fmaxf(top, m);
#pragma unroll
            for (int d = 16; d; d >>= 1) next = fmaxf(next, __shfl_xor_sync(0xFFFFFFFFU, next, d));
            const float old = top == -INFINITY ? 0.0f : exp2_approx(top - next);
            const float weight = m == -INFINITY ? 0.0f : exp2_approx(m - next);
            top = next;
            total = total * old + l * weight;
#pragma unroll
            for (int r = 0; r < kRun; ++r) sum[r].x *= old, sum[r].y *= old;
            for (uint32_t i = 0; i < count; i += kBatch) {  // loaded together, so that they share one latency
                float2 x[kBatch][kRun];
#pragma unroll
                for (uint32_t j = 0; j < kBatch; ++j)
#pragma unroll
                    for (int r = 0; r < kRun; ++r)
                        x[j][r] = i + j < count ? *reinterpret_cast<const float2*>(part(block + (i + j) * shares) + h * kDim +
                                                                                   lane * 2 + r * 64)
                                                : make_float2(0.0f, 0.0f);
#pragma unroll
                for (uint32_t j = 0; j < kBatch; ++j) {
                    const float w = __shfl_sync(0xFFFFFFFFU, weight, (i + j) & 31U);  // 0 behind the last part
#pragma unroll
                    for (int r = 0; r < kRun; ++r) {
                        sum[r].x += x[j][r].x * w;
                        sum[r].y += x[j][r].y * w;
                    }
                }
            }
        }
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xFFFFFFFFU, total, d);
#pragma unroll
    for (int r = 0; r < kRun; ++r) *reinterpret_cast<float2*>(&sums[warp][r * 64 + lane * 2]) = sum[r];
    if (lane == 0) {
        tops[warp] = top;
        totals[warp] = total;
    }
    __syncthreads();
    T* out = nz::device_ptr<T>(a.out) + join.request * a.out_stride[0];
    for (uint32_t i = threadIdx.x; i < each * kDim; i += kJoinWarps * 32U) {
        const uint32_t q = i / kDim, d = i % kDim, head = k * group + from + base + q;
        if (base + q >= heads) break;
        float most = -INFINITY, x = 0.0f, all = 0.0f;
        for (uint32_t v = 0; v < shares; ++v) most = fmaxf(most, tops[q * shares + v]);
        for (uint32_t v = 0; v < shares; ++v) {
            const uint32_t w = q * shares + v;
            const float down = tops[w] == -INFINITY ? 0.0f : exp2_approx(tops[w] - most);
            x += sums[w][d] * down;
            all += totals[w] * down;
        }
        if (d < a.dim) out[head * a.out_stride[1] + d] = from_float<T>(all == 0.0f ? 0.0f : x / all);
        if (d == 0 && a.lse)
            nz::device_ptr<float>(a.lse)[static_cast<uint64_t>(join.request) * a.heads + head] =
                all == 0.0f ? -INFINITY : (most + log2f(all)) * kLn2;
    }
}

// ---- host ------------------------------------------------------------------------------

struct Device {
    int ctas_per_sm = 0;  // of the split kernel
    int sms = 0;
    int clusters[2][4] = {};  // of 1, 2, 4, 8 CTAs of the direct kernel that run at a time, with 4 and 8 warps
};

// How many clusters of each size run at a time: fewer than their CTAs alone
// would allow, as a cluster needs its SMs in one part of the GPU.
template <typename T, int kDim, int kHeadTiles, int kWarps>
cudaError_t count_clusters(int (&counts)[4]) {
    const auto kernel = nz_paged_attention_direct<T, kDim, kHeadTiles, kWarps>;
    constexpr size_t shared = Shape<T, kDim, kHeadTiles, kWarps>::kSharedBytes;
    cudaError_t err =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
    for (int i = 0; i < 4 && err == cudaSuccess; ++i) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(1U << i);
        config.blockDim = dim3(kWarps * 32);
        config.dynamicSmemBytes = shared;
        cudaLaunchAttribute attribute = {};
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = 1U << i;
        attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
        config.attrs = &attribute;
        config.numAttrs = 1;
        err = cudaOccupancyMaxActiveClusters(&counts[i], kernel, &config);
    }
    return err;
}

// The current device's limits, looked up (and the kernels' shared memory
// opted into) once a device.
template <typename T, int kDim, int kHeadTiles>
cudaError_t device_limits(Device* out) {
    static std::mutex lock;
    static Device known[64];
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> hold(lock);
    Device& d = known[device];
    if (!d.sms) {
        const auto split = nz_paged_attention_split<T, kDim, kHeadTiles>;
        constexpr int most = Shape<T, kDim, kHeadTiles, kSplitWarps>::kSharedBytes + NZ_PAGED_MAX_REQUESTS * sizeof(uint32_t);
        constexpr auto attribute = cudaFuncAttributeMaxDynamicSharedMemorySize;
        int sms = 0;
        err = cudaFuncSetAttribute(split, attribute, most);
        if (err == cudaSuccess) err = count_clusters<T, kDim, kHeadTiles, 4>(d.clusters[0]);
        if (err == cudaSuccess) err = count_clusters<T, kDim, kHeadTiles, 8>(d.clusters[1]);
        if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (err == cudaSuccess)
            err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&d.ctas_per_sm, split, kSplitWarps * 32, most);
        if (err != cudaSuccess) return err;
        if (d.ctas_per_sm < 1) return cudaErrorInvalidConfiguration;
        d.sms = sms;
    }
    *out = d;
    return cudaSuccess;
}

// Most chunks that one request can attend to.
uint64_t most_chunks(const nz_attention& a, uint64_t chunk) {
    const uint64_t capacity = static_cast<uint64_t>(a.width) << a.page_shift;
    const uint64_t span = a.window && a.window < capacity ? a.window + chunk - 1 : capacity;  // a window ends anywhere
    return (span + chunk - 1) / chunk;
}

// A launch of one CTA or cluster an item: clusters as large as there are
// chunks, until the CTAs fill the GPU or not all clusters would run at once
// (16 of 8 CTAs, an SM each: 23 us in two waves where 8 of them take 11).
struct Direct {
    uint32_t warps, cluster;
    uint64_t passes;  // of a CTA over its chunks

    Direct(const nz_attention& a, uint64_t items, const Device& device, uint32_t warps_) : warps(warps_), cluster(1) {
        const uint64_t chunks = most_chunks(a, kTile * warps), sms = device.sms;
        const int* most = device.clusters[warps == 8];
        for (int i = 1; cluster < kMostCtas && cluster < chunks && items * cluster < sms && items <= static_cast<uint64_t>(most[i]); ++i)
            cluster *= 2;
        passes = (chunks + cluster - 1) / cluster;
    }
};

// The kernel for these sizes, by what a row of the block table (or the
// window) can hold, since the lengths are on the GPU. (Times of kernels that
// follow one another without overlap; as dependents they take 0.2 us less.)
// 4 warps a CTA, where items alone fill the GPU (512 items of 1024
// positions, 8 key/value heads of 128 in bf16: 40 us, 44 with 8 warps), or
// where a cluster then still reads all in as few passes (8 items of 1024:
// 5.7 us, 6.6); else 8 (8 items of 256, one CTA each: 5.2 us, 5.8 as two of
// 4 warps; of 4096: 8.8, 10.3).
// Split, where a CTA would make many passes: more the more CTAs there are,
// as the joining launch is shared by more work (8 items of 8192: 12.6 us
// direct, 13.2 split; of 16384: 23.6, 21.4; 2 items of 16384: 15.3, 10.0;
// 64 items of 8192: 42.8, 47.5; 512 items of 2048: 76.7, 86.8; fp32 with
// shared heads, 16 items of 8192: 47, 35).
template <typename T, int kDim, int kHeadTiles>
cudaError_t launch(const nz_attention& a, cudaStream_t stream, uint64_t* workspace_only) {
    using S = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    Device device;
    cudaError_t err = device_limits<T, kDim, kHeadTiles>(&device);
    if (err != cudaSuccess) return err;
    const uint32_t group = a.heads / a.kv_heads;
    Plan plan = {0U, (group + S::kHeads - 1U) / S::kHeads, 0U, 2U, 1U, 0U};
    const uint64_t items = static_cast<uint64_t>(a.requests) * a.kv_heads * plan.groups, sms = device.sms;
    const Direct few(a, items, device, 4), many(a, items, device, 8);
    const bool alone = many.cluster == 1 && few.cluster > 1 && many.passes <= few.passes;
    const Direct& direct = items < sms && (many.passes < few.passes || alone) ? many : few;
    constexpr bool kSlow = S::kWide && S::kHeads > 1;  // bound by its arithmetic, which the split spreads evenly
    const uint64_t ctas = items * direct.cluster, most_passes = kSlow || ctas < 32 ? 2 : ctas < 128 ? 4 : 8;
    if (direct.passes * direct.warps > most_passes * 8) {
        const uint64_t all = most_chunks(a, S::kChunk) * items, resident = sms * device.ctas_per_sm;
        plan.workers = static_cast<uint32_t>(all < resident ? all : resident);
        plan.by_item = items <= plan.workers;
        const uint64_t parts = plan.workers / items;  // of an item, where lengths are alike
        plan.shares = parts <= 4 ? 2 : parts <= 16 ? 4 : parts <= 64 ? 8 : 16;
    }
    const uint64_t workspace = plan.workers * (2 * S::kPartFloats * sizeof(float) + sizeof(Join));
    if (workspace_only) {
        *workspace_only = workspace;
        return cudaSuccess;
    }
    if (plan.workers == 0) {
        plan.cluster = direct.cluster;
        // Over several waves of CTAs the next kernel's would crowd these (512 items of 2048: 78 us, 74 without).
        plan.let_next = ctas <= 2 * sms;
        const uint32_t grid = static_cast<uint32_t>(ctas);
        if (direct.warps == 4) {
            const nz::PagedLaunch l(grid, 1, 128, Shape<T, kDim, kHeadTiles, 4>::kSharedBytes, stream, plan.cluster);
            return cudaLaunchKernelEx(&l.config, nz_paged_attention_direct<T, kDim, kHeadTiles, 4>, a, plan);
        }
        const nz::PagedLaunch l(grid, 1, 256, Shape<T, kDim, kHeadTiles, 8>::kSharedBytes, stream, plan.cluster);
        return cudaLaunchKernelEx(&l.config, nz_paged_attention_direct<T, kDim, kHeadTiles, 8>, a, plan);
    }
    if (!a.workspace) return cudaErrorInvalidValue;
    const nz::PagedLaunch split(plan.workers, 1, S::kThreads, S::kSharedBytes + a.requests * sizeof(uint32_t), stream, 1);
    err = cudaLaunchKernelEx(&split.config, nz_paged_attention_split<T, kDim, kHeadTiles>, a, plan);
    if (err != cudaSuccess) return err;
    const uint32_t heads = group < S::kHeads ? group : S::kHeads, each = kJoinWarps / plan.shares;
    const nz::PagedLaunch join(plan.by_item ? static_cast<uint32_t>(items) : plan.workers, (heads + each - 1U) / each,
                               kJoinWarps * 32, 0, stream, 1);
    return cudaLaunchKernelEx(&join.config, nz_paged_attention_join<T, kDim, kHeadTiles>, a, plan);
}

template <typename T>
cudaError_t dispatch(const nz_attention& a, cudaStream_t stream, uint64_t* workspace_only) {
    const bool one = a.heads / a.kv_heads <= (sizeof(T) == 4 ? 1U : 8U);
    if (a.dim <= 64) return one ? launch<T, 64, 1>(a, stream, workspace_only) : launch<T, 64, 2>(a, stream, workspace_only);
    if (a.dim <= 128) return one ? launch<T, 128, 1>(a, stream, workspace_only) : launch<T, 128, 2>(a, stream, workspace_only);
    if (a.dim <= 192) return one ? launch<T, 192, 1>(a, stream, workspace_only) : launch<T, 192, 2>(a, stream, workspace_only);
    return one ? launch<T, 256, 1>(a, stream, workspace_only) : launch<T, 256, 2>(a, stream, workspace_only);
}

int attention(const nz_attention* args, cudaStream_t stream, uint64_t* workspace_only) {
    if (!args) return nz::paged_fail("Null arguments.");
    nz_attention a = *args;
    if (a.pages == 0) a.width = 0;  // no page id is good: nothing to attend to
    if (a.dim == 0 || a.dim > NZ_PAGED_MAX_DIM || a.dim % 8)
        return nz::paged_fail("The head width must be a multiple of 8 up to 256.");
    if (a.kv_heads == 0 || a.heads == 0 || a.heads % a.kv_heads || a.heads > 65536)
        return nz::paged_fail("The query heads must be a multiple of the key/value heads.");
    if (a.requests > NZ_PAGED_MAX_REQUESTS) return nz::paged_fail("At most 4096 requests.");
    if (!nz::paged_sizes_fit(a.pages, a.width, a.page_shift))
        return nz::paged_fail("A cache and a block-table row hold fewer than 2^30 pages and 2^31 tokens.");
    if (a.dtype > NZ_PAGED_FP32) return nz::paged_fail("The type must be bf16, fp16 or fp32.");
    // Chunks (of at least 64 positions) are counted in 32 bits.
    if (((static_cast<uint64_t>(a.width) << a.page_shift) / 64 + 1) * a.requests * a.heads > INT32_MAX)
        return nz::paged_fail("requests * heads * block-table row must stay below 2^37 tokens.");
    if (a.requests == 0) {
        if (workspace_only) *workspace_only = 0;
        return NZ_OK;
    }
    const uint64_t size = a.dtype == NZ_PAGED_FP32 ? 4 : 2;
    uint64_t starts = a.key_pages | a.value_pages | a.workspace;
    const bool stepped[3] = {a.pages > 1, a.page_shift > 0, a.kv_heads > 1};
    for (int i = 0; i < 3; ++i)
        if (stepped[i]) starts |= static_cast<uint64_t>(a.key_stride[i] | a.value_stride[i]) * size;
    if (!workspace_only && starts % 16) return nz::paged_fail("Key and value rows and the workspace must start on 16-byte boundaries.");
    if (!workspace_only && (!a.query || !a.out || !a.lengths || (a.width && !a.block_table) ||
                            (a.pages && (!a.key_pages || !a.value_pages))))
        return nz::paged_fail("Null device array.");
    cudaError_t err;
    switch (a.dtype) {
        case NZ_PAGED_BF16: err = dispatch<__nv_bfloat16>(a, stream, workspace_only); break;
        case NZ_PAGED_FP16: err = dispatch<__half>(a, stream, workspace_only); break;
        default: err = dispatch<float>(a, stream, workspace_only); break;
    }
    return nz::cuda_status(err, "nz_paged_attention");
}

}  // namespace

extern "C" {

int nz_paged_attention_workspace(const nz_attention* args, uint64_t* bytes) {
    if (!bytes) return nz::paged_fail("Null output.");
    return attention(args, nullptr, bytes);
}

int nz_paged_attention(const nz_attention* args, void* cuda_stream) {
    return attention(args, reinterpret_cast<cudaStream_t>(cuda_stream), nullptr);
}

}  // extern "C"
