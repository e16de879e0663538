// Attention of one new token a request over its pages of the cache.
//
// For request b with n tokens, key/value head k and the query heads h that
// share it: s_j = scale * q_h . K_j over the live positions j,
//   out_h = sum_j exp(s_j - max s) V_j / sum_j exp(s_j - max s),
// with the maximum and the sum kept running in 32 bits, so that every key
// and value is read once. Keys and values are all there is to read: the
// kernel is bound by HBM, and by latency where they are few.
//
// Products. A warp takes tiles of 16 or 32 positions of one key/value head.
// Keys and values are the left operand of mma.sync (16 positions, or 16
// elements of the head, by 16) and the up to 8 query heads of a group the
// right one, so that no half-empty tile is multiplied:
//   S^T = K Q^T (positions x heads),  O^T += V^T P^T (elements x heads).
// A left operand of 128 rows, as tcgen05.mma takes, would have to go through
// shared memory; here keys and values go from global memory straight into
// the registers of the mma that uses them. A dot product may sum its terms
// in any order and the rows of O^T may be any elements, so each lane loads
// 16 consecutive bytes of a row: 64 bytes of a key row in 4 lanes, 128 of a
// value row in 8. Pairs of values of two positions are put together with
// byte permutes, P^T is turned with movmatrix.
//
// Precision. 16-bit types: the products are exact, the sums 32-bit; P is
// split into two 16-bit parts (16 or more bits of each weight), because one
// rounding of P would cost as much as the rounding of the result. fp32: each
// operand is split into two tf32 parts and three products are summed (the
// product of the two low parts, 2^-22, is left out); partial sums of 16
// terms leave the tensor core, whose accumulation rounds towards zero,
// and are added in ordinary 32-bit arithmetic.

#include "nz_paged.h"

#include <mutex>
#include <type_traits>

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kDirectWarps = 8, kSplitWarps = 4;
// A block-table row of at most this many chunks gets one CTA a (request,
// head group) and no join.
constexpr uint32_t kDirectChunks = 8;
// Fewest chunks of a CTA where the work is split.
constexpr uint32_t kLeastChunks = 2;

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

// 16 bytes that no other CTA reads again soon.
__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 x;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "l"(p));
    return x;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, float) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t tf32_of(float x) {
    uint32_t y;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
    return y;
}
// x = high + low, each with tf32's 11 significant bits, to 2^-22 of x.
__device__ __forceinline__ void split(uint32_t x, uint32_t& high, uint32_t& low) {
    high = tf32_of(__uint_as_float(x));
    low = tf32_of(__uint_as_float(x) - __uint_as_float(high));
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
// 8 query heads. Rows are read in units of at most 256 bytes of each
// position (32 registers a lane); two units are in registers at a time,
// one used and one on its way.
template <typename T, int kDim, int kHeadTiles, int kWarps_>
struct Shape {
    static constexpr int kWarps = kWarps_;
    static constexpr uint32_t kThreads = kWarps * 32;
    static constexpr int kSize = sizeof(T);
    static constexpr int kUnit = kSize == 4 || kDim % 128 ? 64 : 128;        // elements of a unit
    static constexpr int kUnits = kDim / kUnit;                              // of a tile's keys, and of its values
    static constexpr int kUnitBytes = kUnit * kSize;                         // 128 or 256
    static constexpr int kSteps = 256 / kUnitBytes;                          // 16-position steps of a tile
    static constexpr int kTile = 16 * kSteps;                                // positions of a tile
    static constexpr int kChunk = kTile * kWarps;                            // positions of a CTA's pass
    static constexpr int kKeyBlocks = kUnitBytes / 64;                       // of 64 bytes
    static constexpr int kValueBlocks = kUnitBytes / 128;                    // of 128 bytes
    static constexpr int kVectors = 2 * kKeyBlocks;                          // 16-byte vectors of a step's unit
    static constexpr int kLaneElems = 16 / kSize;                            // elements of a vector
    static constexpr int kHeads = 8 * kHeadTiles;
    static constexpr int kQueryBlocks = kDim * kSize / 64;
    static constexpr int kQueryParts = kSize == 4 ? 2 : 1;
    static constexpr int kRowTiles = kDim / 16;                              // 16-element tiles of O^T
    static constexpr int kSumStride = kDim + 4;
    static constexpr size_t kQueryBytes = static_cast<size_t>(kQueryParts) * kHeadTiles * kQueryBlocks * 32 * 16;
    static constexpr size_t kSumBytes = static_cast<size_t>(kWarps) * kHeads * kSumStride * 4;
    static constexpr size_t kStatBytes = 2 * kWarps * kHeads * 4;
    static constexpr size_t kSharedBytes = kQueryBytes + kSumBytes + kStatBytes;
    static constexpr size_t kPartFloats = static_cast<size_t>(kHeads) * (kDim + 2);  // a partial result
};

// What a split launch adds: the number of CTAs ("workers"), and its
// workspace: two partial results a worker, then one Join a worker.
struct Join {
    uint32_t request, item;  // item: (key/value head, group of kHeads query heads)
    uint32_t parts;          // of workers w, w + 1, ...; 0: nothing that starts here is split
    uint32_t slot;           // of worker w's part (the others' is 0)
};

struct Plan {
    uint32_t workers;   // CTAs of a split launch
    uint32_t groups;    // of kHeads query heads that share a key/value head
};

__device__ __forceinline__ int32_t held_length(const nz_attention& a, uint32_t b) {
    const int32_t n = nz::device_ptr<const int32_t>(a.lengths)[b];
    return max(0, min(n, static_cast<int32_t>(a.width << a.page_shift)));
}
__device__ __forceinline__ int32_t first_position(const nz_attention& a, int32_t length) {
    return a.window && static_cast<uint32_t>(length) > a.window ? length - static_cast<int32_t>(a.window) : 0;
}

template <typename T, int kDim, int kHeadTiles, int kWarps_>
struct Attention {
    using S = Shape<T, kDim, kHeadTiles, kWarps_>;
    static constexpr int kWarps = S::kWarps;
    static constexpr uint32_t kThreads = S::kThreads;

    const nz_attention& a;
    uint4* query;      // shared: fragments [part][head tile][block][lane]
    float* sums;       // shared: [warp][head][kSumStride]
    float* stats;      // shared: [2][warp][head]
    uint32_t warp, lane, row, col;

    __device__ Attention(const nz_attention& args, unsigned char* shared) : a(args) {
        query = reinterpret_cast<uint4*>(shared);
        sums = reinterpret_cast<float*>(shared + S::kQueryBytes);
        stats = reinterpret_cast<float*>(shared + S::kQueryBytes + S::kSumBytes);
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31U;
        row = lane >> 2;
        col = lane & 3U;
    }

    // Query heads [head, head + heads) of request b as right operands: lane
    // (row, col) holds 16 bytes of head `row`, zeros behind the last head
    // and the head's width.
    __device__ void load_query(uint32_t b, uint32_t head, uint32_t heads) {
        const T* source = nz::device_ptr<const T>(a.query) + b * a.query_stride[0];
        for (uint32_t i = threadIdx.x; i < kHeadTiles * S::kQueryBlocks * 32U; i += kThreads) {
            const uint32_t at = i & 31U, block = (i >> 5) % S::kQueryBlocks, tile = (i >> 5) / S::kQueryBlocks;
            const uint32_t h = tile * 8U + (at >> 2), d = (block * 4U + (at & 3U)) * S::kLaneElems;
            alignas(16) T x[S::kLaneElems];
#pragma unroll
            for (int e = 0; e < S::kLaneElems; ++e)
                x[e] = h < heads && d + e < a.dim ? source[(head + h) * a.query_stride[1] + d + e] : T(0.0f);
            if constexpr (S::kSize == 4) {
                uint32_t high[4], low[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split(__float_as_uint(x[e]), high[e], low[e]);
                query[i] = make_uint4(high[0], high[1], high[2], high[3]);
                query[i + kHeadTiles * S::kQueryBlocks * 32] = make_uint4(low[0], low[1], low[2], low[3]);
            } else {
                query[i] = *reinterpret_cast<const uint4*>(x);
            }
        }
    }

    // Page of the lane's position of a tile, -1 where nothing is to be read.
    __device__ int32_t page_of(const int32_t* table, uint32_t tile, uint32_t tiles, int32_t start, int32_t length) const {
        const int32_t position = static_cast<int32_t>(tile * S::kTile + (lane & (S::kTile - 1U)));
        int32_t page = -1;
        if (tile < tiles && position >= start && position < length) {
            page = table[position >> a.page_shift];
            if (page < 0 || static_cast<uint32_t>(page) >= a.pages) page = -1;
        }
        return page;
    }

    using Unit = uint4[S::kSteps][S::kVectors];

    __device__ void load_row(uint4& x, const T* base, const int64_t (&stride)[3], uint32_t tile, uint32_t place,
                             int32_t page, uint32_t element) const {
        x = make_uint4(0U, 0U, 0U, 0U);
        if (page >= 0 && element < a.dim) {
            const uint32_t line = (tile * S::kTile + place) & ((1U << a.page_shift) - 1U);
            x = load_stream(base + page * stride[0] + line * stride[1] + element);
        }
    }

    // Unit u of a tile's keys: vector 2 * block + half is 16 bytes of
    // position row + 8 * half.
    __device__ void load_keys(Unit& x, const T* keys, uint32_t tile, int32_t pages, int u) const {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t place = s * 16 + half * 8 + row;
                const int32_t page = __shfl_sync(0xFFFFFFFFU, pages, place);
#pragma unroll
                for (int block = 0; block < S::kKeyBlocks; ++block)
                    load_row(x[s][2 * block + half], keys, a.key_stride, tile, place, page,
                             u * S::kUnit + (block * 4 + col) * S::kLaneElems);
            }
    }

    // The position, within a step, of vector i of a value block: what the
    // mma's left operand holds in the lane's column.
    __device__ uint32_t value_place(int i) const {
        return S::kSize == 4 ? col + 4U * i : 2U * col + (i & 1) + 8U * (i >> 1);
    }

    // Unit u of a tile's values: vector 4 * block + i is 16 bytes of position value_place(i).
    __device__ void load_values(Unit& x, const T* values, uint32_t tile, int32_t pages, int u) const {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t place = s * 16 + value_place(i);
                const int32_t page = __shfl_sync(0xFFFFFFFFU, pages, place);
#pragma unroll
                for (int block = 0; block < S::kValueBlocks; ++block)
                    load_row(x[s][4 * block + i], values, a.value_stride, tile, place, page,
                             u * S::kUnit + (block * 8 + row) * S::kLaneElems);
            }
    }

    // S^T += K Q^T over unit u.
    __device__ void scores(float (&s)[S::kSteps][kHeadTiles][4], const Unit& x, int u) const {
#pragma unroll
        for (int block = 0; block < S::kKeyBlocks; ++block) {
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t) {
                const uint32_t at = (t * S::kQueryBlocks + u * S::kKeyBlocks + block) * 32U + lane;
                const uint4 q = query[at];
                if constexpr (S::kSize == 4) {
                    const uint4 low = query[at + kHeadTiles * S::kQueryBlocks * 32];
#pragma unroll
                    for (int step = 0; step < S::kSteps; ++step) {
                        const uint4 &k0 = x[step][2 * block], &k1 = x[step][2 * block + 1];
                        uint32_t h[8], l[8];
                        split(k0.x, h[0], l[0]), split(k1.x, h[1], l[1]), split(k0.y, h[2], l[2]), split(k1.y, h[3], l[3]);
                        split(k0.z, h[4], l[4]), split(k1.z, h[5], l[5]), split(k0.w, h[6], l[6]), split(k1.w, h[7], l[7]);
                        float part[3][4] = {};
                        mma(part[0], h[0], h[1], h[2], h[3], q.x, q.y, T());
                        mma(part[1], l[0], l[1], l[2], l[3], q.x, q.y, T());
                        mma(part[2], h[0], h[1], h[2], h[3], low.x, low.y, T());
                        mma(part[0], h[4], h[5], h[6], h[7], q.z, q.w, T());
                        mma(part[1], l[4], l[5], l[6], l[7], q.z, q.w, T());
                        mma(part[2], h[4], h[5], h[6], h[7], low.z, low.w, T());
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[step][t][i] += part[0][i] + (part[1][i] + part[2][i]);
                    }
                } else {
#pragma unroll
                    for (int step = 0; step < S::kSteps; ++step) {
                        const uint4 &k0 = x[step][2 * block], &k1 = x[step][2 * block + 1];
                        mma(s[step][t], k0.x, k1.x, k0.y, k1.y, q.x, q.y, T());
                        mma(s[step][t], k0.z, k1.z, k0.w, k1.w, q.z, q.w, T());
                    }
                }
            }
        }
    }

    // Weights as right operands: [step][head tile][part][2].
    static constexpr int kWeightParts = 2;
    static constexpr int kWeightRegs = S::kSize == 4 ? 4 : 2;
    using Weights = uint32_t[S::kSteps][kHeadTiles][kWeightParts][kWeightRegs];

    __device__ void weights(Weights& w, const float (&p)[S::kSteps][kHeadTiles][4]) const {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t) {
                const float* x = p[s][t];
                if constexpr (S::kSize == 4) {
                    // Register i: position col + 4 * i of head `row`, held by lane 4 * position + row / 2.
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t from = 4U * (col + 4U * (i & 1)) + (row >> 1);
                        const float even = __shfl_sync(0xFFFFFFFFU, x[i < 2 ? 0 : 2], from);
                        const float odd = __shfl_sync(0xFFFFFFFFU, x[i < 2 ? 1 : 3], from);
                        split(__float_as_uint(row & 1U ? odd : even), w[s][t][0][i], w[s][t][1][i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t high = pack(x[2 * i], x[2 * i + 1], T());
                        const float2 back = unpack(high, T());
                        w[s][t][0][i] = transposed(high);
                        w[s][t][1][i] = transposed(pack(x[2 * i] - back.x, x[2 * i + 1] - back.y, T()));
                    }
                }
            }
    }

    // O^T += V^T P^T for the elements of unit u.
    __device__ void products(float (&o)[S::kRowTiles][kHeadTiles][4], const Unit& x, const Weights& w, int u) const {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
            for (int block = 0; block < S::kValueBlocks; ++block) {
                const uint4* v = &x[s][4 * block];
                if constexpr (S::kSize == 4) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t h[8], l[8];  // [position i][element 2j, 2j + 1]
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            split(j ? v[i].z : v[i].x, h[2 * i], l[2 * i]);
                            split(j ? v[i].w : v[i].y, h[2 * i + 1], l[2 * i + 1]);
                        }
#pragma unroll
                        for (int t = 0; t < kHeadTiles; ++t) {
                            float part[3][4] = {};
                            const uint32_t(&high)[4] = w[s][t][0];
                            const uint32_t(&low)[4] = w[s][t][1];
                            mma(part[0], h[0], h[1], h[2], h[3], high[0], high[1], T());
                            mma(part[1], l[0], l[1], l[2], l[3], high[0], high[1], T());
                            mma(part[2], h[0], h[1], h[2], h[3], low[0], low[1], T());
                            mma(part[0], h[4], h[5], h[6], h[7], high[2], high[3], T());
                            mma(part[1], l[4], l[5], l[6], l[7], high[2], high[3], T());
                            mma(part[2], h[4], h[5], h[6], h[7], low[2], low[3], T());
                            float* to = o[(u * S::kValueBlocks + block) * 2 + j][t];
#pragma unroll
                            for (int i = 0; i < 4; ++i) to[i] += part[0][i] + (part[1][i] + part[2][i]);
                        }
                    }
                } else {
                    const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&v[0]);
                    const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&v[1]);
                    const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&v[2]);
                    const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&v[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t a0 = __byte_perm(v0[j], v1[j], 0x5410), a1 = __byte_perm(v0[j], v1[j], 0x7632);
                        const uint32_t a2 = __byte_perm(v2[j], v3[j], 0x5410), a3 = __byte_perm(v2[j], v3[j], 0x7632);
#pragma unroll
                        for (int t = 0; t < kHeadTiles; ++t) {
                            float(&to)[4] = o[(u * S::kValueBlocks + block) * 4 + j][t];
                            mma(to, a0, a1, a2, a3, w[s][t][1][0], w[s][t][1][1], T());
                            mma(to, a0, a1, a2, a3, w[s][t][0][0], w[s][t][0][1], T());
                        }
                    }
                }
            }
    }

    // The first element of the lane's run of O^T's row tile (its rows `row`
    // and `row` + 8 are that element and the next).
    __device__ uint32_t element_of(int tile) const {
        if constexpr (S::kSize == 4) return (tile / 2) * 32 + row * 4 + (tile % 2) * 2;
        else return (tile / 4) * 64 + row * 8 + (tile % 4) * 2;
    }

    // Chunks [chunk, chunk_end) of request b for query heads [head, head +
    // heads) of key/value head k: the joined sums of the CTA's warps end in
    // sums[0] (relative to the maximum), the maximum (of scores times
    // log2 e) and the denominator in stats[0][0] and stats[1][0].
    __device__ void segment(uint32_t b, uint32_t k, uint32_t head, uint32_t heads, uint32_t chunk, uint32_t chunk_end,
                            int32_t start, int32_t length) {
        const int32_t* table = nz::device_ptr<const int32_t>(a.block_table) + b * a.table_stride;
        const T* keys = nz::device_ptr<const T>(a.key_pages) + k * a.key_stride[2];
        const T* values = nz::device_ptr<const T>(a.value_pages) + k * a.value_stride[2];
        const uint32_t tiles = min(chunk_end * kWarps, (static_cast<uint32_t>(length) + S::kTile - 1U) / S::kTile);
        const float scale = a.scale * kLog2e;

        float o[S::kRowTiles][kHeadTiles][4], most[kHeadTiles][2], total[kHeadTiles][2];
#pragma unroll
        for (int i = 0; i < S::kRowTiles; ++i)
#pragma unroll
            for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][t][e] = 0.0f;
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                most[t][e] = -INFINITY;
                total[t][e] = 0.0f;
            }

        // The first loads are on their way before the query is there.
        uint32_t tile = chunk * kWarps + warp;
        Unit x[2];
        int32_t pages = page_of(table, tile, tiles, start, length);
        int32_t after = page_of(table, tile + kWarps, tiles, start, length);
        load_keys(x[0], keys, tile, pages, 0);
        if constexpr (S::kUnits > 1) load_keys(x[1], keys, tile, pages, 1);
        else load_values(x[1], values, tile, pages, 0);
        __syncthreads();  // the previous segment's shared memory is free
        load_query(b, head, heads);
        __syncthreads();
        {
            for (; tile < tiles; tile += kWarps) {
                const uint32_t next = tile + kWarps;
                const int32_t here = pages;
                float s[S::kSteps][kHeadTiles][4];
                Weights w;
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
                    for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[i][t][e] = 0.0f;
#pragma unroll
                for (int u = 0; u < 2 * S::kUnits; ++u) {
                    if (u < S::kUnits) scores(s, x[u % 2], u);
                    else products(o, x[u % 2], w, u - S::kUnits);
                    // The unit after next takes the registers of the one just used.
                    const int ahead = u + 2;
                    if (ahead == 2 * S::kUnits) {
                        pages = after;
                        after = page_of(table, next + kWarps, tiles, start, length);
                    }
                    if (ahead < S::kUnits) load_keys(x[u % 2], keys, tile, here, ahead);
                    else if (ahead < 2 * S::kUnits) load_values(x[u % 2], values, tile, here, ahead - S::kUnits);
                    else if (ahead - 2 * S::kUnits < S::kUnits) load_keys(x[u % 2], keys, next, pages, ahead - 2 * S::kUnits);
                    else load_values(x[u % 2], values, next, pages, ahead - 3 * S::kUnits);
                    if (u == S::kUnits - 1) softmax(s, w, o, most, total, here, scale);
                }
            }
        }
        join_warps(o, most, total);
    }

    // Masks and weighs a tile's scores; rescales the sums when a maximum rose.
    __device__ void softmax(float (&s)[S::kSteps][kHeadTiles][4], Weights& w, float (&o)[S::kRowTiles][kHeadTiles][4],
                            float (&most)[kHeadTiles][2], float (&total)[kHeadTiles][2], int32_t pages, float scale) const {
        float top[kHeadTiles][2];
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t) top[t][0] = most[t][0], top[t][1] = most[t][1];
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const bool live = __shfl_sync(0xFFFFFFFFU, pages, i * 16 + half * 8 + row) >= 0;
#pragma unroll
                for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[i][t][2 * half + e];
                        x = live ? x * scale : -INFINITY;
                        top[t][e] = fmaxf(top[t][e], x);
                    }
            }
        bool rose = false;
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[t][e] = fmaxf(top[t][e], __shfl_xor_sync(0xFFFFFFFFU, top[t][e], d));
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
                for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float& x = s[i][t][2 * half + e];
                        x = exp2_approx(x - base);
                        total[t][e] += x;
                    }
            }
        weights(w, s);
    }

    __device__ void join_warps(float (&o)[S::kRowTiles][kHeadTiles][4], const float (&most)[kHeadTiles][2],
                               float (&total)[kHeadTiles][2]) {
        float* tops = stats;
        float* totals = stats + kWarps * S::kHeads;
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
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kHeadTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t h = t * 8 + 2 * col + e;
                float top = -INFINITY;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) top = fmaxf(top, tops[v * S::kHeads + h]);
                const float down = most[t][e] == -INFINITY ? 0.0f : exp2_approx(most[t][e] - top);
                float* to = sums + (warp * S::kHeads + h) * S::kSumStride;
#pragma unroll
                for (int i = 0; i < S::kRowTiles; ++i)
                    *reinterpret_cast<float2*>(to + element_of(i)) = make_float2(o[i][t][e] * down, o[i][t][2 + e] * down);
            }
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

// One CTA an item: (request, key/value head, group of query heads).
template <typename T, int kDim, int kHeadTiles>
__global__ void __launch_bounds__(kDirectWarps * 32) nz_paged_attention_direct(const nz_attention a, const Plan plan) {
    using S = Shape<T, kDim, kHeadTiles, kDirectWarps>;
    extern __shared__ __align__(16) unsigned char shared[];
    Attention<T, kDim, kHeadTiles, kDirectWarps> run(a, shared);
    const uint32_t group = a.heads / a.kv_heads, items = a.kv_heads * plan.groups;
    const uint32_t b = blockIdx.x / items, item = blockIdx.x % items, k = item / plan.groups;
    const uint32_t first = (item % plan.groups) * S::kHeads, heads = min(group - first, static_cast<uint32_t>(S::kHeads));
    const int32_t length = held_length(a, b), start = first_position(a, length);
    const uint32_t chunk = static_cast<uint32_t>(start) / S::kChunk;
    run.segment(b, k, k * group + first, heads, chunk, chunk + chunk_count(a, b, S::kChunk), start, length);
    run.write(b, k * group + first, heads);
}

// The chunks of all items, request by request and item by item, in equal
// runs, one a CTA, whatever the lengths. A run may end inside an item; then
// its CTAs leave partial results to the join.
template <typename T, int kDim, int kHeadTiles>
__global__ void __launch_bounds__(kSplitWarps * 32) nz_paged_attention_split(const nz_attention a, const Plan plan) {
    using S = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    constexpr int kWarps = kSplitWarps;
    constexpr uint32_t kThreads = S::kThreads;
    extern __shared__ __align__(16) unsigned char shared[];
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
    Join join = {0U, 0U, 0U, 0U};

    // Requests with nothing to attend to, shared out among the CTAs.
    for (uint32_t b = worker; b < a.requests; b += plan.workers) {
        if (ends[b] != (b ? ends[b - 1] : 0U)) continue;
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
                join = {b, item, last - worker + 1U, slot};
            }
        }
        at += taken;
    }
    if (threadIdx.x == 0) joins[worker] = join;
}

// Adds up the partial results of the item that starts, split, in worker
// blockIdx.x's run: 32 warps, a query head each (and, with 8 heads, a
// quarter of the parts), in worker order, so that results do not depend on
// timing.
template <typename T, int kDim, int kHeadTiles>
__global__ void __launch_bounds__(1024) nz_paged_attention_join(const nz_attention a, const Plan plan) {
    using S = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    constexpr uint32_t kShares = 32 / S::kHeads;
    __shared__ float sums[kShares][S::kHeads][kDim];
    __shared__ float tops[kShares][S::kHeads], totals[kShares][S::kHeads];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float* parts = nz::device_ptr<const float>(a.workspace);
    const Join join = reinterpret_cast<const Join*>(parts + 2 * S::kPartFloats * plan.workers)[blockIdx.x];
    if (join.parts == 0) return;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31U, h = warp % S::kHeads, share = warp / S::kHeads;
    const float* mine = parts + 2ULL * blockIdx.x * S::kPartFloats;
    const float* first = mine + join.slot * S::kPartFloats;
    auto part = [&](uint32_t i) { return i ? mine + 2ULL * i * S::kPartFloats : first; };

    float top = -INFINITY;
    for (uint32_t i = lane; i < join.parts; i += 32U) top = fmaxf(top, part(i)[S::kHeads * kDim + h]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFU, top, d));
    constexpr int kRun = kDim / 64;  // float2s of a lane
    float2 sum[kRun];
#pragma unroll
    for (int r = 0; r < kRun; ++r) sum[r] = make_float2(0.0f, 0.0f);
    float total = 0.0f;
#pragma unroll 4
    for (uint32_t i = share; i < join.parts; i += kShares) {
        const float* p = part(i);
        const float m = p[S::kHeads * kDim + h];
        const float down = m == -INFINITY ? 0.0f : exp2_approx(m - top);
        total += p[S::kHeads * (kDim + 1) + h] * down;
#pragma unroll
        for (int r = 0; r < kRun; ++r) {
            const float2 x = *reinterpret_cast<const float2*>(p + h * kDim + r * 64 + lane * 2);
            sum[r].x += x.x * down;
            sum[r].y += x.y * down;
        }
    }
#pragma unroll
    for (int r = 0; r < kRun; ++r) *reinterpret_cast<float2*>(&sums[share][h][r * 64 + lane * 2]) = sum[r];
    if (lane == 0) {
        tops[share][h] = top;
        totals[share][h] = total;
    }
    __syncthreads();
    const uint32_t group = a.heads / a.kv_heads, k = join.item / plan.groups;
    const uint32_t from = (join.item % plan.groups) * S::kHeads, heads = min(group - from, static_cast<uint32_t>(S::kHeads));
    const uint32_t head = k * group + from;
    T* out = nz::device_ptr<T>(a.out) + join.request * a.out_stride[0];
    for (uint32_t i = threadIdx.x; i < heads * kDim; i += 1024U) {
        const uint32_t q = i / kDim, d = i % kDim;
        float x = 0.0f, all = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < kShares; ++v) x += sums[v][q][d], all += totals[v][q];
        if (d < a.dim) out[(head + q) * a.out_stride[1] + d] = from_float<T>(all == 0.0f ? 0.0f : x / all);
        if (d == 0 && a.lse)
            nz::device_ptr<float>(a.lse)[static_cast<uint64_t>(join.request) * a.heads + head + q] =
                all == 0.0f ? -INFINITY : (tops[0][q] + log2f(all)) * kLn2;
    }
}

// ---- host ------------------------------------------------------------------------------

struct Device {
    int ctas_per_sm = 0;
    int sms = 0;
};

// Resident CTAs of the split kernel on the current device, looked up (and
// the kernels' shared memory opted into) once a device.
template <typename T, int kDim, int kHeadTiles>
cudaError_t device_limits(Device* out) {
    using Split = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    using Direct = Shape<T, kDim, kHeadTiles, kDirectWarps>;
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
        const auto direct = nz_paged_attention_direct<T, kDim, kHeadTiles>;
        constexpr size_t most = Split::kSharedBytes + NZ_PAGED_MAX_REQUESTS * sizeof(uint32_t);
        int sms = 0;
        err = cudaFuncSetAttribute(split, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
        if (err == cudaSuccess)
            err = cudaFuncSetAttribute(direct, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(Direct::kSharedBytes));
        if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (err == cudaSuccess)
            err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&d.ctas_per_sm, split, Split::kThreads, most);
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

// The launch for these sizes: `workers` 0 (one CTA an item) where a request
// attends to few chunks, else as many as are resident or as there can be
// chunks.
template <typename T, int kDim, int kHeadTiles>
cudaError_t launch(const nz_attention& a, cudaStream_t stream, uint64_t* workspace_only) {
    using S = Shape<T, kDim, kHeadTiles, kSplitWarps>;
    using Direct = Shape<T, kDim, kHeadTiles, kDirectWarps>;
    Device device;
    cudaError_t err = device_limits<T, kDim, kHeadTiles>(&device);
    if (err != cudaSuccess) return err;
    Plan plan = {0U, (a.heads / a.kv_heads + S::kHeads - 1U) / S::kHeads};
    const uint64_t items = static_cast<uint64_t>(a.requests) * a.kv_heads * plan.groups;
    if (most_chunks(a, Direct::kChunk) > kDirectChunks) {
        const uint64_t all = most_chunks(a, S::kChunk) * items;
        const uint64_t resident = static_cast<uint64_t>(device.sms) * device.ctas_per_sm;
        plan.workers = static_cast<uint32_t>(all < resident ? all : resident);
    }
    const uint64_t workspace = plan.workers * (2 * S::kPartFloats * sizeof(float) + sizeof(Join));
    if (workspace_only) {
        *workspace_only = workspace;
        return cudaSuccess;
    }
    if (plan.workers == 0) {
        nz_paged_attention_direct<T, kDim, kHeadTiles>
            <<<static_cast<uint32_t>(items), Direct::kThreads, Direct::kSharedBytes, stream>>>(a, plan);
        return cudaGetLastError();
    }
    if (!a.workspace) return cudaErrorInvalidValue;
    nz_paged_attention_split<T, kDim, kHeadTiles>
        <<<plan.workers, S::kThreads, S::kSharedBytes + a.requests * sizeof(uint32_t), stream>>>(a, plan);
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    // The join's launch overlaps the first kernel, whose results it waits for.
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(plan.workers);
    config.blockDim = dim3(1024);
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, nz_paged_attention_join<T, kDim, kHeadTiles>, a, plan);
}

template <typename T>
cudaError_t dispatch(const nz_attention& a, cudaStream_t stream, uint64_t* workspace_only) {
    const bool one = a.heads / a.kv_heads <= 8;
    if (a.dim <= 64) return one ? launch<T, 64, 1>(a, stream, workspace_only) : launch<T, 64, 2>(a, stream, workspace_only);
    if (a.dim <= 128) return one ? launch<T, 128, 1>(a, stream, workspace_only) : launch<T, 128, 2>(a, stream, workspace_only);
    if (a.dim <= 192) return one ? launch<T, 192, 1>(a, stream, workspace_only) : launch<T, 192, 2>(a, stream, workspace_only);
    return one ? launch<T, 256, 1>(a, stream, workspace_only) : launch<T, 256, 2>(a, stream, workspace_only);
}

int attention(const nz_attention* args, cudaStream_t stream, uint64_t* workspace_only) {
    if (!args) return nz::paged_fail("Null arguments.");
    const nz_attention& a = *args;
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
