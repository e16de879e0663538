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
//
// Measured: 8191 + 57 rows of 64 + 8 + 8 heads x 128 in bf16 with norms, 340
// MB, in 60 us (5.7 TB/s, 87% of the copy rate; the first form, a thread a
// chunk of a row, took 93: its instructions bound it); 8 tokens of 32 + 8 + 8
// heads in 1.9 us.

#include "nz_paged.h"

namespace {

template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Vec {
    T v[VEC];
};

// ONCE: bytes that nobody reads soon are the first to leave L2.
template <typename T, int VEC, bool ONCE = false>
__device__ __forceinline__ Vec<T, VEC> load(const T* p) {
    if constexpr (ONCE && sizeof(Vec<T, VEC>) == 16) {
        const int4 bits = __ldcs(reinterpret_cast<const int4*>(p));
        return *reinterpret_cast<const Vec<T, VEC>*>(&bits);
    } else {
        return *reinterpret_cast<const Vec<T, VEC>*>(p);
    }
}
template <typename T, int VEC, bool ONCE = false>
__device__ __forceinline__ void store(T* p, const Vec<T, VEC>& x) {
    if constexpr (ONCE && sizeof(Vec<T, VEC>) == 16)
        __stcs(reinterpret_cast<int4*>(p), *reinterpret_cast<const int4*>(&x));
    else
        *reinterpret_cast<Vec<T, VEC>*>(p) = x;
}

// VEC values in 32 bits, by whole registers where two values share one.
template <int VEC>
__device__ __forceinline__ void widen(float* f, const Vec<float, VEC>& x) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = x.v[i];
}
template <int VEC>
__device__ __forceinline__ void widen(float* f, const Vec<__nv_bfloat16, VEC>& x) {
    if constexpr (VEC == 1) f[0] = __bfloat162float(x.v[0]);
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) {
        const uint32_t both = *reinterpret_cast<const uint32_t*>(&x.v[i]);
        f[i] = __uint_as_float(both << 16);
        f[i + 1] = __uint_as_float(both & 0xFFFF0000U);
    }
}
template <int VEC>
__device__ __forceinline__ void widen(float* f, const Vec<__half, VEC>& x) {
    if constexpr (VEC == 1) f[0] = __half2float(x.v[0]);
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) {
        const float2 both = __half22float2(*reinterpret_cast<const __half2*>(&x.v[i]));
        f[i] = both.x;
        f[i + 1] = both.y;
    }
}

// Rounds VEC values, two at a time where the type has a paired conversion.
template <int VEC>
__device__ __forceinline__ void round_to(Vec<float, VEC>& x, const float* f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x.v[i] = f[i];
}
template <int VEC>
__device__ __forceinline__ void round_to(Vec<__nv_bfloat16, VEC>& x, const float* f) {
    if constexpr (VEC == 1) x.v[0] = __float2bfloat16_rn(f[0]);
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) *reinterpret_cast<__nv_bfloat162*>(&x.v[i]) = __floats2bfloat162_rn(f[i], f[i + 1]);
}
template <int VEC>
__device__ __forceinline__ void round_to(Vec<__half, VEC>& x, const float* f) {
    if constexpr (VEC == 1) x.v[0] = __float2half_rn(f[0]);
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) *reinterpret_cast<__half2*>(&x.v[i]) = __floats2half2_rn(f[i], f[i + 1]);
}

// Two products, or products and sums, in one instruction.
__device__ __forceinline__ float2 mul(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// A lane's N pairs (a, b) of a chunk in 32 bits, two pairs to an
// instruction where N is even.
template <int N>
struct Pairs {
    static constexpr int kTwos = (N + 1) / 2;
    float2 a[kTwos], b[kTwos];

    __device__ float& first(int i) { return i % 2 ? a[i / 2].y : a[i / 2].x; }
    __device__ float& second(int i) { return i % 2 ? b[i / 2].y : b[i / 2].x; }
    // From the elements of the chunk's two vectors: (i, N + i), or neighbours.
    __device__ void set(const float* f, bool neighbours) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            first(i) = neighbours ? f[2 * i] : f[i];
            second(i) = neighbours ? f[2 * i + 1] : f[N + i];
        }
        if constexpr (N % 2) a[kTwos - 1].y = b[kTwos - 1].y = 0.0f;
    }
    __device__ void get(float* f, bool neighbours) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            f[neighbours ? 2 * i : i] = first(i);
            f[neighbours ? 2 * i + 1 : N + i] = second(i);
        }
    }
};

constexpr uint32_t kThreads = 256;

// Rows of one kind: queries, keys or values. Which one is uniform in a
// warp, so a thread holds the pointers and strides of one kind only.
struct Kind {
    uint64_t source, weight, out, pages;
    int64_t source_stride[2], out_stride[2], pages_stride[3];
    uint32_t heads, turns;
    uint32_t before;  // blocks, or steps of a token, of the kinds before
};

struct Kinds {
    Kind kind[3];
    uint32_t steps;  // of a token
    float mean;      // 1 / width
};

// What a lane multiplies its chunk of a row of one kind at one position by,
// the norm's weights w included: a' = a (w_a cos) - b (w_b sin), b' =
// b (w_b cos) + a (w_a sin). Elements behind the rotated part keep only
// their weights.
template <typename T, int VEC, bool INTERLEAVED>
struct Factors {
    Pairs<VEC> along, across;

    __device__ void set(const nz_rotary& a, const Kind& k, uint32_t token, uint32_t pair, const uint32_t (&at)[2],
                        bool have) {
        float w[2 * VEC];
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) w[i] = 1.0f;
        if (k.weight && have) {
            widen(w, load<T, VEC>(nz::device_ptr<const T>(k.weight) + at[0]));
            widen(w + VEC, load<T, VEC>(nz::device_ptr<const T>(k.weight) + at[1]));
        }
        along.set(w, INTERLEAVED);
        across = along;
        if (!have || pair >= a.rot / 2) return;
        const int32_t position = nz::device_ptr<const int32_t>(a.positions)[token];
        Vec<float, VEC> cosine, sine;
        if (position >= 0 && static_cast<uint32_t>(position) < a.table_rows) {
            const float* angles = nz::device_ptr<const float>(a.table) + position * a.table_stride + pair;
            cosine = load<float, VEC>(angles);
            sine = load<float, VEC>(angles + a.rot / 2);
        } else {  // NaN where a position outside the table would rotate
#pragma unroll
            for (int i = 0; i < VEC; ++i) cosine.v[i] = sine.v[i] = __int_as_float(0x7FFFFFFF);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            along.first(i) *= cosine.v[i];
            along.second(i) *= cosine.v[i];
            across.first(i) *= sine.v[i];
            across.second(i) *= -sine.v[i];
        }
    }

    __device__ void apply(Pairs<VEC>& p, bool rotates, bool normed, float scale) const {
        const float2 both = make_float2(scale, scale);
#pragma unroll
        for (int i = 0; i < Pairs<VEC>::kTwos; ++i) {
            float2 u = mul(p.a[i], along.a[i]), v = mul(p.b[i], along.b[i]);
            if (rotates) {
                u = fma(p.b[i], across.b[i], u);
                v = fma(p.a[i], across.a[i], v);
            }
            p.a[i] = normed ? mul(u, both) : u;
            p.b[i] = normed ? mul(v, both) : v;
        }
    }
};

// Where the two vectors of the chunk of pairs that starts at `pair` lie in a row.
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ void place(const nz_rotary& a, uint32_t pair, uint32_t (&at)[2]) {
    const uint32_t turned = a.rot / 2;
    if (pair >= turned) {
        at[0] = turned + pair;
        at[1] = a.dim / 2 + pair;
    } else if (INTERLEAVED) {
        at[0] = 2U * pair;
        at[1] = 2U * pair + VEC;
    } else {
        at[0] = pair;
        at[1] = turned + pair;
    }
}

template <int N>
__device__ __forceinline__ float squares_of(const Pairs<N>& p) {
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < Pairs<N>::kTwos; ++i) sum = fma(p.b[i], p.b[i], fma(p.a[i], p.a[i], sum));
    return sum.x + sum.y;
}

// The sum over a group; its lanes hold one row, so they are all here.
__device__ __forceinline__ float group_sum(float x, uint32_t group) {
    const uint32_t mask = (0xFFFFFFFFU >> (32U - group)) << (threadIdx.x & 31U & ~(group - 1U));
    for (uint32_t d = 1; d < group; d <<= 1) x += __shfl_xor_sync(mask, x, d);
    return x;
}

// The rows of a token's kind: where query_out or key_out and the cache want them (null: not).
template <typename T>
struct Targets {
    T *out, *pages;

    __device__ Targets(const nz_rotary& a, const Kind& k, uint32_t token) : out(nullptr), pages(nullptr) {
        if (k.out) out = nz::device_ptr<T>(k.out) + token * k.out_stride[0];
        if (k.pages) {
            const int32_t slot = nz::device_ptr<const int32_t>(a.slots)[token];
            const int64_t page = slot >> a.page_shift, line = slot & ((1 << a.page_shift) - 1);
            if (slot >= 0 && page < a.pages)
                pages = nz::device_ptr<T>(k.pages) + page * k.pages_stride[0] + line * k.pages_stride[1];
        }
    }
    template <bool ONCE, int VEC>
    __device__ void write(const Kind& k, uint32_t head, uint32_t at, const Vec<T, VEC>& x) const {
        if (out) store<T, VEC, ONCE>(out + head * k.out_stride[1] + at, x);
        if (pages) store<T, VEC, ONCE>(pages + head * k.pages_stride[2] + at, x);
    }
};

// A group takes one row. CHUNKS: pair chunks of VEC a lane owns; group_log:
// lanes of a group; MANY: rows, read and written as bytes that go ONCE.
template <typename T, int VEC, int CHUNKS, bool INTERLEAVED, bool MANY>
__global__ void __launch_bounds__(kThreads) nz_rotary_kernel(const nz_rotary a, const __grid_constant__ Kinds kinds,
                                                             uint32_t group_log) {
    nz::after_predecessor();
    const uint32_t which = blockIdx.x >= kinds.kind[2].before ? 2U : blockIdx.x >= kinds.kind[1].before ? 1U : 0U;
    const Kind& k = kinds.kind[which];
    const uint32_t group = 1U << group_log, lane = threadIdx.x & (group - 1U);
    const uint32_t unit = ((blockIdx.x - k.before) << (8U - group_log)) + (threadIdx.x >> group_log);
    const uint32_t token = unit / k.heads, head = unit - token * k.heads;
    if (token >= a.tokens) return;  // whole groups
    const T* row = nz::device_ptr<const T>(k.source) + token * k.source_stride[0] + head * k.source_stride[1];
    uint32_t at[CHUNKS][2];
    bool have[CHUNKS];
    Vec<T, VEC> x[CHUNKS][2];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t pair = (c * group + lane) * VEC;
        have[c] = pair < a.dim / 2;
        place<VEC, INTERLEAVED>(a, pair, at[c]);
        if (have[c]) {
            x[c][0] = load<T, VEC, MANY>(row + at[c][0]);
            x[c][1] = load<T, VEC, MANY>(row + at[c][1]);
        }
    }
    const Targets<T> targets(a, k, token);
    if (k.turns) {
        Factors<T, VEC, INTERLEAVED> factors[CHUNKS];
        Pairs<VEC> p[CHUNKS];
        float scale = 0.0f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            factors[c].set(a, k, token, (c * group + lane) * VEC, at[c], have[c]);
            if (!have[c]) continue;
            float f[2 * VEC];
            widen(f, x[c][0]);
            widen(f + VEC, x[c][1]);
            p[c].set(f, INTERLEAVED);
            scale += squares_of(p[c]);
        }
        if (k.weight) scale = rsqrtf(group_sum(scale, group) * kinds.mean + a.eps);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            if (!have[c]) continue;
            factors[c].apply(p[c], (c * group + lane) * VEC < a.rot / 2, k.weight, scale);
            float f[2 * VEC];
            p[c].get(f, INTERLEAVED);
            round_to(x[c][0], f);
            round_to(x[c][1], f + VEC);
        }
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        if (!have[c]) continue;
        targets.template write<MANY>(k, head, at[c][0], x[c][0]);
        targets.template write<MANY>(k, head, at[c][1], x[c][1]);
    }
}

// Into shared memory, for ONCE.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* shared, const void* global, uint64_t policy) {
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(shared));
    static_assert(BYTES % 16 == 0);
#pragma unroll
    for (int i = 0; i < BYTES; i += 16)
        asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to + i),
                     "l"(static_cast<const char*>(global) + i), "l"(policy)
                     : "memory");
}
__device__ __forceinline__ uint64_t leave_first() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}

constexpr uint32_t kStreamThreads = 128, kStreamCtas = 5;
constexpr uint32_t kRing = 4096;  // bytes of rows a warp has on their way

// Many rows: the steps of all tokens (a step: the rows of one kind that a
// warp's groups hold at a time, 4 for a 128-wide 16-bit head) are shared out
// in equal runs, one a warp, so that factors are made once for all heads of
// a token. A lane copies its own vectors of the coming steps into its own
// part of shared memory, which only it reads: a ring without barriers that
// keeps kRing bytes a warp on their way, where registers alone could not.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kStreamThreads, kStreamCtas) nz_rotary_stream(const nz_rotary a, const __grid_constant__ Kinds kinds,
                                                             uint32_t group_log) {
    using V = Vec<T, VEC>;
    constexpr int kDepth = kRing / (32 * 2 * sizeof(V));
    nz::after_predecessor();
    extern __shared__ __align__(16) unsigned char shared[];
    V* ring = reinterpret_cast<V*>(shared) + (threadIdx.x >> 5) * (kDepth * 64) + (threadIdx.x & 31U);
    const uint32_t group = 1U << group_log, lane = threadIdx.x & (group - 1U);
    const uint32_t groups = 32U >> group_log, mine = (threadIdx.x & 31U) >> group_log;
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (kStreamThreads / 32);
    const uint64_t warp = static_cast<uint64_t>(blockIdx.x) * (kStreamThreads / 32) + (threadIdx.x >> 5);
    const uint64_t all = static_cast<uint64_t>(a.tokens) * kinds.steps;
    const uint32_t begin = static_cast<uint32_t>(all * warp / warps), end = static_cast<uint32_t>(all * (warp + 1) / warps);
    const uint32_t pair = lane * VEC;
    const bool have = pair < a.dim / 2, rotates = pair < a.rot / 2;
    uint32_t at[2];
    place<VEC, INTERLEAVED>(a, pair, at);

    const uint64_t policy = leave_first();
    // The loads run kDepth - 1 steps ahead. Both walks keep pointers that
    // step from row to row, and look at the kinds only when one ends.
    const T* source = nullptr;
    int64_t source_step = 0;
    uint32_t ahead_token = begin / kinds.steps, ahead_step = begin % kinds.steps, ahead_last = 0, ahead_head = 0, ahead_heads = 0;
    auto kind_of = [&](uint32_t step) { return step >= kinds.kind[2].before ? 2U : step >= kinds.kind[1].before ? 1U : 0U; };
    auto fetch = [&](uint32_t index) {  // into the ring's place for `index`
        if (index < end) {
            if (ahead_step >= ahead_last) {
                if (ahead_step == kinds.steps) {
                    ahead_step = 0;
                    ++ahead_token;
                }
                const uint32_t which = kind_of(ahead_step);
                const Kind& k = kinds.kind[which];
                ahead_last = which == 2U ? kinds.steps : kinds.kind[which + 1U].before;
                ahead_head = (ahead_step - k.before) * groups + mine;
                ahead_heads = have ? k.heads : 0U;
                source = nz::device_ptr<const T>(k.source) + ahead_token * k.source_stride[0] + ahead_head * k.source_stride[1];
                source_step = groups * k.source_stride[1];
            }
            if (ahead_head < ahead_heads) {
                V* to = ring + (index % kDepth) * 64;
                copy_async<sizeof(V)>(to, source + at[0], policy);
                copy_async<sizeof(V)>(to + 32, source + at[1], policy);
            }
            source += source_step;
            ahead_head += groups;
            ++ahead_step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (uint32_t i = begin; i < begin + kDepth - 1; ++i) fetch(i);

    Factors<T, VEC, INTERLEAVED> factors;
    uint32_t token = begin / kinds.steps, step = begin % kinds.steps;
    for (uint32_t i = begin; i < end;) {  // a kind of a token
        const uint32_t which = kind_of(step);
        const Kind& k = kinds.kind[which];
        const uint32_t last = which == 2U ? kinds.steps : kinds.kind[which + 1U].before;
        const uint32_t stop = min(end, i + last - step), heads = k.heads;
        uint32_t head = (step - k.before) * groups + mine;
        const Targets<T> targets(a, k, token);
        const bool turns = k.turns, normed = k.weight != 0;
        T* out = targets.out ? targets.out + head * k.out_stride[1] : nullptr;
        T* pages = targets.pages ? targets.pages + head * k.pages_stride[2] : nullptr;
        const int64_t out_step = groups * k.out_stride[1], pages_step = groups * k.pages_stride[2];
        if (turns) factors.set(a, k, token, pair, at, have);
        step += stop - i;
        if (step == kinds.steps) {
            step = 0;
            ++token;
        }
#pragma unroll 1
        for (; i < stop; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
            if (head < heads) {  // whole groups
                V x[2] = {ring[(i % kDepth) * 64], ring[(i % kDepth) * 64 + 32]};
                if (turns) {
                    float f[2 * VEC];
                    widen(f, x[0]);
                    widen(f + VEC, x[1]);
                    Pairs<VEC> p;
                    p.set(f, INTERLEAVED);
                    float scale = 1.0f;
                    if (normed) scale = rsqrtf(group_sum(have ? squares_of(p) : 0.0f, group) * kinds.mean + a.eps);
                    factors.apply(p, rotates, normed, scale);
                    p.get(f, INTERLEAVED);
                    round_to(x[0], f);
                    round_to(x[1], f + VEC);
                }
                if (have && out) {
                    store<T, VEC, true>(out + at[0], x[0]);
                    store<T, VEC, true>(out + at[1], x[1]);
                }
                if (have && pages) {
                    store<T, VEC, true>(pages + at[0], x[0]);
                    store<T, VEC, true>(pages + at[1], x[1]);
                }
            }
            out += out ? out_step : 0;
            pages += pages ? pages_step : 0;
            head += groups;
            fetch(i + kDepth - 1);
        }
    }
}

bool many_elements(const nz_rotary& a) {
    const uint64_t least = a.dtype == NZ_PAGED_FP32 ? 6U << 20 : 4U << 20;
    return static_cast<uint64_t>(a.tokens) * (a.heads + 2ULL * a.kv_heads) * a.dim >= least;
}

template <typename T, int VEC, bool INTERLEAVED>
cudaError_t launch_stream(const nz_rotary& a, Kinds& kinds, uint32_t group_log, cudaStream_t stream) {
    const uint32_t groups = 32U >> group_log;
    kinds.steps = 0;
    for (Kind& k : kinds.kind) {
        k.before = kinds.steps;
        kinds.steps += (k.heads + groups - 1U) / groups;
    }
    const auto kernel = nz_rotary_stream<T, VEC, INTERLEAVED>;
    constexpr size_t shared = kRing * (kStreamThreads / 32);
    int device = 0, sms = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
    if (err != cudaSuccess) return err;
    const nz::PagedLaunch l(static_cast<uint32_t>(sms) * kStreamCtas, 1, kStreamThreads, shared, stream, 1);
    return cudaLaunchKernelEx(&l.config, kernel, a, kinds, group_log);
}

template <typename T, int VEC, int CHUNKS, bool INTERLEAVED, bool MANY>
cudaError_t launch_kernel(const nz_rotary& a, bool streaming, cudaStream_t stream) {
    const uint32_t chunks = (a.dim / 2 + VEC - 1) / VEC;
    uint32_t group_log = 0;
    while ((1U << group_log) * CHUNKS < chunks) ++group_log;
    Kinds kinds = {};
    kinds.mean = 1.0f / static_cast<float>(a.dim);
    uint32_t blocks = 0;
    auto set = [&](int which, uint64_t source, const int64_t* stride, uint64_t weight, uint64_t out, const int64_t* out_stride,
                   uint64_t pages, const int64_t* pages_stride, uint32_t heads, uint32_t turns) {
        Kind& k = kinds.kind[which];
        k.source = source, k.weight = weight, k.out = out, k.pages = pages;
        for (int i = 0; i < 2; ++i) k.source_stride[i] = stride[i], k.out_stride[i] = out_stride ? out_stride[i] : 0;
        for (int i = 0; i < 3; ++i) k.pages_stride[i] = pages_stride ? pages_stride[i] : 0;
        k.heads = heads, k.turns = turns, k.before = blocks;
        blocks += static_cast<uint32_t>((((static_cast<uint64_t>(a.tokens) * heads) << group_log) + kThreads - 1) / kThreads);
    };
    set(0, a.query, a.query_stride, a.query_norm, a.query_out, a.query_out_stride, 0, nullptr, a.heads, 1);
    set(1, a.key, a.key_stride, a.key_norm, a.key_out, a.key_out_stride, a.key_pages, a.key_pages_stride, a.kv_heads, 1);
    set(2, a.value, a.value_stride, 0, 0, nullptr, a.value_pages, a.value_pages_stride, a.kv_heads, 0);
    if constexpr (MANY)
        if (streaming) return launch_stream<T, VEC, INTERLEAVED>(a, kinds, group_log, stream);
    const nz::PagedLaunch l(blocks, 1, kThreads, 0, stream, 1);
    return cudaLaunchKernelEx(&l.config, nz_rotary_kernel<T, VEC, CHUNKS, INTERLEAVED, MANY>, a, kinds, group_log);
}

template <typename T, int VEC, int CHUNKS, bool MANY = false>
cudaError_t launch(const nz_rotary& a, cudaStream_t stream, bool streaming = false) {
    return a.interleaved ? launch_kernel<T, VEC, CHUNKS, true, MANY>(a, streaming, stream)
                         : launch_kernel<T, VEC, CHUNKS, false, MANY>(a, streaming, stream);
}

// Whether vectors of `vec` elements divide both kinds of pair chunks and
// every address.
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

// From 4M elements on (fp32: 6M), the streaming kernel, where a token's rows keep at
// least three fifths of its lanes busy: 32 + 8 heads of 128 in bf16 with
// norms take 5.5 us of the other kernel and 5.9 us of this one at 512 tokens
// (3M), 7.2 and 6.9 at 768, 57 and 39 at 8192; 32 + 8 heads of 80 (62% of
// the lanes) 48 and 29 us at 8000 tokens; 14 + 2 heads of 64 (56%) 9.9 and
// 15.4 us at 8192, 39 and 52 at 32000; in fp32 12 + 12 heads of 96 7.8 and
// 9.0 us at 1300 (4.5M), 11.4 and 11.1 at 1800.
// Either kernel then reads and writes with the hint that nothing of it is
// needed soon (ONCE): 8248 tokens of 64 + 8 heads of 128 62.2 us without,
// 59.7 with; 14 + 2 of 64 at 32000 42 and 39.
template <typename T>
bool streams(const nz_rotary& a, uint32_t vec) {
    const uint64_t rows = a.heads + 2ULL * a.kv_heads, chunks = a.dim / 2 / vec;
    uint32_t lanes = 1;
    while (lanes < chunks) lanes *= 2;
    const uint32_t groups = 32U / lanes;
    const uint64_t steps = (a.heads + groups - 1) / groups + 2ULL * ((a.kv_heads + groups - 1) / groups);
    return rows * chunks * 5 >= steps * 32 * 3;
}

// The streaming kernel takes 16-byte vectors, which need the fewest
// instructions, the other one 4 elements a vector, which shares a row among
// more lanes (a step of 8 tokens: 2.0 us, 2.2 with 8). Rotated widths or
// strides that 4 does not divide take 2 or 1.
template <typename T>
cudaError_t launch_type(const nz_rotary& a, cudaStream_t stream) {
    constexpr int kWide = 16 / sizeof(T);
    if (many_elements(a) && vector_fits(a, kWide, sizeof(T))) return launch<T, kWide, 1, true>(a, stream, streams<T>(a, kWide));
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
