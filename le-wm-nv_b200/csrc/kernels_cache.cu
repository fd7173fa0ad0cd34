// kernels_cache.cu — the paged cache's writes and reads: append with the
// rotary turn on the way (lwm_cache_append_device) and gather
// (lwm_cache_gather_device).  Bound: memory.
//
// 16 bits: a block per 16 new tokens of a sequence (a page holds whole runs
// of 16): their angles are computed once into shared memory and serve every
// head; a thread has four units' loads in flight before it uses one.
// 8 bits: a block per page that gets new tokens; a group of lanes owns a
// (page, head): the new tokens' largest value first, then the scale, the
// earlier tokens' codes where the scale grew, and the new codes, so that no
// scale is shared between groups.
//
// Measured (one B200): 16 sequences x up to 1568 new tokens, 16 heads of 64
// channels, bf16, queries turned along: 215 MB read and written in 49 us, 165
// MB of them in DRAM; gathering 151 MB back 24 us, 99 MB of them in DRAM (the
// rest hit the L2, which the append before has filled).  8 bits, one token
// for each of 1024 sequences: 16 to 24 us, the chain lengths -> page ->
// tokens -> scale -> codes twice over (80 registers: three blocks a SM);
// gathering 17 tokens of each, 35 MB of codes to 70 MB: 23 us, two thirds of
// the issue slots.  Left, as they cost more than they gave: more blocks a SM
// with 64 registers or fewer (spills, +2 %), 16 codes a load in the gather
// (+6 %), eight loads in flight (+2 %).
#include "lwm_blocks.cuh"

namespace lwm {

namespace {

constexpr int kThreads = 256;

// The new tokens of one page of a sequence.
struct PagePart {
    uint32_t row, slot, count;  // first packed row and slot (the page's earlier tokens), tokens
    uint32_t index;             // cache index of the first
    int page;                   // -1: nothing to do
};
// (or of one run of 1 << shift tokens inside a page)
__device__ __forceinline__ PagePart page_part(const CacheArgs& c, const SeqView& v, uint32_t s, uint32_t ordinal,
                                              uint32_t shift) {
    PagePart p{0, 0, 0, 0, -1};
    if (!v.ok || v.n == 0 || v.n > v.length) return p;
    const uint32_t first = v.length - v.n, run = (first >> shift) + ordinal;
    if (static_cast<uint64_t>(run) << shift >= v.length) return p;
    const uint32_t begin = max(first, run << shift);
    const uint32_t end = static_cast<uint32_t>(min(static_cast<uint64_t>(v.length), static_cast<uint64_t>(run + 1) << shift));
    const uint32_t j = begin >> c.page_shift;
    p.index = begin;
    p.slot = begin & (c.page_tokens - 1);
    p.count = end - begin;
    p.row = v.start + (begin - first);
    p.page = c.table[static_cast<size_t>(s) * c.table_stride + j];
    if (static_cast<uint32_t>(p.page) >= c.pages) {
        if (threadIdx.x == 0) cache_report(c.err, kCacheErrPage, s, p.page);
        p.page = -1;
    }
    return p;
}

// Divisions of a launch: units of a head, heads that turn, vectors of a head.
struct CacheDivs {
    FastDiv units, turning, vecs, kv, ordinals;
};

// A turning or passing unit of one head row: loads, turns, hands the one or
// two vectors to `put(channel, values)`.
template <typename T, class Put>
__device__ __forceinline__ void head_unit(const lwm_rotary& r, uint32_t pairs, const HeadUnits& hu, uint32_t u,
                                          const T* row, const float2* cs, Put put) {
    float v[8];
    if (u >= hu.turned) {
        const uint32_t ch = 2 * pairs + 8 * (u - hu.turned);
        unpack(load8(row + ch), v);
        put(ch, v);
        return;
    }
    uint32_t ch, apart, pair;
    unit_place(r, u, ch, apart, pair);
    unpack(load8(row + ch), v);
    if (r.interleaved) {
        turn_pairs(v, cs + pair);
        put(ch, v);
    } else {
        float w[8];
        unpack(load8(row + ch + apart), w);
        turn_halves(v, w, cs + pair);
        put(ch, v);
        put(ch + apart, w);
    }
}

template <int kLanes> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = min(kLanes, 32) / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (kLanes > 32) {  // the block
        __shared__ float parts[kThreads / 32];
        __syncthreads();
        if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) v = fmaxf(v, parts[w]);
    }
    return v;
}
__device__ __forceinline__ float finite_abs(float v) { return isfinite(v) ? fabsf(v) : 0.0f; }

// One (page, head) of an 8-bit pool, by kLanes lanes; `on` false: nothing but
// the shuffles that the warp's other groups need.
template <typename T, int kLanes>
__device__ __forceinline__ void append_codes(const AppendArgs& a, const PagePart& p, uint32_t held, uint32_t h, bool keys,
                                             const float2* trig, int lane, bool on) {
    const HeadUnits hu(keys ? a.pairs : 0, a.r.interleaved, a.c.head_dim);
    const uint32_t pairs = keys ? a.pairs : 0;
    const T* src = static_cast<const T*>(keys ? a.k : a.v);
    const size_t ts = keys ? a.k_ts : a.v_ts, hs = keys ? a.k_hs : a.v_hs;
    float* scale_at = (keys ? a.c.k_scale : a.c.v_scale) + static_cast<size_t>(p.page) * a.c.kv_heads + h;
    uint8_t* pool = static_cast<uint8_t*>(keys ? a.c.k : a.c.v) + pool_at(a.c, p.page, h, 0);
    const uint32_t work = on ? p.count * hu.count : 0;
    float amax = 0.0f;
    for (uint32_t i = lane; i < work; i += kLanes) {
        const uint32_t t = i / hu.count, u = i - t * hu.count;
        head_unit<T>(a.r, pairs, hu, u, src + (p.row + t) * ts + h * hs, trig + t * a.pairs,
                     [&](uint32_t, const float(&v)[8]) {
#pragma unroll
                         for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[e]));
                     });
    }
    float scale = page_scale(lanes_max<kLanes>(amax));
    if (!on) return;
    if (held) {
        // the page holds earlier tokens: its scale never falls, and their
        // codes are rounded again where it grows
        const float old = *scale_at;
        if (!(old >= scale)) {
            const float again = old / scale;
            for (uint32_t i = lane; i < held * (a.c.head_dim / 8); i += kLanes) {
                uint2* at = reinterpret_cast<uint2*>(pool) + i;
                float f[8];
                from_e4m3(*at, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= again;
                *at = to_e4m3(f);
            }
        } else {
            scale = old;
        }
    }
    const float inv = 1.0f / scale;
    for (uint32_t i = lane; i < work; i += kLanes) {
        const uint32_t t = i / hu.count, u = i - t * hu.count;
        uint8_t* row = pool + static_cast<size_t>(p.slot + t) * a.c.head_dim;
        head_unit<T>(a.r, pairs, hu, u, src + (p.row + t) * ts + h * hs, trig + t * a.pairs,
                     [&](uint32_t ch, float(&v)[8]) {
#pragma unroll
                         for (int e = 0; e < 8; ++e) v[e] *= inv;
                         *reinterpret_cast<uint2*>(row + ch) = to_e4m3(v);
                     });
    }
    // every lane of the group has read the old scale
    if constexpr (kLanes > 32) __syncthreads();
    else __syncwarp(kLanes == 32 ? 0xffffffffu : ((1u << (kLanes & 31)) - 1u) << ((threadIdx.x & 31) / kLanes * kLanes));
    if (lane == 0) *scale_at = scale;
}

// cos and sin of the part's tokens.
__device__ __forceinline__ void part_angles(const AppendArgs& a, const PagePart& p, const PairTurns& turns, float2* trig) {
    __syncthreads();  // turns
    for (uint32_t i = threadIdx.x; i < p.count * a.pairs; i += kThreads) {
        const uint32_t t = i / a.pairs, pr = i - t * a.pairs;
        const int32_t pos = a.positions
                                ? a.positions[static_cast<size_t>(p.row + t) * a.axes + turns.axis[pr]]
                                : static_cast<int32_t>(p.index + t);
        trig[i] = turn_of(pos, turns.turn[pr]);
    }
    __syncthreads();
}

// Turns heads [0, heads) of the part's tokens: queries, then (16 bits) keys.
// Both vectors of a unit are read before either is written: q_out may be q.
// The work of the part's blocks (blockIdx.y) is dealt out by loads in flight.
template <typename T>
__device__ __forceinline__ void turn_heads(const AppendArgs& a, const CacheDivs& d, const PagePart& p, uint32_t q_heads,
                                           uint32_t heads, const float2* trig) {
    const HeadUnits hu(a.pairs, a.r.interleaved, a.c.head_dim);
    const uint32_t work = p.count * heads * hu.count;
    for (uint32_t base = blockIdx.y * 4 * kThreads + threadIdx.x; base < work; base += gridDim.y * 4 * kThreads) {
        Vec8<T> x[4], y[4];
        T* dst[4];
        uint32_t apart[4], pair[4], at[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t i = base + b * kThreads;
            dst[b] = nullptr;
            if (i >= work) continue;
            const uint32_t row = d.units.div(i), u = i - row * hu.count, t = d.turning.div(row), h = row - t * heads;
            const size_t r = p.row + t;
            const bool is_q = h < q_heads;
            const T* src = is_q ? static_cast<const T*>(a.q) + r * a.q_ts + h * a.q_hs
                                : static_cast<const T*>(a.k) + r * a.k_ts + (h - q_heads) * a.k_hs;
            dst[b] = is_q ? static_cast<T*>(a.q_out) + r * a.qo_ts + h * a.qo_hs
                          : static_cast<T*>(a.c.k) + pool_at(a.c, p.page, h - q_heads, p.slot + t);
            uint32_t ch = 2 * a.pairs + 8 * (u - hu.turned);
            apart[b] = 0;
            pair[b] = 0xffffffffu;  // passes through
            if (u < hu.turned) unit_place(a.r, u, ch, apart[b], pair[b]);
            at[b] = t * a.pairs;
            x[b] = load8(src + ch);
            if (apart[b]) y[b] = load8(src + ch + apart[b]);
            dst[b] += ch;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (!dst[b]) continue;
            if (pair[b] != 0xffffffffu) {
                const float2* cs = trig + at[b] + pair[b];
                float v[8];
                unpack(x[b], v);
                if (apart[b]) {
                    float w[8];
                    unpack(y[b], w);
                    turn_halves(v, w, cs);
                    store8(dst[b] + apart[b], pack<T>(w));
                } else {
                    turn_pairs(v, cs);
                }
                x[b] = pack<T>(v);
            }
            store8(dst[b], x[b]);
        }
    }
}

// (80 registers a thread are three blocks a SM; at 81, two blocks, 215 MB and the gather took 84 us, not 79)
template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a, const CacheDivs d,
                                                          uint32_t runs) {
    extern __shared__ float2 trig[];  // [16][pairs]
    __shared__ PairTurns turns;
    fill_turns(a.r, a.pairs, turns);
    const uint32_t s = d.ordinals.div(blockIdx.x), ordinal = blockIdx.x - s * runs;
    const SeqView v = sequence(a.c, s, true, threadIdx.x == 0 && ordinal == 0);
    const PagePart p = page_part(a.c, v, s, ordinal, 4);
    if (p.page < 0) return;
    part_angles(a, p, turns, trig);
    const uint32_t kv = a.c.kv_heads, vecs = a.c.head_dim / 8, q_heads = a.q ? a.heads : 0;
    turn_heads<T>(a, d, p, q_heads, q_heads + kv, trig);
    const uint32_t work = p.count * kv * vecs;
    for (uint32_t base = threadIdx.x; base < work; base += 4 * kThreads) {
        Vec8<T> x[4];
        T* dst[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t i = base + b * kThreads;
            dst[b] = nullptr;
            if (i >= work) continue;
            const uint32_t row = d.vecs.div(i), c8 = 8 * (i - row * vecs), t = d.kv.div(row), h = row - t * kv;
            x[b] = load8(static_cast<const T*>(a.v) + (p.row + t) * a.v_ts + h * a.v_hs + c8);
            dst[b] = static_cast<T*>(a.c.v) + pool_at(a.c, p.page, h, p.slot + t) + c8;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (dst[b]) store8(dst[b], x[b]);
    }
}

// 8 bits; kLanes lanes a (page, head): 8 when a call brings a token or two a
// sequence (a head's units fill no more), the whole block when pages are few
// and full, else a warp.  blockIdx.y: parts of the heads, where the
// pages alone are too few blocks.
template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads, 3) append_codes_kernel(const __grid_constant__ AppendArgs a, const CacheDivs d,
                                                                uint32_t pages) {
    extern __shared__ float2 trig[];  // [page_tokens][pairs]
    __shared__ PairTurns turns;
    fill_turns(a.r, a.pairs, turns);
    const uint32_t s = d.ordinals.div(blockIdx.x), ordinal = blockIdx.x - s * pages;
    const SeqView v = sequence(a.c, s, true, threadIdx.x == 0 && ordinal == 0 && blockIdx.y == 0);
    const PagePart p = page_part(a.c, v, s, ordinal, a.c.page_shift);
    if (p.page < 0) return;
    part_angles(a, p, turns, trig);
    if (a.q) turn_heads<T>(a, d, p, a.heads, a.heads, trig);
    const uint32_t kv = a.c.kv_heads, group = threadIdx.x / kLanes, groups = kThreads / kLanes;
    const uint32_t stride = groups * gridDim.y, rounds = (2 * kv + stride - 1) / stride;
    for (uint32_t i = 0; i < rounds; ++i) {
        const uint32_t job = (i * gridDim.y + blockIdx.y) * groups + group;
        const bool on = job < 2 * kv, keys = job < kv;
        append_codes<T, kLanes>(a, p, p.slot, on ? (keys ? job : job - kv) : 0, keys, trig, threadIdx.x % kLanes, on);
    }
}

template <typename T, bool kCodes>
__global__ void __launch_bounds__(kThreads) gather_kernel(const __grid_constant__ GatherArgs a, const CacheDivs d,
                                                          uint32_t runs) {
    const uint32_t s = d.ordinals.div(blockIdx.x), ordinal = blockIdx.x - s * runs;
    const SeqView v = sequence(a.c, s, true, threadIdx.x == 0 && ordinal == 0);
    const PagePart p = page_part(a.c, v, s, ordinal, 4);
    if (p.page < 0) return;
    const uint32_t kv = a.c.kv_heads, vecs = a.c.head_dim / 8, half = p.count * kv, work = 2 * half * vecs;
    for (uint32_t base = threadIdx.x; base < work; base += 4 * kThreads) {
        uint4 x[4];
        float scale[4];
        T* dst[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t i = base + b * kThreads;
            dst[b] = nullptr;
            if (i >= work) continue;
            uint32_t row = d.vecs.div(i);
            const uint32_t c8 = 8 * (i - row * vecs);
            const bool keys = row < half;
            if (!keys) row -= half;
            const uint32_t t = d.kv.div(row), h = row - t * kv;
            const size_t r = p.row + t, at = pool_at(a.c, p.page, h, p.slot + t) + c8;
            dst[b] = (keys ? static_cast<T*>(a.k_out) + r * a.k_ts + h * a.k_hs
                           : static_cast<T*>(a.v_out) + r * a.v_ts + h * a.v_hs) + c8;
            const void* pool = keys ? a.c.k : a.c.v;
            if constexpr (kCodes) {
                const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at);
                x[b] = make_uint4(c.x, c.y, 0, 0);
                scale[b] = (keys ? a.c.k_scale : a.c.v_scale)[static_cast<size_t>(p.page) * kv + h];
            } else {
                x[b] = load8(static_cast<const T*>(pool) + at).a;
            }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (!dst[b]) continue;
            if constexpr (kCodes) {
                float f[8];
                from_e4m3(make_uint2(x[b].x, x[b].y), f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= scale[b];
                store8(dst[b], pack<T>(f));
            } else {
                store8(dst[b], Vec8<T>{x[b]});
            }
        }
    }
}

// Runs of `tokens` that up to max_new tokens of a sequence can lie in.
uint32_t runs_of(const CacheArgs& c, uint32_t tokens) { return (c.max_new + tokens - 2) / tokens + 1; }

CacheDivs divs_of(const CacheArgs& c, uint32_t units, uint32_t turning, uint32_t ordinals) {
    return {FastDiv(units), FastDiv(turning ? turning : 1), FastDiv(c.head_dim / 8), FastDiv(c.kv_heads), FastDiv(ordinals)};
}

template <typename T> cudaError_t append(const AppendArgs& a, bool codes, cudaStream_t s) {
    const HeadUnits hu(a.pairs, a.r.interleaved, a.c.head_dim);
    const uint32_t q_heads = a.q ? a.heads : 0;
    const uint32_t tokens = codes ? a.c.page_tokens : 16, runs = runs_of(a.c, tokens), blocks = runs * a.c.sequences;
    const size_t smem = static_cast<size_t>(min(tokens, a.c.max_new)) * a.pairs * sizeof(float2);
    if (!codes) {
        append_kernel<T><<<blocks, kThreads, smem, s>>>(a, divs_of(a.c, hu.count, q_heads + a.c.kv_heads, runs), runs);
        return cudaGetLastError();
    }
    const bool few = a.c.max_new <= 2;
    // A block a (page, head) where pages are full enough for all its threads and too few for the GPU's warps; us with
    // the events around them, a block and a warp each: 413 tokens of 3 sequences, 8 heads of 128, pages of 128, 42 and
    // 86; 316 of 23, 16 of 64, 128, 72 and 94; 1024 of 64, 16 of 64, 128, 327 and 301; 19 of 146, 8 of 32, 32, 38 and 30.
    const bool block = !few && min(tokens, a.c.max_new) * hu.count >= kThreads &&
                       static_cast<uint64_t>(blocks) * 2 * a.c.kv_heads < 148 * 32;
    auto* kernel = few ? append_codes_kernel<T, 8> : block ? append_codes_kernel<T, kThreads> : append_codes_kernel<T, 32>;
    if (smem > 40 * 1024) {  // with the static part beyond the 48 KB that need no leave
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
        if (e != cudaSuccess) return e;
    }
    // heads in parts until there are four blocks a SM, or a group has one head
    const uint32_t groups = kThreads / (few ? 8 : block ? kThreads : 32);
    uint32_t parts = 1;
    while (parts < 64 && static_cast<uint64_t>(blocks) * parts < 148 * 4 && 2 * a.c.kv_heads > groups * parts) parts *= 2;
    kernel<<<dim3(blocks, parts), kThreads, smem, s>>>(a, divs_of(a.c, hu.count, q_heads, runs), runs);
    return cudaGetLastError();
}
template <typename T, bool kCodes> cudaError_t gather(const GatherArgs& a, cudaStream_t s) {
    const uint32_t runs = runs_of(a.c, 16);
    gather_kernel<T, kCodes><<<runs * a.c.sequences, kThreads, 0, s>>>(a, divs_of(a.c, 1, 1, runs), runs);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cache_append(const AppendArgs& a, int dtype, int storage, cudaStream_t s) {
    const bool codes = storage == LWM_CACHE_E4M3;
    return dtype == LWM_DTYPE_BF16 ? append<bf16>(a, codes, s) : append<__half>(a, codes, s);
}
cudaError_t launch_cache_gather(const GatherArgs& a, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? gather<bf16, true>(a, s) : gather<__half, true>(a, s);
    return dtype == LWM_DTYPE_BF16 ? gather<bf16, false>(a, s) : gather<__half, false>(a, s);
}

}  // namespace lwm
