// kernels_cache.cu — the paged cache's writes and reads: append with the
// rotary turn on the way (lwm_cache_append_device) and gather
// (lwm_cache_gather_device).  Bound: memory.
//
// One block per (sequence, page that gets new tokens): the angles of the
// page's new tokens are computed once into shared memory and serve every
// head.  16-bit storage is element-wise from there.  In 8 bits a warp owns a
// (page, head): the new tokens' largest value first, then the scale, the
// earlier tokens' codes where the scale grew, and the new codes, so that no
// scale is shared between warps.
#include "lwm_blocks.cuh"

namespace lwm {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// The new tokens of one page of a sequence.
struct PagePart {
    uint32_t row, slot, count;  // first packed row and slot (the page's earlier tokens), tokens
    uint32_t index;             // cache index of the first
    int page;                   // -1: nothing to do
};
__device__ __forceinline__ PagePart page_part(const CacheArgs& c, const SeqView& v, uint32_t s, uint32_t ordinal) {
    PagePart p{0, 0, 0, 0, -1};
    if (!v.ok || v.n == 0 || v.n > v.length) return p;
    const uint32_t first = v.length - v.n, j = (first >> c.page_shift) + ordinal;
    if (static_cast<uint64_t>(j) << c.page_shift >= v.length) return p;
    const uint32_t begin = max(first, j << c.page_shift), end = min(v.length, (j + 1) << c.page_shift);
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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float finite_abs(float v) { return isfinite(v) ? fabsf(v) : 0.0f; }

// One (page, head) of an 8-bit pool, by one warp.
template <typename T>
__device__ void append_codes(const AppendArgs& a, const PagePart& p, uint32_t held, uint32_t h, bool keys,
                             const float2* trig, int lane) {
    const HeadUnits hu(keys ? a.pairs : 0, a.r.interleaved, a.c.head_dim);
    const uint32_t pairs = keys ? a.pairs : 0;
    const T* src = static_cast<const T*>(keys ? a.k : a.v);
    const size_t ts = keys ? a.k_ts : a.v_ts, hs = keys ? a.k_hs : a.v_hs;
    float* scale_at = (keys ? a.c.k_scale : a.c.v_scale) + static_cast<size_t>(p.page) * a.c.kv_heads + h;
    uint8_t* pool = static_cast<uint8_t*>(keys ? a.c.k : a.c.v) + pool_at(a.c, p.page, h, 0);
    const uint32_t work = p.count * hu.count;
    float amax = 0.0f;
    for (uint32_t i = lane; i < work; i += 32) {
        const uint32_t t = i / hu.count, u = i - t * hu.count;
        head_unit<T>(a.r, pairs, hu, u, src + (p.row + t) * ts + h * hs, trig + t * a.pairs,
                     [&](uint32_t, const float(&v)[8]) {
#pragma unroll
                         for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[e]));
                     });
    }
    float scale = page_scale(warp_max(amax));
    if (held) {
        // the page holds earlier tokens: its scale never falls, and their
        // codes are rounded again where it grows
        const float old = *scale_at;
        if (!(old >= scale)) {
            const float again = old / scale;
            for (uint32_t i = lane; i < held * (a.c.head_dim / 8); i += 32) {
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
    for (uint32_t i = lane; i < work; i += 32) {
        const uint32_t t = i / hu.count, u = i - t * hu.count;
        uint8_t* row = pool + static_cast<size_t>(p.slot + t) * a.c.head_dim;
        head_unit<T>(a.r, pairs, hu, u, src + (p.row + t) * ts + h * hs, trig + t * a.pairs,
                     [&](uint32_t ch, float(&v)[8]) {
#pragma unroll
                         for (int e = 0; e < 8; ++e) v[e] *= inv;
                         *reinterpret_cast<uint2*>(row + ch) = to_e4m3(v);
                     });
    }
    __syncwarp();
    if (lane == 0) *scale_at = scale;
}

template <typename T, bool kCodes>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, uint32_t ordinals) {
    extern __shared__ float2 trig[];  // [page_tokens][pairs]
    const uint32_t s = blockIdx.x / ordinals, ordinal = blockIdx.x - s * ordinals;
    const SeqView v = sequence(a.c, s, true, threadIdx.x == 0 && ordinal == 0);
    const PagePart p = page_part(a.c, v, s, ordinal);
    if (p.page < 0) return;
    for (uint32_t i = threadIdx.x; i < p.count * a.pairs; i += kThreads) {
        const uint32_t t = i / a.pairs, pr = i - t * a.pairs;
        const int32_t pos = a.positions
                                ? a.positions[static_cast<size_t>(p.row + t) * a.axes + axis_of(a.r, pr)]
                                : static_cast<int32_t>(p.index + t);
        trig[i] = turn_of(pos, a.r.turn[pr]);
    }
    __syncthreads();
    const uint32_t kv = a.c.kv_heads, d = a.c.head_dim;
    const HeadUnits hu(a.pairs, a.r.interleaved, d);
    const uint32_t q_heads = a.q ? a.heads : 0, turning = q_heads + (kCodes ? 0 : kv);
    // queries, and in 16 bits keys: (token, head, unit)
    for (uint32_t i = threadIdx.x; i < p.count * turning * hu.count; i += kThreads) {
        const uint32_t row = i / hu.count, u = i - row * hu.count;
        const uint32_t t = row / turning, h = row - t * turning;
        const bool is_q = h < q_heads;
        const size_t r = p.row + t;
        const T* src = is_q ? static_cast<const T*>(a.q) + r * a.q_ts + h * a.q_hs
                            : static_cast<const T*>(a.k) + r * a.k_ts + (h - q_heads) * a.k_hs;
        T* dst = is_q ? static_cast<T*>(a.q_out) + r * a.qo_ts + h * a.qo_hs
                      : static_cast<T*>(a.c.k) + pool_at(a.c, p.page, h - q_heads, p.slot + t);
        // both vectors are read before either is written: q_out may be q
        head_unit<T>(a.r, a.pairs, hu, u, src, trig + t * a.pairs,
                     [&](uint32_t ch, const float(&x)[8]) { store8(dst + ch, pack<T>(x)); });
    }
    if constexpr (kCodes) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (uint32_t job = warp; job < 2 * kv; job += kWarps)
            append_codes<T>(a, p, p.slot, job < kv ? job : job - kv, job < kv, trig, lane);
    } else {
        const uint32_t vecs = d / 8;
        for (uint32_t i = threadIdx.x; i < p.count * kv * vecs; i += kThreads) {
            const uint32_t row = i / vecs, c8 = 8 * (i - row * vecs);
            const uint32_t t = row / kv, h = row - t * kv;
            const T* src = static_cast<const T*>(a.v) + (p.row + t) * a.v_ts + h * a.v_hs + c8;
            store8(static_cast<T*>(a.c.v) + pool_at(a.c, p.page, h, p.slot + t) + c8, load8(src));
        }
    }
}

template <typename T, bool kCodes>
__global__ void __launch_bounds__(kThreads) gather_kernel(GatherArgs a, uint32_t ordinals) {
    const uint32_t s = blockIdx.x / ordinals, ordinal = blockIdx.x - s * ordinals;
    const SeqView v = sequence(a.c, s, true, threadIdx.x == 0 && ordinal == 0);
    const PagePart p = page_part(a.c, v, s, ordinal);
    if (p.page < 0) return;
    const uint32_t kv = a.c.kv_heads, vecs = a.c.head_dim / 8;
    for (uint32_t i = threadIdx.x; i < 2 * p.count * kv * vecs; i += kThreads) {
        uint32_t row = i / vecs;
        const uint32_t c8 = 8 * (i - row * vecs);
        const bool keys = row < p.count * kv;
        if (!keys) row -= p.count * kv;
        const uint32_t t = row / kv, h = row - t * kv;
        const size_t r = p.row + t, at = pool_at(a.c, p.page, h, p.slot + t) + c8;
        T* dst = keys ? static_cast<T*>(a.k_out) + r * a.k_ts + h * a.k_hs
                      : static_cast<T*>(a.v_out) + r * a.v_ts + h * a.v_hs;
        const void* pool = keys ? a.c.k : a.c.v;
        if constexpr (kCodes) {
            const float scale = (keys ? a.c.k_scale : a.c.v_scale)[static_cast<size_t>(p.page) * kv + h];
            float f[8];
            from_e4m3(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= scale;
            store8(dst + c8, pack<T>(f));
        } else {
            store8(dst + c8, load8(static_cast<const T*>(pool) + at));
        }
    }
}

// Pages that up to max_new tokens of a sequence can lie in.
uint32_t page_ordinals(const CacheArgs& c) { return (c.max_new + c.page_tokens - 2) / c.page_tokens + 1; }

template <typename T, bool kCodes> cudaError_t append(const AppendArgs& a, cudaStream_t s) {
    const size_t smem = static_cast<size_t>(min(a.c.page_tokens, a.c.max_new)) * a.pairs * sizeof(float2);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(append_kernel<T, kCodes>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
        if (e != cudaSuccess) return e;
    }
    const uint32_t ord = page_ordinals(a.c);
    append_kernel<T, kCodes><<<ord * a.c.sequences, kThreads, smem, s>>>(a, ord);
    return cudaGetLastError();
}
template <typename T, bool kCodes> cudaError_t gather(const GatherArgs& a, cudaStream_t s) {
    const uint32_t ord = page_ordinals(a.c);
    gather_kernel<T, kCodes><<<ord * a.c.sequences, kThreads, 0, s>>>(a, ord);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cache_append(const AppendArgs& a, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? append<bf16, true>(a, s) : append<__half, true>(a, s);
    return dtype == LWM_DTYPE_BF16 ? append<bf16, false>(a, s) : append<__half, false>(a, s);
}
cudaError_t launch_cache_gather(const GatherArgs& a, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? gather<bf16, true>(a, s) : gather<__half, true>(a, s);
    return dtype == LWM_DTYPE_BF16 ? gather<bf16, false>(a, s) : gather<__half, false>(a, s);
}

}  // namespace lwm
