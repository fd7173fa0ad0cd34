// lwm_blocks.cuh — device helpers of the transformer-block kernels: 16-byte
// vectors of 8 values, the 8-bit codes, rotary angles, and the checked view
// of a batch of paged sequences.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lwm_blocks.hpp"

namespace lwm {

using bf16 = __nv_bfloat16;

// ---------------------------------------------------------- 8-value vectors

template <typename T> struct Vec8;  // 8 values: one 16-byte word, two for f32
template <> struct Vec8<float> { float4 a, b; };
template <> struct Vec8<bf16> { uint4 a; };
template <> struct Vec8<__half> { uint4 a; };

__device__ __forceinline__ Vec8<float> load8(const float* p) {
    return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
}
__device__ __forceinline__ Vec8<bf16> load8(const bf16* p) { return {*reinterpret_cast<const uint4*>(p)}; }
__device__ __forceinline__ Vec8<__half> load8(const __half* p) { return {*reinterpret_cast<const uint4*>(p)}; }
__device__ __forceinline__ void store8(float* p, const Vec8<float>& v) {
    reinterpret_cast<float4*>(p)[0] = v.a;
    reinterpret_cast<float4*>(p)[1] = v.b;
}
__device__ __forceinline__ void store8(bf16* p, const Vec8<bf16>& v) { *reinterpret_cast<uint4*>(p) = v.a; }
__device__ __forceinline__ void store8(__half* p, const Vec8<__half>& v) { *reinterpret_cast<uint4*>(p) = v.a; }

__device__ __forceinline__ void unpack(const Vec8<float>& v, float (&f)[8]) {
    f[0] = v.a.x; f[1] = v.a.y; f[2] = v.a.z; f[3] = v.a.w;
    f[4] = v.b.x; f[5] = v.b.y; f[6] = v.b.z; f[7] = v.b.w;
}
__device__ __forceinline__ void unpack(const Vec8<bf16>& v, float (&f)[8]) {
    const uint32_t w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const Vec8<__half>& v, float (&f)[8]) {
    const uint32_t w[4] = {v.a.x, v.a.y, v.a.z, v.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bf16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}
template <typename T> __device__ __forceinline__ Vec8<T> pack(const float (&f)[8]) {
    if constexpr (sizeof(T) == 4)
        return {make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7])};
    else
        return {make_uint4(pack2(f[0], f[1], T{}), pack2(f[2], f[3], T{}), pack2(f[4], f[5], T{}),
                           pack2(f[6], f[7], T{}))};
}

// ------------------------------------------------------------- 8-bit codes

// 8 values, already divided by the scale, as e4m3 codes (round to nearest
// even).  The conversion saturates; infinities become NaN here, so that what
// the format cannot hold stays visible.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float no_inf(float v) { return isinf(v) ? __int_as_float(0x7fc00000) : v; }
__device__ __forceinline__ uint2 to_e4m3(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = e4m3x2(no_inf(f[2 * i]), no_inf(f[2 * i + 1]));
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}
// Two codes as a pair of halves (exact).
__device__ __forceinline__ uint32_t f16x2_from_e4m3x2(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
    return r;
}
__device__ __forceinline__ void from_e4m3(uint2 c, float (&f)[8]) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t h = f16x2_from_e4m3x2(w[i >> 1] >> (16 * (i & 1)));
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
}
// The least 2^e, e in [-120, 120], with amax <= 448 * 2^e (448 = 1.75 * 2^8).
__device__ __forceinline__ float page_scale(float amax) {
    const uint32_t b = __float_as_uint(amax);
    int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = min(max(e, -120), 120);
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// ----------------------------------------------------------- rotary angles

// cos and sin of position * frequency.  The frequency is in 2^-64 turns, so
// the product modulo 2^64 is the angle's fraction of a turn with an error of
// 2^-65 turns per position whatever the position; its top 32 bits, signed,
// are half-turns in [-1, 1).
__device__ __forceinline__ float2 turn_of(int32_t position, uint64_t turn) {
    const uint64_t t = static_cast<uint64_t>(static_cast<int64_t>(position)) * turn;
    float s, c;
    sincospif(static_cast<float>(static_cast<int32_t>(t >> 32)) * 4.656612873077393e-10f, &s, &c);  // * 2^-31
    return make_float2(c, s);
}
__device__ __forceinline__ uint32_t axis_of(const lwm_rotary& r, uint32_t pair) {
    uint32_t a = 0, end = r.dims[0] / 2;
    while (pair >= end) end += r.dims[++a] / 2;
    return a;
}
// A launch's frequencies and axes by pair, in shared memory: in the kernel's
// parameters they are constants, which a warp reads one address at a time
// (61316 tokens of one head: 24 us so, 15.5 from shared memory).
struct PairTurns {
    uint64_t turn[LWM_ROTARY_MAX_PAIRS];
    uint8_t axis[LWM_ROTARY_MAX_PAIRS];
};
// (the caller synchronises the block)
__device__ __forceinline__ void fill_turns(const lwm_rotary& r, uint32_t pairs, PairTurns& to) {
    for (uint32_t p = threadIdx.x; p < pairs; p += blockDim.x) {
        to.turn[p] = r.turn[p];
        to.axis[p] = static_cast<uint8_t>(axis_of(r, p));
    }
}

// A head as units of work: with halves, unit u < pairs / 8 is two vectors,
// channels [c, c + 8) and [c + n/2, c + n/2 + 8) of an axis with n channels;
// interleaved, unit u < pairs / 4 is the vector at 8 u.  The units behind
// are single vectors that pass through.
struct HeadUnits {
    uint32_t turned, count;  // units that turn, and all units
    __host__ __device__ HeadUnits(uint32_t pairs, int interleaved, uint32_t head_dim)
        : turned(interleaved ? pairs / 4 : pairs / 8), count(turned + (head_dim - 2 * pairs) / 8) {}
};
// First channel of a turning unit and the distance to its second vector
// (halves); trig of its pairs starts at `pair`.
__device__ __forceinline__ void unit_place(const lwm_rotary& r, uint32_t u, uint32_t& channel, uint32_t& apart,
                                           uint32_t& pair) {
    if (r.interleaved) {
        channel = 8 * u;
        apart = 0;
        pair = 4 * u;
        return;
    }
    pair = 8 * u;
    uint32_t a = 0, base = 0, p0 = 0;
    while (pair >= p0 + r.dims[a] / 2) {
        p0 += r.dims[a] / 2;
        base += r.dims[a];
        ++a;
    }
    channel = base + (pair - p0);
    apart = r.dims[a] / 2;
}
// Turns a unit's values: halves a[i], b[i] by cs[i]; interleaved a[2i],
// a[2i + 1] by cs[i].
__device__ __forceinline__ void turn_halves(float (&a)[8], float (&b)[8], const float2* cs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 t = cs[i];
        const float x = a[i], y = b[i];
        a[i] = x * t.x - y * t.y;
        b[i] = x * t.y + y * t.x;
    }
}
__device__ __forceinline__ void turn_pairs(float (&a)[8], const float2* cs) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = cs[i];
        const float x = a[2 * i], y = a[2 * i + 1];
        a[2 * i] = x * t.x - y * t.y;
        a[2 * i + 1] = x * t.y + y * t.x;
    }
}

// ------------------------------------------------------- paged sequences

__device__ __forceinline__ void cache_report(uint64_t* err, int code, uint32_t seq, int detail) {
    const uint64_t word = cache_report_word({code, seq, detail});
    const uint32_t lo = static_cast<uint32_t>(word), hi = static_cast<uint32_t>(word >> 32);
    // (joined here: as a 64-bit operand it cost the append's kernels the register that their third block a SM needs)
    asm volatile("{\n\t.reg .b64 w;\n\tmov.b64 w, {%1, %2};\n\tst.volatile.global.u64 [%0], w;\n\t}" ::"l"(err), "r"(lo), "r"(hi)
                 : "memory");
}

struct SeqView {
    uint32_t start = 0, n = 0, length = 0;  // packed rows [start, start + n), cached tokens
    bool ok = false;
};
// Sequence s as the batch's arrays give it; one that does not fit the batch
// comes back with ok false (reported once per calling thread).
__device__ __forceinline__ SeqView sequence(const CacheArgs& c, uint32_t s, bool append, bool report) {
    SeqView v;
    const int st = c.starts[s], en = c.starts[s + 1], len = c.lengths[s];
    int code = 0, detail = 0;
    if (st < 0 || en < st || static_cast<uint32_t>(en) > c.tokens) {
        code = kCacheErrStarts;
        detail = en;
    } else if (len < 0 || static_cast<uint64_t>(len) > (static_cast<uint64_t>(c.table_stride) << c.page_shift)) {
        code = kCacheErrLength;
        detail = len;
    } else if (static_cast<uint32_t>(en - st) > c.max_new || (append && en - st > len)) {
        code = kCacheErrNew;
        detail = en - st;
    }
    if (code) {
        if (report) cache_report(c.err, code, s, detail);
        return v;
    }
    v.start = static_cast<uint32_t>(st);
    v.n = static_cast<uint32_t>(en - st);
    v.length = static_cast<uint32_t>(len);
    v.ok = true;
    return v;
}
// The page of table entry `j`, or -1 (reported) when it is not in the pool.
__device__ __forceinline__ int page_of(const CacheArgs& c, uint32_t s, uint32_t j) {
    const int p = c.table[static_cast<size_t>(s) * c.table_stride + j];
    if (static_cast<uint32_t>(p) < c.pages) return p;
    cache_report(c.err, kCacheErrPage, s, p);
    return -1;
}
// Elements before (page, head, slot) of a pool.
__device__ __forceinline__ size_t pool_at(const CacheArgs& c, uint32_t page, uint32_t head, uint32_t slot) {
    return ((static_cast<size_t>(page) * c.kv_heads + head) * c.page_tokens + slot) * c.head_dim;
}

}  // namespace lwm
