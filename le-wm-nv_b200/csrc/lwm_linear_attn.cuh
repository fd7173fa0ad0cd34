// lwm_linear_attn.cuh — device helpers of the linear-attention kernels: the
// checked view of a sequence and its state slots, tiles in shared memory,
// tensor-core fragments.
#pragma once

#include <type_traits>

#include "lwm_blocks.cuh"

namespace lwm {

struct StateView {
    uint32_t start = 0, n = 0;  // packed rows [start, start + n)
    int source = -1, target = -1;  // slots, -1: zero, not kept
    bool ok = false;
};
// Sequence s as the batch's arrays give it; one that does not fit comes back
// with ok false.
__device__ __forceinline__ StateView state_view(const LinearArgs& a, uint32_t s, bool report) {
    StateView v;
    const int st = a.starts[s], en = a.starts[s + 1];
    const int src = a.source ? a.source[s] : static_cast<int>(s), dst = a.target ? a.target[s] : static_cast<int>(s);
    int code = 0, detail = 0;
    if (st < 0 || en < st || static_cast<uint32_t>(en) > a.tokens) {
        code = kStateErrStarts;
        detail = en;
    } else if (static_cast<uint32_t>(en - st) > a.max_new) {
        code = kStateErrNew;
        detail = en - st;
    } else if (src >= static_cast<int>(a.slots) || dst >= static_cast<int>(a.slots)) {
        code = kStateErrSlot;
        detail = src >= static_cast<int>(a.slots) ? src : dst;
    }
    if (code) {
        if (report) cache_report(a.err, code, s, detail);
        return v;
    }
    v.start = static_cast<uint32_t>(st);
    v.n = static_cast<uint32_t>(en - st);
    v.source = src;
    v.target = dst;
    v.ok = true;
    return v;
}

// e^x, x at most zero, as a sum of two floats: the one below the nearest float,
// and what is left of it.  Near one a single float is off by up to 2^-25, which
// a state that is multiplied again and again would forget more or less by; far
// from one, e^x - 1 alone would keep only 2^-24 of one, not of e^x.  (Both are
// positive, so an infinite state stays infinite.)
struct Fade {
    float most, rest;
};
__device__ __forceinline__ Fade fade_of(float x) {
    const float less = expm1f(x);
    const bool near = x > -0.5f;
    const float all = near ? 1.0f + less : expf(x);
    const float lost = near ? less - (all - 1.0f) : 0.0f;  // (exact)
    const float most = all > 0.0f ? __uint_as_float(__float_as_uint(all) - 1u) : all;
    return {most, (all - most) + lost};
}
// y e^x + added, rounded at y's size once.
__device__ __forceinline__ float faded(const Fade& f, float y, float added) { return fmaf(y, f.most, fmaf(y, f.rest, added)); }

// Two products and sums at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r)
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)), "l"(reinterpret_cast<const uint64_t&>(c)));
    return reinterpret_cast<const float2&>(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
    return reinterpret_cast<const float2&>(r);
}
__device__ __forceinline__ float2 faded(const Fade& f, float2 y, float2 added) {
    return fma2(y, make_float2(f.most, f.most), fma2(y, make_float2(f.rest, f.rest), added));
}
__device__ __forceinline__ float2 faded(const Fade& f, float2 y, float2 added, float2 times) {  // added times times
    return fma2(y, make_float2(f.most, f.most), fma2(added, times, mul2(y, make_float2(f.rest, f.rest))));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    // a dead row's 16 bytes are filled with zeros, its address is not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte chunk c of row r of a tile of D 16-bit channels:
// 128-byte lines whose chunks are permuted, so that 8 rows of one chunk touch
// every bank once.
template <int D> __device__ __forceinline__ uint32_t tile_at(uint32_t r, uint32_t c) {
    if constexpr (D >= 64) return r * D * 2 + ((c ^ (r & 7)) << 4);
    else return (r >> 1) * 128 + (((((r & 1) << 2) + c) ^ ((r >> 1) & 3)) << 4);
}
template <typename T, int D> __device__ __forceinline__ float tile_value(const uint8_t* tile, uint32_t r, uint32_t ch) {
    return static_cast<float>(*reinterpret_cast<const T*>(tile + tile_at<D>(r, ch >> 3) + (ch & 7) * 2));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, bf16>)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float2 half2_at(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T> __device__ __forceinline__ float2 pair_at(uint32_t w) {
    if constexpr (std::is_same_v<T, bf16>) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return half2_at(w);
}
// Whether a pair of 16-bit values holds an infinity or a NaN; the pair with
// those as zeros.
template <typename T> __device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t e = std::is_same_v<T, bf16> ? 0x7f80u : 0x7c00u;
    return (w & e) == e || ((w >> 16) & e) == e;
}
template <typename T> __device__ __forceinline__ uint32_t finite2(uint32_t w) {
    constexpr uint32_t e = std::is_same_v<T, bf16> ? 0x7f80u : 0x7c00u;
    if ((w & e) == e) w &= 0xffff0000u;
    if (((w >> 16) & e) == e) w &= 0x0000ffffu;
    return w;
}
// Powers of two (x, 1 / x) with top * x in [2^14, 2^15); ones where top is
// zero or not finite.
__device__ __forceinline__ float2 row_scale(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23);  // (top >= 0)
    if (e == 0 || e == 255) return make_float2(1.0f, 1.0f);
    const int by = min(max(127 + 14 - e, -100), 100);
    return make_float2(__uint_as_float(static_cast<uint32_t>(127 + by) << 23), __uint_as_float(static_cast<uint32_t>(127 - by) << 23));
}

}  // namespace lwm
