// lwm_cache_attn.cuh — what the attention kernels over the paged cache
// share: which keys a token sees, and the softmax's exponential.
#pragma once

#include <type_traits>

#include "lwm_blocks.cuh"

namespace lwm {

// A row's maximum is raised only when a score passes it by this many powers
// of two, so that most steps need no rescaling; weights stay below 2^8.
constexpr float kRaise = 8.0f;

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// The keys that packed token `tok` of a sequence sees: [0, first) and
// [lo, hi), first <= lo.  All three only grow with the token.
struct VisibleRange {
    uint32_t lo, hi, first;
};
__device__ __forceinline__ VisibleRange visible(const CacheAttnArgs& a, const SeqView& v, uint32_t tok) {
    const int64_t p = static_cast<int64_t>(v.length) - v.n + tok;
    if (p < 0) return {0, 0, 0};  // before the first cached token
    const uint64_t after = (static_cast<uint64_t>(a.frame_div.div(static_cast<uint32_t>(p))) + 1) * a.frame;
    const uint64_t back = static_cast<uint64_t>(a.window) * a.frame;
    VisibleRange r;
    r.hi = a.causal && after < v.length ? static_cast<uint32_t>(after) : v.length;
    r.lo = a.window && after > back ? static_cast<uint32_t>(after - back) : 0u;
    r.first = min(a.sinks, r.lo);
    return r;
}

// Whether a 32-bit word of pool values (two of T, or four codes) holds an
// infinity or a NaN.
template <typename T, bool kCodes> __device__ __forceinline__ bool any_not_finite(uint32_t w) {
    if constexpr (kCodes) {
        const uint32_t x = w | 0x80808080u;  // a code is NaN when its low 7 bits are set
        return __vcmpeq4(x, 0xffffffffu) != 0;
    } else {
        constexpr uint32_t e = std::is_same_v<T, bf16> ? 0x7f80u : 0x7c00u;
        return (w & e) == e || ((w >> 16) & e) == e;
    }
}

}  // namespace lwm
