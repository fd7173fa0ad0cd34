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

// ------------------------------------------------------- shared prefixes

struct GroupView {
    uint32_t first = 0, end = 0;  // sequences
    uint32_t start = 0, n = 0;    // packed rows [start, start + n)
    uint32_t shared = 0;          // tokens of the prefix
    bool ok = false;
};
// Group g as the arrays give it; one that does not fit comes back with ok
// false, and so does every sequence that would belong to it.
__device__ __forceinline__ GroupView group_view(const CacheAttnArgs& a, uint32_t g, bool report) {
    GroupView v;
    const int first = a.groups[g], end = a.groups[g + 1], len = a.shared[g];
    int detail = end;
    bool fits = first >= 0 && end >= first && static_cast<uint32_t>(end) <= a.c.sequences;
    if (fits) {
        const int st = a.c.starts[first], en = a.c.starts[end];
        fits = st >= 0 && en >= st && static_cast<uint32_t>(en) <= a.c.tokens && static_cast<uint32_t>(en - st) <= a.max_tokens;
        detail = en;
        v.start = static_cast<uint32_t>(st);
        v.n = static_cast<uint32_t>(en - st);
        if (fits) {
            fits = len >= 0 && static_cast<uint64_t>(len) <= (static_cast<uint64_t>(a.c.table_stride) << a.c.page_shift);
            detail = len;
        }
    }
    if (!fits) {
        if (report) cache_report(a.c.err, kCacheErrGroup, g, detail);
        return v;
    }
    v.first = static_cast<uint32_t>(first);
    v.end = static_cast<uint32_t>(end);
    v.shared = static_cast<uint32_t>(len);
    v.ok = true;
    return v;
}
// The last entry of a sorted array [lo, hi) that is at most x (lo: there is
// none); any contents end the search in bounds.
__device__ __forceinline__ uint32_t last_at_most(const int32_t* a, uint32_t lo, uint32_t hi, int x) {
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
// What packed row `tok` of a group sees of its prefix.
__device__ __forceinline__ VisibleRange visible_prefix(const CacheAttnArgs& a, const GroupView& v, uint32_t tok) {
    VisibleRange r = {0, v.shared, 0};
    if (!a.window) return r;
    const uint32_t row = v.start + tok;
    const uint32_t s = last_at_most(a.c.starts, v.first, v.end, static_cast<int>(row));
    const int64_t p = static_cast<int64_t>(a.c.lengths[s]) - (static_cast<int64_t>(a.c.starts[s + 1]) - row);
    if (p < v.shared) return r;  // (a sequence that is skipped)
    const uint64_t after = (static_cast<uint64_t>(a.frame_div.div(static_cast<uint32_t>(p))) + 1) * a.frame;
    const uint64_t back = static_cast<uint64_t>(a.window) * a.frame;
    r.lo = after > back ? static_cast<uint32_t>(min(after - back, static_cast<uint64_t>(v.shared))) : 0u;
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
