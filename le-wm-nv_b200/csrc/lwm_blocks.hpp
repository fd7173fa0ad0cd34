// lwm_blocks.hpp — argument blocks and launchers of the transformer-block
// kernels: rotary positions, the paged cache, its attention, gated norms.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/lewm_b200.h"

namespace lwm {

// Division by a launch constant: q = (n * mul) >> 32 >> shift, exact for
// n < 2^31 and 0 < d <= 2^31 (mul = ceil(2^(32 + shift) / d) - 2^32, shift =
// ceil(log2 d), which is 32 for larger d and no shift of 32 bits).
struct FastDiv {
    uint32_t d = 1, mul = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((1ull << shift) < d) ++shift;
        const uint64_t m = ((1ull << 32) * ((1ull << shift) - d)) / d + 1;
        mul = static_cast<uint32_t>(m);
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
        const uint32_t t = __umulhi(n, mul);
#else
        const uint32_t t = static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> 32);
#endif
        return (t + n) >> shift;
    }
};

// Codes of the paged-cache kernels' error word.  It is one 64-bit store (code
// above 27 bits of sequence above 32 of detail), so that of many threads that
// report at once one is read whole, not one's page with another's sequence.
constexpr int kCacheErrStarts = 1, kCacheErrNew = 2, kCacheErrLength = 3, kCacheErrPage = 4, kCacheErrWait = 5;
constexpr uint32_t kCacheErrSequences = 1u << 27;  // as many as a batch may have
struct CacheReport {
    int code;
    uint32_t sequence;
    int detail;
};
__host__ __device__ inline uint64_t cache_report_word(const CacheReport& r) {
    const uint32_t high = static_cast<uint32_t>(r.code) * kCacheErrSequences + r.sequence;
    return static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(r.detail);
}
inline CacheReport cache_report_of(uint64_t word) {
    const uint32_t high = static_cast<uint32_t>(word >> 32);
    return {static_cast<int>(high / kCacheErrSequences), high % kCacheErrSequences, static_cast<int>(static_cast<uint32_t>(word))};
}

struct RotaryArgs {
    lwm_rotary r;
    uint32_t pairs, turned;  // rotated pairs and channels (2 * pairs)
    const void* x;
    void* out;
    size_t x_ts, x_hs, o_ts, o_hs;
    const int32_t* positions;
    uint32_t tokens, heads, head_dim;
    int inverse;
};
cudaError_t launch_rotary(const RotaryArgs& a, int dtype, cudaStream_t s);

// The cache, its batch and the error word, as the kernels see them.
struct CacheArgs {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    uint32_t pages, kv_heads, page_tokens, page_shift, head_dim;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    uint32_t sequences, table_stride, tokens, max_new, max_length;
    uint64_t* err;
};
struct AppendArgs {
    CacheArgs c;
    lwm_rotary r;
    uint32_t axes, pairs, turned;  // pairs 0: nothing is turned
    const void* q;
    void* q_out;
    const void* k;
    const void* v;
    size_t q_ts, q_hs, qo_ts, qo_hs, k_ts, k_hs, v_ts, v_hs;
    const int32_t* positions;
    uint32_t heads;
};
cudaError_t launch_cache_append(const AppendArgs& a, int dtype, int storage, cudaStream_t s);
struct GatherArgs {
    CacheArgs c;
    void* k_out;
    void* v_out;
    size_t k_ts, k_hs, v_ts, v_hs;
};
cudaError_t launch_cache_gather(const GatherArgs& a, int dtype, int storage, cudaStream_t s);

struct CacheAttnArgs {
    CacheArgs c;
    const void* q;
    void* out;
    size_t q_ts, q_hs, o_ts, o_hs;
    uint32_t heads, group;   // query heads, and those of a kv head
    float scale_log2;        // scale * log2(e)
    int causal;
    uint32_t window, sinks, frame;
    FastDiv group_div, frame_div;
    FastDiv tile_div, kv_div;  // set by the launch
};
// Keys that a tile of query rows can see, by the sizes that the host knows.
inline uint64_t visible_span(const CacheAttnArgs& a, uint32_t tile_rows) {
    const uint64_t reach = a.c.max_length ? a.c.max_length : static_cast<uint64_t>(a.c.table_stride) << a.c.page_shift;
    if (!a.window) return reach;
    // the window of the tile's first token, up to the end of its last one's frame (or of the sequence)
    const uint64_t tokens = static_cast<uint64_t>(tile_rows) / a.group + 1 + a.frame;
    const uint64_t beyond = a.causal && tokens < a.c.max_new ? tokens : a.c.max_new;
    const uint64_t keys = static_cast<uint64_t>(a.window) * a.frame + a.sinks + beyond;
    return keys < reach ? keys : reach;
}
// Few query rows a kv head, and many.
cudaError_t launch_cache_attention(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s);
bool cache_attention_many_rows(const CacheAttnArgs& a);  // which of the two
cudaError_t launch_cache_attention_tc(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s);

struct GatedNormArgs {
    lwm_gated_norm_args a;
    FastDiv cond_div;
    int out_norm;
};
cudaError_t launch_gated_norm(const GatedNormArgs& a, cudaStream_t s);

}  // namespace lwm
