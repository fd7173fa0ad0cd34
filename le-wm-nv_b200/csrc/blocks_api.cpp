// blocks_api.cpp — the C ABI of the transformer blocks (include/lewm_b200.h):
// argument checks and launches of the rotary, paged-cache, attention and
// gated-norm kernels.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "../../include/lewm_b200.h"
#include "lwm_blocks.hpp"
#include "lwm_host.hpp"

namespace {

using lwm::CtxView;

lwm_status fail(lwm_status s, const std::string& m) { return lwm::set_last_error(s, m); }
lwm_status bad(const std::string& m) { return fail(LWM_INVALID_ARGUMENT, m); }

#define LWM_TRY(expr)                \
    do {                             \
        lwm_status s_ = (expr);      \
        if (s_ != LWM_OK) return s_; \
    } while (0)

// Runs `launch` with the context's device current and gives the caller's back.
template <class F> lwm_status on_device(lwm_ctx* ctx, const CtxView& c, const char* what, F launch) {
    int before = 0;
    cudaError_t e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != c.device) e = cudaSetDevice(c.device);
    if (e == cudaSuccess) e = launch(static_cast<cudaStream_t>(c.stream));
    if (before != c.device) cudaSetDevice(before);
    if (e != cudaSuccess) return fail(LWM_CUDA_ERROR, std::string(what) + " failed: " + cudaGetErrorString(e));
    lwm::ctx_add_launches(ctx, 1);
    return LWM_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// A [rows, heads, head_dim] tensor: aligned, strides in whole vectors.
lwm_status check_heads(const char* name, const void* p, uint64_t ts, uint64_t hs) {
    if (!p) return bad(std::string(name) + " is null");
    if (!aligned16(p)) return bad(std::string(name) + " is not 16-byte aligned");
    if (ts % 8 || hs % 8) return bad(std::string(name) + " strides must be multiples of 8 elements");
    return LWM_OK;
}

// Rotated pairs of a filled lwm_rotary, checked against a head's width.
lwm_status check_rotary(const lwm_rotary* r, uint32_t head_dim, uint32_t* pairs) {
    const uint32_t unit = r->interleaved ? 8 : 16;
    if (r->axes == 0 || r->axes > LWM_ROTARY_MAX_AXES) return bad("rotary axes must be 1 to 4");
    uint64_t sum = 0;
    for (uint32_t a = 0; a < r->axes; ++a) {
        if (r->dims[a] == 0 || r->dims[a] % unit)
            return bad("rotary dims[" + std::to_string(a) + "]=" + std::to_string(r->dims[a]) +
                       " must be a positive multiple of " + std::to_string(unit));
        sum += r->dims[a];
    }
    if (sum > 2 * LWM_ROTARY_MAX_PAIRS) return bad("rotary dims exceed 128 channels");
    if (head_dim && sum > head_dim)
        return bad("rotary dims (" + std::to_string(sum) + " channels) exceed head_dim " + std::to_string(head_dim));
    *pairs = static_cast<uint32_t>(sum / 2);
    return LWM_OK;
}

lwm_status check_cache(const lwm_paged_cache* c, const lwm_cache_batch* b, lwm::CacheArgs* out) {
    if (!c || !b) return bad("null cache or batch");
    if (c->dtype != LWM_DTYPE_BF16 && c->dtype != LWM_DTYPE_F16) return bad("cache dtype must be bf16 or f16");
    if (c->storage != LWM_CACHE_16BIT && c->storage != LWM_CACHE_E4M3) return bad("unknown cache storage");
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)
        return fail(LWM_UNSUPPORTED, "cache head_dim " + std::to_string(c->head_dim) + " is not 32, 64 or 128");
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
        return fail(LWM_UNSUPPORTED, "cache page_tokens " + std::to_string(c->page_tokens) + " is not 16, 32, 64 or 128");
    if (c->kv_heads == 0) return bad("cache kv_heads must be greater than zero");
    if (c->pages == 0) return bad("cache pages must be greater than zero");
    if (c->pages > 0x7fffffffu || c->kv_heads > 65535) return bad("cache pages or kv_heads out of range");
    if (!c->k || !c->v) return bad("cache pools are null");
    if (!aligned16(c->k) || !aligned16(c->v)) return bad("cache pools are not 16-byte aligned");
    if (c->storage == LWM_CACHE_E4M3 && (!c->k_scale || !c->v_scale)) return bad("an 8-bit cache needs its scales");
    if (c->storage == LWM_CACHE_E4M3 && (!aligned4(c->k_scale) || !aligned4(c->v_scale)))
        return bad("cache scales are not 4-byte aligned");
    if (b->sequences && (!b->table || !b->lengths || !b->starts)) return bad("batch arrays are null");
    if (b->sequences && (!aligned4(b->table) || !aligned4(b->lengths) || !aligned4(b->starts)))
        return bad("batch arrays are not 4-byte aligned");
    if (b->sequences && b->table_stride == 0) return bad("batch table_stride must be greater than zero");
    if (b->sequences > 0x7ffffffu || b->tokens > 0x7fffffffu || b->max_new > b->tokens)
        return bad("batch sizes out of range (max_new " + std::to_string(b->max_new) + ", tokens " +
                   std::to_string(b->tokens) + ")");
    lwm::CacheArgs a{};
    a.k = c->k;
    a.v = c->v;
    a.k_scale = c->k_scale;
    a.v_scale = c->v_scale;
    a.pages = c->pages;
    a.kv_heads = c->kv_heads;
    a.page_tokens = c->page_tokens;
    while ((1u << a.page_shift) < c->page_tokens) ++a.page_shift;
    a.head_dim = c->head_dim;
    a.table = b->table;
    a.lengths = b->lengths;
    a.starts = b->starts;
    a.sequences = b->sequences;
    a.table_stride = b->table_stride;
    a.tokens = b->tokens;
    a.max_new = b->max_new;
    a.max_length = b->max_length;
    *out = a;
    return LWM_OK;
}

// Blocks of a launch with one block per (sequence, run of 16 new tokens).
lwm_status check_run_blocks(const lwm::CacheArgs& a) {
    const uint64_t per = (static_cast<uint64_t>(a.max_new) + 14) / 16 + 1;
    if (per * a.sequences > 0x7fffffffull) return fail(LWM_UNSUPPORTED, "batch is too large for one call");
    return LWM_OK;
}

}  // namespace

extern "C" {

lwm_status lwm_rotary_init(uint32_t axes, const uint32_t* dims, const double* bases, int32_t interleaved,
                           lwm_rotary* out) {
    if (!dims || !bases || !out) return bad("null argument");
    lwm_rotary r;
    std::memset(&r, 0, sizeof r);
    r.axes = axes;
    r.interleaved = interleaved ? 1 : 0;
    if (axes == 0 || axes > LWM_ROTARY_MAX_AXES) return bad("rotary axes must be 1 to 4");
    for (uint32_t a = 0; a < axes; ++a) {
        r.dims[a] = dims[a];
        if (!std::isfinite(bases[a]) || bases[a] <= 0.0)
            return bad("rotary base " + std::to_string(a) + " must be finite and greater than zero");
    }
    uint32_t pairs = 0;
    LWM_TRY(check_rotary(&r, 0, &pairs));
    uint32_t p = 0;
    for (uint32_t a = 0; a < axes; ++a)
        for (uint32_t i = 0; i < dims[a] / 2; ++i, ++p) {
            // whole turns per position do not matter; the rest in 2^-64 turns
            const long double turns = std::pow(static_cast<long double>(bases[a]),
                                               -2.0L * i / static_cast<long double>(dims[a])) /
                                      6.283185307179586476925286766559L;
            long double part = turns - std::floor(turns);
            part = std::nearbyint(std::ldexp(part, 64));
            r.turn[p] = part >= 18446744073709551616.0L ? 0u : static_cast<uint64_t>(part);
        }
    *out = r;
    return LWM_OK;
}

lwm_status lwm_rotary_device(lwm_ctx* ctx, const lwm_rotary* rotary, const lwm_rotary_args* x) {
    if (!rotary || !x) return bad("null argument");
    lwm::RotaryArgs a{};
    a.r = *rotary;
    LWM_TRY(check_rotary(rotary, x->head_dim, &a.pairs));
    if (x->head_dim == 0 || x->head_dim % 8 || x->head_dim > 256)
        return fail(LWM_UNSUPPORTED, "rotary head_dim " + std::to_string(x->head_dim) + " must be a multiple of 8 up to 256");
    if (x->dtype < LWM_DTYPE_F32 || x->dtype > LWM_DTYPE_F16) return bad("unknown dtype");
    if (x->heads == 0) return bad("rotary heads must be greater than zero");
    if (x->tokens > 0x7fffffffu || x->heads > 65535) return bad("rotary tokens or heads out of range");
    if (x->tokens) {
        LWM_TRY(check_heads("x", x->x, x->x_token_stride, x->x_head_stride));
        LWM_TRY(check_heads("out", x->out, x->out_token_stride, x->out_head_stride));
        if (!x->positions) return bad("positions are null");
        if (!aligned4(x->positions)) return bad("positions are not 4-byte aligned");
    }
    CtxView c;
    if (!lwm::ctx_view(ctx, &c)) return bad("null context");
    if (x->tokens == 0) return LWM_OK;
    a.turned = 2 * a.pairs;
    a.x = x->x;
    a.out = x->out;
    a.x_ts = x->x_token_stride;
    a.x_hs = x->x_head_stride;
    a.o_ts = x->out_token_stride;
    a.o_hs = x->out_head_stride;
    a.positions = x->positions;
    a.tokens = x->tokens;
    a.heads = x->heads;
    a.head_dim = x->head_dim;
    a.inverse = x->inverse != 0;
    return on_device(ctx, c, "rotary", [&](cudaStream_t s) { return lwm::launch_rotary(a, x->dtype, s); });
}

lwm_status lwm_cache_append_device(lwm_ctx* ctx, const lwm_paged_cache* cache, const lwm_cache_batch* batch,
                                   const lwm_rotary* rotary, const lwm_cache_append_args* x) {
    if (!x) return bad("null argument");
    lwm::AppendArgs a{};
    LWM_TRY(check_cache(cache, batch, &a.c));
    LWM_TRY(check_run_blocks(a.c));
    if (rotary) {
        LWM_TRY(check_rotary(rotary, cache->head_dim, &a.pairs));
        a.r = *rotary;
        a.axes = rotary->axes;
    }
    if (x->q && x->heads == 0) return bad("query heads must be greater than zero");
    if (x->q && x->heads > 65535) return bad("query heads out of range");
    if (!x->q && x->q_out) return bad("q_out needs q");
    const bool work = a.c.sequences && a.c.max_new;
    if (!aligned4(x->positions)) return bad("positions are not 4-byte aligned");
    if (work) {
        LWM_TRY(check_heads("k", x->k, x->k_token_stride, x->k_head_stride));
        LWM_TRY(check_heads("v", x->v, x->v_token_stride, x->v_head_stride));
    }
    if (work && x->q) {
        LWM_TRY(check_heads("q", x->q, x->q_token_stride, x->q_head_stride));
        LWM_TRY(check_heads("q_out", x->q_out, x->q_out_token_stride, x->q_out_head_stride));
    }
    CtxView c;
    if (!lwm::ctx_view(ctx, &c)) return bad("null context");
    if (!work) return LWM_OK;
    a.c.err = c.cache_err;
    a.turned = 2 * a.pairs;
    a.q = x->q;
    a.q_out = x->q_out;
    a.k = x->k;
    a.v = x->v;
    a.q_ts = x->q_token_stride;
    a.q_hs = x->q_head_stride;
    a.qo_ts = x->q_out_token_stride;
    a.qo_hs = x->q_out_head_stride;
    a.k_ts = x->k_token_stride;
    a.k_hs = x->k_head_stride;
    a.v_ts = x->v_token_stride;
    a.v_hs = x->v_head_stride;
    a.positions = x->positions;
    a.heads = x->heads;
    return on_device(ctx, c, "cache append",
                     [&](cudaStream_t s) { return lwm::launch_cache_append(a, cache->dtype, cache->storage, s); });
}

lwm_status lwm_cache_gather_device(lwm_ctx* ctx, const lwm_paged_cache* cache, const lwm_cache_batch* batch,
                                   const lwm_cache_gather_args* x) {
    if (!x) return bad("null argument");
    lwm::GatherArgs a{};
    LWM_TRY(check_cache(cache, batch, &a.c));
    LWM_TRY(check_run_blocks(a.c));
    const bool work = a.c.sequences && a.c.max_new;
    if (work) {
        LWM_TRY(check_heads("k_out", x->k_out, x->k_token_stride, x->k_head_stride));
        LWM_TRY(check_heads("v_out", x->v_out, x->v_token_stride, x->v_head_stride));
    }
    CtxView c;
    if (!lwm::ctx_view(ctx, &c)) return bad("null context");
    if (!work) return LWM_OK;
    a.c.err = c.cache_err;
    a.k_out = x->k_out;
    a.v_out = x->v_out;
    a.k_ts = x->k_token_stride;
    a.k_hs = x->k_head_stride;
    a.v_ts = x->v_token_stride;
    a.v_hs = x->v_head_stride;
    return on_device(ctx, c, "cache gather",
                     [&](cudaStream_t s) { return lwm::launch_cache_gather(a, cache->dtype, cache->storage, s); });
}

lwm_status lwm_cache_attention_device(lwm_ctx* ctx, const lwm_paged_cache* cache, const lwm_cache_batch* batch,
                                      const lwm_cache_attention_args* x) {
    if (!x) return bad("null argument");
    lwm::CacheAttnArgs a{};
    LWM_TRY(check_cache(cache, batch, &a.c));
    if (x->heads == 0 || x->heads % cache->kv_heads || x->heads > 65535)
        return bad("query heads " + std::to_string(x->heads) + " must be a positive multiple of kv_heads " +
                   std::to_string(cache->kv_heads));
    if (!std::isfinite(x->scale)) return bad("attention scale must be finite");
    if (x->frame_tokens > (1u << 30)) return bad("frame_tokens out of range");
    a.heads = x->heads;
    a.group = x->heads / cache->kv_heads;
    if (static_cast<uint64_t>(a.c.max_new) * a.group > 0x7fffffffull)
        return fail(LWM_UNSUPPORTED, "batch is too large for one call");
    const uint64_t jobs = static_cast<uint64_t>(a.c.sequences) * cache->kv_heads *
                          ((static_cast<uint64_t>(a.c.max_new) * a.group + 15) / 16);
    if (jobs > (0x7fffffffull >> 4)) return fail(LWM_UNSUPPORTED, "batch is too large for one call");
    const bool work = a.c.sequences && a.c.max_new;
    if (work) {
        LWM_TRY(check_heads("q", x->q, x->q_token_stride, x->q_head_stride));
        LWM_TRY(check_heads("out", x->out, x->out_token_stride, x->out_head_stride));
    }
    CtxView c;
    if (!lwm::ctx_view(ctx, &c)) return bad("null context");
    if (!work) return LWM_OK;
    a.c.err = c.cache_err;
    a.q = x->q;
    a.out = x->out;
    a.q_ts = x->q_token_stride;
    a.q_hs = x->q_head_stride;
    a.o_ts = x->out_token_stride;
    a.o_hs = x->out_head_stride;
    a.scale_log2 = x->scale * 1.4426950408889634f;
    a.causal = x->causal != 0;
    a.window = x->window;
    a.sinks = x->sinks;
    a.frame = x->frame_tokens ? x->frame_tokens : 1;
    a.group_div = lwm::FastDiv(a.group);
    a.frame_div = lwm::FastDiv(a.frame);
    return on_device(ctx, c, "cache attention",
                     [&](cudaStream_t s) {
                         return lwm::cache_attention_many_rows(a)
                                    ? lwm::launch_cache_attention_tc(a, cache->dtype, cache->storage, s)
                                    : lwm::launch_cache_attention(a, cache->dtype, cache->storage, s);
                     });
}

lwm_status lwm_gated_norm_device(lwm_ctx* ctx, const lwm_gated_norm_args* x) {
    if (!x) return bad("null argument");
    const auto dtype_ok = [](int32_t d) { return d >= LWM_DTYPE_F32 && d <= LWM_DTYPE_F16; };
    if (!dtype_ok(x->residual_dtype) || !dtype_ok(x->dtype)) return bad("unknown dtype");
    const bool cond = x->gate || x->shift || x->scale;
    if (cond && !dtype_ok(x->cond_dtype)) return bad("unknown conditioning dtype");
    if (x->width == 0 || x->width > 8192)
        return fail(LWM_UNSUPPORTED, "gated norm width " + std::to_string(x->width) + " must be 1 to 8192");
    if (x->rows > 0x7fffffffu) return bad("gated norm rows out of range");
    const auto kind_ok = [](int32_t k) { return k == LWM_NORM_LAYER || k == LWM_NORM_RMS || k == LWM_NORM_NONE; };
    if (!kind_ok(x->post_kind) || !kind_ok(x->pre_kind)) return bad("gated norm kinds are layer, rms or none");
    const auto eps_ok = [](float e) { return std::isfinite(e) && e >= 0.0f; };
    if ((x->post_kind != LWM_NORM_NONE && !eps_ok(x->post_eps)) || (x->pre_kind != LWM_NORM_NONE && !eps_ok(x->pre_eps)) ||
        (x->out_weight && !eps_ok(x->out_eps)))
        return bad("gated norm eps must be finite and non-negative");
    if (x->out_bias && !x->out_weight) return bad("out_bias needs out_weight");
    if (cond && x->rows_per_cond == 0) return bad("rows_per_cond must be greater than zero");
    if (x->rows && !x->x_out && !x->h) return bad("gated norm has no output");
    if (x->rows && !x->x) return bad("x is null");
    const auto size = [](int32_t d) { return d == LWM_DTYPE_F32 ? 4u : 2u; };
    const auto natural = [](const void* p, unsigned e) { return reinterpret_cast<uintptr_t>(p) % e == 0; };
    if (!natural(x->x, size(x->residual_dtype)) || !natural(x->x_out, size(x->residual_dtype)) ||
        !natural(x->y, size(x->dtype)) || !natural(x->h, size(x->dtype)) ||
        (cond && (!natural(x->gate, size(x->cond_dtype)) || !natural(x->shift, size(x->cond_dtype)) ||
                  !natural(x->scale, size(x->cond_dtype)))))
        return bad("gated norm tensors must be aligned to their element size");
    for (const float* p : {x->residual_scale, x->post_weight, x->post_bias, x->pre_weight, x->pre_bias, x->out_weight,
                           x->out_bias})
        if (!aligned4(p)) return bad("gated norm weights must be aligned to 4 bytes");
    CtxView c;
    if (!lwm::ctx_view(ctx, &c)) return bad("null context");
    if (x->rows == 0) return LWM_OK;
    lwm::GatedNormArgs a{};
    a.a = *x;
    a.out_norm = x->out_weight != nullptr;
    a.cond_div = lwm::FastDiv(cond ? std::min(x->rows_per_cond, x->rows) : 1);  // (more rows than there are: one for all)
    return on_device(ctx, c, "gated norm", [&](cudaStream_t s) { return lwm::launch_gated_norm(a, s); });
}

}  // extern "C"
