// kernels_linear_attn_tc.cu — linear attention with decay over whole histories
// of bf16 on the tcgen05 tensor cores (lwm_linear_attention_device).
//
// A block takes a sequence and head (or, of few long ones, a part along time,
// the parts of a sequence in a cluster) in chunks of 128 tokens:
//   P  = Q K^T                     (TMEM), times lambda^(i-j) where j <= i, to bf16 in place
//   O1 = Q S, O2 = P V             (TMEM), out = scale (lambda^(i+1) O1 + O2)
//   S  = lambda^m S + K'^T V       (TMEM, 32 bits; a bf16 copy in shared memory for O1)
// with K' = lambda^(m-1-j) k_j in three parts of 8 bits, so that S keeps them
// as 32-bit products would.
//
// Warpgroups: outputs (a token a thread: P, O1, O2), two for the state (a key
// channel a thread, half of the value channels: K' 64 tokens at a time, the
// first part in place of K once P is done, S between its two uses), and one
// that loads (cp.async: rows behind the sequence's end are zeros).  K and V
// have two stages, Q is loaded again as soon as both its products are done.
// All tiles are rows of 64 channels (128 bytes, 128-byte swizzle); K' is an
// M-major A operand, V and S N-major B operands of that layout.  64 channels
// have a second half of K' that is zero, as an A operand of 128 rows wants.
//
// Infinities and NaN among the values are taken out of the tiles and added
// where they belong, one by one.  Every wait is bounded: one that gives up
// marks the block, which unwinds.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "lwm_linear_attn.cuh"
#include "lwm_tc.cuh"

namespace lwm {

namespace {

namespace cg = cooperative_groups;

constexpr int kChunk = 128, kHalf = 64;
constexpr int kThreads = 512, kOut = 128, kState = 256, kLoad = 128;
constexpr uint32_t kMostParts = 16;
constexpr uint32_t kPCol = 0, kO1Col = 128;

template <int D> struct Shape {
    static constexpr int kPanels = D / 64;
    static constexpr int kTile = kPanels * kChunk * 128;    // bytes of 128 tokens
    static constexpr int kPart = kPanels * kHalf * 128;     // of 64
    static constexpr int kS = D * D * 2;
    static constexpr int kQ = 0, kK = kTile, kV = kK + 2 * kTile, kMid = kV + 2 * kTile, kLow = kMid + kPart, kSAt = kLow + kPart;
    static constexpr int kZero = kSAt + kS;                 // 64 channels: the empty half of K'
    static constexpr int kBytes = kZero + (D == 64 ? kHalf * 128 : 0) + 1024;  // + alignment
    static constexpr uint32_t kO2Col = kO1Col + D, kSCol = kO2Col + D;
};

struct Control {
    uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], scores[2], between, pv, s_full, kv, drain;
    uint32_t tmem;
    int dead;     // a wait gave up
    int bad[4];   // infinities or NaN were taken out of a V tile (four, as a flag is read after the tile may be free)
    float power[kChunk + 1];  // lambda^i
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Control* c, int site, uint64_t* err, uint32_t seq) {
    bool done = tc::mbar_try(bar, parity);
    for (uint32_t i = 0; i < tc::kWaitLimit && !done; ++i) {
        done = tc::mbar_try(bar, parity);
        if ((i & 255u) == 255u && *static_cast<volatile int*>(&c->dead)) break;
    }
    if (__all_sync(0xffffffffu, done)) return true;
    if (atomicExch(&c->dead, 1) == 0) cache_report(err, kStateErrWait, seq, site);
    return false;
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// Whether any thread of a group says so: a group goes on, or gives up, as one, so that none waits for another there.
__device__ __forceinline__ bool named_any(int id, int threads, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(x)), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}

// kind::f16 of bf16 with f32 accumulation, M 128: operands K-major, or transposed (bits 15 and 16).
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool a_turned, bool b_turned) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_turned ? 1u : 0u) << 15) | ((b_turned ? 1u : 0u) << 16) | ((n >> 3) << 17) |
           ((128u >> 4) << 24);
}
// Descriptor of a tile: start, distance of its panels of 64 channels.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t panel) { return tc::smem_desc(addr, panel, 1024, tc::kSwizzle128); }

// Offset of 16-byte chunk c of row r of a tile whose panels have `rows` rows.
__device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c, uint32_t rows) {
    return (c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) linear_tc_kernel(const __grid_constant__ LinearArgs a, uint32_t parts) {
    using S = Shape<D>;
    constexpr int kSteps = D / 16, kRowChunks = D / 8;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Control ctl_s;
    Control* const ctl = &ctl_s;
    uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t base = tc::smem_u32(smem);
    const int warp = threadIdx.x >> 5;
    const uint32_t rank = blockIdx.x % parts, job = blockIdx.x / parts;
    const uint32_t s = a.head_div.div(job), h = job - s * a.heads;
    const StateView v = state_view(a, s, h == 0 && rank == 0 && threadIdx.x == 0);
    if (!v.ok) return;  // (the same in a whole cluster)
    const uint32_t hk = a.group_div.div(h);
    float decay = a.log_decay[h];
    if (decay < -200.0f) decay = -200.0f;  // (e^-200 is zero; minus infinity times zero would be NaN)
    const uint32_t chunks = (v.n + kChunk - 1) / kChunk, per = (chunks + parts - 1) / parts;
    const uint32_t first = min(rank * per, chunks), end = min(first + per, chunks);

    if (threadIdx.x == 0) {
        tc::mbar_init(&ctl->q_full, kLoad);
        tc::mbar_init(&ctl->q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&ctl->k_full[i], kLoad);
            tc::mbar_init(&ctl->v_full[i], kLoad);
            tc::mbar_init(&ctl->k_empty[i], 1);
            tc::mbar_init(&ctl->v_empty[i], 2);
            tc::mbar_init(&ctl->scores[i], 1);
        }
        tc::mbar_init(&ctl->between, 1);
        tc::mbar_init(&ctl->s_full, kState);
        tc::mbar_init(&ctl->kv, 1);
        tc::mbar_init(&ctl->pv, 1);
        tc::mbar_init(&ctl->drain, 2);
        ctl->dead = 0;
        tc::mbar_fence_init();
    }
    for (int i = threadIdx.x; i <= kChunk; i += kThreads) ctl->power[i] = expf(decay * i);
    if constexpr (D == 64)
        for (int i = threadIdx.x; i < kHalf * 8; i += kThreads) *reinterpret_cast<uint4*>(smem + S::kZero + i * 16) = make_uint4(0, 0, 0, 0);
    tc::fence_async_smem();
    if (warp == 0) tc::tmem_alloc(&ctl->tmem, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = ctl->tmem;
    uint64_t* const err = a.err;
    const auto* const q_at = static_cast<const bf16*>(a.q) + h * a.q_hs;
    const auto* const k_at = static_cast<const bf16*>(a.k) + hk * a.k_hs;
    const auto* const v_at = static_cast<const bf16*>(a.v) + hk * a.v_hs;
    auto tokens_of = [&](uint32_t i) { return min(static_cast<uint32_t>(kChunk), v.n - i * kChunk); };
    auto row_at = [&](uint32_t i) { return static_cast<size_t>(v.start) + i * kChunk; };

    // ------------------------------------------------------------ loads
    // One tile of the chunk's rows into `to`; the caller commits.
    auto load = [&](const bf16* src, size_t stride, uint32_t i, uint32_t to) {
        const int t = threadIdx.x - kOut - kState;
        const uint32_t m = tokens_of(i);
#pragma unroll 4
        for (int c = 0; c < kChunk * kRowChunks / kLoad; ++c) {
            const uint32_t x = c * kLoad + t, r = x / kRowChunks, ch = x % kRowChunks;
            const bool live = r < m;
            cp_async16(to + chunk_at(r, ch, kChunk), src + (row_at(i) + (live ? r : 0)) * stride + 8 * ch, live);
        }
    };
    auto loads = [&](bool whole, uint32_t from, uint32_t& use) {
        // use: chunks that the rings have seen before
        bool fine = true;
        const int t = threadIdx.x - kOut - kState;
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t st = use & 1, round = use >> 1;
            if (use >= 2) fine = wait(&ctl->k_empty[st], (round - 1) & 1, ctl, 1, err, s);
            if (fine) load(k_at, a.k_ts, i, base + S::kK + st * S::kTile);
            cp_commit();
            if (fine && use >= 2) fine = wait(&ctl->v_empty[st], (round - 1) & 1, ctl, 2, err, s);
            if (fine) load(v_at, a.v_ts, i, base + S::kV + st * S::kTile);
            cp_commit();
            if (fine && whole && i > from) fine = wait(&ctl->q_empty, (i - from - 1) & 1, ctl, 3, err, s);
            if (fine && whole) load(q_at, a.q_ts, i, base + S::kQ);
            cp_commit();
            cp_wait<2>();
            tc::fence_async_smem();
            if (fine) tc::mbar_arrive(&ctl->k_full[st]);
            cp_wait<1>();
            if (t == 0) ctl->bad[use & 3] = 0;
            named_sync(3, kLoad);
            if (fine) {
#pragma unroll 4
                for (int c = 0; c < kChunk * kRowChunks / kLoad; ++c) {
                    const uint32_t x = c * kLoad + t;
                    uint4* at = reinterpret_cast<uint4*>(smem + S::kV + st * S::kTile + chunk_at(x / kRowChunks, x % kRowChunks, kChunk));
                    uint4 y = *at;
                    if (not_finite2<bf16>(y.x) | not_finite2<bf16>(y.y) | not_finite2<bf16>(y.z) | not_finite2<bf16>(y.w)) {
                        ctl->bad[use & 3] = 1;
                        *at = make_uint4(finite2<bf16>(y.x), finite2<bf16>(y.y), finite2<bf16>(y.z), finite2<bf16>(y.w));
                    }
                }
                tc::fence_async_smem();
                tc::mbar_arrive(&ctl->v_full[st]);
            }
            cp_wait<0>();
            tc::fence_async_smem();
            if (fine && whole) tc::mbar_arrive(&ctl->q_full);
            fine = !named_any(3, kLoad, !fine);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    };

    // ------------------------------------------------------------ state
    const int t_state = threadIdx.x - kOut, wg = t_state >> 7, row = t_state & 127;  // key channel, half of the value channels
    const int col0 = wg * (D / 2);
    const bool has_row = row < D;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    // the bf16 copy of this thread's part of the state
    auto copy16 = [&](int c, const float(&x)[16]) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = x[8 * b + e];
            *reinterpret_cast<uint4*>(smem + S::kSAt + chunk_at(row, (col0 + c) / 8 + b, D)) = pack<bf16>(f).a;
        }
    };
    // The state's steps over the chunks from `from` on (TMEM holds it, times the first chunk's decay).  whole: beside
    // the outputs, else alone.
    auto states = [&](bool whole, uint32_t from, uint32_t& use, uint32_t& kv_use, float* final_state) {
        bool fine = true;
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t st = use & 1, round = use >> 1, m = tokens_of(i);
            uint8_t* const kt = smem + S::kK + st * S::kTile;
            const uint32_t v_a = base + S::kV + st * S::kTile;
            fine = wait(&ctl->k_full[st], round & 1, ctl, 10, err, s);
            if (fine && whole) fine = wait(&ctl->scores[(i - from) & 1], ((i - from) >> 1) & 1, ctl, 11, err, s);  // K is read: its place may change
            if (fine) fine = wait(&ctl->v_full[st], round & 1, ctl, 12, err, s);
            const uint32_t halves = m > kHalf ? 2 : 1;
            for (uint32_t half = 0; half < halves; ++half) {
                if (fine) {
#pragma unroll
                for (int c = 0; c < kHalf * kRowChunks / kState; ++c) {
                    const uint32_t x = c * kState + t_state, r = x / kRowChunks, ch = x % kRowChunks;
                    const uint32_t tok = half * kHalf + r;
                    const float w = tok < m ? ctl->power[m - 1 - tok] : 0.0f;
                    uint4* const at = reinterpret_cast<uint4*>(kt + chunk_at(tok, ch, kChunk));
                    float f[8], g[8];
                    unpack(Vec8<bf16>{*at}, f);
                    Vec8<bf16> part[3];
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= w;
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        part[p] = pack<bf16>(f);
                        unpack(part[p], g);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] -= g[e];
                    }
                    *at = part[0].a;
                    *reinterpret_cast<uint4*>(smem + S::kMid + chunk_at(r, ch, kHalf)) = part[1].a;
                    *reinterpret_cast<uint4*>(smem + S::kLow + chunk_at(r, ch, kHalf)) = part[2].a;
                }
                }
                tc::fence_async_smem();
                tc::fence_before();  // (the state's stores, too)
                fine = !named_any(2, kState, !fine);
                if (warp == 4 && fine) {
                    tc::fence_after();
                    constexpr uint32_t kI = idesc(D, true, true);
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const uint32_t from_a = p == 0 ? base + S::kK + st * S::kTile + half * kHalf * 128 : base + (p == 1 ? S::kMid : S::kLow);
                        const uint32_t panel = D == 64 ? base + S::kZero - from_a : (p == 0 ? kChunk : kHalf) * 128;
#pragma unroll
                        for (int k = 0; k < kHalf / 16; ++k)
                            tc::mma_bf16_w(tmem + S::kSCol, tile_desc(from_a + k * 2048, panel),
                                           tile_desc(v_a + half * kHalf * 128 + k * 2048, kChunk * 128), kI, 1);
                    }
                    tc::commit_w(&ctl->kv);
                    if (half + 1 == halves) {
                        tc::commit_w(&ctl->k_empty[st]);
                        tc::commit_w(&ctl->v_empty[st]);
                        if (!whole) tc::commit_w(&ctl->v_empty[st]);
                    }
                    __syncwarp();
                }
                if (fine) fine = wait(&ctl->kv, kv_use & 1, ctl, 13, err, s);
                ++kv_use;
            }
            tc::fence_after();
            // its bf16 copy's last reader is the product of this chunk
            if (fine && whole) fine = wait(&ctl->between, (i - from) & 1, ctl, 14, err, s);
            const bool more = i + 1 < end;
            const float fade = more ? expm1f(decay * tokens_of(i + 1)) : 0.0f;
            const bool bad = *static_cast<volatile int*>(&ctl->bad[use & 3]) != 0;
            if (has_row && fine) {
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 16) {
                    float x[16];
                    tc::tmem_ld16(t_lane + S::kSCol + col0 + c, x);
                    tc::tmem_ld_wait();
                    if (bad)
                        for (uint32_t j = 0; j < m; ++j)
                            for (int e = 0; e < 16; ++e) {
                                const float y = static_cast<float>(v_at[(row_at(i) + j) * a.v_ts + col0 + c + e]);
                                if (!isfinite(y)) x[e] += static_cast<float>(k_at[(row_at(i) + j) * a.k_ts + row]) * ctl->power[m - 1 - j] * y;
                            }
                    if (whole && more) copy16(c, x);
                    if (final_state && !more) {
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<float4*>(final_state + static_cast<size_t>(row) * D + col0 + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                    }
                    if (more || !whole) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = fmaf(x[e], fade, x[e]);
                        tc::tmem_st16(t_lane + S::kSCol + col0 + c, x);
                    }
                }
                tc::tmem_st_wait();
            }
            tc::fence_before();
            tc::fence_async_smem();
            if (whole && more && fine) tc::mbar_arrive(&ctl->s_full);
            fine = !named_any(2, kState, !fine);
        }
    };

    // ---------------------------------------------------------- outputs
    auto outputs = [&](uint32_t from, uint32_t use) {
        const uint32_t r = threadIdx.x;  // token of the chunk
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        bool fine = true;
        const uint32_t q_a = base + S::kQ, s_a = base + S::kSAt;
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t st = use & 1, round = use >> 1, m = tokens_of(i), turn = (i - from) & 1;
            const uint32_t k_a = base + S::kK + st * S::kTile, v_a = base + S::kV + st * S::kTile;
            if (warp == 0) {
                fine = wait(&ctl->q_full, turn, ctl, 20, err, s) && wait(&ctl->k_full[st], round & 1, ctl, 21, err, s);
                if (fine) {
                    tc::fence_after();
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        const uint32_t off = (k >> 2) * kChunk * 128 + (k & 3) * 32;
                        tc::mma_bf16_w(tmem + kPCol, tile_desc(q_a + off, 16), tile_desc(k_a + off, 16), idesc(kChunk, false, false), k > 0);
                    }
                    tc::commit_w(&ctl->scores[turn]);
                    fine = wait(&ctl->s_full, turn, ctl, 22, err, s);
                }
                if (fine) {
                    tc::fence_after();
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        const uint32_t off = (k >> 2) * kChunk * 128 + (k & 3) * 32;
                        tc::mma_bf16_w(tmem + kO1Col, tile_desc(q_a + off, 16), tile_desc(s_a + k * 2048, D * 128), idesc(D, false, true), k > 0);
                    }
                    tc::commit_w(&ctl->between);
                    tc::commit_w(&ctl->q_empty);
                }
            }
            if (fine) fine = wait(&ctl->scores[turn], ((i - from) >> 1) & 1, ctl, 23, err, s);
            tc::fence_after();
            // weights: what a token does not see is zero
#pragma unroll 1
            for (int c = 0; c < kChunk; c += 16) {
                uint32_t p[8];
                if (c > warp * 32 + 31) {  // none of the warp's tokens
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = 0u;
                    tc::tmem_st8u(lanes + kPCol + c / 2, p);
                    continue;
                }
                float x[16];
                tc::tmem_ld16(lanes + kPCol + c, x);
                tc::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int apart = static_cast<int>(r) - (c + e);
                    const float w = ctl->power[max(apart, 0)];
                    x[e] = apart >= 0 ? x[e] * w : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = pack2(x[2 * e], x[2 * e + 1], bf16{});
                tc::tmem_st8u(lanes + kPCol + c / 2, p);
            }
            tc::tmem_st_wait();
            tc::fence_before();
            fine = !named_any(1, kOut, !fine);
            if (warp == 0 && fine) {
                fine = wait(&ctl->v_full[st], round & 1, ctl, 24, err, s);
                if (fine) {
                    tc::fence_after();
#pragma unroll
                    for (int k = 0; k < kChunk / 16; ++k)
                        tc::mma_bf16_ta_w(tmem + S::kO2Col, tmem + kPCol + 8 * k, tile_desc(v_a + k * 2048, kChunk * 128),
                                          idesc(D, false, true), k > 0);
                    tc::commit_w(&ctl->v_empty[st]);
                    tc::commit_w(&ctl->pv);
                }
            }
            if (fine) fine = wait(&ctl->between, turn, ctl, 25, err, s) && wait(&ctl->pv, turn, ctl, 26, err, s);
            tc::fence_after();
            const bool live = fine && r < m, bad = *static_cast<volatile int*>(&ctl->bad[use & 3]) != 0;
            const float grow = ctl->power[r + 1] * a.scale;
            bf16* const to = static_cast<bf16*>(a.out) + (row_at(i) + r) * a.o_ts + h * a.o_hs;
            if (bad) {
                // the values that were left out, for the tokens that see them (before any output, which may be where q is)
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    float y[16];
                    tc::tmem_ld16(lanes + S::kO2Col + c, y);
                    tc::tmem_ld_wait();
                    for (uint32_t j = 0; live && j <= r; ++j) {
                        float dot = 0.0f;
                        bool any = false;
                        for (int e = 0; e < 16; ++e) {
                            const float z = static_cast<float>(v_at[(row_at(i) + j) * a.v_ts + c + e]);
                            if (isfinite(z)) continue;
                            if (!any)
                                for (int ch = 0; ch < D; ++ch)
                                    dot = fmaf(static_cast<float>(q_at[(row_at(i) + r) * a.q_ts + ch]), static_cast<float>(k_at[(row_at(i) + j) * a.k_ts + ch]), dot);
                            any = true;
                            y[e] += dot * ctl->power[r - j] * z;
                        }
                    }
                    __syncwarp();
                    tc::tmem_st16(lanes + S::kO2Col + c, y);
                    tc::tmem_st_wait();
                }
            }
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                float x[16], y[16];
                tc::tmem_ld16(lanes + kO1Col + c, x);
                tc::tmem_ld16(lanes + S::kO2Col + c, y);
                tc::tmem_ld_wait();
                if (live) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = fmaf(x[8 * b + e], grow, y[8 * b + e] * a.scale);
                        store8(to + c + 8 * b, pack<bf16>(f));
                    }
                }
            }
            tc::fence_before();
            fine = !named_any(1, kOut, !fine);
        }
    };

    // A state into TMEM, times the decay of the first chunk, and its bf16 copy.
    const float fade0 = first < end ? expm1f(decay * tokens_of(first)) : 0.0f;
    auto begin = [&](int c, float(&x)[16], bool copy) {
        if (copy) copy16(c, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = fmaf(x[e], fade0, x[e]);
        tc::tmem_st16(t_lane + S::kSCol + col0 + c, x);
    };
    const bool is_state = warp >= 4 && warp < 12;
    const size_t size = static_cast<size_t>(D) * D;
    const float* const before = a.states + (static_cast<size_t>(v.source < 0 ? 0 : v.source) * a.heads + h) * size;
    // the block with the last tokens has the state after them (where there are none, the first)
    const bool last = end == chunks && (first < end || (chunks == 0 && rank == 0));
    float* const after = last && v.target >= 0 ? a.states + (static_cast<size_t>(v.target) * a.heads + h) * size : nullptr;
    uint32_t use = 0, kv_use = 0;
    float* const shared = reinterpret_cast<float*>(smem);
    if (parts > 1) {
        // What each block's tokens add to a state, then the states before them: element by element, each block a
        // share of the elements for all of them, over distributed shared memory.
        const bool walks = rank + 1 < parts && first < end;
        if (walks) {
            if (is_state) {
                float x[16];
                for (int c = 0; has_row && c < D / 2; c += 16) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = 0.0f;
                    begin(c, x, false);
                }
                tc::tmem_st_wait();
                states(false, first, use, kv_use, nullptr);
            } else if (warp >= 12) {
                loads(false, first, use);
            }
            use = end - first;  // (for the warps that did neither)
        }
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
        if (is_state && has_row) {
            for (int c = 0; c < D / 2; c += 16) {
                float x[16];
                if (walks) {
                    tc::tmem_ld16(t_lane + S::kSCol + col0 + c, x);
                    tc::tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) shared[(col0 + c + e) * D + row] = walks ? x[e] : 0.0f;
            }
        }
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const uint32_t share = D * D / parts + 1;
        for (uint32_t x = threadIdx.x; x < share; x += kThreads) {
            const uint32_t at = rank * share + x;
            if (at >= D * D) break;
            float y = v.source < 0 ? 0.0f : before[(at % D) * D + at / D];
            float added[kMostParts];
#pragma unroll
            for (uint32_t b = 0; b < kMostParts; ++b) added[b] = b + 1 < parts ? cluster.map_shared_rank(shared, b)[at] : 0.0f;
#pragma unroll
            for (uint32_t b = 0; b < kMostParts; ++b) {
                if (b >= parts) break;
                cluster.map_shared_rank(shared, b)[at] = y;
                const uint32_t done = min(b * per * kChunk, v.n), tokens = min(v.n - done, per * kChunk);
                y = fmaf(y, expm1f(decay * tokens), y) + added[b];
            }
        }
        cluster.sync();
    }
    if (is_state && has_row) {
        for (int c = 0; c < D / 2; c += 16) {
            float x[16];
            if (parts > 1) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = shared[(col0 + c + e) * D + row];
            } else if (v.source >= 0) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(before + static_cast<size_t>(row) * D + col0 + c + e);
                    x[e] = y.x, x[e + 1] = y.y, x[e + 2] = y.z, x[e + 3] = y.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = 0.0f;
            }
            if (after && first == end) {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(after + static_cast<size_t>(row) * D + col0 + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            }
            begin(c, x, true);
        }
        tc::tmem_st_wait();
    }
    tc::fence_before();
    tc::fence_async_smem();
    __syncthreads();  // (the tiles go where the states were)
    tc::fence_after();
    if (is_state) {
        if (first < end) tc::mbar_arrive(&ctl->s_full);
        states(true, first, use, kv_use, after);
    } else if (warp < 4) {
        outputs(first, use);
    } else {
        loads(true, first, use);
    }
    // every product has read its operands before the block ends
    if (warp == 0 || warp == 4) {
        tc::commit_w(&ctl->drain);
        tc::mbar_wait_landing(&ctl->drain, 0);
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 0) tc::tmem_free(tmem, 512);
}

// Blocks that a sequence and head are cut into along time: as many as run at once (clusters of blocks that fill an SM
// each: a GPU of 148 has room for fewer than 148 / parts), with two chunks each at least.
uint32_t parts_of(const LinearArgs& a) {
    constexpr uint32_t kRoom[] = {0, 148, 74, 44, 33, 25, 22, 16, 15, 8, 8, 8, 8, 8, 8, 7, 7};
    const uint64_t jobs = static_cast<uint64_t>(a.sequences) * a.heads;
    const uint32_t chunks = (a.max_new + kChunk - 1) / kChunk;
    uint32_t best = 1;
    double least = 1e30;
    for (uint32_t parts = 1; parts <= kMostParts && parts * 2 <= std::max(chunks, 2u); ++parts) {
        const double cost = std::ceil(static_cast<double>(jobs) / kRoom[parts]) * ((chunks + parts - 1) / parts * (parts > 1 ? 1.6 : 1.0) + (parts > 1 ? 4.0 : 2.0));
        if (cost < least) least = cost, best = parts;
    }
    return best;
}

template <int D> cudaError_t launch(const LinearArgs& a, cudaStream_t s) {
    using S = Shape<D>;
    static_assert(S::kBytes + sizeof(Control) <= 227 * 1024, "shared memory");
    auto* kernel = linear_tc_kernel<D>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    uint32_t parts = parts_of(a);
    if (getenv("LWM_PARTS")) parts = atoi(getenv("LWM_PARTS"));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.sequences * a.heads * parts);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, parts);
}

}  // namespace

bool linear_attention_tensor(const LinearArgs& a, int dtype) {
    return dtype == LWM_DTYPE_BF16 && a.head_dim >= 64 && a.max_new > 64;
}

cudaError_t launch_linear_attention_tc(const LinearArgs& a, cudaStream_t s) {
    return a.head_dim == 64 ? launch<64>(a, s) : launch<128>(a, s);
}

}  // namespace lwm
