// kernels_linear_attn.cu — linear attention with a decay for each head
// (lwm_linear_attention_device):
//   S_t = lambda S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,
// S one f32 [head_dim, head_dim] state a head.
//
// A few tokens a sequence (linear_step_kernel): the state is read once, kept
// in registers over the tokens, and written once.  Where every sequence has a
// state of its own that is bound by those bytes: 1024 sequences of 16 heads of
// 64, a token each, 537 MB in 84.2 us, 6.4 TB/s.  256 that fork from one state,
// 16 heads of 128, write 268 MB in 61 us, which a plain fill would do in 38:
// there each block's way from its state (in the L2) over the sums to its stores
// is the bound, one after the other, with two blocks of 8 warps an SM for their
// 107 registers (DRAM 41 %, L2 45 %).  Up to 8 tokens: 8 of those 1024 take 186
// us, in chunks 283, and each token more 17, the latency of its loads.
//
// Whole histories (linear_chunk_kernel): chunks of 64 tokens,
//   O = lambda^(i+1) Q S + (Q K^T . lambda^(i-j), j <= i) V,
//   S' = lambda^m S + sum_j lambda^(m-1-j) k_j v_j^T   (m tokens),
// all four products on mma.sync with the state in registers: half of the warps
// keep it, the others compute the outputs of the chunk before.  For f16 (whose
// states and weights need powers of two a row, and tf32 for Q S), 32 channels,
// short sequences, strides that a tensor map does not take, and an out that may
// lie on keys or values; long ones of bf16 with 64 or 128 channels go on
// tcgen05.  Bound by the products' issue and the fragments' way to them: 16
// sequences of 1568 tokens, 16 heads, f16, of 32 channels 62 us, of 64 109, of
// 128 (one block a SM) 359; one of 65536 tokens 367, 609, 2669.
//
// What is rounded to 16 bits: a row's weights, as operands of their product
// with v (a rounding costs them half a step each, of either sign, as that of
// the output does), and the state's copy for the product with q (f16: 11 bits
// by tf32).  The state itself and what enters it keep 22 bits and more.
#include <cooperative_groups.h>

#include <algorithm>

#include "lwm_blocks.cuh"
#include "lwm_linear_attn.cuh"

namespace lwm {

namespace {

namespace cg = cooperative_groups;

// -------------------------------------------------------------- few tokens

// A block takes (sequence, head): thread (r, c) keeps rows r, r + kRowGroups,
// ... of the state at value channels 4 c .. 4 c + 3.
template <int D> struct StepShape {
    static constexpr int kCols = D / 4, kThreads = D == 128 ? 256 : D == 64 ? 128 : 64;
    static constexpr int kRowGroups = kThreads / kCols, kRows = D / kRowGroups;
};

template <int D> struct alignas(16) Channels {  // of a token, read four at a time
    float x[D];
};

template <typename T, int D>
__global__ void __launch_bounds__(StepShape<D>::kThreads) linear_step_kernel(const __grid_constant__ LinearArgs a) {
    using S = StepShape<D>;
    __shared__ Channels<D> q_s, k_s, v_s;
    static_assert(alignof(decltype(v_s)) == sizeof(float4), "read as float4");
    __shared__ float4 part[S::kRowGroups][S::kCols];
    const uint32_t s = a.head_div.div(blockIdx.x), h = blockIdx.x - s * a.heads;
    const StateView v = state_view(a, s, h == 0 && threadIdx.x == 0);
    if (!v.ok) return;
    const int c = threadIdx.x % S::kCols, r = threadIdx.x / S::kCols;
    float4 st[S::kRows];
    const size_t size = static_cast<size_t>(D) * D;
    const float* from = a.states + (static_cast<size_t>(v.source < 0 ? 0 : v.source) * a.heads + h) * size + 4 * c;
#pragma unroll
    for (int i = 0; i < S::kRows; ++i)
        st[i] = v.source < 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                             : *reinterpret_cast<const float4*>(from + (r + i * S::kRowGroups) * D);
    // As the chunks do it: with lambda rounded to 32 bits a head that forgets 1 / 4096 a token would be off by 1e-4 of
    // that.  (What a token fades by less than 2^-25 of the state is lost in the state's own rounding.)
    const Fade fade = fade_of(a.log_decay[h]);
    const uint32_t hk = a.group_div.div(h);
    for (uint32_t i = 0; i < v.n; ++i) {
        const size_t tok = v.start + i;
        for (int e = threadIdx.x; e < 3 * D; e += S::kThreads) {
            const int w = e / D, ch = e % D;
            const T* src = w == 0 ? static_cast<const T*>(a.q) + tok * a.q_ts + h * a.q_hs
                           : w == 1 ? static_cast<const T*>(a.k) + tok * a.k_ts + hk * a.k_hs
                                    : static_cast<const T*>(a.v) + tok * a.v_ts + hk * a.v_hs;
            (w == 0 ? q_s : w == 1 ? k_s : v_s).x[ch] = static_cast<float>(src[ch]);
        }
        __syncthreads();
        const float4 x = *reinterpret_cast<const float4*>(v_s.x + 4 * c);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < S::kRows; ++j) {
            const float k = k_s.x[r + j * S::kRowGroups], q = q_s.x[r + j * S::kRowGroups];
            auto next = [&](float& s0, float& s1, float x0, float x1, float& o0, float& o1) {
                const float2 y = faded(fade, make_float2(s0, s1), make_float2(x0, x1), make_float2(k, k));
                const float2 z = fma2(make_float2(q, q), y, make_float2(o0, o1));
                s0 = y.x, s1 = y.y, o0 = z.x, o1 = z.y;
            };
            next(st[j].x, st[j].y, x.x, x.y, o.x, o.y);
            next(st[j].z, st[j].w, x.z, x.w, o.z, o.w);
        }
        part[r][c] = o;
        __syncthreads();
        for (int e = threadIdx.x; e < D; e += S::kThreads) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < S::kRowGroups; ++j) sum += reinterpret_cast<const float*>(part[j])[e];
            static_cast<T*>(a.out)[tok * a.o_ts + h * a.o_hs + e] = static_cast<T>(sum * a.scale);
        }
    }
    if (v.target < 0) return;
    float* to = a.states + (static_cast<size_t>(v.target) * a.heads + h) * size + 4 * c;
#pragma unroll
    for (int i = 0; i < S::kRows; ++i) *reinterpret_cast<float4*>(to + (r + i * S::kRowGroups) * D) = st[i];
}

// --------------------------------------------------------- whole histories

constexpr int kChunk = 64;
constexpr uint32_t kMostParts = 16;  // blocks of a cluster

template <typename T, int D> struct ChunkShape {
    static constexpr bool kHalf = std::is_same_v<T, __half>;
    static constexpr int kOutWarps = D == 128 ? 8 : 4, kStateWarps = D / 16, kWarps = 2 * kOutWarps, kThreads = kWarps * 32;
    static constexpr int kSplit = kOutWarps / 4;     // warps that share 16 tokens, each with its value channels
    static constexpr int kTile = kChunk * D * 2;     // bytes of a chunk of Q, K or V
    static constexpr int kPitch = D + 4;             // floats of a row of an f32 state
    static constexpr int kState = kHalf ? D * kPitch * 4 : D * D * 2;
    static constexpr int kStages = kHalf && D == 128 ? 2 : 3, kStates = kHalf && D == 128 ? 1 : 2;
    static constexpr int kBytes = kStages * 3 * kTile + kStates * kState;
    static constexpr int kBlocks = D == 128 ? 1 : 2;
    static_assert(kStages * 3 * kTile >= D * D * 4, "a state goes where the tiles are");
};

template <typename T, int D>
__global__ void __launch_bounds__(ChunkShape<T, D>::kThreads, ChunkShape<T, D>::kBlocks)
    linear_chunk_kernel(const __grid_constant__ LinearArgs a, uint32_t parts) {
    using S = ChunkShape<T, D>;
    constexpr int kSteps = D / 16, kTiles = D / 8, kCols = kTiles / S::kSplit;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float power[kChunk + 1];  // lambda^i
    __shared__ Fade fades[2 + kMostParts];      // of a whole chunk, of the last one, of each block's tokens
    __shared__ uint32_t bad_chunk[S::kStages];  // the last chunk there whose values are not all finite
    if (threadIdx.x < S::kStages) bad_chunk[threadIdx.x] = 0xffffffffu;
    // (called from either kind of warp)
    auto meet = [] { asm volatile("bar.sync 0;" ::: "memory"); };
    auto meet_cluster = [] { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t rank = blockIdx.x % parts, job = blockIdx.x / parts;
    const uint32_t s = a.head_div.div(job), h = job - s * a.heads;
    const StateView v = state_view(a, s, h == 0 && rank == 0 && threadIdx.x == 0);
    if (!v.ok) return;
    const uint32_t hk = a.group_div.div(h);
    float decay = a.log_decay[h];
    if (decay < -200.0f) decay = -200.0f;  // (e^-200 is zero; minus infinity times zero would be NaN)
    for (int i = threadIdx.x; i <= kChunk; i += S::kThreads) power[i] = expf(decay * i);
    const uint32_t smem_a = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    // this block's chunks of the sequence
    const uint32_t chunks = (v.n + kChunk - 1) / kChunk, per = (chunks + parts - 1) / parts;
    const uint32_t first = min(rank * per, chunks), end = min(first + per, chunks);
    if (threadIdx.x < 2 + parts) {
        const uint32_t b = threadIdx.x - 2, before = min(b * per * kChunk, v.n);
        const uint32_t tokens = threadIdx.x == 0 ? kChunk : threadIdx.x == 1 ? (v.n + kChunk - 1) % kChunk + 1 : min(v.n - before, per * kChunk);
        fades[threadIdx.x] = fade_of(decay * tokens);
    }
    meet();  // (what is set up so far, before any warp uses it, or marks a chunk)
    constexpr int kRowChunks = D / 8, kEach = kChunk * kRowChunks / S::kThreads;
    auto load = [&](uint32_t i, bool with_q) {
        if (i < end) {
            const uint32_t dst = smem_a + (i - first) % S::kStages * 3 * S::kTile;
            const T* src[3] = {static_cast<const T*>(a.q) + h * a.q_hs, static_cast<const T*>(a.k) + hk * a.k_hs,
                               static_cast<const T*>(a.v) + hk * a.v_hs};
            const size_t ts[3] = {a.q_ts, a.k_ts, a.v_ts};
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                if (w == 0 && !with_q) continue;
#pragma unroll
                for (int c = 0; c < kEach; ++c) {
                    const uint32_t x = c * S::kThreads + threadIdx.x, r = x / kRowChunks, ch = x % kRowChunks;
                    const uint32_t tok = i * kChunk + r;
                    const bool live = tok < v.n;
                    cp_async16(dst + w * S::kTile + tile_at<D>(r, ch), src[w] + (v.start + (live ? tok : 0)) * ts[w] + 8 * ch, live);
                }
            }
        }
        cp_commit();
    };

    // state (the second half of the warps): rows 16 sw + g (+ 8), channels 8 n + 2 t (+ 1)
    const int sw = warp - S::kOutWarps;
    const bool holds = sw >= 0 && sw < S::kStateWarps;
    float st[kTiles][4];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) st[n][0] = st[n][1] = st[n][2] = st[n][3] = 0.0f;

    // S' = lambda^m S + sum of lambda^(m - 1 - j) k_j v_j^T
    auto update = [&](uint32_t i) {
        const uint32_t k_a = smem_a + (i - first) % S::kStages * 3 * S::kTile + S::kTile, v_a = k_a + S::kTile;
        const uint32_t m = min(static_cast<uint32_t>(kChunk), v.n - i * kChunk);
        const Fade fade = fades[m < kChunk];
        float scale[2] = {1.0f, 1.0f}, back[2] = {1.0f, 1.0f};
        auto weight = [&](int k, int e) {  // of tokens 16 k + 2 t, + 1, + 8, + 9
            const int left = static_cast<int>(m) - 1 - (16 * k + 2 * t + (e & 1) + 8 * (e >> 1));
            return left >= 0 ? power[left] : 0.0f;
        };
        auto keys = [&](int k, uint32_t(&raw)[4]) {
            ldsm4t(raw, k_a + tile_at<D>(16 * k + (lane & 7) + ((lane >> 4) << 3), 2 * sw + ((lane >> 3) & 1)));
        };
        if constexpr (S::kHalf) {
            // f16: the rows of K by powers of two, so that small keys keep their bits
            float top[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t raw[4];
                keys(k, raw);
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 x = half2_at(raw[r + 2 * e]);
                        top[r] = fmaxf(top[r], fmaxf(fabsf(x.x) * weight(k, 2 * e), fabsf(x.y) * weight(k, 2 * e + 1)));
                    }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                const float2 f = row_scale(top[r]);
                scale[r] = f.x, back[r] = f.y;
            }
        }
        // Tensor cores cut off what does not fit a sum, step by step, so a chunk's sums start at zero and are added to
        // the state with rounding (16384 tokens that hardly fade: off by 6e-6 of the state when summed in place, 6e-7 so).
        constexpr int kGroup = D == 64 ? 8 : 4;  // tiles at once, for the registers
#pragma unroll
        for (int n0 = 0; n0 < kTiles; n0 += kGroup) {
            float sum[kGroup][4];
#pragma unroll
            for (int n = 0; n < kGroup; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // keys times their decay in parts (bf16 three of 8 bits, f16 two of 11), so that the state keeps them
                // as a 32-bit product would
                constexpr int kParts = S::kHalf ? 2 : 3;
                uint32_t raw[4], x[kParts][4];
                keys(k, raw);
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // register e: row g + 8 (e & 1), tokens 2 t (+ 1) + 8 (e >> 1)
                    float2 r = pair_at<T>(raw[e]);
                    r.x *= weight(k, 2 * (e >> 1)) * scale[e & 1], r.y *= weight(k, 2 * (e >> 1) + 1) * scale[e & 1];
#pragma unroll
                    for (int q = 0; q < kParts; ++q) {
                        x[q][e] = pack2(r.x, r.y, T{});
                        const float2 y = pair_at<T>(x[q][e]);
                        r.x -= y.x, r.y -= y.y;
                    }
                }
#pragma unroll
                for (int n = 0; n < kGroup; n += 2) {
                    uint32_t b[4];
                    ldsm4t(b, v_a + tile_at<D>(16 * k + (lane & 15), n0 + n + (lane >> 4)));
#pragma unroll
                    for (int q = 0; q < kParts; ++q) {
                        mma<T>(sum[n], x[q], b[0], b[1]);
                        mma<T>(sum[n + 1], x[q], b[2], b[3]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < kGroup; ++n)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float* const y = &st[n0 + n][e];
                    if constexpr (S::kHalf && D == 128) {  // (pairs: 4 % for the registers that hold them)
                        y[0] = faded(fade, y[0], sum[n][e] * back[e >> 1]);
                        y[1] = faded(fade, y[1], sum[n][e + 1] * back[e >> 1]);
                    } else {
                        const float2 x = make_float2(y[0], y[1]), added = make_float2(sum[n][e], sum[n][e + 1]);
                        const float2 z = S::kHalf ? faded(fade, x, added, make_float2(back[e >> 1], back[e >> 1])) : faded(fade, x, added);
                        y[0] = z.x, y[1] = z.y;
                    }
                }
        }
    };
    // the state to shared memory, for the product with Q: bf16, or tf32 for f16 (which has no room for its range)
    auto publish = [&](uint32_t i) {
        uint8_t* const to = smem + S::kStages * 3 * S::kTile + (i - first) % S::kStates * S::kState;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 16 * sw + g + 8 * r;
                if constexpr (S::kHalf)
                    *reinterpret_cast<uint2*>(to + (row * S::kPitch + 8 * n + 2 * t) * 4) =
                        make_uint2(to_tf32(st[n][2 * r]), to_tf32(st[n][2 * r + 1]));
                else
                    *reinterpret_cast<uint32_t*>(to + tile_at<D>(row, n) + 4 * t) = pack2(st[n][2 * r], st[n][2 * r + 1], T{});
            }
    };
    // The outputs of a chunk: this warp's 16 tokens and value channels.
    const int tile = warp / S::kSplit, col0 = (warp % S::kSplit) * kCols;
    auto outputs = [&](uint32_t i, bool bad) {
        const uint8_t* const base = smem + (i - first) % S::kStages * 3 * S::kTile;
        const uint8_t* const state_s = smem + S::kStages * 3 * S::kTile + (i - first) % S::kStates * S::kState;
        const uint32_t q_a = static_cast<uint32_t>(__cvta_generic_to_shared(base)), k_a = q_a + S::kTile, v_a = k_a + S::kTile;
        const uint32_t state_a = static_cast<uint32_t>(__cvta_generic_to_shared(state_s));
        const uint32_t m = min(static_cast<uint32_t>(kChunk), v.n - i * kChunk);
        if (16u * tile >= m) return;
        // scores of tokens 16 tile + g (+ 8) with keys up to their own
        float p[8][4], o[kCols][4];
#pragma unroll
        for (int n = 0; n < 8; ++n) p[n][0] = p[n][1] = p[n][2] = p[n][3] = 0.0f;
#pragma unroll
        for (int n = 0; n < kCols; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            uint32_t q[4];
            ldsm4(q, q_a + tile_at<D>(16 * tile + (lane & 15), 2 * k + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if (n > tile) continue;
                uint32_t b[4];  // keys 16 n + 0-7 at both halves of the channels, then keys 8-15
                ldsm4(b, k_a + tile_at<D>(16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                mma<T>(p[2 * n], q, b[0], b[1]);
                mma<T>(p[2 * n + 1], q, b[2], b[3]);
            }
            if constexpr (!S::kHalf) {
#pragma unroll
                for (int n = 0; n < kCols; n += 2) {
                    uint32_t b[4];  // state rows 16 k + 0-15 at 8 channels, then at the next 8
                    ldsm4t(b, state_a + tile_at<D>(16 * k + (lane & 15), col0 + n + (lane >> 4)));
                    mma<T>(o[n], q, b[0], b[1]);
                    mma<T>(o[n + 1], q, b[2], b[3]);
                }
            } else {
                // halves have no room for a state's range: tf32, exact for q, with f16's precision for the state
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 r0 = half2_at(q[2 * e]), r1 = half2_at(q[2 * e + 1]);
                    const uint32_t x[4] = {__float_as_uint(r0.x), __float_as_uint(r1.x), __float_as_uint(r0.y),
                                           __float_as_uint(r1.y)};
                    const float* rows = reinterpret_cast<const float*>(state_s) + (16 * k + 8 * e + 2 * t) * S::kPitch + 8 * col0 + g;
#pragma unroll
                    for (int n = 0; n < kCols; ++n)
                        mma_tf32(o[n], x, __float_as_uint(rows[8 * n]), __float_as_uint(rows[S::kPitch + 8 * n]));
                }
            }
        }
        // decays; what a token does not see is zero
        float up[2] = {1.0f, 1.0f};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = 16 * tile + g + 8 * r;
            float top = 0.0f;
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = 8 * n + 2 * t + e;
                    float& x = p[n][2 * r + e];
                    x = key <= row && n <= 2 * tile + 1 ? x * power[max(row - key, 0)] : 0.0f;
                    top = fmaxf(top, fabsf(x));
                }
            float down = 1.0f;
            if constexpr (S::kHalf) {
                // weights become halves below 2^15, by a power of two a row
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float2 f = row_scale(top);
                down = f.x, up[r] = f.y;
#pragma unroll
                for (int n = 0; n < 8; ++n) p[n][2 * r] *= down, p[n][2 * r + 1] *= down;
            }
            const float grow = power[row + 1] * down;
#pragma unroll
            for (int n = 0; n < kCols; ++n) o[n][2 * r] *= grow, o[n][2 * r + 1] *= grow;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k > tile) continue;
            const uint32_t x[4] = {pack2(p[2 * k][0], p[2 * k][1], T{}), pack2(p[2 * k][2], p[2 * k][3], T{}),
                                   pack2(p[2 * k + 1][0], p[2 * k + 1][1], T{}), pack2(p[2 * k + 1][2], p[2 * k + 1][3], T{})};
#pragma unroll
            for (int n = 0; n < kCols; n += 2) {
                uint32_t b[4];
                ldsm4t(b, v_a + tile_at<D>(16 * k + (lane & 15), col0 + n + (lane >> 4)));
                if (bad) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) b[e] = finite2<T>(b[e]);
                }
                mma<T>(o[n], x, b[0], b[1]);
                mma<T>(o[n + 1], x, b[2], b[3]);
            }
        }
        if (bad) {
            // the values that were left out, one by one, for the tokens that see them
#pragma unroll 1
            for (int r = 0; r < 2; ++r) {
                const int row = 16 * tile + g + 8 * r;
#pragma unroll 1
                for (int key = 0; key <= row && key < static_cast<int>(m); ++key) {
                    float dot = 0.0f;
#pragma unroll 1
                    for (int ch = 0; ch < D; ++ch)
                        dot = fmaf(tile_value<T, D>(base, row, ch), tile_value<T, D>(base + S::kTile, key, ch), dot);
                    dot *= power[row - key];
#pragma unroll
                    for (int n = 0; n < kCols; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x = tile_value<T, D>(base + 2 * S::kTile, key, 8 * (col0 + n) + 2 * t + e);
                            if (!isfinite(x)) o[n][r ? 2 + e : e] += dot * x;
                        }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = 16 * tile + g + 8 * r;
            if (row >= m) continue;
            T* to = static_cast<T*>(a.out) + (v.start + i * kChunk + row) * a.o_ts + h * a.o_hs + 8 * col0 + 2 * t;
            const float f = a.scale * up[r];
#pragma unroll
            for (int n = 0; n < kCols; ++n)
                *reinterpret_cast<uint32_t*>(to + 8 * n) = pack2(o[n][2 * r] * f, o[n][2 * r + 1] * f, T{});
        }
    };

    // A walk over the block's chunks: the outputs beside the state's next step, or the state alone.  The two kinds of
    // warps have loops of their own (so that neither holds the other's registers), with the same barriers.
    auto walk = [&](auto whole, auto state_warp) {
        constexpr bool kWhole = decltype(whole)::value, kStateWarp = decltype(state_warp)::value;
        auto arrived = [&](uint32_t i) {
            // infinities and NaN among the values must not reach earlier tokens as zero times them
            bool bad = false;
            if (kWhole && i < end) {
                const uint8_t* const vs = smem + (i - first) % S::kStages * 3 * S::kTile + 2 * S::kTile;
#pragma unroll
                for (int c = 0; c < kEach; ++c) {
                    const uint32_t x = c * S::kThreads + threadIdx.x;
                    const uint4 w = *reinterpret_cast<const uint4*>(vs + tile_at<D>(x / kRowChunks, x % kRowChunks));
                    bad |= not_finite2<T>(w.x) | not_finite2<T>(w.y) | not_finite2<T>(w.z) | not_finite2<T>(w.w);
                }
                if (bad) bad_chunk[(i - first) % S::kStages] = i;
            }
            meet();
            return kWhole && i < end && bad_chunk[(i - first) % S::kStages] == i;
        };
#pragma unroll 1
        for (uint32_t x = 0; x + 1 < S::kStages; ++x) load(first + x, kWhole);
        if (kWhole && kStateWarp && holds) publish(first);
        cp_wait<S::kStages - 2>();
        bool bad = arrived(first);
#pragma unroll 1
        for (uint32_t i = first; i < end; ++i) {
            load(i + S::kStages - 1, kWhole);
            if constexpr (!kStateWarp) {
                if (kWhole) outputs(i, bad);
            } else if (holds) {
                update(i);
                if (kWhole && S::kStates == 2) publish(i + 1);
            }
            cp_wait<S::kStages - 2>();
            if (kWhole && S::kStates == 1) {
                meet();  // the state has been read
                if (kStateWarp && holds) publish(i + 1);
            }
            bad = arrived(i + 1);
        }
        cp_wait<0>();
    };

    const size_t size = static_cast<size_t>(D) * D;
    const float* const from = a.states + (static_cast<size_t>(v.source < 0 ? 0 : v.source) * a.heads + h) * size;
    const size_t at = static_cast<size_t>(16 * sw + g) * D + 2 * t;
    auto run = [&](auto state_warp) {
        constexpr bool kStateWarp = decltype(state_warp)::value;
        if (parts > 1) {
            // What each block's tokens add to a state, then the states before them: element by element, each block a
            // share of the elements for all of them, over distributed shared memory.
            cg::cluster_group cluster = cg::this_cluster();
            if (rank + 1 < parts) walk(std::false_type{}, state_warp);
            meet();
            float* const shared = reinterpret_cast<float*>(smem);
            constexpr int kHolders = S::kStateWarps * 32;
            const int id = threadIdx.x - S::kOutWarps * 32;
            if (kStateWarp && holds) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) shared[(4 * n + e) * kHolders + id] = st[n][e];
            }
            meet_cluster();
            const uint32_t share = D * D / parts;
            for (uint32_t x = threadIdx.x; x < share; x += S::kThreads) {
                const uint32_t at_x = rank * share + x, who = at_x % kHolders, ne = at_x / kHolders, l = who & 31;
                const uint32_t row = 16 * (who >> 5) + (l >> 2) + 8 * ((ne >> 1) & 1), col = 8 * (ne >> 2) + 2 * (l & 3) + (ne & 1);
                float y = v.source < 0 ? 0.0f : from[row * D + col];
                float added[kMostParts];
#pragma unroll
                for (uint32_t b = 0; b < kMostParts; ++b)
                    added[b] = b + 1 < parts ? cluster.map_shared_rank(shared, b)[at_x] : 0.0f;
#pragma unroll
                for (uint32_t b = 0; b < kMostParts; ++b) {
                    if (b >= parts) break;
                    cluster.map_shared_rank(shared, b)[at_x] = y;
                    y = faded(fades[2 + b], y, added[b]);
                }
            }
            meet_cluster();
            if (kStateWarp && holds) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st[n][e] = shared[(4 * n + e) * kHolders + id];
            }
            meet();  // the tiles go there
        } else if (kStateWarp && holds && v.source >= 0) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                const float2 x = *reinterpret_cast<const float2*>(from + at + 8 * n);
                const float2 y = *reinterpret_cast<const float2*>(from + at + 8 * D + 8 * n);
                st[n][0] = x.x, st[n][1] = x.y, st[n][2] = y.x, st[n][3] = y.y;
            }
        }
        walk(std::true_type{}, state_warp);
        // the block with the last tokens has the state after them (all of them where there are none: the first)
        const bool last = end == chunks && (first < end || (chunks == 0 && rank == 0));
        if (kStateWarp && holds && last && v.target >= 0) {
            float* to = a.states + (static_cast<size_t>(v.target) * a.heads + h) * size + at;
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                *reinterpret_cast<float2*>(to + 8 * n) = make_float2(st[n][0], st[n][1]);
                *reinterpret_cast<float2*>(to + 8 * D + 8 * n) = make_float2(st[n][2], st[n][3]);
            }
        }
    };
    if (sw >= 0) run(std::true_type{});
    else run(std::false_type{});
}

// Blocks that a sequence and head are cut into along time (a cluster): as many as run at once, where they have two
// chunks each at least.  A cut costs a second walk for the state, so two parts gain nothing (128 heads of 64 channels
// over 1024 tokens: 51 us in two, 41 uncut); 16 heads of 64 over 1024 tokens in 8 parts 15.4 us, 16 heads of 128 channels
// of bf16 over 65536 tokens 2529 in 16 (before a chunk's sums were rounded into the state: 5382 uncut, 1979 in 4, or in
// 8, as a GPU has room for 15 clusters of 8 such blocks, 1502 in 16).
uint32_t parts_of(const LinearArgs& a, int resident) {
    const uint64_t jobs = static_cast<uint64_t>(a.sequences) * a.heads, chunks = (a.max_new + kChunk - 1) / kChunk;
    uint32_t parts = 1;
    while (parts < kMostParts && jobs * parts <= 74ull * resident && chunks >= parts * 4) parts *= 2;
    return parts < 4 ? 1 : parts;
}

template <typename T, int D> cudaError_t launch(const LinearArgs& a, cudaStream_t s) {
    const uint32_t blocks = a.sequences * a.heads;
    if (a.max_new <= kStepTokens) {
        linear_step_kernel<T, D><<<blocks, StepShape<D>::kThreads, 0, s>>>(a);
        return cudaGetLastError();
    }
    using S = ChunkShape<T, D>;
    static_assert(S::kBytes <= 226 * 1024, "shared memory");
    auto* kernel = linear_chunk_kernel<T, D>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    const uint32_t parts = parts_of(a, S::kBlocks);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks * parts);
    cfg.blockDim = dim3(S::kThreads);
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

template <typename T> cudaError_t by_dim(const LinearArgs& a, cudaStream_t s) {
    switch (a.head_dim) {
        case 32: return launch<T, 32>(a, s);
        case 64: return launch<T, 64>(a, s);
        default: return launch<T, 128>(a, s);
    }
}

}  // namespace

cudaError_t launch_linear_attention(const LinearArgs& a, int dtype, cudaStream_t s, uint32_t* launches) {
    bool taken = false;
    *launches = 1;
    const cudaError_t e = launch_linear_attention_tc(a, dtype, s, &taken, launches);
    if (taken || e != cudaSuccess) return e;
    return dtype == LWM_DTYPE_BF16 ? by_dim<bf16>(a, s) : by_dim<__half>(a, s);
}

}  // namespace lwm
