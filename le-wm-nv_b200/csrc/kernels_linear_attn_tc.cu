// kernels_linear_attn_tc.cu — linear attention with decay over whole histories
// of bf16 on the tcgen05 tensor cores (lwm_linear_attention_device).
//
// A block takes a sequence and head, or, of few long ones, a part along time,
// in chunks of 128 tokens:
//   P  = Q K^T                     (TMEM), times lambda^(i-j) where j <= i, to bf16 in place
//   O1 = Q S, O2 = P V             (TMEM), out = scale (lambda^(i+1) O1 + O2)
//   S  = lambda^m S + K'^T V       (the product in TMEM, S in registers; a bf16 copy in shared memory for O1)
// with K' = lambda^(m-1-j) k_j in three parts of 8 bits, so that S keeps them
// as 32-bit products would.  P and the copy of S are rounded to bf16 as operands
// have to be: half a step each, of either sign, which in a sum costs about what
// rounding the output does (errors of 0.0023 against 0.0017 for the latter alone).
//
// Warps: four for the outputs (a token a thread: P, O1, O2), eight for the
// state (a key channel a thread, half of the value channels: K' some tokens at
// a time, computed while the products before it run, then S), one that loads
// by TMA, and an issuer of products for each of the two chains.  V has two
// stages; Q and K are loaded again as soon as their products are done (the state
// reads its keys from memory, with L2's help).  With 64 channels there is room
// for two stages of Q and of P, so a chunk's weights are computed beside the
// product of the one before with V.  All
// tiles are rows of 64 channels (128 bytes, 128-byte swizzle); K' is an M-major
// A operand, V and S N-major B operands of that layout.  64 channels have a
// second half of K' that is zero, as an A operand of 128 rows wants.
//
// What bounds it (one B200): the instructions of the two chains, one after
// another in few warps.  A chunk of 64 channels takes about 3.3 us, 4000 of its
// cycles in the output warps and as many in the state's; one of 128 channels
// 4.6, the state's warps (K' in parts, waits for the products, the state).  16
// sequences of up to 1568 tokens, 16 heads of 64: 68.5 us, 256 blocks on 148
// SMs, where the bytes would take 23; one of 65536 tokens, 16 heads of 128: 458
// to 474 us (the states 192, the joining 9, the outputs 270), where its bytes
// (keys and values read twice, 1.6 GB in DRAM) would take 250.  Measured
// otherwise, when these took 69.5 and 475:
// mma.sync with the state in registers 98 and 1502; one stage of Q and P 72;
// two sums of keys and values in TMEM by turns, so that no wait is left in the
// state's warps, 73 and 470 (fewer cycles, more of them in each other's way);
// the state in TMEM alone, summed there, 71 and 456, but off by 2e-5 where
// nothing fades, as those sums are cut off (now 6e-7).
//
// A head's factor for a chunk is the sum of two floats (Fade), the same for a
// chunk, a part and a single token, whatever is left of a state.
//
// Parts: a first launch walks them for the state alone, each from zero, a
// second one turns what they add into the states before them, and a third one
// walks them for the outputs.  In between, a part's state (32 bits) lies in the
// rows of `out` that are the part's own, where nothing is kept yet; so no part is
// shorter than that many rows, and a call whose out overlaps its inputs is not
// cut here (most of those go by clusters on mma.sync, and all whose out may lie
// on keys or values).
//
// Rows behind the sequence's end are another's: their keys weigh zero, their
// values are zeroed.  Infinities and NaN among the values make outputs that
// are not finite, also of tokens that do not see them; such rows of their chunk
// are computed again, term by term (about 2.5 ms a chunk).  Every wait is bounded: one that gives up marks the
// block, which unwinds.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <algorithm>
#include <cmath>
#include <numeric>

#include "lwm_linear_attn.cuh"
#include "lwm_tc.cuh"

namespace lwm {

namespace {

constexpr int kChunk = 128;
constexpr int kThreads = 480, kOut = 128, kState = 256, kOutWarps = 4, kStateWarps = 8;
constexpr int kLoadWarp = 12, kStateIssuer = 13, kOutIssuer = 14;
constexpr uint32_t kMostParts = 64;
// What a launch does: the whole, the state that a part adds, or the outputs of a part.
constexpr int kWhole = 0, kAdds = 1, kGoesOn = 2;

template <int D> struct Shape {
    static constexpr int kPanels = D / 64;
    static constexpr int kTile = kPanels * kChunk * 128;    // bytes of 128 tokens
    static constexpr int kRound = 4096 / D;                 // tokens of a round of K', twice 16 bytes a thread
    static constexpr int kPart = kPanels * kRound * 128;    // of a part of it
    static constexpr int kS = D * D * 2;
    static constexpr int kAhead = D == 64 ? 2 : 1;          // stages of Q, and of scores and weights: room is there
    static constexpr int kQ = 0, kK = kAhead * kTile, kV = kK + kTile, kParts = kV + 2 * kTile, kSAt = kParts + 6 * kPart;
    static constexpr int kStage = kSAt + kS;                // outputs on their way, 32 rows of 32 channels a warp
    static constexpr int kZero = kStage + 4 * 2048;         // 64 channels: the empty half of K'
    static constexpr int kBytes = kZero + (D == 64 ? kRound * 128 : 0) + 1024;  // + alignment
    static constexpr uint32_t kPCol = 0, kO1Col = kAhead * 128, kO2Col = kO1Col + D, kSCol = kO2Col + D;  // of TMEM
    static_assert(kSCol + D <= 512, "TMEM");
};

struct Control {
    uint64_t q_full[2], q_empty[2], k_full, k_empty, v_full[2], v_empty[2], v_raw, scores[2], weights[2], between, pv, o_free, parts[2], kv[2], s_copy, drain;
    uint32_t tmem;
    int dead;     // a wait gave up
    float power[kChunk + 1];  // lambda^i
    Fade fades[2];            // of a whole chunk, and of the sequence's last one
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
// kind::f16 of bf16 with f32 accumulation, M 128: operands K-major, or transposed (bits 15 and 16).
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool a_turned, bool b_turned) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_turned ? 1u : 0u) << 15) | ((b_turned ? 1u : 0u) << 16) | ((n >> 3) << 17) |
           ((128u >> 4) << 24);
}
// A warp's arrival, by one lane (32 arrivals at one barrier wait for each other).
__device__ __forceinline__ void arrive_w(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(bar);
}
// Descriptors: the low word holds the start and the distance of the panels of 64 channels (in 16 bytes), the high one
// is a constant (8-row groups 1024 bytes apart, 128-byte swizzle).
constexpr uint32_t kHigh = (1024u >> 4) | (1u << 14) | (tc::kSwizzle128 << 29);
__device__ __forceinline__ uint32_t low_desc(uint32_t addr, uint32_t panel) { return (addr >> 4) | ((panel >> 4) << 16); }
// Two K = 16 steps by a whole warp (one elected lane), the second's operands at fixed distances: issued one by one, a
// step costs the warp about 100 cycles for its descriptors.
__device__ __forceinline__ void mma2(uint32_t d, uint32_t al, uint32_t a_step, uint32_t bl, uint32_t b_step, uint32_t id, uint32_t more) {
    asm volatile(
        "{\n\t.reg .pred e, m;\n\t.reg .b32 a2, b2;\n\t.reg .b64 x, y;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 m, %7, 0;\n\t"
        "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%3, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %6, m;\n\t"
        "add.u32 a2, %1, %2;\n\tadd.u32 b2, %3, %4;\n\tmov.b64 x, {a2, %5};\n\tmov.b64 y, {b2, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %6, 1;\n\t}\n" ::"r"(d),
        "r"(al), "r"(a_step), "r"(bl), "r"(b_step), "r"(kHigh), "r"(id), "r"(more)
        : "memory");
}
// The same with A in TMEM (8 columns a step).
__device__ __forceinline__ void mma2_t(uint32_t d, uint32_t at, uint32_t bl, uint32_t b_step, uint32_t id, uint32_t more) {
    asm volatile(
        "{\n\t.reg .pred e, m;\n\t.reg .b32 a2, b2;\n\t.reg .b64 y;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 m, %6, 0;\n\t"
        "mov.b64 y, {%2, %4};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %5, m;\n\t"
        "add.u32 a2, %1, 8;\n\tadd.u32 b2, %2, %3;\n\tmov.b64 y, {b2, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], y, %5, 1;\n\t}\n" ::"r"(d),
        "r"(at), "r"(bl), "r"(b_step), "r"(kHigh), "r"(id), "r"(more)
        : "memory");
}
// 64 channels of 128 rows of a head to shared memory (no multicast).
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int channel, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(tc::smem_u32(bar)), "r"(channel), "r"(head), "r"(row)
        : "memory");
}
// The same rows into L2.
__device__ __forceinline__ void prefetch_rows(const CUtensorMap* map, int channel, int head, int row) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(channel), "r"(head), "r"(row) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// Offset of 16-byte chunk c of row r of a tile whose panels have `rows` rows.
__device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c, uint32_t rows) {
    return (c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The part of a sequence's chunks that one of `parts` blocks has: `per` of them, the last part what is left, and
// another 2 D - 1 tokens at most, so that each part has rows of `out` for a state.
struct Part {
    uint32_t chunks, first, end, count;  // of the sequence; chunks of this part; parts with tokens
};
__host__ __device__ __forceinline__ uint32_t chunks_a_part(uint32_t max_new, uint32_t parts) {
    return ((max_new + kChunk - 1) / kChunk + parts - 1) / parts;
}
__device__ __forceinline__ Part part_of(uint32_t n, uint32_t per, uint32_t parts, uint32_t rank, uint32_t d) {
    Part p;
    const uint32_t tokens = per * kChunk, full = n / tokens, rest = n - full * tokens;
    p.chunks = (n + kChunk - 1) / kChunk;
    p.count = parts == 1 ? 1 : max(1u, rest >= 2 * d ? full + 1 : full);
    p.first = rank < p.count ? rank * per : p.chunks;
    p.end = rank + 1 < p.count ? p.first + per : p.chunks;
    return p;
}
// Element i of a part's state in the rows of `out` from `row` on.
template <int D> __device__ __forceinline__ float* stash(const LinearArgs& a, size_t row, uint32_t h, uint32_t i) {
    return reinterpret_cast<float*>(static_cast<bf16*>(a.out) + (row + i / (D / 2)) * a.o_ts + h * a.o_hs) + i % (D / 2);
}

template <int D, int kMode>
__global__ void __launch_bounds__(kThreads, 1)
    linear_tc_kernel(const __grid_constant__ LinearArgs a, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map, uint32_t per, uint32_t parts) {
    using S = Shape<D>;
    constexpr int kSteps = D / 16, kRowChunks = D / 8;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Control ctl_s;
    Control* const ctl = &ctl_s;
    uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t base = tc::smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % parts, job = blockIdx.x / parts;
    const uint32_t s = a.head_div.div(job), h = job - s * a.heads;
    const StateView v = state_view(a, s, kMode != kGoesOn && h == 0 && rank == 0 && threadIdx.x == 0);
    if (!v.ok) return;
    const Part part = part_of(v.n, per, parts, rank, D);
    const uint32_t chunks = part.chunks, first = part.first, end = part.end;
    if (rank >= part.count || (kMode == kAdds && rank + 1 == part.count)) return;
    const uint32_t hk = a.group_div.div(h);
    float decay = a.log_decay[h];
    if (decay < -200.0f) decay = -200.0f;  // (e^-200 is zero; minus infinity times zero would be NaN)

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&ctl->q_full[i], 1);
            tc::mbar_init(&ctl->q_empty[i], 2);
            tc::mbar_init(&ctl->scores[i], 1);
            tc::mbar_init(&ctl->weights[i], kOutWarps);
            tc::mbar_init(&ctl->v_full[i], 1);
            tc::mbar_init(&ctl->v_empty[i], 2);
            tc::mbar_init(&ctl->parts[i], kStateWarps);
            tc::mbar_init(&ctl->kv[i], 1);
        }
        for (uint64_t* b : {&ctl->k_full, &ctl->k_empty, &ctl->v_raw, &ctl->between, &ctl->pv}) tc::mbar_init(b, 1);
        tc::mbar_init(&ctl->o_free, kOutWarps);
        tc::mbar_init(&ctl->s_copy, kStateWarps);
        tc::mbar_init(&ctl->drain, 2);
        ctl->dead = 0;
        tc::mbar_fence_init();
    }
    for (int i = threadIdx.x; i <= kChunk; i += kThreads) ctl->power[i] = expf(decay * i);
    if (threadIdx.x < 2) ctl->fades[threadIdx.x] = fade_of(decay * (threadIdx.x ? (v.n + kChunk - 1) % kChunk + 1 : kChunk));
    if constexpr (D == 64)
        for (int i = threadIdx.x; i < S::kRound * 8; i += kThreads) *reinterpret_cast<uint4*>(smem + S::kZero + i * 16) = make_uint4(0, 0, 0, 0);
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
    // chunk i's stage of Q, scores and weights, and the parity of its turn there
    constexpr uint32_t kAhead = S::kAhead;
    auto stage_of = [&](uint32_t i) { return (i - first) % kAhead; };
    auto turn_of = [&](uint32_t i) { return (i - first) / kAhead & 1; };
    auto row_at = [&](uint32_t i) { return static_cast<size_t>(v.start) + i * kChunk; };

    // ------------------------------------------------------------ loads
    auto loads = [&] {
        constexpr bool whole = kMode != kAdds;
        const uint32_t from = first;
        uint32_t use = 0;
        bool fine = true;
        auto tile = [&](const CUtensorMap* map, uint32_t head, uint32_t i, uint32_t to, uint64_t* bar) {
            if (lane == 0) {
                tc::mbar_expect_tx(bar, S::kTile);
#pragma unroll
                for (int p = 0; p < S::kPanels; ++p) tma_rows(to + p * kChunk * 128, map, 64 * p, head, static_cast<int>(row_at(i)), bar);
            }
            __syncwarp();
        };
        // keys (which the state reads from memory) and queries come to L2 two chunks ahead
        auto ahead = [&](uint32_t i) {
            if (i >= end || lane >= S::kPanels * (whole ? 2 : 1)) return;
            if (lane < S::kPanels) prefetch_rows(&k_map, 64 * lane, hk, static_cast<int>(row_at(i)));
            else prefetch_rows(&q_map, 64 * (lane - S::kPanels), h, static_cast<int>(row_at(i)));
        };
        ahead(from + 1);
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t st = use & 1, round = use >> 1, m = tokens_of(i);
            ahead(i + 2);
            if (whole) {
                if (i > from) fine = wait(&ctl->k_empty, (i - from - 1) & 1, ctl, 1, err, s);
                if (!fine) break;
                tile(&k_map, hk, i, base + S::kK, &ctl->k_full);
                const uint32_t at = stage_of(i);
                if (i - from >= kAhead) fine = wait(&ctl->q_empty[at], turn_of(i) ^ 1, ctl, 3, err, s);
                if (!fine) break;
                tile(&q_map, h, i, base + S::kQ + at * S::kTile, &ctl->q_full[at]);
            }
            if (use >= 2) fine = wait(&ctl->v_empty[st], (round - 1) & 1, ctl, 2, err, s);
            if (!fine) break;
            const uint32_t v_a = S::kV + st * S::kTile;
            tile(&v_map, hk, i, base + v_a, m == kChunk ? &ctl->v_full[st] : &ctl->v_raw);
            if (m < kChunk) {  // (the sequence's last chunk) rows behind it
                fine = wait(&ctl->v_raw, 0, ctl, 4, err, s);
                if (!fine) break;
                for (uint32_t x = m * kRowChunks + lane; x < kChunk * kRowChunks; x += 32)
                    *reinterpret_cast<uint4*>(smem + v_a + chunk_at(x / kRowChunks, x % kRowChunks, kChunk)) = make_uint4(0, 0, 0, 0);
                tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctl->v_full[st]);
            }
        }
        // a block that gave up: its boxes in flight land long before this
        if (!fine)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    };

    // ------------------------------------------------------------ state
    const int t_state = threadIdx.x - kOut, wg = t_state >> 7, row = t_state & 127;  // key channel, half of the value channels
    const int col0 = wg * (D / 2);
    const bool has_row = row < D;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    // the bf16 copy of this thread's part of the state
    auto copy16 = [&](int c, const float* x) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = x[8 * b + e];
            *reinterpret_cast<uint4*>(smem + S::kSAt + chunk_at(row, (col0 + c) / 8 + b, D)) = pack<bf16>(f).a;
        }
    };
    // The state's steps; x is this thread's part of it.  The parts of K' are computed while the products before them run.
    auto states = [&](float(&x)[D / 2]) {
        constexpr bool whole = kMode != kAdds;
        const uint32_t from = first;
        uint32_t use = 0, turn = 0;  // chunks and rounds so far
        bool fine = true;
        // Keys come straight from memory, a round ahead (their tile in shared memory is for P).
        uint4 raw[2];
        const int at_tok = t_state / kRowChunks, at_ch = t_state % kRowChunks;  // and kApart tokens later
        constexpr int kApart = kState / kRowChunks;
        auto ask = [&](uint32_t i, uint32_t round) {
            const uint32_t m = tokens_of(i), tok = round * S::kRound + at_tok;
            const bf16* const k = k_at + (row_at(i) + tok) * a.k_ts + 8 * at_ch;
#pragma unroll
            for (int c = 0; c < 2; ++c)
                raw[c] = tok + c * kApart < m ? *reinterpret_cast<const uint4*>(k + c * kApart * a.k_ts) : make_uint4(0, 0, 0, 0);
        };
        ask(from, 0);
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t m = tokens_of(i), rounds = (m + S::kRound - 1) / S::kRound;
            const bool more = i + 1 < end;
            for (uint32_t round = 0; round < rounds; ++round, ++turn) {
                // three parts of 8 bits are all of a 32-bit product: its high half, and twice that of what is left
                uint4 part[3][2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float f[8];
                    unpack(Vec8<bf16>{raw[c]}, f);
                    const uint32_t tok = round * S::kRound + at_tok + c * kApart;
                    const float w = ctl->power[tok < m ? m - 1 - tok : 0];
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= w;
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        uint32_t* const y = &part[p][c].x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t lo = __float_as_uint(f[2 * e]), hi = __float_as_uint(f[2 * e + 1]);
                            y[e] = __byte_perm(lo, hi, 0x7632);
                            f[2 * e] -= __uint_as_float(lo & 0xffff0000u);
                            f[2 * e + 1] -= __uint_as_float(hi & 0xffff0000u);
                        }
                    }
                }
                if (round + 1 < rounds) ask(i, round + 1);
                else if (more) ask(i + 1, 0);
                const uint32_t b = turn & 1;
                if (turn >= 2) fine = wait(&ctl->kv[b], ((turn >> 1) - 1) & 1, ctl, 13, err, s);  // the round before last is done
                if (!fine) break;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        *reinterpret_cast<uint4*>(smem + S::kParts + (3 * b + p) * S::kPart + chunk_at(at_tok + c * kApart, at_ch, S::kRound)) = part[p][c];
                tc::fence_async_smem();
                if (round == 0) tc::fence_before();  // (the state's stores, too)
                arrive_w(&ctl->parts[b]);
            }
            if (fine) fine = wait(&ctl->kv[(turn - 1) & 1], ((turn - 1) >> 1) & 1, ctl, 19, err, s);
            // the bf16 copy's last reader is the product of this chunk
            if (fine && whole) fine = wait(&ctl->between, (i - from) & 1, ctl, 14, err, s);
            if (!fine) break;
            tc::fence_after();
            // Sums in TMEM are cut off, not rounded, at each step: a chunk's are added to the state here.
            const Fade fade = ctl->fades[m < kChunk];
            if (has_row) {
#pragma unroll
                for (int c = 0; c < D / 2; c += 32) {
                    float y[32];
                    tmem_ld32(t_lane + S::kSCol + col0 + c, y);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 z = faded(fade, make_float2(x[c + e], x[c + e + 1]), make_float2(y[e], y[e + 1]));
                        x[c + e] = z.x, x[c + e + 1] = z.y;
                    }
                    if (whole && more) {
                        copy16(c, x + c);
                        copy16(c + 16, x + c + 16);
                    }
                }
            }
            tc::fence_before();
            tc::fence_async_smem();
            if (whole && more) arrive_w(&ctl->s_copy);
        }
    };
    // The state's products: O1 = Q S of a chunk, then K'^T V of it in rounds.
    auto state_products = [&] {
        constexpr bool whole = kMode != kAdds;
        const uint32_t from = first;
        uint32_t use = 0, turn = 0;
        constexpr uint32_t kI = idesc(D, true, true), kB = idesc(D, false, true);
        bool fine = true;
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t st = use & 1, m = tokens_of(i), rounds = (m + S::kRound - 1) / S::kRound;
            if (whole) {
                fine = wait(&ctl->s_copy, (i - from) & 1, ctl, 17, err, s) && wait(&ctl->q_full[stage_of(i)], turn_of(i), ctl, 15, err, s);
                if (fine && i > from) fine = wait(&ctl->o_free, (i - from - 1) & 1, ctl, 16, err, s);
                if (!fine) break;
                tc::fence_after();
#pragma unroll
                for (int k = 0; k < kSteps; k += 2)
                    mma2(tmem + S::kO1Col, low_desc(base + S::kQ + stage_of(i) * S::kTile + (k >> 2) * kChunk * 128 + (k & 3) * 32, 16), 2,
                         low_desc(base + S::kSAt + k * 2048, D * 128), 128, kB, k > 0);
                tc::commit_w(&ctl->between);
                tc::commit_w(&ctl->q_empty[stage_of(i)]);
            }
            fine = wait(&ctl->v_full[st], (use >> 1) & 1, ctl, 12, err, s);
            for (uint32_t round = 0; round < rounds && fine; ++round, ++turn) {
                const uint32_t b = turn & 1;
                fine = wait(&ctl->parts[b], (turn >> 1) & 1, ctl, 18, err, s);
                if (!fine) break;
                tc::fence_after();
                const uint32_t k_a = base + S::kParts + 3 * b * S::kPart, v_low = low_desc(base + S::kV + st * S::kTile + round * S::kRound * 128, kChunk * 128);
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const uint32_t k_p = k_a + p * S::kPart, panel = D == 64 ? base + S::kZero - k_p : S::kRound * 128;
#pragma unroll
                    for (int k = 0; k < S::kRound / 16; k += 2)
                        mma2(tmem + S::kSCol, low_desc(k_p + k * 2048, panel), 128, v_low + k * 128, 128, kI, round || p || k);
                }
                tc::commit_w(&ctl->kv[b]);
            }
            if (!fine) break;
            tc::commit_w(&ctl->v_empty[st]);
            if (!whole) tc::commit_w(&ctl->v_empty[st]);
        }
    };

    // ---------------------------------------------------------- outputs
    auto out_products = [&] {
        const uint32_t from = first;
        uint32_t use = 0;
        constexpr uint32_t kP = idesc(kChunk, false, false), kO = idesc(D, false, true);
        bool fine = true;
        auto scores = [&](uint32_t i) {
            fine = wait(&ctl->q_full[stage_of(i)], turn_of(i), ctl, 20, err, s) && wait(&ctl->k_full, (i - from) & 1, ctl, 21, err, s);
            if (!fine) return;
            tc::fence_after();
#pragma unroll
            for (int k = 0; k < kSteps; k += 2) {
                const uint32_t off = (k >> 2) * kChunk * 128 + (k & 3) * 32;
                mma2(tmem + S::kPCol + stage_of(i) * 128, low_desc(base + S::kQ + stage_of(i) * S::kTile + off, 16), 2, low_desc(base + S::kK + off, 16), 2, kP, k > 0);
            }
            tc::commit_w(&ctl->scores[stage_of(i)]);
            tc::commit_w(&ctl->q_empty[stage_of(i)]);
            tc::commit_w(&ctl->k_empty);
        };
        scores(from);
        for (uint32_t i = from; i < end && fine; ++i, ++use) {
            const uint32_t st = use & 1;
            // (over the weights of the chunk before, which their product has read)
            if (kAhead == 2 && i + 1 < end) scores(i + 1);
            if (!fine) break;
            fine = wait(&ctl->v_full[st], (use >> 1) & 1, ctl, 24, err, s) && wait(&ctl->weights[stage_of(i)], turn_of(i), ctl, 27, err, s);
            if (fine && i > from) fine = wait(&ctl->o_free, (i - from - 1) & 1, ctl, 28, err, s);
            if (!fine) break;
            tc::fence_after();
#pragma unroll
            for (int k = 0; k < kChunk / 16; k += 2)
                mma2_t(tmem + S::kO2Col, tmem + S::kPCol + stage_of(i) * 128 + 8 * k, low_desc(base + S::kV + st * S::kTile + k * 2048, kChunk * 128), 128, kO, k > 0);
            tc::commit_w(&ctl->v_empty[st]);
            tc::commit_w(&ctl->pv);
            if (kAhead == 1 && i + 1 < end) scores(i + 1);  // (over the weights, which the product before it has read)
        }
    };
    auto outputs = [&] {
        const uint32_t from = first;
        const uint32_t r = threadIdx.x;  // token of the chunk
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        bool fine = true;
        auto weigh = [&](uint32_t i) {
            fine = wait(&ctl->scores[stage_of(i)], turn_of(i), ctl, 23, err, s);
            if (!fine) return;
            tc::fence_after();
            const uint32_t p_at = lanes + S::kPCol + stage_of(i) * 128;
            // weights: what a token does not see is zero
#pragma unroll 1
            for (int c = 0; c < kChunk; c += 32) {
                uint32_t p[16];
                if (c > warp * 32) {  // none of the warp's tokens
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = 0u;
                } else {
                    float x[32];
                    tmem_ld32(p_at + c, x);
                    tc::tmem_ld_wait();
                    const float* const w = ctl->power + (r - c);
                    if (c < warp * 32) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] *= w[-e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = e <= lane ? x[e] * w[e <= lane ? -e : 0] : 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = pack2(x[2 * e], x[2 * e + 1], bf16{});
                }
                tc::tmem_st8u(p_at + c / 2, reinterpret_cast<const uint32_t(&)[8]>(p[0]));
                tc::tmem_st8u(p_at + c / 2 + 8, reinterpret_cast<const uint32_t(&)[8]>(p[8]));
            }
            tc::tmem_st_wait();
            tc::fence_before();
            arrive_w(&ctl->weights[stage_of(i)]);
        };
        auto write = [&](uint32_t i) {
            const uint32_t m = tokens_of(i), turn = (i - from) & 1;
            fine = wait(&ctl->between, turn, ctl, 25, err, s) && wait(&ctl->pv, turn, ctl, 26, err, s);
            if (!fine) return;
            tc::fence_after();
            const bool live = r < m;
            const float grow = ctl->power[r + 1] * a.scale;
            bf16* const out_at = static_cast<bf16*>(a.out) + h * a.o_hs;
            // a row of O2 that is not finite is computed again, from what it sees, if values of the chunk are not finite
            // (before any output, which may be where q is)
            float zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float y[32];
                tmem_ld32(lanes + S::kO2Col + c, y);
                tc::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) zeros[e & 3] = fmaf(y[e], 0.0f, zeros[e & 3]);
            }
            const float zero = (zeros[0] + zeros[1]) + (zeros[2] + zeros[3]);
            const bool again = live && zero != 0.0f;  // (then it is NaN)
            bool bad = __any_sync(0xffffffffu, again);
            if (bad) {  // (with finite values it is right as it is)
                bad = false;
                for (uint32_t x = lane; x < m * kRowChunks; x += 32) {
                    float f[8];
                    unpack(load8(v_at + (row_at(i) + x / kRowChunks) * a.v_ts + 8 * (x % kRowChunks)), f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) bad |= !isfinite(f[e]);
                }
                bad = __any_sync(0xffffffffu, bad);
            }
            if (bad) {
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    float y[16];
                    tc::tmem_ld16(lanes + S::kO2Col + c, y);
                    tc::tmem_ld_wait();
                    if (again) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) y[e] = 0.0f;
                        for (uint32_t j = 0; j <= r; ++j) {
                            float dot = 0.0f;
                            for (int ch = 0; ch < D; ++ch)
                                dot = fmaf(static_cast<float>(q_at[(row_at(i) + r) * a.q_ts + ch]), static_cast<float>(k_at[(row_at(i) + j) * a.k_ts + ch]), dot);
                            dot *= ctl->power[r - j];
#pragma unroll
                            for (int e = 0; e < 16; ++e) y[e] = fmaf(dot, static_cast<float>(v_at[(row_at(i) + j) * a.v_ts + c + e]), y[e]);
                        }
                    }
                    __syncwarp();
                    tc::tmem_st16(lanes + S::kO2Col + c, y);
                    tc::tmem_st_wait();
                }
            }
            // 32 channels at a time through shared memory, so that a store takes whole runs of 64 bytes
            uint8_t* const stage = smem + S::kStage + warp * 2048;
            bf16* to[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t rr = warp * 32 + 8 * k + (lane >> 2);
                to[k] = rr < m ? out_at + (row_at(i) + rr) * a.o_ts + 8 * (lane & 3) : nullptr;
            }
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float x[32], y[32];
                tmem_ld32(lanes + S::kO1Col + c, x);
                tmem_ld32(lanes + S::kO2Col + c, y);
                tc::tmem_ld_wait();
                __syncwarp();  // (the rows before these have been read)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float f[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = fmaf(x[8 * b + e], grow, y[8 * b + e] * a.scale);
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((b ^ ((lane >> 1) & 3)) << 4)) = pack<bf16>(f).a;
                }
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t rr = 8 * k + (lane >> 2), b = lane & 3;
                    if (to[k]) *reinterpret_cast<uint4*>(to[k] + c) = *reinterpret_cast<const uint4*>(stage + rr * 64 + ((b ^ ((rr >> 1) & 3)) << 4));
                }
            }
            tc::fence_before();
            arrive_w(&ctl->o_free);
        };
        if (kAhead == 2) weigh(from);
        for (uint32_t i = from; i < end && fine; ++i) {
            // the next chunk's weights beside this one's product with V
            if (kAhead == 1) weigh(i);
            else if (i + 1 < end) weigh(i + 1);
            if (fine) write(i);
        }
    };

    constexpr bool whole = kMode != kAdds;
    const bool is_state = warp >= 4 && warp < 12;
    const size_t size = static_cast<size_t>(D) * D;
    const float* const before = a.states + (static_cast<size_t>(v.source < 0 ? 0 : v.source) * a.heads + h) * size;
    // the part with the last tokens has the state after them
    float* const after = whole && end == chunks && v.target >= 0 ? a.states + (static_cast<size_t>(v.target) * a.heads + h) * size : nullptr;
    const size_t row0 = static_cast<size_t>(v.start) + first * kChunk;
    const bool stashed = kMode == kGoesOn && part.count > 1;
    float x[D / 2];
    if (is_state && has_row) {
#pragma unroll
        for (int c = 0; c < D / 2; c += 16) {
            if (stashed) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[c + e] = *stash<D>(a, row0, h, (col0 + c + e) * D + row);
            } else if (kMode != kAdds && v.source >= 0) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(before + static_cast<size_t>(row) * D + col0 + c + e);
                    x[c + e] = y.x, x[c + e + 1] = y.y, x[c + e + 2] = y.z, x[c + e + 3] = y.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[c + e] = 0.0f;
            }
            if (whole) copy16(c, x + c);
        }
    }
    tc::fence_async_smem();
    __syncthreads();  // (before any output: rows of `out` may hold the state)
    if (is_state) {
        if (first < end) {
            if (whole) arrive_w(&ctl->s_copy);
            states(x);
        }
        if (has_row && (kMode == kAdds || after)) {
#pragma unroll
            for (int c = 0; c < D / 2; c += 4) {
                if constexpr (kMode == kAdds) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) *stash<D>(a, row0, h, (col0 + c + e) * D + row) = x[c + e];
                } else {
                    *reinterpret_cast<float4*>(after + static_cast<size_t>(row) * D + col0 + c) = make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]);
                }
            }
        }
    } else if (first < end) {
        if (warp < 4) {
            if (whole) outputs();
        } else if (warp == kLoadWarp) {
            loads();
        } else if (warp == kStateIssuer) {
            state_products();
        } else {
            if (whole) out_products();
        }
    }
    // every product has read its operands before the block ends
    if (warp == kStateIssuer || warp == kOutIssuer) {
        tc::commit_w(&ctl->drain);
        tc::mbar_wait_landing(&ctl->drain, 0);
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 0) tc::tmem_free(tmem, 512);
}

// What the parts of a sequence and head add, into the states before them, element by element.
template <int D>
__global__ void __launch_bounds__(256) linear_parts_kernel(const __grid_constant__ LinearArgs a, uint32_t per, uint32_t parts) {
    constexpr uint32_t kSlices = D * D / 256;
    const uint32_t job = blockIdx.x / kSlices, i = (blockIdx.x - job * kSlices) * 256 + threadIdx.x;
    const uint32_t s = a.head_div.div(job), h = job - s * a.heads;
    const StateView v = state_view(a, s, false);
    if (!v.ok) return;
    const uint32_t count = part_of(v.n, per, parts, 0, D).count;
    if (count == 1) return;
    float decay = a.log_decay[h];
    if (decay < -200.0f) decay = -200.0f;
    const Fade fade = fade_of(decay * (per * kChunk));  // (all but the last part are that long)
    const size_t size = static_cast<size_t>(D) * D;
    float y = v.source < 0 ? 0.0f : a.states[(static_cast<size_t>(v.source) * a.heads + h) * size + (i % D) * D + i / D];
    // (eight parts are read before the first of them is written)
    for (uint32_t r0 = 0; r0 < count; r0 += 8) {
        float* at[8];
        float added[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            at[e] = stash<D>(a, static_cast<size_t>(v.start) + (r0 + e) * per * kChunk, h, i);
            added[e] = r0 + e + 1 < count ? *at[e] : 0.0f;
        }
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            if (r0 + e < count) *at[e] = y;
            y = faded(fade, y, added[e]);
        }
    }
}

// A [tokens, heads, head_dim] tensor in boxes of 128 rows of 64 channels of a head, 128-byte swizzle.
bool rows_map(const void* p, uint32_t tokens, uint32_t heads, uint32_t d, size_t ts, size_t hs, CUtensorMap* map) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    if (!encode || ts == 0 || hs == 0 || ts >> 38 || hs >> 38) return false;
    const cuuint64_t dims[3] = {d, heads, tokens}, strides[2] = {hs * 2, ts * 2};
    const cuuint32_t box[3] = {64, 1, kChunk}, ones[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int kMode>
cudaError_t launch_mode(const LinearArgs& a, const CUtensorMap (&maps)[3], uint32_t per, uint32_t parts, cudaStream_t s) {
    using S = Shape<D>;
    static_assert(S::kBytes + sizeof(Control) <= 227 * 1024, "shared memory");
    auto* kernel = linear_tc_kernel<D, kMode>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (e != cudaSuccess) return e;
    kernel<<<a.sequences * a.heads * parts, kThreads, S::kBytes, s>>>(a, maps[0], maps[1], maps[2], per, parts);
    return cudaGetLastError();
}

// Parts that a sequence and head are cut into: where that is quicker by the blocks that a GPU runs at once and the
// chunks they have one after another (a chunk costs about as much for the state alone as with its outputs), with four
// chunks each at least.
uint32_t parts_of(const LinearArgs& a) {
    const double jobs = static_cast<double>(a.sequences) * a.heads, chunks = (a.max_new + kChunk - 1) / kChunk;
    const double chunk_us = a.head_dim == 128 ? 4.6 : 3.3;
    uint32_t best = 1;
    double least = std::max(1.0, jobs / 148) * chunks * chunk_us;
    for (uint32_t parts = 2; parts <= kMostParts && parts * 4 <= chunks; ++parts) {
        const double cost = std::ceil(jobs * parts / 148) * (std::ceil(chunks / parts) * 1.7 * chunk_us + 8.0) + 12.0;
        if (cost < least) least = cost, best = parts;
    }
    return best;
}

// Whether two tensors' extents are apart.
bool apart(const void* x, size_t x_ts, size_t x_hs, uint32_t x_heads, const void* y, size_t y_ts, size_t y_hs, uint32_t y_heads, const LinearArgs& a) {
    const auto end = [&](const void* p, size_t ts, size_t hs, uint32_t heads) {
        return reinterpret_cast<uintptr_t>(p) + ((a.tokens - 1) * ts + (heads - 1) * hs + a.head_dim) * sizeof(bf16);
    };
    return end(x, x_ts, x_hs, x_heads) <= reinterpret_cast<uintptr_t>(y) || end(y, y_ts, y_hs, y_heads) <= reinterpret_cast<uintptr_t>(x);
}

// Whether an element of out may be one of x's (k or v): not where the extents are apart, nor where they interleave in a
// way that strides show (a fused projection's rows: what a token, or a head, has of each lies apart; heads that have
// q, k, v and out side by side: so it is for each of them).
bool may_share(const void* x, size_t x_ts, size_t x_hs, uint32_t x_heads, const LinearArgs& a) {
    if (apart(x, x_ts, x_hs, x_heads, a.out, a.o_ts, a.o_hs, a.heads, a)) return false;
    const size_t d = a.head_dim;
    const auto by = (static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.out)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(x))) /
                    static_cast<int64_t>(sizeof(bf16));
    const auto turn = [&](size_t n) { return static_cast<size_t>((by % static_cast<int64_t>(n) + static_cast<int64_t>(n)) % static_cast<int64_t>(n)); };
    // repeated every `outer` elements, with this much of either in between
    const auto beside = [&](size_t outer, size_t x_span, size_t o_span) {
        return outer && x_span <= turn(outer) && turn(outer) + o_span <= outer;
    };
    if (x_ts == a.o_ts && beside(x_ts, (x_heads - 1) * x_hs + d, (a.heads - 1) * a.o_hs + d)) return false;
    if (x_hs == a.o_hs && beside(x_hs, (a.tokens - 1) * x_ts + d, (a.tokens - 1) * a.o_ts + d)) return false;
    const size_t all = std::gcd(std::gcd(x_ts, a.o_ts), std::gcd(x_heads > 1 ? x_hs : 0, a.heads > 1 ? a.o_hs : 0));
    return !beside(all, d, d);
}

// Whether out's rows may not hold a state, as an input's lie among them.
bool overlaps(const LinearArgs& a) {
    const uint32_t kv = a.heads / a.group_div.d;
    return !apart(a.q, a.q_ts, a.q_hs, a.heads, a.out, a.o_ts, a.o_hs, a.heads, a) || !apart(a.k, a.k_ts, a.k_hs, kv, a.out, a.o_ts, a.o_hs, a.heads, a) ||
           !apart(a.v, a.v_ts, a.v_hs, kv, a.out, a.o_ts, a.o_hs, a.heads, a);
}

template <int D> cudaError_t launch(const LinearArgs& a, const CUtensorMap (&maps)[3], cudaStream_t s, uint32_t* launches) {
    const uint32_t parts = overlaps(a) ? 1 : parts_of(a);
    const uint32_t per = chunks_a_part(a.max_new, parts);
    if (parts == 1) return launch_mode<D, kWhole>(a, maps, per, 1, s);
    *launches = 3;
    cudaError_t e = launch_mode<D, kAdds>(a, maps, per, parts, s);
    if (e != cudaSuccess) return e;
    linear_parts_kernel<D><<<a.sequences * a.heads * (D * D / 256), 256, 0, s>>>(a, per, parts);
    e = cudaGetLastError();
    return e == cudaSuccess ? launch_mode<D, kGoesOn>(a, maps, per, parts, s) : e;
}

// 64 channels: the mma.sync kernel has two blocks a SM, chunks of 64 tokens and cuts that cost less (us, here and there):
// 64 sequences of 16 heads with 128 tokens 53 and 36, 256 77 and 62, 512 120 and 111, 1024 187 and 208; one of 16 heads
// with 128 tokens 8.3 and 7.4, 256 10.7 and 12.1, 512, cut along time, 15.6 and 12.8, 1024 26 and 15.4, 2048 29 and 28.
// With 128 channels it has one block a SM: 16 heads with 128 tokens 14.7 and 17.8, 1024 sequences and heads 112 and 143.
// Its cuts along time need no room in `out`, so it has the long sequences of a call whose out overlaps its inputs (65536
// tokens, uncut here and there: 16 heads of 64 channels 1239 and 537, 16 of 128 2015 and 2529, 4 of 128 2057 and 657).
// All with heads of their own keys and sequences of one length; ragged batches and shared heads go by the same rule.
bool rather_there(const LinearArgs& a) {
    const uint64_t jobs = static_cast<uint64_t>(a.sequences) * a.heads;
    if (parts_of(a) > 1 && (a.head_dim == 64 || jobs * 16 <= 148) && overlaps(a)) return true;
    if (a.head_dim != 64) return false;
    return a.max_new <= 192 || (a.max_new <= 512 && jobs > 148) || (a.max_new >= 384 && a.max_new <= 1024 && jobs * 4 <= 148);
}

}  // namespace

cudaError_t launch_linear_attention_tc(const LinearArgs& a, int dtype, cudaStream_t s, bool* taken, uint32_t* launches) {
    *taken = false;
    if (dtype != LWM_DTYPE_BF16 || a.head_dim < 64 || a.max_new <= 64 || rather_there(a)) return cudaSuccess;
    CUtensorMap maps[3];
    const uint32_t kv = a.heads / a.group_div.d;
    // (the state reads its keys from memory beside the outputs of the same chunk, and rows that are computed again
    // read values; the other kernel has a chunk's in shared memory before it writes)
    if (may_share(a.k, a.k_ts, a.k_hs, kv, a) || may_share(a.v, a.v_ts, a.v_hs, kv, a)) return cudaSuccess;
    if (!rows_map(a.q, a.tokens, a.heads, a.head_dim, a.q_ts, a.q_hs, &maps[0]) || !rows_map(a.k, a.tokens, kv, a.head_dim, a.k_ts, a.k_hs, &maps[1]) ||
        !rows_map(a.v, a.tokens, kv, a.head_dim, a.v_ts, a.v_hs, &maps[2]))
        return cudaSuccess;  // (strides that a tensor map does not take)
    *taken = true;
    return a.head_dim == 64 ? launch<64>(a, maps, s, launches) : launch<128>(a, maps, s, launches);
}

}  // namespace lwm
