// kernels_cache_attn_tc.cu — attention over the paged cache for many query
// rows a kv head (whole histories, frames, chunks): both products on the
// tcgen05 tensor cores.
//
// A block takes 256 query rows (tokens x heads of the group) of one sequence
// and kv head as two tiles of 128 (or one, where that fills more SMs), and
// walks the visible keys 128 at a time.
// S = Q K^T goes to TMEM, a softmax warpgroup a tile (one row a thread, so no
// shuffles) reads it, writes P back over it in the operands' type, and O +=
// P V accumulates in TMEM with P as the A operand there.  The two tiles
// alternate: while one is in its softmax the tensor cores work for the other,
// and both use each K and V tile that is loaded.  The weights go to the
// product with V in two halves of 64 keys, which shortens the chain of
// scores, softmax and product that bounds a tile.  Measured and left: an
// issuing warp for each tile (their products interleave and delay each other:
// 427 us on whole histories against 373), and 64 keys a step with two buffers
// of S (375: an N = 64 product reads A as an N = 128 one does and takes three
// quarters of its time); four softmax warpgroups (397 in two passes over the
// scores, 379 in one); part of the exponentials as polynomials (375 to 381).
//
// Measured: 2 sequences of 8192 tokens, 16 heads over 4 kv heads of 128
// channels, causal, bf16: 398 us a call one after another, 897 TFLOP/s (373
// with pauses between, as the alternatives above were timed), tensor pipe 47
// %, issue slots 41 %: bound by a tile's chain of scores, softmax and product.
// 8 sequences of 394 new tokens over 1700 visible ones, 12 heads of 64
// channels, 8-bit codes: 68 us; 192 blocks on 148 SMs, a third of their 16
// steps at edges of the masks (a 16-bit cache: 61).  The producers of codes
// bounded a tile (4800 cycles) until they located their chunks once for K and
// V, looked pages up a tile ahead and kept the test for NaN scales out of the
// plain expansion: 86.
// Left: three buffers of scores for 64 channels (16-bit cache 7 % faster,
// codes 2 %, but 128 channels 5 % slower).
//
// 32 channels run as 64 whose upper half is zero (by TMA's fill beyond the
// tensor, or copies of no bytes): the softmax bounds them all the same.
//
// A prefix that sequences share (kPrefixKeys) is attended by all rows of its
// group as if they were one sequence's, in parts of its keys: a part's rows
// leave in 32 bits, divided by their sum, with that sum's logarithm, and the
// tails' kernels join them.  Figures stand at shared_plan.
//
// TMEM: S (and P) of tile t at column 128 t, O at 256 and 256 + D.  Shared
// memory: Q, two stages of K and of V, all rows of 64 channels (128 bytes,
// 128-byte swizzle); K is a K-major operand, V the transposed (N-major) one
// with the same layout.
//
// Producers (a warpgroup): a tile that every row sees comes by TMA, a box of
// 64 channels for each page; the few tiles at the edges of the masks are
// gathered row by row with cp.async, rows that no query sees as zeros.
// 8-bit codes are copied tiles ahead (four for 64 channels; shared memory has
// room for one of 128) and become halves (exact) on the way to the operands;
// each thread expands what it copied itself.  Their scales stay out of the
// products: a page's key scale multiplies its 16-key groups' scores, its value
// scale, relative to the block's largest (which the warps beside the issuer
// find meanwhile), enters the exponent of the weight, before a row's maximum m
// is taken.  The row's sum takes it out again, by a factor for each 16 keys;
// where a page lies more than 2^60 below the largest (kFar) its weights may
// vanish although the softmax gives them all, so their sum is taken from the
// scores once more, against a maximum of its own that is never below m.  Only
// a block that sees such pages runs that form of the loop (frames on codes:
// 67.7 us; one loop for both, with more registers alive, 69.7).
//
// O is rescaled only when a score passes a row's maximum by more than kRaise
// (a factor of 2^8).  Weights that become halves are 2^kLift times as large, at
// most 2^15: halves end at 2^-25, so a weight loses 2^-32 of the row's largest
// at most, less than rounding the output costs in sums of 2^18 keys too.
// Every wait is bounded: one that gives up marks the block, which unwinds.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "lwm_blocks.cuh"
#include "lwm_cache_attn.cuh"
#include "lwm_tc.cuh"

namespace lwm {

namespace {

constexpr int kTile = 128;           // rows of a tile, keys of a step
constexpr int kHalf = 64;            // keys whose weights go to the product at once
constexpr int kThreads = 512;        // two softmax warpgroups, producers, MMA issuers
constexpr int kProducers = 128;
constexpr int kScaleThreads = 96;    // of the warps beside the MMA issuer
constexpr int kPanel = kTile * 128;  // bytes of 128 rows x 64 channels
constexpr int kInfos = 4;
constexpr uint32_t kOCol = 256;
constexpr float kFar = 0x1p-60f;     // ratio of a value scale to the largest below which its sum goes by itself

// What the softmax needs of a key tile, by 16-key groups.
struct TileInfo {
    float k_scale[8];  // codes: key scales
    float v_log[8];    // log2 of the value scale relative to the block's
    float v_inv[8];    // that ratio's reciprocal, 0 below kFar
    uint32_t ok;       // groups whose page is in the pool
    uint32_t far;      // groups below kFar
    uint32_t pad[6];
};

// A tile of codes in flight, by 16-key groups, a copy for each producer warp.
struct TileNotes {
    int page[8];
    float k_scale[8], v_scale[8];
};

struct Control {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], o_half[2], o_done[2], info_full[kInfos], drain;
    uint32_t tmem;
    int dead;        // a wait gave up
    int poisoned;    // infinities or NaN were taken out of a V tile
    uint32_t lo_min, lo_max;  // a prefix: first keys in the window of the block's rows
    float v_ref;     // codes: the largest value scale of the visible pages
    int wide;        // codes: some visible page lies below kFar of it
    float high[3], low[3];
    TileInfo info[kInfos];
};

template <int D, bool kCodes> struct Shape {
    static constexpr int kPanels = D / 64;
    static constexpr int kTileBytes = kPanels * kPanel;
    static constexpr int kRaw = kCodes ? (D == 64 ? 4 : 1) : 0;      // tiles of codes in flight
    static constexpr int kRawBytes = kTile * D;                     // of K, and of V
    static constexpr int kQ = 0, kK = 2 * kTileBytes, kV = kK + 2 * kTileBytes, kCodesAt = kV + 2 * kTileBytes;
    static constexpr int kControl = kCodesAt + kRaw * 2 * kRawBytes, kNotes = kControl + static_cast<int>(sizeof(Control));
    static constexpr int kBytes = kNotes + (kCodes ? 4 * (kRaw + 1) * static_cast<int>(sizeof(TileNotes)) : 0) + 1024;  // + alignment
};

// Called by whole warps; the answer is the warp's, so that its lanes stay together.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Control* c, int site, uint64_t* err, uint32_t seq) {
    bool done = tc::mbar_try(bar, parity);
    for (uint32_t i = 0; i < tc::kWaitLimit && !done; ++i) {
        done = tc::mbar_try(bar, parity);
        if ((i & 255u) == 255u && *static_cast<volatile int*>(&c->dead)) break;
    }
    if (__all_sync(0xffffffffu, done)) return true;
    if (atomicExch(&c->dead, 1) == 0) cache_report(err, kCacheErrWait, seq, site);
    return false;
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// A product's K = 16 steps as one run of instructions by a whole warp (one
// elected lane): D (+)= A B^T.  The descriptors' low words advance by
// constants, so that between two instructions there is next to nothing; a
// call a step cost the issuing warp about 55 cycles each, as long as the
// tensor core takes for it.
#define LWM_SS(on)                                                                                      \
    "add.u32 al, %1, " on ";\n\tadd.u32 bl, %2, " on ";\n\tmov.b64 x, {al, %3};\n\tmov.b64 y, {bl, %3};\n\t" \
    "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, "
// S: 4 or 8 steps; 16 channels are 2 units of 16 bytes, a panel 1024.
template <int kSteps>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t high, uint32_t idesc) {
    if constexpr (kSteps == 8)
        asm volatile(
            "{\n\t.reg .pred e;\n\t.reg .b32 al, bl;\n\t.reg .b64 x, y;\n\telect.sync _|e, 0xffffffff;\n\t"
            LWM_SS("0") "0;\n\t" LWM_SS("2") "1;\n\t" LWM_SS("4") "1;\n\t" LWM_SS("6") "1;\n\t"
            LWM_SS("1024") "1;\n\t" LWM_SS("1026") "1;\n\t" LWM_SS("1028") "1;\n\t" LWM_SS("1030") "1;\n\t}\n" ::"r"(d),
            "r"(a_low), "r"(b_low), "r"(high), "r"(idesc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred e;\n\t.reg .b32 al, bl;\n\t.reg .b64 x, y;\n\telect.sync _|e, 0xffffffff;\n\t"
            LWM_SS("0") "0;\n\t" LWM_SS("2") "1;\n\t" LWM_SS("4") "1;\n\t" LWM_SS("6") "1;\n\t}\n" ::"r"(d),
            "r"(a_low), "r"(b_low), "r"(high), "r"(idesc)
            : "memory");
}
#undef LWM_SS
// O: the four steps of 64 keys; 16 keys are 8 columns of P and 128 units of V.
__device__ __forceinline__ void mma_weighted(uint32_t d, uint32_t a, uint32_t b_low, uint32_t high, uint32_t idesc, bool more) {
#define LWM_TS(p, on) \
    "add.u32 al, %1, " p ";\n\tadd.u32 bl, %2, " on ";\n\tmov.b64 y, {bl, %3};\n\t" \
    "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [al], y, %4, "
    asm volatile(
        "{\n\t.reg .pred e, m;\n\t.reg .b32 al, bl;\n\t.reg .b64 y;\n\telect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 m, %5, 0;\n\t"
        LWM_TS("0", "0") "m;\n\t" LWM_TS("8", "128") "1;\n\t" LWM_TS("16", "256") "1;\n\t" LWM_TS("24", "384") "1;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b_low), "r"(high), "r"(idesc), "r"(static_cast<uint32_t>(more))
        : "memory");
#undef LWM_TS
}
// Packed pairs and the three-operand maximum.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(r)
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
          "l"(reinterpret_cast<const uint64_t&>(c)));
    return reinterpret_cast<const float2&>(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
    return reinterpret_cast<const float2&>(r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Bits e of the keys k32 + e below `end`.
__device__ __forceinline__ uint32_t below(uint32_t end, uint32_t k32) {
    return end <= k32 ? 0u : end - k32 >= 32 ? 0xffffffffu : (1u << (end - k32)) - 1u;
}

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(dst)), "l"(src) : "memory");
}

// 64 channels of the rows of a box to shared memory (no multicast).
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int channel, int row, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            dst),
        "l"(map), "r"(tc::smem_u32(bar)), "r"(channel), "r"(row), "r"(page)
        : "memory");
}

// kind::f16 descriptor: f32 accumulation, both operands of type M; B
// transposed (N-major) for V.
template <typename M> __device__ __forceinline__ constexpr uint32_t idesc(uint32_t n, bool b_transposed) {
    constexpr uint32_t t = std::is_same_v<M, bf16> ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((b_transposed ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// The keys a block walks: tiles [0, sink_tiles) and from win_tile on.
struct Walk {
    uint32_t lo_min, lo_max, hi_min, hi_max, sinks_end, sink_tiles, win_tile, tiles, skip = 0;
    __device__ __forceinline__ uint32_t key0(uint32_t i) const {
        return (i < sink_tiles ? i + skip : i - sink_tiles + win_tile) * kTile;
    }
    __device__ __forceinline__ void count(uint32_t sinks) {
        sinks_end = min(sinks, min(lo_min, hi_max));
        sink_tiles = (sinks_end + kTile - 1) / kTile;
        win_tile = max(lo_min / kTile, sink_tiles);
        tiles = sink_tiles + (hi_max > win_tile * kTile ? (hi_max - win_tile * kTile + kTile - 1) / kTile : 0);
    }
    // only the share-th of so many parts of the tiles
    __device__ __forceinline__ void cut(uint32_t share, uint32_t shares) {
        const uint32_t per = (tiles + shares - 1) / shares, first = min(share * per, tiles);
        const uint32_t sink = min(first, sink_tiles);
        tiles = min(per, tiles - first);
        skip = sink;
        win_tile += first - sink;
        sink_tiles -= sink;
    }
    // whether every row sees all 128 keys from `key`
    __device__ __forceinline__ bool whole(uint32_t key) const {
        return (key >= lo_max || key + kTile <= sinks_end) && key + kTile <= hi_min;
    }
};
__device__ __forceinline__ Walk walk_of(const CacheAttnArgs& a, const SeqView& v, uint32_t row0, uint32_t last) {
    const VisibleRange r0 = visible(a, v, a.group_div.div(row0)), r1 = visible(a, v, a.group_div.div(last));
    Walk w;
    w.lo_min = r0.lo, w.lo_max = r1.lo, w.hi_min = r0.hi, w.hi_max = r1.hi;
    w.count(a.sinks);
    return w;
}

// Zeroes the infinities and NaN of eight values; true if there were any.
template <typename T> __device__ __forceinline__ bool take_out(uint4& x) {
    uint32_t* w = &x.x;
    constexpr uint32_t e = std::is_same_v<T, bf16> ? 0x7f80u : 0x7c00u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & e) == e) w[i] &= 0xffff0000u, any = true;
        if (((w[i] >> 16) & e) == e) w[i] &= 0x0000ffffu, any = true;
    }
    return any;
}

// The weights exp2(score - maximum) of a row's 64 keys, packed for the
// product, their sum (the value scales taken out again, far groups left out)
// and the largest exponent.  kMasked: only the keys that the row sees.
template <typename M, bool kCodes, bool kMasked>
__device__ __forceinline__ float weights(const float (&x)[64], uint32_t (&p)[32], float2& sum, const TileInfo& info,
                                         int half, float mul, float sub, const VisibleRange& rr, uint32_t key, uint32_t ok) {
    float top0 = -INFINITY, top1 = -INFINITY;
    sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int group = 4 * half + g;
        const float gm = kCodes ? info.k_scale[group] * mul : mul;
        const float add = kCodes ? sub + info.v_log[group] : sub;
        uint32_t seen = 0xffffu;
        if constexpr (kMasked) {
            // (rows of a warp mostly see all or none of 16 keys: a frame's rows see alike)
            const uint32_t k16 = key + 16 * group;
            seen = (ok >> group) & 1 ? below(rr.hi, k16) & (~below(rr.lo, k16) | below(rr.first, k16)) & 0xffffu : 0u;
            if (__all_sync(0xffffffffu, seen == 0)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) p[8 * g + e] = 0u;
                continue;
            }
        }
        float2 part = make_float2(0.0f, 0.0f);
        auto weigh = [&](auto masked) {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float2 y = fma2(make_float2(x[16 * g + e], x[16 * g + e + 1]), make_float2(gm, gm), make_float2(add, add));
                if constexpr (decltype(masked)::value) {
                    if (!((seen >> e) & 1)) y.x = -INFINITY;
                    if (!((seen >> (e + 1)) & 1)) y.y = -INFINITY;
                }
                if (e & 2) top1 = max3(top1, y.x, y.y);
                else top0 = max3(top0, y.x, y.y);
                y = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                part = add2(part, y);
                p[8 * g + e / 2] = pack2(y.x, y.y, M{});
            }
        };
        if (!kMasked || __all_sync(0xffffffffu, seen == 0xffffu)) weigh(std::false_type{});
        else weigh(std::true_type{});
        if constexpr (kCodes) sum = fma2(part, make_float2(info.v_inv[group], info.v_inv[group]), sum);
        else sum = add2(sum, part);
    }
    return fmaxf(top0, top1);
}

// Adds the far groups' weights of a row's 64 keys (scores at `t_scores`) to
// l, which is in units of 2^(ml - lift).
__device__ __forceinline__ void far_sum(uint32_t t_scores, const TileInfo& info, int half, float mul, const VisibleRange& rr,
                                     uint32_t key, float& l, float& ml, float lift) {
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        const int group = 4 * half + g;
        if (!((info.far >> group) & 1)) continue;
        float x[16];
        tc::tmem_ld16(t_scores + 16 * g, x);
        tc::tmem_ld_wait();
        const uint32_t k16 = key + 16 * group, seen = below(rr.hi, k16) & (~below(rr.lo, k16) | below(rr.first, k16));
        const float gm = info.k_scale[group] * mul;
        float top = ml;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[e] = (seen >> e) & 1 ? x[e] * gm : -INFINITY;
            top = fmaxf(top, x[e]);
        }
        if (top > ml) l *= exp2_fast(ml - top), ml = top;
        const float sub = ml == -INFINITY ? 0.0f : ml - lift;
#pragma unroll
        for (int e = 0; e < 16; ++e) l += exp2_fast(x[e] - sub);
    }
}

template <typename T, int D, bool kCodes, int kKeys>
__global__ void __launch_bounds__(kThreads, 1)
    cache_attn_tc_kernel(const __grid_constant__ CacheAttnArgs a, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map, uint32_t block_rows) {
    using M = std::conditional_t<kCodes, __half, T>;
    using S = Shape<D, kCodes>;
    constexpr int kSteps = D / 16;
    constexpr float kLift = std::is_same_v<M, __half> ? 7.0f : 0.0f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
    Control* ctl = reinterpret_cast<Control*>(smem + S::kControl);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (the tails' kernel may start when every block has)
    if constexpr (kKeys == kPrefixKeys) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // The last rows of the sequences first, where causal rows see the most keys, and blocks counted from the last row,
    // so that the one that is not full is the shortest and starts last.
    // A prefix: a group's rows as one sequence, over a part of the keys, which its first sequence's table names.
    constexpr bool kPrefix = kKeys == kPrefixKeys;
    const uint32_t lots = kPrefix ? a.group_count * a.splits : a.c.sequences;
    const uint32_t pairs = lots * a.c.kv_heads, turn = blockIdx.x / pairs, hs = blockIdx.x - turn * pairs;
    const uint32_t h = hs % a.c.kv_heads, lot = hs / a.c.kv_heads, share = kPrefix ? lot % a.splits : 0;
    SeqView v;
    GroupView group;
    uint32_t s = lot;
    if constexpr (kPrefix) {
        group = group_view(a, lot / a.splits, threadIdx.x == 0 && h == 0 && turn == 0 && share == 0);
        s = group.first;
        v.start = group.start, v.n = group.ok ? group.n : 0, v.length = group.shared, v.ok = group.ok;
    } else {
        v = sequence(a.c, s, false, threadIdx.x == 0 && h == 0 && turn == 0);
    }
    const uint32_t later = turn * block_rows;
    if (later >= v.n * a.group) return;
    const uint32_t rows = v.n * a.group - later;  // the end of this block's
    const uint32_t row0 = max(rows, block_rows) - block_rows, last = rows - 1;
    const bool two = last >= row0 + kTile;  // the second tile has rows
    Walk w;
    if constexpr (kPrefix) {
        // rows of many sequences: the ends of what they see, over the block
        if (threadIdx.x == 0) ctl->lo_min = a.window ? v.length : 0u, ctl->lo_max = 0u;
        if (a.window) {
            __syncthreads();
            if (threadIdx.x < 256 && row0 + threadIdx.x < rows) {
                const uint32_t lo = visible_prefix(a, group, a.group_div.div(row0 + threadIdx.x)).lo;
                atomicMin(&ctl->lo_min, lo);
                atomicMax(&ctl->lo_max, lo);
            }
        }
        __syncthreads();
        w.lo_min = ctl->lo_min, w.lo_max = ctl->lo_max, w.hi_min = w.hi_max = v.length;
        w.count(a.sinks);
        w.cut(share, a.splits);
    } else {
        w = walk_of(a, v, row0, last);
    }

    if (threadIdx.x == 0) {
        const int softmax = two ? 256 : 128;
        tc::mbar_init(&ctl->q_full, softmax);
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&ctl->k_full[i], kProducers);
            tc::mbar_init(&ctl->v_full[i], kProducers);
            tc::mbar_init(&ctl->k_empty[i], 1);
            tc::mbar_init(&ctl->v_empty[i], 1);
            tc::mbar_init(&ctl->s_full[i], 1);
            for (int b = 0; b < 2; ++b) tc::mbar_init(&ctl->p_full[i][b], 4);
            tc::mbar_init(&ctl->o_half[i], 1);
            tc::mbar_init(&ctl->o_done[i], 1);
        }
        for (int i = 0; i < kInfos; ++i) tc::mbar_init(&ctl->info_full[i], 8);
        tc::mbar_init(&ctl->drain, 1);
        ctl->dead = 0;
        ctl->poisoned = 0;
        ctl->v_ref = 1.0f;
        ctl->wide = 0;
        tc::mbar_fence_init();
    }
    if (warp == 12) tc::tmem_alloc(&ctl->tmem, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = ctl->tmem;
    uint64_t* const err = a.c.err;

    if (warp < 8) {
        // ---------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(184));
        const int tile = warp >> 2, r = threadIdx.x & 127;
        const uint32_t R = row0 + tile * kTile + r;
        if (tile == 0 || two) {
            const bool live = R < rows;
            const uint32_t tok = live ? a.group_div.div(R) : 0;
            VisibleRange rr = {0, 0, 0};
            float mul = a.scale_log2;
            if (live) {
                if constexpr (kPrefix) rr = visible_prefix(a, group, tok);
                else rr = visible(a, v, tok);
            }
            // Q: the warp's 32 rows into the swizzled tile, whole rows at a time
            {
                constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;  // lanes a row, rows a load
                const int c = lane % kLanes;
                uint8_t* dst = smem + S::kQ + tile * S::kTileBytes + (c >> 3) * kPanel;
                Vec8<T> x[kLanes];
#pragma unroll
                for (int k = 0; k < kLanes; ++k) {
                    const uint32_t Rk = row0 + tile * kTile + (warp & 3) * 32 + k * kAtOnce + lane / kLanes;
                    const uint32_t tk = Rk < rows ? a.group_div.div(Rk) : 0;
                    x[k].a = make_uint4(0, 0, 0, 0);
                    if (Rk < rows && 8u * c < a.c.head_dim)
                        x[k] = load8(static_cast<const T*>(a.q) + (v.start + tk) * a.q_ts +
                                     (h * a.group + (Rk - tk * a.group)) * a.q_hs + 8 * c);
                }
#pragma unroll
                for (int k = 0; k < kLanes; ++k) {
                    const int rk = (warp & 3) * 32 + k * kAtOnce + lane / kLanes;
                    uint4 y = x[k].a;
                    if constexpr (kCodes && std::is_same_v<T, bf16>) {
                        // to fp16 by a power of two a row, which the scores' factor takes back
                        float f[8], amax = 0.0f;
                        unpack(x[k], f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
#pragma unroll
                        for (int o = kLanes / 2; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                        int e2 = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
                        if (amax == 0.0f || e2 == 128) e2 = 0;
                        e2 = min(max(e2, -126), 126);
                        const float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] *= down;
                        y = pack<__half>(f).a;
                        // the factor of row k * kAtOnce + j to the lane that owns the row
                        const float up = __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
#pragma unroll
                        for (int j = 0; j < kAtOnce; ++j) {
                            const float u = __shfl_sync(0xffffffffu, up, j * kLanes);
                            if (lane == k * kAtOnce + j) mul *= u;
                        }
                    }
                    *reinterpret_cast<uint4*>(dst + rk * 128 + (((c & 7) ^ (rk & 7)) << 4)) = y;
                }
                tc::fence_async_smem();
                tc::mbar_arrive(&ctl->q_full);
            }
            Walk mine = w;
            if constexpr (!kPrefix) mine = walk_of(a, v, row0 + tile * kTile, min(row0 + (tile + 1) * kTile - 1, last));
            const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t t_s = t_lane + tile * kTile, t_o = t_lane + kOCol + tile * D;
            float m = -INFINITY, l = 0.0f;
            float ml_end = -INFINITY;  // wide: what l is in units of, at the end
            bool fine = true;
            // a warp without rows leaves its part of P as it is: a row of P enters its own row of O alone
            const bool idle = row0 + tile * kTile + (warp & 3) * 32 >= rows;
            for (uint32_t i = 0; i < w.tiles && fine && idle; ++i) {
                fine = wait(&ctl->s_full[tile], i & 1, ctl, 10 + tile, err, s);
                if (fine && lane < 2) tc::mbar_arrive(&ctl->p_full[tile][lane]);
            }
            // the tiles one after another; returns the root of O's unit over l's
            auto walk = [&](auto far_apart) {
            constexpr bool kWide = decltype(far_apart)::value;
            float ml = -INFINITY;  // wide: l is in units of 2^(ml - kLift), O in those of 2^(m - kLift), ml >= m
            for (uint32_t i = 0; i < w.tiles && fine; ++i) {
                // (the producers' notes are there long before the scores)
                const TileInfo& info = ctl->info[i % kInfos];
                fine = wait(&ctl->info_full[i % kInfos], (i / kInfos) & 1, ctl, 12 + tile, err, s);
                if (!fine) break;
                const uint32_t key = w.key0(i), ok = info.ok;
                const bool whole = mine.whole(key) && ok == 0xffu;
                fine = wait(&ctl->s_full[tile], i & 1, ctl, 10 + tile, err, s);
                tc::fence_after();
#pragma unroll 1
                for (int half = 0; half < 2 && fine; ++half) {
                    // The weights are taken against the row's old maximum while the new one is found; only when a
                    // score passes it by kRaise (or it is the first) are they taken again.
                    float x[kHalf];
                    tmem_ld32(t_s + kHalf * half, x);
                    tmem_ld32(t_s + kHalf * half + 32, x + 32);
                    tc::tmem_ld_wait();
                    uint32_t p[32];
                    float2 sum;
                    bool again = false;
                    while (true) {
                        const bool first = m == -INFINITY;
                        const float sub = first ? 0.0f : kLift - m;
                        const float top = whole ? weights<M, kCodes, false>(x, p, sum, info, half, mul, sub, rr, key, ok)
                                                : weights<M, kCodes, true>(x, p, sum, info, half, mul, sub, rr, key, ok);
                        if (again || !__any_sync(0xffffffffu, top > (first ? -INFINITY : kRaise + kLift))) break;
                        again = true;
                        const float up = first ? top : fmaxf(top - kLift, 0.0f), down = first ? 0.0f : exp2_fast(-up);
                        m = first ? top : m + up;
                        if constexpr (kWide) {
                            if (m > ml) l *= exp2_fast(ml - m), ml = m;
                        } else {
                            l *= down;
                        }
                        if (i > 0 || half) {  // O holds every product up to here once the last one is done
                            fine = half ? wait(&ctl->o_half[tile], i & 1, ctl, 14 + tile, err, s)
                                        : wait(&ctl->o_done[tile], (i - 1) & 1, ctl, 14 + tile, err, s);
                            if (!fine) break;
                            tc::fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                float o[16];
                                tc::tmem_ld16(t_o + c, o);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] *= down;
                                tc::tmem_st16(t_o + c, o);
                            }
                        }
                        tmem_ld32(t_s + kHalf * half, x);  // still there: P covers what has been read
                        tmem_ld32(t_s + kHalf * half + 32, x + 32);
                        tc::tmem_ld_wait();
                    }
                    if (!fine) break;
                    if constexpr (kWide) {
                        l += (sum.x + sum.y) * (m == ml ? 1.0f : exp2_fast(m - ml));
                        if ((info.far >> (4 * half)) & 0xfu) far_sum(t_s + kHalf * half, info, half, mul, rr, key, l, ml, kLift);
                    } else {
                        l += sum.x + sum.y;
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 8)
                        tc::tmem_st8u(t_s + 32 * half + c, reinterpret_cast<const uint32_t(&)[8]>(p[c]));
                    tc::tmem_st_wait();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&ctl->p_full[tile][half]);
                }
            }
            if (kPrefix) ml_end = kWide ? ml : m;
            // (twice the root of 2^(m - ml), as the whole may be below the smallest float)
            return kWide && m != ml ? exp2_fast(0.5f * (m - ml)) : 1.0f;
            };
            float root = 1.0f;
            if constexpr (kCodes) {
                bool wide = false;
                if (w.tiles && !idle) {
                    fine = wait(&ctl->info_full[0], 0, ctl, 12 + tile, err, s);
                    wide = fine && ctl->wide != 0;
                }
                if (wide) root = walk(std::true_type{});
                else if (!idle) walk(std::false_type{});
            } else if (!idle) {
                walk(std::false_type{});
            }
            if (fine && w.tiles) fine = wait(&ctl->o_done[tile], (w.tiles - 1) & 1, ctl, 16 + tile, err, s);
            tc::fence_after();
            const float inv = l == 0.0f ? 0.0f : 1.0f / l, v_ref = ctl->v_ref;
            const bool poisoned = *static_cast<volatile int*>(&ctl->poisoned) != 0;
            // rows go through the tile's Q, which no product reads any more, and out in whole 16-byte runs
            uint8_t* stage = smem + S::kQ + tile * S::kTileBytes;
#pragma unroll 1
            for (int c = 0; c < static_cast<int>(a.c.head_dim); c += 16) {
                float o[16];
                if (w.tiles) {
                    tc::tmem_ld16(t_o + c, o);
                    tc::tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = l == 0.0f ? 0.0f : kCodes ? o[e] * inv * root * v_ref * root : o[e] * inv;
                if (poisoned && live && l != 0.0f) {
                    // a value that is not finite, in a tile where rows differ in what they see: its weight is
                    // positive, so it decides its channel for the rows that see it
                    for (uint32_t i = 0; i < w.tiles; ++i) {
                        const uint32_t key = w.key0(i);
                        if (w.whole(key)) continue;
                        for (uint32_t j = key; j < min(key + kTile, rr.hi); ++j) {
                            if (!(j >= rr.lo || j < rr.first)) continue;
                            const int page = a.c.table[static_cast<size_t>(s) * a.c.table_stride + (j >> a.c.page_shift)];
                            if (static_cast<uint32_t>(page) >= a.c.pages) continue;
                            const size_t at = pool_at(a.c, page, h, j & (a.c.page_tokens - 1)) + c;
#pragma unroll
                            for (int b = 0; b < 16; b += 8) {
                                float f[8];
                                if constexpr (kCodes) {
                                    from_e4m3(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.c.v) + at + b), f);
                                    const float vs = a.c.v_scale[static_cast<size_t>(page) * a.c.kv_heads + h];
                                    if (!isfinite(vs)) f[0] = f[1] = f[2] = f[3] = f[4] = f[5] = f[6] = f[7] = __int_as_float(0x7fc00000);
                                } else {
                                    unpack(load8(static_cast<const T*>(a.c.v) + at + b), f);
                                }
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    if (!isfinite(f[e])) o[b + e] += f[e];
                            }
                        }
                    }
                }
                if constexpr (kPrefix) {
                    // a part: in 32 bits, joined with the others where the tails are read
                    if (live && fine) {
                        const size_t row = (static_cast<size_t>(share) * a.c.tokens + v.start + tok) * a.heads + h * a.group + (R - tok * a.group);
                        float4* to = reinterpret_cast<float4*>(a.part_out + row * a.c.head_dim + c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) to[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                        if (c == 0) a.part_log[row] = l == 0.0f ? -INFINITY : ml_end - kLift + log2f(l);
                    }
                } else {
                float f[8];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = o[8 * b + e];
                    const int ch = c / 8 + b;
                    *reinterpret_cast<uint4*>(stage + (ch >> 3) * kPanel + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = pack<T>(f).a;
                }
                }
            }
            __syncwarp();
            if (!kPrefix && fine) {
                constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
                const int c = lane % kLanes;
#pragma unroll
                for (int k = 0; k < kLanes; ++k) {
                    const int rk = (warp & 3) * 32 + k * kAtOnce + lane / kLanes;
                    const uint32_t Rk = row0 + tile * kTile + rk;
                    if (Rk >= rows || 8u * c >= a.c.head_dim) continue;
                    const uint32_t tk = a.group_div.div(Rk);
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (v.start + tk) * a.o_ts +
                                              (h * a.group + (Rk - tk * a.group)) * a.o_hs + 8 * c) =
                        *reinterpret_cast<const uint4*>(stage + (c >> 3) * kPanel + rk * 128 + (((c & 7) ^ (rk & 7)) << 4));
                }
            }
        }
    } else if (warp < 12) {
        // -------------------------------------------------------- producers
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(88));
        const int t = threadIdx.x - 256;
        constexpr int kRowChunks = kCodes ? D / 16 : D / 8;  // 16-byte chunks of a cached row
        constexpr int kEach = kTile * kRowChunks / kProducers, kRowStep = kProducers / kRowChunks;
        const int ch = t % kRowChunks, r0 = t / kRowChunks;
        constexpr size_t kElem = kCodes ? 1 : 2;
        const bool inside = ch * 16 < static_cast<int>(a.c.head_dim * kElem);  // (32 channels: half of a row)
        // the page of group g of tile i, -1: nothing visible or no page
        auto group_page = [&](uint32_t i, uint32_t g) {
            const uint32_t j = w.key0(i) + 16 * g;
            return i < w.tiles && j < w.hi_max && (j + 16 > w.lo_min || j < w.sinks_end) ? page_of(a.c, s, j >> a.c.page_shift) : -1;
        };
        auto page_ids = [&](uint32_t i) { return lane < 8 ? group_page(i, lane) : -1; };  // lane g: of group g
        auto row_live = [&](uint32_t j) { return inside && j < w.hi_max && (j >= w.lo_min || j < w.sinks_end); };
        auto source = [&](const void* pool, int page, uint32_t j) {
            return static_cast<const uint8_t*>(pool) +
                   (pool_at(a.c, page < 0 ? 0 : page, h, j & (a.c.page_tokens - 1)) * kElem + ch * 16);
        };
        bool fine = true;
        int pages = kCodes ? -1 : page_ids(0);
        // codes in flight: this thread's chunks, and its warp's notes of the tiles
        TileNotes* notes = reinterpret_cast<TileNotes*>(smem + S::kNotes) + (warp - 8) * (S::kRaw + 1);
        uint8_t* raw = smem + S::kCodesAt + t * 16;
        uint32_t note_in = 0, note_out = 0;  // slots of the notes written and read next
        auto copy_notes = [&](int p) {
            TileNotes& n = notes[note_in];
            note_in = note_in == S::kRaw ? 0 : note_in + 1;
            if (lane < 8) {
                n.page[lane] = p;
                if (p >= 0) {
                    const size_t at = static_cast<size_t>(p) * a.c.kv_heads + h;
                    cp_async4(&n.k_scale[lane], a.c.k_scale + at);
                    cp_async4(&n.v_scale[lane], a.c.v_scale + at);
                }
            }
        };
        // where this thread's chunks of tile i lie in either pool (all ones: not to be read), before any is asked for
        constexpr int kMine = kCodes ? kEach : 1;
        size_t from[kMine];
        auto locate = [&](uint32_t i, int p) {
#pragma unroll
            for (int c = 0; c < kMine; ++c) {
                const uint32_t r = r0 + c * kRowStep, j = w.key0(i) + r;
                const int page = __shfl_sync(0xffffffffu, p, r >> 4);
                from[c] = page >= 0 && row_live(j) ? pool_at(a.c, page, h, j & (a.c.page_tokens - 1)) + ch * 16 : ~size_t{0};
            }
        };
        auto copy_codes = [&](uint32_t i, const void* pool, int which) {
            const uint32_t dst = tc::smem_u32(raw) + ((i % max(S::kRaw, 1)) * 2 + which) * S::kRawBytes;
#pragma unroll
            for (int c = 0; c < kMine; ++c) {
                const bool live = from[c] != ~size_t{0};
                cp_async16(dst + c * kProducers * 16, static_cast<const uint8_t*>(pool) + (live ? from[c] : 0), live);
            }
        };
        // 16 codes to two chunks of halves; NaN codes of a mixed tile are taken out
        auto expand = [&](uint8_t* dst, uint32_t r, uint4 x, bool mixed, bool nan) {
            const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t y = wd[e];
                if (mixed) {
                    const uint32_t bad = __vcmpeq4(y | 0x80808080u, 0xffffffffu) | (nan ? 0xffffffffu : 0u);
                    if (bad) ctl->poisoned = 1;
                    y &= ~bad;
                } else if (nan) {
                    y = 0x7f7f7f7fu;
                }
                o[2 * e] = f16x2_from_e4m3x2(y);
                o[2 * e + 1] = f16x2_from_e4m3x2(y >> 16);
            }
            const int c0 = 2 * ch;
            uint8_t* row = dst + (c0 >> 3) * kPanel + r * 128;
            *reinterpret_cast<uint4*>(row + (((c0 & 7) ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(row + ((((c0 + 1) & 7) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
        };
        if constexpr (kCodes) {
            const int first = lane < 8 * S::kRaw ? group_page(lane >> 3, lane & 7) : -1;  // of all of them at once
#pragma unroll 1
            for (uint32_t i = 0; i < S::kRaw; ++i) {
                const int p = __shfl_sync(0xffffffffu, first, 8 * i + (lane & 7));
                if (i < w.tiles) {
                    copy_notes(p);
                    locate(i, p);
                    copy_codes(i, a.c.k, 0);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (i < w.tiles) copy_codes(i, a.c.v, 1);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        }
        float v_ref_inv = 1.0f;
        int ahead = kCodes ? page_ids(S::kRaw) : -1;  // codes: pages of the next tile to copy, looked up a tile earlier
        for (uint32_t i = 0; i < w.tiles && fine; ++i) {
            const uint32_t st = i & 1, use = (i >> 1) & 1, key = w.key0(i);
            const bool mixed = !w.whole(key);
            const int next_pages = kCodes ? -1 : page_ids(i + 1);
            float k_scale = 1.0f, v_scale = 1.0f;
            uint32_t nan_groups = 0;
            if constexpr (kCodes) {
                asm volatile("cp.async.wait_group %0;" ::"n"(2 * S::kRaw - 1) : "memory");  // K of this tile
                __syncwarp();
                const TileNotes& n = notes[note_out];
                note_out = note_out == S::kRaw ? 0 : note_out + 1;
                pages = lane < 8 ? n.page[lane] : -1;
                if (pages >= 0) k_scale = n.k_scale[lane], v_scale = n.v_scale[lane];
                nan_groups = __ballot_sync(0xffffffffu, !isfinite(v_scale));
            }
            uint8_t* kd = smem + S::kK + st * S::kTileBytes;
            uint8_t* vd = smem + S::kV + st * S::kTileBytes;
            if (i >= 2 && !wait(&ctl->k_empty[st], use ^ 1, ctl, 20, err, s)) { fine = false; break; }
            // what the softmax needs to know, a warp in turn; the ring is four tiles deep, the stages two
            auto inform = [&] {
                if (warp != 8 + static_cast<int>(i & 3) || lane >= 8) return;
                TileInfo& info = ctl->info[i % kInfos];
                if constexpr (kCodes) {
                    const float ratio = isfinite(v_scale) && pages >= 0 ? v_scale * v_ref_inv : 1.0f;
                    const bool is_far = ratio < kFar;
                    const uint32_t far = __ballot_sync(0xffu, is_far);
                    info.k_scale[lane] = k_scale;
                    info.v_log[lane] = log2f(ratio);
                    info.v_inv[lane] = is_far ? 0.0f : 1.0f / ratio;
                    if (is_far) info.v_log[lane] = log2f(v_scale) + log2f(v_ref_inv);  // (the ratio may vanish)
                    if (lane == 0) info.far = far;
                }
                const uint32_t ok = __ballot_sync(0xffu, pages >= 0);
                if (lane == 0) info.ok = ok;
                tc::mbar_arrive(&ctl->info_full[i % kInfos]);
            };
            if constexpr (!kCodes) inform();
            if constexpr (kCodes) {
                const uint8_t* kr = raw + (i % max(S::kRaw, 1)) * 2 * S::kRawBytes;
                const uint8_t* vr = kr + S::kRawBytes;
#pragma unroll
                for (int c = 0; c < kEach; ++c)
                    expand(kd, r0 + c * kRowStep, *reinterpret_cast<const uint4*>(kr + c * kProducers * 16), false, false);
                tc::fence_async_smem();
                tc::mbar_arrive(&ctl->k_full[st]);
                if (i == 0) {  // the idle warps' maximum
                    asm volatile("bar.sync 1, %0;" ::"n"(kProducers + kScaleThreads) : "memory");
                    float top = fmaxf(fmaxf(ctl->high[0], ctl->high[1]), ctl->high[2]);
                    const float low = fminf(fminf(ctl->low[0], ctl->low[1]), ctl->low[2]);
                    top = fmaxf(top, 0x1p-126f);  // (zero, or so small that its reciprocal is infinite)
                    v_ref_inv = 1.0f / top;
                    if (t == 0) ctl->v_ref = top, ctl->wide = low * v_ref_inv < kFar;
                }
                inform();
                const bool more = i + S::kRaw < w.tiles;
                if (more) {
                    copy_notes(ahead);
                    locate(i + S::kRaw, ahead);
                    copy_codes(i + S::kRaw, a.c.k, 0);
                    ahead = page_ids(i + S::kRaw + 1);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group %0;" ::"n"(2 * S::kRaw - 1) : "memory");  // V of this tile
                if (i >= 2 && !wait(&ctl->v_empty[st], use ^ 1, ctl, 21, err, s)) { fine = false; break; }
                if (!mixed && nan_groups == 0) {
#pragma unroll
                    for (int c = 0; c < kEach; ++c)
                        expand(vd, r0 + c * kRowStep, *reinterpret_cast<const uint4*>(vr + c * kProducers * 16), false, false);
                } else {
#pragma unroll
                    for (int c = 0; c < kEach; ++c) {
                        const uint32_t r = r0 + c * kRowStep;
                        expand(vd, r, *reinterpret_cast<const uint4*>(vr + c * kProducers * 16), mixed, (nan_groups >> (r >> 4)) & 1);
                    }
                }
                tc::fence_async_smem();
                tc::mbar_arrive(&ctl->v_full[st]);
                if (more) copy_codes(i + S::kRaw, a.c.v, 1);
                asm volatile("cp.async.commit_group;" ::: "memory");
            } else if (!mixed && __all_sync(0xffffffffu, lane >= 8 || pages >= 0)) {
                // (the lookups of all warps agree, so all of them come here)
                const uint32_t box = min(a.c.page_tokens, static_cast<uint32_t>(kTile));  // rows a box
                const uint32_t g = lane * box / 16;  // this lane's box starts at this group
                const int page = __shfl_sync(0xffffffffu, pages, g & 7);
                if (warp == 8 && lane == 0) tc::mbar_expect_tx(&ctl->k_full[st], S::kTileBytes);
                __syncwarp();
                const int row = h * a.c.page_tokens + (key & (a.c.page_tokens - 1));
                if (warp == 8 && g < 8)
#pragma unroll
                    for (int p = 0; p < S::kPanels; ++p)
                        tma_rows(tc::smem_u32(kd) + p * kPanel + lane * box * 128, &k_map, 64 * p, row, page, &ctl->k_full[st]);
                if (t != 0) tc::mbar_arrive(&ctl->k_full[st]);
                if (i >= 2 && !wait(&ctl->v_empty[st], use ^ 1, ctl, 21, err, s)) { fine = false; break; }
                if (warp == 8 && lane == 0) tc::mbar_expect_tx(&ctl->v_full[st], S::kTileBytes);
                __syncwarp();
                if (warp == 8 && g < 8)
#pragma unroll
                    for (int p = 0; p < S::kPanels; ++p)
                        tma_rows(tc::smem_u32(vd) + p * kPanel + lane * box * 128, &v_map, 64 * p, row, page, &ctl->v_full[st]);
                if (t != 0) tc::mbar_arrive(&ctl->v_full[st]);
            } else {
                const uint32_t ka = tc::smem_u32(kd) + (ch >> 3) * kPanel, va = tc::smem_u32(vd) + (ch >> 3) * kPanel;
#pragma unroll 4
                for (int c = 0; c < kEach; ++c) {
                    const uint32_t r = r0 + c * kRowStep, j = key + r;
                    const int page = __shfl_sync(0xffffffffu, pages, r >> 4);
                    cp_async16(ka + r * 128 + (((ch & 7) ^ (r & 7)) << 4), source(a.c.k, page, j), page >= 0 && row_live(j));
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (i >= 2 && !wait(&ctl->v_empty[st], use ^ 1, ctl, 21, err, s)) { fine = false; break; }
#pragma unroll 4
                for (int c = 0; c < kEach; ++c) {
                    const uint32_t r = r0 + c * kRowStep, j = key + r;
                    const int page = __shfl_sync(0xffffffffu, pages, r >> 4);
                    cp_async16(va + r * 128 + (((ch & 7) ^ (r & 7)) << 4), source(a.c.v, page, j), page >= 0 && row_live(j));
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                tc::fence_async_smem();
                tc::mbar_arrive(&ctl->k_full[st]);
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                if (mixed) {
#pragma unroll 4
                    for (int c = 0; c < kEach; ++c) {
                        const uint32_t r = r0 + c * kRowStep;
                        uint4* at = reinterpret_cast<uint4*>(vd + (ch >> 3) * kPanel + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                        uint4 x = *at;
                        if (take_out<T>(x)) {
                            *at = x;
                            ctl->poisoned = 1;
                        }
                    }
                }
                tc::fence_async_smem();
                tc::mbar_arrive(&ctl->v_full[st]);
            }
            pages = next_pages;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // a block that gave up: its TMA boxes in flight land long before this
        if (!fine)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(56));
        if (warp == 12) {
            // ------------------------------------------------------ MMA issuer
            constexpr uint32_t kS = idesc<M>(kTile, false), kO = idesc<M>(D, true);
            // the descriptors' high words are constants; their low words hold the address in 16-byte units, which
            // the steps' offsets only add to
            constexpr uint32_t kHigh = (1024u >> 4) | (1u << 14) | (tc::kSwizzle128 << 29);
            const uint32_t q_low = (tc::smem_u32(smem + S::kQ) >> 4) | ((16u >> 4) << 16);
            const uint32_t k_low = (tc::smem_u32(smem + S::kK) >> 4) | ((16u >> 4) << 16);
            const uint32_t v_low = (tc::smem_u32(smem + S::kV) >> 4) | ((static_cast<uint32_t>(kPanel) >> 4) << 16);
            auto scores = [&](int tile, uint32_t i) {
                mma_scores<kSteps>(tmem + tile * kTile, q_low + tile * (S::kTileBytes >> 4),
                                   k_low + (i & 1) * (S::kTileBytes >> 4), kHigh, kS);
                tc::commit_w(&ctl->s_full[tile]);
            };
            // the product of a tile's weights with V, half by half as they come
            auto weighted = [&](int tile, uint32_t i) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!wait(&ctl->p_full[tile][half], i & 1, ctl, 33 + tile, err, s)) return false;
                    tc::fence_after();
                    mma_weighted(tmem + kOCol + tile * D, tmem + tile * kTile + 32 * half,
                                 v_low + (i & 1) * (S::kTileBytes >> 4) + half * (kHalf * 128 >> 4), kHigh, kO, i > 0 || half);
                    tc::commit_w(half ? &ctl->o_done[tile] : &ctl->o_half[tile]);
                }
                return true;
            };
            bool fine = w.tiles == 0 || (wait(&ctl->q_full, 0, ctl, 30, err, s) && wait(&ctl->k_full[0], 0, ctl, 31, err, s));
            if (fine && w.tiles) {
                tc::fence_after();
                scores(0, 0);
                if (two) scores(1, 0);
                tc::commit_w(&ctl->k_empty[0]);
            }
            for (uint32_t i = 0; i < w.tiles && fine; ++i) {
                // K and V are there early as a rule: nothing but the weights is waited for between two products.
                // The next scores overwrite this step's weights; a thread's products run in the order of issue.
                const uint32_t st = i & 1, next = i + 1;
                fine = wait(&ctl->v_full[st], (i >> 1) & 1, ctl, 32, err, s);
                if (fine && next < w.tiles) fine = wait(&ctl->k_full[next & 1], (next >> 1) & 1, ctl, 31, err, s);
                fine = fine && weighted(0, i);
                if (!fine) break;
                if (next < w.tiles) scores(0, next);
                if (two) {
                    fine = weighted(1, i);
                    if (!fine) break;
                }
                tc::commit_w(&ctl->v_empty[st]);
                if (next < w.tiles) {
                    if (two) scores(1, next);
                    tc::commit_w(&ctl->k_empty[next & 1]);
                }
            }
            // every MMA has read its operands before the block ends
            tc::commit_w(&ctl->drain);
            tc::mbar_wait_landing(&ctl->drain, 0);
            tc::fence_before();
        } else if (kCodes && w.tiles) {
            // ------- the largest and smallest value scale of the visible pages
            float top = 0.0f, low = INFINITY;
            for (uint32_t i = threadIdx.x - 13 * 32; i < w.tiles * 8; i += kScaleThreads) {
                const uint32_t j = w.key0(i / 8) + 16 * (i % 8);
                if (j < w.hi_max && (j + 16 > w.lo_min || j < w.sinks_end)) {
                    const int p = a.c.table[static_cast<size_t>(s) * a.c.table_stride + (j >> a.c.page_shift)];
                    if (static_cast<uint32_t>(p) < a.c.pages) {
                        const float x = a.c.v_scale[static_cast<size_t>(p) * a.c.kv_heads + h];
                        if (isfinite(x)) top = fmaxf(top, x), low = fminf(low, x);
                    }
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
            }
            if (lane == 0) ctl->high[warp - 13] = top, ctl->low[warp - 13] = low;
            __syncwarp();
            asm volatile("bar.arrive 1, %0;" ::"n"(kProducers + kScaleThreads) : "memory");
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 12) tc::tmem_free(tmem, 512);
}

// The pool as [pages][kv_heads x page_tokens][head_dim], boxes of one page's
// rows and 64 channels, 128-byte swizzle.
cudaError_t page_map(const CacheArgs& c, void* pool, bool is_bf16, CUtensorMap* map) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    if (!encode) return cudaErrorNotSupported;
    const uint64_t row = c.head_dim * 2ull, rows = static_cast<uint64_t>(c.kv_heads) * c.page_tokens;
    const cuuint64_t dims[3] = {c.head_dim, rows, c.pages};
    const cuuint64_t strides[2] = {row, row * rows};
    const cuuint32_t box[3] = {64, c.page_tokens, 1}, ones[3] = {1, 1, 1};
    const CUresult r = encode(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, pool,
                              dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Which kernel is faster, and whether a block here takes one row tile or two,
// by what each was measured to cost (us, one B200, 16 heads over 8 kv heads,
// 1 to 256 sequences of 64 to 4096 tokens).  Here: a block costs 6.5 (64
// channels) or 9 (128) and 1.25 or 1.6 a tile of 128 keys, half again with
// two row tiles, one block a SM at a time (32 channels cost what 64 do): two
// tiles share what is loaded, one a block fills the SMs where rows are few.
// The other kernel: 6 a call, and 1580, 3100 or (32 channels) 3700 (16 rows x
// 16 keys) a us, 4 of them lost a job.  E.g. 256 sequences, 128 rows a kv
// head, 64 channels: 64 tokens 50 there and 101 here, 1024 tokens 335 there
// and 201 here; 16 sequences of 4096 tokens, 32 rows 40 and 56, 128 rows 109
// and 56; 32 channels: 256 sequences of 640 tokens, 256 rows 355 and 195, 32
// rows of 1024 tokens 83 and 190.
struct Costs {
    double here, there;
    uint32_t rows;  // of a block here
};
Costs costs_of(const CacheAttnArgs& a) {
    const bool wide = a.c.head_dim == 128;
    const double rows = static_cast<double>(a.c.max_new) * a.group, lots = static_cast<double>(a.c.sequences) * a.c.kv_heads;
    const auto blocks_cost = [&](uint32_t block, double factor) {
        const double waves = std::max(1.0, lots * std::ceil(rows / block) / 148);
        const double tiles = std::ceil(static_cast<double>(visible_span(a, block)) / kTile);
        return waves * ((wide ? 9.0 : 6.5) + (wide ? 1.6 : 1.25) * factor * tiles);
    };
    const double one = blocks_cost(kTile, 1.0), both = blocks_cost(2 * kTile, rows > kTile ? 1.5 : 1.0);
    const double there = 6.0 + lots * std::ceil(rows / 16) * (std::ceil(static_cast<double>(visible_span(a, 16)) / 16) + 4) /
                                   (wide ? 1580.0 : a.c.head_dim == 64 ? 3100.0 : 3700.0);
    return {std::min(one, both), there, one < both ? kTile : 2u * kTile};
}

template <typename T, int D, bool kCodes, int kKeys>
cudaError_t launch(const CacheAttnArgs& a, uint32_t block_rows, cudaStream_t s) {
    using S = Shape<D, kCodes>;
    static_assert(S::kBytes <= 227 * 1024, "shared memory");
    const uint32_t most = kKeys == kPrefixKeys ? a.max_tokens : a.c.max_new, row_blocks = (most * a.group + block_rows - 1) / block_rows;
    const uint32_t lots = kKeys == kPrefixKeys ? a.group_count * a.splits : a.c.sequences;
    auto* kernel = cache_attn_tc_kernel<T, D, kCodes, kKeys>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    CUtensorMap k_map{}, v_map{};
    if constexpr (!kCodes) {
        if (e == cudaSuccess) e = page_map(a.c, a.c.k, std::is_same_v<T, bf16>, &k_map);
        if (e == cudaSuccess) e = page_map(a.c, a.c.v, std::is_same_v<T, bf16>, &v_map);
    }
    if (e != cudaSuccess) return e;
    kernel<<<row_blocks * lots * a.c.kv_heads, kThreads, S::kBytes, s>>>(a, k_map, v_map, block_rows);
    return cudaGetLastError();
}

template <int kKeys, typename T, bool kCodes> cudaError_t by_dim(const CacheAttnArgs& a, uint32_t rows, cudaStream_t s) {
    return a.c.head_dim == 128 ? launch<T, 128, kCodes, kKeys>(a, rows, s) : launch<T, 64, kCodes, kKeys>(a, rows, s);
}
template <int kKeys> cudaError_t by_type(const CacheAttnArgs& a, uint32_t rows, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? by_dim<kKeys, bf16, true>(a, rows, s) : by_dim<kKeys, __half, true>(a, rows, s);
    return dtype == LWM_DTYPE_BF16 ? by_dim<kKeys, bf16, false>(a, rows, s) : by_dim<kKeys, __half, false>(a, rows, s);
}

}  // namespace

bool cache_attention_many_rows(const CacheAttnArgs& a) {
    const Costs c = costs_of(a);
    return c.here < c.there;
}

double cache_attention_cost(const CacheAttnArgs& a) {
    const Costs c = costs_of(a);
    return std::min(c.here, c.there);
}

cudaError_t launch_cache_attention_tc(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s) {
    return by_type<kAllKeys>(a, costs_of(a).rows, dtype, storage, s);
}

// The prefix's blocks by the same costs: row tiles a block, and parts of the
// keys, each of which writes 32-bit results that the tails' kernel reads.
// What bounds the prefix (one B200): with few keys the chain of a block's steps and its start (1024 candidates of 16
// heads behind 1568 tokens: 26 us, tensor pipe 15 %; its flops alone 3.4), with many the chain of scores, softmax and
// product as in a sequence's own attention (64 candidates of 4 tokens and 32 heads behind 65536: 208 us, pipe 53 %, 106
// at its peak).  8-bit codes: 16 groups of 64 with a window of 4096 75 us, expanding the codes beside that chain.  A part
// more costs its results in 32 bits, written here and read by the tails; the choice made here was the quickest
// of all (block, parts) pairs in the cases tried.
SharedPlan shared_plan(const CacheAttnArgs& a, uint32_t most_splits) {
    const bool wide = a.c.head_dim == 128;
    const uint64_t rows = static_cast<uint64_t>(a.max_tokens) * a.group;
    uint64_t span = a.c.max_length ? a.c.max_length : static_cast<uint64_t>(a.c.table_stride) << a.c.page_shift;
    if (a.window)  // rows of several lengths: as if they were as far apart as their tails allow
        span = std::min(span, static_cast<uint64_t>(a.window) * a.frame + a.sinks + (a.max_tail ? a.max_tail : 128));
    const uint64_t tiles = std::max<uint64_t>(1, (span + kTile - 1) / kTile);
    const double part = static_cast<double>(a.c.tokens) * a.heads * a.c.head_dim * 8 / 4e6;  // written and read, us
    SharedPlan best;
    for (uint32_t block = kTile; block <= 2 * kTile; block += kTile)
        for (uint32_t splits = 1; splits <= std::min<uint64_t>(std::min<uint64_t>(tiles, most_splits), 64); ++splits) {
            const double blocks = static_cast<double>(a.group_count) * a.c.kv_heads * ((rows + block - 1) / block) * splits;
            const double factor = block > kTile && rows > kTile ? 1.5 : 1.0, steps = static_cast<double>((tiles + splits - 1) / splits);
            const double cost = std::ceil(blocks / 148) * ((wide ? 9.0 : 6.5) + (wide ? 1.6 : 1.25) * factor * steps) + part * splits;
            if (best.cost == 0.0 || cost < best.cost) best = {block, splits, cost};
        }
    return best;
}

cudaError_t launch_cache_attention_prefix(const CacheAttnArgs& a, uint32_t block_rows, int dtype, int storage, cudaStream_t s) {
    return by_type<kPrefixKeys>(a, block_rows, dtype, storage, s);
}

}  // namespace lwm
