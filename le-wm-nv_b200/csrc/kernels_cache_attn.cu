// kernels_cache_attn.cu — attention over the paged cache for few query rows
// a kv head (lwm_cache_attention_device).
//
// A job is (sequence, kv head, 8 or 16 query rows = tokens x heads of the
// group).  A warp walks 16-key units: scores S^T = K Q^T on mma.sync m16n8k16
// (the keys are the wide side: a single token's few rows fill half of a
// 16-row tile at best), a running maximum and sum in 32 bits, O^T += V^T P^T,
// P turned over by movmatrix.  The units of a job are dealt to the four warps
// of a block and, for long contexts, to the blocks of a cluster; their
// (maximum, sum, O) are joined in shared memory and over distributed shared
// memory, so a call needs no workspace and no second kernel and its sums have
// one order.  Where contexts are short and jobs many, a warp has some heads of a
// sequence alone, their units one stream through its ring: the sequence's
// lengths and pages are looked up once and no head waits for its first load.
//
// Bound: memory (each K and V byte is used by at most 16 rows, 32 flops a
// byte).  Every warp keeps its own ring of units in flight with cp.async, so
// no barrier stands between a load and its use.  Measured (one B200, DRAM
// bytes as ncu counts them): four sequences of up to 65536 tokens, 8 kv heads
// of 128 channels, bf16: 910 MB in 146 us, 6.2 TB/s; 48 sequences, windows
// of 4096 tokens in 8-bit codes: 178 MB in 42 us, 4.2 TB/s, half of the issue
// slots in use for the codes; 1024 sequences of 34 tokens, 16 heads of 64
// channels: 50 MB in 33 us, bound by instructions and by the chain lengths ->
// page -> keys -> scores of a sequence, not by memory; one sequence of 37
// tokens: 5.9 us, a launch and that chain.  Left: holding the scores of all
// keys of a short context before one maximum (73 us against 44, both with the
// events around them: the unrolled steps miss the instruction cache).
//
// Tails (kTailKeys): what lies behind a prefix that a group shares, joined with
// the prefix's parts, which another kernel leaves in the workspace; it may
// start beside that one and waits for it only before the join, of the first head
// where a warp has several (64 candidates of 4 tokens with tails up to 64 tokens,
// 32 heads over 8 of 128, a head a block: 50 us, most of them beside a prefix of
// 208).
//
// 8-bit codes become halves in registers: e4m3 is exact in fp16.  The
// contraction's order is free, so a thread's 16 bytes of a key are the four
// channels each of four k-steps, and Q is loaded in the same order; V's
// bytes are interleaved by key pairs with byte permutes.  The key scale
// multiplies the scores.  A value scale 2^e f (f in [1, 2)) goes into the
// weight before it is rounded: a row keeps, beside its maximum m and sum, the
// power of two E of its largest weighted scale, and its weights for the
// product are exp2(score - m + e - E) f, at most 2^9 (2^14 as rounded, see
// kLift) and near one for the page that counts most, whatever the scales of
// the others.  So a weight has two exponentials, one for the sum and one for
// the product (one, times the row's power of two, measured the same or slower;
// the ratio of the scales on the finished weight, 0 to 8 % faster, loses what
// lies 2^14 below the largest scale).  bf16 queries are brought to fp16 by a
// power of two a row, exactly down to 2^-17 of the row's largest.
#include <cooperative_groups.h>

#include "lwm_blocks.cuh"
#include "lwm_cache_attn.cuh"

namespace lwm {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kUnit = 16;    // keys a step

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    // a dead row's 16 bytes are filled with zeros, its address is not read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
// An 8 x 8 tile of 16-bit values turned over.
__device__ __forceinline__ uint32_t turn_over(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <typename M>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(M) == 2 && std::is_same_v<M, bf16>)
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

// Byte offset of 16-byte chunk `c` of row `r` in a unit: 128-byte lines whose
// chunks are permuted so that ldmatrix (16 bits: 8 rows of one chunk) and the
// code reads (8 bits: K 16 bytes of 2 rows a phase, V 32 bytes of rows 0, 2,
// 4, 6) touch every bank once.
template <int D, bool kCodes> __device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c) {
    constexpr uint32_t kChunks = kCodes ? D / 16 : D / 8;  // of a row
    if constexpr (kChunks >= 16) {
        return r * kChunks * 16 + ((c ^ (r & 7)) << 4);
    } else {
        constexpr uint32_t kRows = 8 / kChunks;            // rows of a line
        const uint32_t line = r / kRows, at = (r % kRows) * kChunks + c;
        uint32_t x;
        if constexpr (!kCodes) x = kRows == 1 ? (r & 7) : (line & 3);
        else if constexpr (kRows == 1) x = (((r >> 1) & 3) << 1) ^ ((r & 1) << 2);
        else if constexpr (kRows == 2) x = (line & 3) << 1;
        else x = (line & 1) << 1;
        return line * 128 + ((at ^ x) << 4);
    }
}

// Value (key, channel) of a unit in shared memory.
template <typename T, int D, bool kCodes>
__device__ __forceinline__ float value_at(const uint8_t* unit, uint32_t key, uint32_t ch) {
    if constexpr (kCodes) {
        const uint8_t code = unit[chunk_at<D, true>(key, ch >> 4) + (ch & 15)];
        const uint32_t h = f16x2_from_e4m3x2(code);
        return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
    } else {
        return static_cast<float>(*reinterpret_cast<const T*>(unit + chunk_at<D, false>(key, ch >> 3) + (ch & 7) * 2));
    }
}

// kRows: query rows of a job, 8 or 16.
template <int D, bool kCodes, int kRows, bool kShared> struct Shape {
    static constexpr int kUnitBytes = kUnit * D * (kCodes ? 1 : 2);  // of K, and of V
    static constexpr int kStages = 3;
    static constexpr int kWarpBytes = kStages * 2 * kUnitBytes;
    static constexpr int kPitch = D + 4;                             // floats of a row of O in shared memory
    static constexpr int kPartFloats = kRows * kPitch;               // a warp's O
    static constexpr int kPart = kPartFloats + (kCodes ? 3 : 2) * kRows;  // maxima, sums (and powers of two) too
    static constexpr int kPartBytes = kShared ? kPart * 4 : 0;
    static constexpr int kRings = kWarps * (kWarpBytes > kPartBytes ? kWarpBytes : kPartBytes);
    // and the units' pages and scales; alone, a warp's output rows
    static constexpr int kBytes = kRings + kWarps * kStages * 16 + (kShared ? 0 : kWarps * kRows * D * 2);
    // blocks a SM, by shared memory and registers
    static constexpr int kBySmem = 220 * 1024 / (kBytes + 1024), kByRegs = kRows == 8 ? (D == 128 ? 4 : 5) : (D == 128 ? 3 : 4);
    static constexpr int kBlocks = kBySmem < kByRegs ? kBySmem : kByRegs;
};

// 2^e of a whole number in [-126, 127] (any other: the nearer end).
__device__ __forceinline__ float power_of_two(float e) {
    return __uint_as_float(static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(e, -126.0f), 127.0f)) + 127) << 23);
}

// A unit in flight: its page (-1: none) and, of codes, the page's scales.
struct UnitNote {
    int page;
    float k_scale, v_scale, pad;
};

// Visible keys of one row: [0, first) and [lo, hi).
struct RowRange { uint32_t lo, hi, first; };

template <typename T, int D, bool kCodes, int kRows, bool kShared, int kKeys>
__global__ void __launch_bounds__(kThreads, Shape<D, kCodes, kRows, kShared>::kBlocks)
    cache_attn_kernel(const __grid_constant__ CacheAttnArgs a, uint32_t tiles, uint32_t split) {
    using M = std::conditional_t<kCodes, __half, T>;  // the operands' type
    using S = Shape<D, kCodes, kRows, kShared>;
    constexpr int kSteps = D / 16, kQ = kRows / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // job: four warps (and `split` blocks) share one head's, or a warp has `split` heads' (the last: fewer)
    const uint32_t rank = kShared ? blockIdx.x % split : 0;
    const uint32_t job = kShared ? blockIdx.x / split : blockIdx.x * kWarps + warp;
    const uint32_t hs = a.tile_div.div(job), tile = job - hs * tiles, s = a.kv_div.div(hs);
    const uint32_t h0 = (hs - s * a.kv_div.d) * (kShared ? 1 : split);
    const uint32_t h_end = kShared ? h0 + 1 : min(h0 + split, a.c.kv_heads);
    // a short table's row comes along with the lengths
    int entry = -1;
    const bool small_table = !kShared && a.c.table_stride <= 32;
    SeqView v;
    if (s < a.c.sequences) {
        if (small_table && lane < a.c.table_stride)
            entry = a.c.table[static_cast<size_t>(s) * a.c.table_stride + lane];
        v = sequence(a.c, s, false, h0 == 0 && tile == 0 && rank == 0 && lane == 0);
    }
    // A tail: what lies behind the prefix that the sequence's group shares (no group: everything).
    constexpr bool kTail = kKeys == kTailKeys;
    uint32_t shared = 0;
    bool joined = false;  // with the prefix's parts
    if constexpr (kTail) {
        if (v.ok && a.group_count && static_cast<int>(s) >= a.groups[0]) {
            const uint32_t g = last_at_most(a.groups, 0, a.group_count, static_cast<int>(s));
            if (static_cast<int>(s) < a.groups[g + 1]) {
                const GroupView group = group_view(a, g, false);
                // (the prefix's rows are the group's)
                joined = group.ok && v.start >= group.start && v.start + v.n <= group.start + group.n;
                shared = group.shared;
                const bool reaches = joined && shared && v.n && static_cast<uint64_t>(v.n) + shared > v.length;
                if (reaches && h0 == 0 && tile == 0 && rank == 0 && lane == 0) cache_report(a.c.err, kCacheErrShared, s, shared);
                if (!joined || reaches) v.n = 0;
            }
        }
    }
    const uint32_t rows = v.n * a.group, row0 = tile * kRows;
    const bool live = row0 < rows;
    if (!live && (!kShared || split == 1)) {  // uniform over what waits together
        // (this grid is not done before the prefix's is)
        if constexpr (kTail) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }

    // the keys that this thread's queries 8 n + 2 t + e see, and the tile's union
    RowRange rr[kQ][2];
    uint32_t lo_min = 0, lo_max = 0, hi_min = 0, hi_max = 0;
    if (live) {
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t R = row0 + 8 * n + 2 * t + e;
                rr[n][e] = {0, 0, 0};
                if (R < rows) {
                    const VisibleRange vr = visible(a, v, a.group_div.div(R));
                    rr[n][e] = {kTail ? max(vr.lo, shared) : vr.lo, vr.hi, vr.first};
                }
            }
        const uint32_t tok0 = a.group_div.div(row0), tok1 = a.group_div.div(min(row0 + kRows - 1, rows - 1));
        const VisibleRange r0 = visible(a, v, tok0), r1 = visible(a, v, tok1);
        lo_min = r0.lo, hi_min = r0.hi;
        lo_max = r1.lo, hi_max = r1.hi;
        if (kTail) lo_min = max(lo_min, shared), lo_max = max(lo_max, shared);
    }
    const bool mixed = lo_min != lo_max || hi_min != hi_max;  // rows that differ in what they see
    const uint32_t sinks_end = min(a.sinks, min(lo_min, hi_max));
    const uint32_t sink0 = kTail ? min(shared, sinks_end) / kUnit : 0;  // (a tail's first unit may hold keys of the prefix)
    const uint32_t sink_units = kTail && sinks_end <= shared ? 0 : (sinks_end + kUnit - 1) / kUnit - sink0;
    const uint32_t win_unit = max(lo_min / kUnit, sink_units ? sink0 + sink_units : 0);
    const uint32_t win_units = hi_max > win_unit * kUnit ? (hi_max - win_unit * kUnit + kUnit - 1) / kUnit : 0;
    const uint32_t units = sink_units + win_units;
    // this warp's units: walk, walk + step, ... below end
    const uint32_t per = kShared ? (units + split - 1) / split : units;
    const uint32_t end = kShared ? min(units, (rank + 1) * per) : units;
    const uint32_t walk = kShared ? rank * per + warp : 0;
    const uint32_t step = kShared ? kWarps : 1;

    uint8_t* ring = smem + warp * S::kWarpBytes;
    const uint32_t ring_a = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    const uint32_t count = walk < end ? (end - walk + step - 1) / step : 0;
    auto key_of = [&](uint32_t i) {
        const uint32_t u = walk + i * step;
        return (u < sink_units ? u + sink0 : u - sink_units + win_unit) * kUnit;
    };
    // page of the warp's unit i: from the table's row, or looked up 32 units at a time
    int pages_ahead = -1;
    auto page_at = [&](uint32_t i) {
        if (small_table) {
            const int p = __shfl_sync(0xffffffffu, entry, key_of(i) >> a.c.page_shift);
            if (static_cast<uint32_t>(p) < a.c.pages) return p;
            if (lane == 0) cache_report(a.c.err, kCacheErrPage, s, p);
            return -1;
        }
        if ((i & 31) == 0) pages_ahead = i + lane < count ? page_of(a.c, s, key_of(i + lane) >> a.c.page_shift) : -1;
        return __shfl_sync(0xffffffffu, pages_ahead, i & 31);
    };
    UnitNote* notes = reinterpret_cast<UnitNote*>(smem + S::kRings) + warp * S::kStages;
    auto load = [&](uint32_t h, uint32_t i, uint32_t slot) {
        const int page = page_at(i);
        const uint32_t key = key_of(i);
        constexpr int kRowChunks = S::kUnitBytes / kUnit / 16;
        const size_t base = pool_at(a.c, page < 0 ? 0 : page, h, key & (a.c.page_tokens - 1)) * (kCodes ? 1 : 2);
        const uint32_t dst = ring_a + slot * 2 * S::kUnitBytes;
        if (lane == 0) notes[slot].page = page;
        if (kCodes && lane < 2 && page >= 0) {
            const float* scale = (lane ? a.c.v_scale : a.c.k_scale) + static_cast<size_t>(page) * a.c.kv_heads + h;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                             static_cast<uint32_t>(__cvta_generic_to_shared(lane ? &notes[slot].v_scale : &notes[slot].k_scale))),
                         "l"(scale)
                         : "memory");
        }
        const uint8_t* kp = static_cast<const uint8_t*>(a.c.k) + base + lane * 16;
        const uint8_t* vp = static_cast<const uint8_t*>(a.c.v) + base + lane * 16;
        // rows that no query sees come as zeros
        const bool all = page >= 0 && key + kUnit <= hi_max && (key >= lo_min || (key + kUnit <= sinks_end && key >= shared));
#pragma unroll
        for (int c = 0; c < kUnit * kRowChunks / 32; ++c) {
            const uint32_t x = c * 32 + lane, r = x / kRowChunks, ch = x % kRowChunks;
            const uint32_t j = key + r;
            const bool ok = all || (page >= 0 && j < hi_max && (j >= lo_min || (j < sinks_end && j >= shared)));
            cp_async16(dst + chunk_at<D, kCodes>(r, ch), kp + c * 512, ok);
            cp_async16(dst + S::kUnitBytes + chunk_at<D, kCodes>(r, ch), vp + c * 512, ok);
        }
    };
    // the next unit of the stream: of this head, then of the next one
    uint32_t load_h = count ? h0 : h_end, load_i = 0;
    auto load_next = [&](uint32_t slot) {
        if (load_h < h_end) {
            load(load_h, load_i, slot);
            if (++load_i == count) load_i = 0, ++load_h;
        }
        cp_commit();
    };
#pragma unroll 1
    for (uint32_t i = 0; i < S::kStages - 1; ++i) load_next(i);

    // queries 8 n + g as they lie, in the order of the contraction
    auto fetch_q = [&](uint32_t h, uint32_t(&raw)[kQ][kSteps][2]) {
#pragma unroll
        for (int n = 0; n < kQ; ++n) {
            const uint32_t R = row0 + 8 * n + g;
            const T* qr = nullptr;
            if (live && R < rows) {
                const uint32_t tok = a.group_div.div(R);
                qr = static_cast<const T*>(a.q) + (v.start + tok) * a.q_ts + (h * a.group + (R - tok * a.group)) * a.q_hs;
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                if constexpr (!kCodes) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        raw[n][k][i] = qr ? *reinterpret_cast<const uint32_t*>(qr + 16 * k + 8 * i + 2 * t) : 0u;
                } else {
                    constexpr int kRun = D >= 64 ? 16 : 8;  // channels a thread reads of each 4 * kRun
                    const int ch = (k / (kRun / 4)) * 4 * kRun + t * kRun + (k % (kRun / 4)) * 4;
                    uint2 w = make_uint2(0, 0);
                    if (qr) w = *reinterpret_cast<const uint2*>(qr + ch);
                    raw[n][k][0] = w.x;
                    raw[n][k][1] = w.y;
                }
            }
        }
    };
    uint32_t raw[kQ][kSteps][2];
    fetch_q(h0, raw);
    uint32_t slot = 0;
    auto channel = [&](int d, int half) {  // of row g + 8 half of channel tile d
        return kCodes ? 32 * (d >> 1) + 4 * g + 2 * (d & 1) + half : 16 * d + 8 * half + g;
    };

#pragma unroll 1
    for (uint32_t h = h0; h < h_end; ++h) {
    uint32_t q[kQ][kSteps][2];
    float row_mul[kQ][2];  // of queries 8 n + 2 t + e
#pragma unroll
    for (int n = 0; n < kQ; ++n) {
        row_mul[n][0] = row_mul[n][1] = a.scale_log2;
        if constexpr (!(kCodes && std::is_same_v<T, bf16>)) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) q[n][k][0] = raw[n][k][0], q[n][k][1] = raw[n][k][1];
        } else {
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(raw[n][k][i] << 16)),
                                             fabsf(__uint_as_float(raw[n][k][i] & 0xffff0000u))));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
            if (amax == 0.0f || e == 128) e = 0;
            e = min(max(e, -126), 126);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
            for (int i = 0; i < 2; ++i) row_mul[n][i] *= __shfl_sync(0xffffffffu, up, (2 * t + i) * 4);
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    q[n][k][i] = pack2(__uint_as_float(raw[n][k][i] << 16) * down,
                                       __uint_as_float(raw[n][k][i] & 0xffff0000u) * down, __half{});
        }
    }
    if (!kShared && h + 1 < h_end) fetch_q(h + 1, raw);

    // O^T: tile n of queries, tile d of channels; element i is query 2 t + (i & 1), channel of row g + 8 (i >> 1)
    float o[kQ][kSteps][4];
    float m[kQ][2], l[kQ][2];
#pragma unroll
    for (int n = 0; n < kQ; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int d = 0; d < kSteps; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][d][e] = 0.0f;
    }
    float vx[kQ][2];  // 8 bits: O is in units of 2^vx (a whole number) times the weights' 2^m
#pragma unroll
    for (int n = 0; n < kQ; ++n) vx[n][0] = vx[n][1] = INFINITY;  // (no key yet)

    // (not unrolled over the ring: copies of the body missed the instruction cache)
#pragma unroll 1
    for (uint32_t i = 0; i < count; ++i) {
        cp_wait<S::kStages - 2>();
        __syncwarp();
        const int page = notes[slot].page;
        const uint32_t key = key_of(i);
        const uint32_t k_at = ring_a + slot * 2 * S::kUnitBytes, v_at = k_at + S::kUnitBytes;
        float k_scale = 1.0f, v_exp = 0.0f, v_frac = 1.0f;
        if constexpr (kCodes) {
            k_scale = notes[slot].k_scale;
            float v_scale = page < 0 ? 1.0f : notes[slot].v_scale;
            if (!isfinite(v_scale)) v_scale = __int_as_float(0x7fc00000);
            const int e = min(max(static_cast<int>((__float_as_uint(v_scale) >> 23) & 255) - 127, -126), 126);
            v_exp = static_cast<float>(e);
            v_frac = v_scale * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        }
        // scores: element e is key g + 8 (e >> 1), query 2 t + (e & 1); two chains of products
        float sc[kQ][4], odd[kQ][4];
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = odd[n][e] = 0.0f;
        if constexpr (!kCodes) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];  // keys 0-7 and 8-15 of channels 0-7, then of channels 8-15
                ldsm4(b, k_at + chunk_at<D, false>(lane & 15, 2 * k + (lane >> 4)));
#pragma unroll
                for (int n = 0; n < kQ; ++n) mma<M>(k & 1 ? odd[n] : sc[n], b, q[n][k][0], q[n][k][1]);
            }
        } else {
            uint32_t w[2][kSteps];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if constexpr (D == 32) {
                    const uint32_t at = k_at + chunk_at<D, true>(g + 8 * r, t >> 1) + (t & 1) * 8;
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[r][0]), "=r"(w[r][1]) : "r"(at) : "memory");
                } else {
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {
                        const uint32_t at = k_at + chunk_at<D, true>(g + 8 * r, 4 * c + t);
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(w[r][4 * c]), "=r"(w[r][4 * c + 1]), "=r"(w[r][4 * c + 2]), "=r"(w[r][4 * c + 3])
                                     : "r"(at)
                                     : "memory");
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const uint32_t b[4] = {f16x2_from_e4m3x2(w[0][k]), f16x2_from_e4m3x2(w[1][k]),
                                       f16x2_from_e4m3x2(w[0][k] >> 16), f16x2_from_e4m3x2(w[1][k] >> 16)};
#pragma unroll
                for (int n = 0; n < kQ; ++n) mma<M>(k & 1 ? odd[n] : sc[n], b, q[n][k][0], q[n][k][1]);
            }
        }
        // in units of log2, masked where a query does not see the key
        const bool whole = page >= 0 && (key >= lo_max || (key + kUnit <= sinks_end && key >= shared)) && key + kUnit <= hi_min;
        auto sees = [&](int n, int e) {
            const uint32_t j = key + g + 8 * (e >> 1);
            return page >= 0 && j < rr[n][e & 1].hi && (j >= rr[n][e & 1].lo || (j < rr[n][e & 1].first && j >= shared));
        };
        bool above = false;
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[n][e] = (sc[n][e] + odd[n][e]) * (k_scale * row_mul[n][e & 1]);
                if (!whole && !sees(n, e)) sc[n][e] = -INFINITY;
                const float lift = kCodes ? fmaxf(v_exp - vx[n][e & 1], 0.0f) : 0.0f;
                above |= sc[n][e] > m[n][e & 1] + (kRaise - lift);
            }
        // the maximum (of the scores, and of them with their scales) moves
        // only when a score passes it by kRaise: until then exp2(score - m),
        // scaled or not, stays below 2^kRaise
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int n = 0; n < kQ; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(sc[n][e], sc[n][e + 2]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float here = x;  // this unit's largest
                    x = fmaxf(x, m[n][e]);
                    const bool first = m[n][e] == -INFINITY;
                    const float down = first ? 0.0f : exp2_fast(m[n][e] - x);
                    float o_down = down;
                    if constexpr (kCodes) {
                        // (m - x and the powers of two are differences of near numbers, so nothing is lost far from zero)
                        const float kept = first ? -INFINITY : (m[n][e] - x) + vx[n][e];
                        const float to = x == -INFINITY ? INFINITY : ceilf(fmaxf(kept, (here - x) + v_exp));
                        o_down = first ? 0.0f : exp2_fast(kept - to);
                        vx[n][e] = to;
                    }
                    m[n][e] = x;
                    if (i == 0) continue;
                    l[n][e] *= down;
#pragma unroll
                    for (int d = 0; d < kSteps; ++d) {
                        o[n][d][e] *= o_down;
                        o[n][d][e + 2] *= o_down;
                    }
                }
        }
        // P in the operands' type: 2^-9 (bf16) or 2^-12 (fp16) of itself, no
        // more than rounding the output costs.  Halves end at 2^-25, so theirs
        // are 2^kLift times as large (below 2^15): what a weight can lose, 2^-32
        // (codes 2^-29) of the row's largest, stays below that rounding in sums
        // of 2^18 keys too
        constexpr float kLift = !std::is_same_v<M, __half> ? 0.0f : kCodes ? 5.0f : 7.0f;
        float p[kQ][4];
        uint32_t pb[kQ][2];
#pragma unroll
        for (int n = 0; n < kQ; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float over = sc[n][e] - (m[n][e & 1] == -INFINITY ? 0.0f : m[n][e & 1] - kLift);
                p[n][e] = exp2_fast(over);
                l[n][e & 1] += p[n][e];
                if constexpr (kCodes) p[n][e] = exp2_fast(over + (v_exp - vx[n][e & 1])) * v_frac;
            }
            pb[n][0] = turn_over(pack2(p[n][0], p[n][1], M{}));
            pb[n][1] = turn_over(pack2(p[n][2], p[n][3], M{}));
        }
        // a key that some rows of the tile see and others do not: zero
        // times an infinity or NaN would reach the others
        bool poison = false;
        if (!whole && mixed) {
            constexpr int kVecs = S::kUnitBytes / 16 / 32;
#pragma unroll
            for (int c = 0; c < kVecs; ++c) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(v_at + (c * 32 + lane) * 16)
                             : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) poison |= any_not_finite<T, kCodes>(w[e]);
            }
            poison |= kCodes && v_frac != v_frac;
            poison = __any_sync(0xffffffffu, poison);
        }
        if (!poison) {
            if constexpr (!kCodes) {
#pragma unroll
                for (int d = 0; d < kSteps; ++d) {
                    uint32_t b[4];  // channels 0-7 and 8-15 of keys 0-7, then of keys 8-15
                    ldsm4t(b, v_at + chunk_at<D, false>((lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1)));
#pragma unroll
                    for (int n = 0; n < kQ; ++n) mma<M>(o[n][d], b, pb[n][0], pb[n][1]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t w[4];  // channels 32 c + 4 g .. + 3 of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t r = 2 * t + (e & 1) + 8 * (e >> 1);
                        const uint32_t at = v_at + chunk_at<D, true>(r, 2 * c + (g >> 2)) + (g & 3) * 4;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[e]) : "r"(at) : "memory");
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t sel = j == 0 ? 0x5140 : 0x7362;
                        const uint32_t lo2 = __byte_perm(w[0], w[1], sel), hi2 = __byte_perm(w[2], w[3], sel);
                        const uint32_t b[4] = {f16x2_from_e4m3x2(lo2), f16x2_from_e4m3x2(lo2 >> 16),
                                               f16x2_from_e4m3x2(hi2), f16x2_from_e4m3x2(hi2 >> 16)};
#pragma unroll
                        for (int n = 0; n < kQ; ++n) mma<M>(o[n][2 * c + j], b, pb[n][0], pb[n][1]);
                    }
                }
            }
        } else {
            // one key after another, for the rows that see it
#pragma unroll 1
            for (int r = 0; r < kUnit; ++r) {
                const uint32_t j = key + r;
#pragma unroll
                for (int n = 0; n < kQ; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float low = __shfl_sync(0xffffffffu, p[n][e], (r & 7) * 4 + t);
                        const float high = __shfl_sync(0xffffffffu, p[n][e + 2], (r & 7) * 4 + t);
                        const float pk = r < 8 ? low : high;
                        if (!(page >= 0 && j < rr[n][e].hi && (j >= rr[n][e].lo || (j < rr[n][e].first && j >= shared)))) continue;
#pragma unroll
                        for (int d = 0; d < kSteps; ++d)
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                o[n][d][2 * x + e] += pk * value_at<T, D, kCodes>(ring + slot * 2 * S::kUnitBytes + S::kUnitBytes,
                                                                                  r, channel(d, x));
                    }
            }
        }
        __syncwarp();
        // this slot's unit is done: the one kStages - 1 ahead goes to the slot before it
        load_next(slot == 0 ? S::kStages - 1 : slot - 1);
        if (++slot == S::kStages) slot = 0;
    }
#pragma unroll
    for (int n = 0; n < kQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
        }

    constexpr float kUnitLog = !std::is_same_v<M, __half> ? 0.0f : kCodes ? 5.0f : 7.0f;  // (the weights' kLift)
    if constexpr (kTail) asm volatile("griddepcontrol.wait;" ::: "memory");  // the prefix's parts are there
    // a row's share of each part: the sum of weights behind it, relative to the whole (`tail` its own log2, and its
    // share when it returns); parts are read one after another
    auto part_row = [&](uint32_t R, uint32_t hh) {
        const uint32_t tok = a.group_div.div(R);
        return (static_cast<size_t>(v.start) + tok) * a.heads + hh * a.group + (R - tok * a.group);
    };
    const size_t part_rows = static_cast<size_t>(a.c.tokens) * a.heads;
    auto join = [&](size_t row, float& tail, float& top) {
        top = tail;
        bool nan = tail != tail;
        if (joined)
            for (uint32_t x = 0; x < a.splits; ++x) {
                const float log = a.part_log[x * part_rows + row];
                top = fmaxf(top, log);
                nan |= log != log;
            }
        if (top == -INFINITY && !nan) {
            tail = 0.0f;
            return 0.0f;
        }
        if (nan) top = __int_as_float(0x7fc00000);
        float sum = tail = exp2_fast(tail - top);
        if (joined)
            for (uint32_t x = 0; x < a.splits; ++x) sum += exp2_fast(a.part_log[x * part_rows + row] - top);
        const float inv = 1.0f / sum;
        tail *= inv;
        return inv;
    };

    if constexpr (!kShared) {
        // the warp's own rows: through shared memory to whole 16-byte stores
        T* part = reinterpret_cast<T*>(smem + S::kRings + kWarps * S::kStages * 16 + warp * kRows * D * 2);
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool none = l[n][e] == 0.0f;  // nothing weighs, not even against infinities in O
                const float inv = none ? 0.0f : 1.0f / l[n][e];
                const float unit = kCodes ? power_of_two(vx[n][e]) : 1.0f;
                if constexpr (kTail) {
                    const uint32_t R = row0 + 8 * n + 2 * t + e;
                    float tail = none ? -INFINITY : m[n][e] - kUnitLog + log2f(l[n][e]), top = -INFINITY, all = 0.0f;
                    const size_t row = R < rows ? part_row(R, h) : 0;
                    if (R < rows) all = join(row, tail, top);
#pragma unroll
                    for (int d = 0; d < kSteps; ++d)
#pragma unroll
                        for (int x = 0; x < 2; ++x) o[n][d][2 * x + e] = none ? 0.0f : o[n][d][2 * x + e] * inv * unit * tail;
                    if (R < rows && joined) {
                        for (uint32_t y = 0; y < a.splits; ++y) {
                            const float w = all == 0.0f ? 0.0f : exp2_fast(a.part_log[y * part_rows + row] - top) * all;
                            if (w == 0.0f) continue;
                            const float* from = a.part_out + (y * part_rows + row) * D;
#pragma unroll
                            for (int d = 0; d < kSteps; ++d)
#pragma unroll
                                for (int x = 0; x < 2; ++x) o[n][d][2 * x + e] += w * from[channel(d, x)];
                        }
                    }
#pragma unroll
                    for (int d = 0; d < kSteps; ++d)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            part[(8 * n + 2 * t + e) * D + channel(d, x)] = static_cast<T>(o[n][d][2 * x + e]);
                } else {
#pragma unroll
                for (int d = 0; d < kSteps; ++d)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        part[(8 * n + 2 * t + e) * D + channel(d, x)] = static_cast<T>(none ? 0.0f : o[n][d][2 * x + e] * inv * unit);
                }
            }
        __syncwarp();
        for (int x = lane; x < kRows * D / 8; x += 32) {
            const uint32_t R = row0 + x / (D / 8), c8 = 8 * (x % (D / 8));
            if (R >= rows) continue;
            const uint32_t tok = a.group_div.div(R), head = h * a.group + (R - tok * a.group);
            store8(static_cast<T*>(a.out) + (v.start + tok) * a.o_ts + head * a.o_hs + c8,
                   *reinterpret_cast<const Vec8<T>*>(part + x * 8));
        }
        __syncwarp();  // the next head's rows go there
    } else {
        // join the warps, then the blocks of the cluster
        cp_wait<0>();
        __syncthreads();  // every ring is done with
        float* parts = reinterpret_cast<float*>(smem);
        constexpr int kPart = S::kPart;
        float* mine = parts + warp * kPart;
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * t + e;
#pragma unroll
                for (int d = 0; d < kSteps; ++d)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        mine[r * S::kPitch + channel(d, x)] = o[n][d][2 * x + e];
                if (g == 0) {
                    mine[S::kPartFloats + r] = m[n][e];
                    mine[S::kPartFloats + kRows + r] = l[n][e];
                    if constexpr (kCodes) mine[S::kPartFloats + 2 * kRows + r] = vx[n][e];
                }
            }
        if (split > 1) cg::this_cluster().sync();
        else __syncthreads();
        if (live) {
            // this block finishes every split-th vector of 4 channels
            const uint32_t stride = split * kThreads;
            for (uint32_t x = rank * kThreads + threadIdx.x; x < kRows * D / 4; x += stride) {
                const uint32_t r = x / (D / 4), c4 = 4 * (x % (D / 4)), R = row0 + r;
                if (R >= rows) continue;
                float top = -INFINITY;
                for (uint32_t b = 0; b < split; ++b) {
                    const float* p = split > 1 ? cg::this_cluster().map_shared_rank(parts, b) : parts;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, p[w * kPart + S::kPartFloats + r]);
                }
                float unit = -INFINITY;  // 8 bits: the power of two of the joined O
                if constexpr (kCodes) {
                    for (uint32_t b = 0; b < split; ++b) {
                        const float* p = split > 1 ? cg::this_cluster().map_shared_rank(parts, b) : parts;
#pragma unroll
                        for (int w = 0; w < kWarps; ++w) {
                            const float* pw = p + w * kPart + S::kPartFloats + r;
                            if (pw[kRows] != 0.0f) unit = fmaxf(unit, (pw[0] - top) + pw[2 * kRows]);
                        }
                    }
                    unit = ceilf(unit);
                }
                float sum = 0.0f;
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (uint32_t b = 0; b < split; ++b) {
                    const float* p = split > 1 ? cg::this_cluster().map_shared_rank(parts, b) : parts;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float* pw = p + w * kPart;
                        const float mw = pw[S::kPartFloats + r], lw = pw[S::kPartFloats + kRows + r];
                        if (lw == 0.0f) continue;  // saw nothing
                        const float lf = exp2_fast(mw - top);
                        const float f = kCodes ? exp2_fast((mw - top) + (pw[S::kPartFloats + 2 * kRows + r] - unit)) : lf;
                        const float4 ov = *reinterpret_cast<const float4*>(pw + r * S::kPitch + c4);
                        sum += lw * lf;
                        acc.x += ov.x * f;
                        acc.y += ov.y * f;
                        acc.z += ov.z * f;
                        acc.w += ov.w * f;
                    }
                }
                float inv = sum == 0.0f ? 0.0f : 1.0f / sum, up = kCodes ? power_of_two(unit) : 1.0f;
                if constexpr (kTail) {
                    float tail = sum == 0.0f ? -INFINITY : top - kUnitLog + log2f(sum), high = -INFINITY;
                    const size_t row = part_row(R, h);
                    const float all = join(row, tail, high);
                    if (sum == 0.0f) acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    acc.x = acc.x * inv * up * tail, acc.y = acc.y * inv * up * tail;
                    acc.z = acc.z * inv * up * tail, acc.w = acc.w * inv * up * tail;
                    if (joined) {
                        for (uint32_t y = 0; y < a.splits; ++y) {
                            const float w = all == 0.0f ? 0.0f : exp2_fast(a.part_log[y * part_rows + row] - high) * all;
                            if (w == 0.0f) continue;
                            const float4 x = *reinterpret_cast<const float4*>(a.part_out + (y * part_rows + row) * D + c4);
                            acc.x += w * x.x, acc.y += w * x.y, acc.z += w * x.z, acc.w += w * x.w;
                        }
                    }
                    inv = up = 1.0f;
                }
                const uint32_t tok = a.group_div.div(R), head = h * a.group + (R - tok * a.group);
                uint2 w2 = make_uint2(pack2(acc.x * inv * up, acc.y * inv * up, T{}), pack2(acc.z * inv * up, acc.w * inv * up, T{}));
                *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (v.start + tok) * a.o_ts + head * a.o_hs + c4) = w2;
            }
        }
        if (split > 1) cg::this_cluster().sync();  // a block's parts stay until all have read them
    }
    }
}

// The tails' kernel may start while the prefix's runs: it waits for that one before it reads its parts.
cudaLaunchAttribute beside_the_prefix() {
    cudaLaunchAttribute x{};
    x.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    x.val.programmaticStreamSerializationAllowed = 1;
    return x;
}

template <typename T, int D, bool kCodes, int kRows, int kKeys> cudaError_t launch(CacheAttnArgs a, cudaStream_t s) {
    const uint32_t tiles = (a.c.max_new * a.group + kRows - 1) / kRows;
    const uint64_t jobs = static_cast<uint64_t>(a.c.sequences) * a.c.kv_heads * tiles;
    a.tile_div = FastDiv(tiles);
    const uint64_t span = kKeys == kTailKeys && a.max_tail ? min(visible_span(a, kRows), uint64_t{a.max_tail}) : visible_span(a, kRows);
    const uint64_t units = (span + kUnit - 1) / kUnit;
    // A warp alone or four a job (bf16, 1024 sequences, 16 heads of 64 channels, one new token; us with the events
    // around them): 16-bit pools, 192 tokens 109 and 140, 400 tokens 201 and 195; codes 138 and 132, 260 and 186.
    if (units <= (kCodes ? 8 : 16) && jobs >= 148 * 4) {
        using S = Shape<D, kCodes, kRows, false>;
        // the heads in as many parts as run at once, evenly
        const uint64_t lots = static_cast<uint64_t>(a.c.sequences) * tiles, slots = 148 * kWarps * S::kBlocks;
        uint32_t parts = static_cast<uint32_t>(min(uint64_t{a.c.kv_heads}, max(uint64_t{1}, slots / lots)));
        const uint32_t heads = (a.c.kv_heads + parts - 1) / parts;
        parts = (a.c.kv_heads + heads - 1) / heads;
        a.kv_div = FastDiv(parts);
        auto* kernel = cache_attn_kernel<T, D, kCodes, kRows, false, kKeys>;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e != cudaSuccess) return e;
        const uint64_t warps = lots * parts;
        const uint32_t blocks = static_cast<uint32_t>((warps + kWarps - 1) / kWarps);
        if constexpr (kKeys == kTailKeys) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(blocks);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = S::kBytes;
            cfg.stream = s;
            cudaLaunchAttribute early = beside_the_prefix();
            cfg.attrs = &early;
            cfg.numAttrs = 1;
            return cudaLaunchKernelEx(&cfg, kernel, a, tiles, heads);
        }
        kernel<<<blocks, kThreads, S::kBytes, s>>>(a, tiles, heads);
        return cudaGetLastError();
    }
    // as many blocks a job as fit the GPU at once (above 8: 16, a cluster of a whole GPC), at least four units a warp
    using S = Shape<D, kCodes, kRows, true>;
    a.kv_div = FastDiv(a.c.kv_heads);
    const uint64_t fit = min(static_cast<uint64_t>(148 * S::kBlocks) / max(jobs, uint64_t{1}), units / (kWarps * 4));
    const uint32_t split = fit >= 16 ? 16 : fit > 8 ? 8 : fit > 1 ? static_cast<uint32_t>(fit) : 1;
    auto* kernel = cache_attn_kernel<T, D, kCodes, kRows, true, kKeys>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<uint32_t>(jobs * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2] = {};
    cfg.attrs = attr;
    if (split > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = split;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    if (kKeys == kTailKeys) attr[cfg.numAttrs++] = beside_the_prefix();
    return cudaLaunchKernelEx(&cfg, kernel, a, tiles, split);
}

template <int kKeys, typename T, int D, bool kCodes> cudaError_t by_rows(const CacheAttnArgs& a, cudaStream_t s) {
    return a.c.max_new * a.group <= 8 ? launch<T, D, kCodes, 8, kKeys>(a, s) : launch<T, D, kCodes, 16, kKeys>(a, s);
}

template <int kKeys, typename T, bool kCodes> cudaError_t by_dim(const CacheAttnArgs& a, cudaStream_t s) {
    switch (a.c.head_dim) {
        case 32: return by_rows<kKeys, T, 32, kCodes>(a, s);
        case 64: return by_rows<kKeys, T, 64, kCodes>(a, s);
        default: return by_rows<kKeys, T, 128, kCodes>(a, s);
    }
}

template <int kKeys> cudaError_t by_type(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? by_dim<kKeys, bf16, true>(a, s) : by_dim<kKeys, __half, true>(a, s);
    return dtype == LWM_DTYPE_BF16 ? by_dim<kKeys, bf16, false>(a, s) : by_dim<kKeys, __half, false>(a, s);
}

}  // namespace

cudaError_t launch_cache_attention(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s) {
    return by_type<kAllKeys>(a, dtype, storage, s);
}

cudaError_t launch_cache_attention_tail(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s) {
    return by_type<kTailKeys>(a, dtype, storage, s);
}

// What the tails cost here, by the measured rates of this kernel (us); where nothing is said of them, as 128 tokens.
double shared_tail_cost(const CacheAttnArgs& a) {
    const double jobs = static_cast<double>(a.c.sequences) * a.c.kv_heads * ((static_cast<double>(a.c.max_new) * a.group + 15) / 16);
    const uint64_t span = min(visible_span(a, 16), uint64_t{a.max_tail ? a.max_tail : 128});
    return 4.0 + jobs * (static_cast<double>((span + 15) / 16) + 4) / (a.c.head_dim == 128 ? 1580.0 : a.c.head_dim == 64 ? 3100.0 : 3700.0);
}

}  // namespace lwm
