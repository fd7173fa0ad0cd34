// kernels_cache_attn.cu — attention over the paged cache for few query rows
// a kv head (lwm_cache_attention_device).
//
// A job is (sequence, kv head, 16 query rows = tokens x heads of the group).
// A warp walks 16-key units: scores = Q K^T on mma.sync m16n8k16, a running
// maximum and sum in 32 bits, O += P V.  The units of a job are dealt to the
// four warps of a block and, for long contexts, to the blocks of a cluster;
// their (maximum, sum, O) are joined in shared memory and over distributed
// shared memory, so a call needs no workspace and no second kernel and its
// sums have one order.
//
// Bound: memory (each K and V byte is used by at most 16 rows, 32 flops a
// byte).  Every warp keeps its own ring of units in flight with cp.async, so
// no barrier stands between a load and its use.
//
// 8-bit codes become halves in registers: e4m3 is exact in fp16.  The
// contraction's order is free, so a thread's 16 bytes of a key are the four
// channels each of four k-steps, and Q is loaded in the same order; V's
// bytes are interleaved by key pairs with byte permutes.  The key scale
// multiplies the scores; the value scales are kept relative to the largest
// so far, which multiplies O once at the end.  bf16 queries are brought to
// fp16 by a power of two a row, exactly down to 2^-17 of the row's largest.
#include <cooperative_groups.h>

#include "lwm_blocks.cuh"
#include "lwm_cache_attn.cuh"

namespace lwm {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kUnit = 16;    // keys a step
constexpr int kMaxSplit = 16;

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

template <int D, bool kCodes> struct Shape {
    static constexpr int kUnitBytes = kUnit * D * (kCodes ? 1 : 2);  // of K, and of V
    static constexpr int kStages = kCodes ? (D == 128 ? 6 : 8) : (D == 128 ? 4 : 6);
    static constexpr int kWarpBytes = kStages * 2 * kUnitBytes;
    static constexpr int kPartFloats = 16 * D;                       // a warp's O
    static constexpr int kPartBytes = (kPartFloats + 32) * 4;        // and its maxima and sums
    static constexpr int kBytes = kWarps * (kWarpBytes > kPartBytes ? kWarpBytes : kPartBytes);
};

// Visible keys of one row: [0, first) and [lo, hi).
struct RowRange { uint32_t lo, hi, first; };

template <typename T, int D, bool kCodes, bool kShared>
__global__ void __launch_bounds__(kThreads) cache_attn_kernel(CacheAttnArgs a, uint32_t tiles, uint32_t split) {
    using M = std::conditional_t<kCodes, __half, T>;  // the operands' type
    using S = Shape<D, kCodes>;
    constexpr int kSteps = D / 16, kTiles = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // job: four warps (and `split` blocks) share one, or a warp has its own
    const uint32_t rank = kShared ? blockIdx.x % split : 0;
    const uint32_t job = kShared ? blockIdx.x / split : blockIdx.x * kWarps + warp;
    const uint32_t tile = job % tiles, hs = job / tiles, h = hs % a.c.kv_heads, s = hs / a.c.kv_heads;
    SeqView v;
    if (s < a.c.sequences) v = sequence(a.c, s, false, h == 0 && tile == 0 && rank == 0 && lane == 0);
    const uint32_t rows = v.n * a.group, row0 = tile * 16;
    const bool live = row0 < rows;
    if (!live && (!kShared || split == 1)) return;  // uniform over what waits together

    // this thread's rows g and g + 8, and the tile's union
    RowRange rr[2];
    const void* q_row[2] = {nullptr, nullptr};
    uint32_t lo_min = 0, lo_max = 0, hi_min = 0, hi_max = 0;
    if (live) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t R = row0 + g + 8 * i;
            rr[i] = {0, 0, 0};
            if (R < rows) {
                const uint32_t tok = a.group_div.div(R), head = h * a.group + (R - tok * a.group);
                const VisibleRange vr = visible(a, v, tok);
                rr[i] = {vr.lo, vr.hi, vr.first};
                q_row[i] = static_cast<const T*>(a.q) + (v.start + tok) * a.q_ts + head * a.q_hs;
            }
        }
        const uint32_t tok0 = a.group_div.div(row0), tok1 = a.group_div.div(min(row0 + 15, rows - 1));
        const VisibleRange r0 = visible(a, v, tok0), r1 = visible(a, v, tok1);
        lo_min = r0.lo, hi_min = r0.hi;
        lo_max = r1.lo, hi_max = r1.hi;
    }
    const uint32_t sinks_end = min(a.sinks, min(lo_min, hi_max));
    const uint32_t sink_units = (sinks_end + kUnit - 1) / kUnit;
    const uint32_t win_unit = max(lo_min / kUnit, sink_units);
    const uint32_t win_units = hi_max > win_unit * kUnit ? (hi_max - win_unit * kUnit + kUnit - 1) / kUnit : 0;
    const uint32_t units = sink_units + win_units;
    // this warp's units: walk, walk + step, ... below end
    const uint32_t per = kShared ? (units + split - 1) / split : units;
    const uint32_t end = kShared ? min(units, (rank + 1) * per) : units;
    uint32_t walk = kShared ? rank * per + warp : 0;
    const uint32_t step = kShared ? kWarps : 1;

    uint8_t* ring = smem + warp * S::kWarpBytes;
    const uint32_t ring_a = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    const uint32_t count = walk < end ? (end - walk + step - 1) / step : 0;
    // page and first key of the warp's unit i, looked up 32 units at a time
    int pages_ahead = -1;
    auto key_of = [&](uint32_t i) {
        const uint32_t u = walk + i * step;
        return (u < sink_units ? u : u - sink_units + win_unit) * kUnit;
    };
    auto look_ahead = [&](uint32_t i) {
        pages_ahead = i + lane < count ? page_of(a.c, s, key_of(i + lane) >> a.c.page_shift) : -1;
    };
    int unit_pages[S::kStages];  // of the units in flight, by ring slot (8 bits: their scales)
    auto load = [&](uint32_t i, int slot) {
        if ((i & 31) == 0) look_ahead(i);
        const int page = __shfl_sync(0xffffffffu, pages_ahead, i & 31);
        const uint32_t key = key_of(i);
        const uint32_t at = key & (a.c.page_tokens - 1);
        constexpr int kRowChunks = S::kUnitBytes / kUnit / 16;
        const size_t base = pool_at(a.c, page < 0 ? 0 : page, h, at) * (kCodes ? 1 : 2);
        const uint32_t dst = ring_a + slot * 2 * S::kUnitBytes;
#pragma unroll
        for (int c = 0; c < kUnit * kRowChunks / 32; ++c) {
            const uint32_t x = c * 32 + lane, r = x / kRowChunks, ch = x % kRowChunks;
            const uint32_t j = key + r;
            const bool ok = page >= 0 && j < hi_max && (j >= lo_min || j < sinks_end);
            cp_async16(dst + chunk_at<D, kCodes>(r, ch), static_cast<const uint8_t*>(a.c.k) + base + x * 16, ok);
            cp_async16(dst + S::kUnitBytes + chunk_at<D, kCodes>(r, ch),
                       static_cast<const uint8_t*>(a.c.v) + base + x * 16, ok);
        }
        return page;
    };
#pragma unroll
    for (int i = 0; i < S::kStages; ++i) unit_pages[i] = -1;
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) {
        if (i < count) unit_pages[i] = load(i, i);
        cp_commit();
    }

    // queries, in the order of the contraction
    uint32_t q[kSteps][4];
    float row_mul[2] = {a.scale_log2, a.scale_log2};
    if (live) {
        if constexpr (!kCodes) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    q[k][i] = q_row[i & 1] ? *reinterpret_cast<const uint32_t*>(static_cast<const T*>(q_row[i & 1]) +
                                                                               16 * k + 8 * (i >> 1) + 2 * t)
                                           : 0u;
        } else {
            constexpr int kRun = D >= 64 ? 16 : 8;  // channels a thread reads of each 4 * kRun
            float f[2][kSteps][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float amax = 0.0f;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const int ch = (k / (kRun / 4)) * 4 * kRun + t * kRun + (k % (kRun / 4)) * 4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f[i][k][e] = q_row[i] ? static_cast<float>(static_cast<const T*>(q_row[i])[ch + e]) : 0.0f;
                        amax = fmaxf(amax, fabsf(f[i][k][e]));
                    }
                }
                if constexpr (std::is_same_v<T, bf16>) {
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
                    if (amax == 0.0f || e == 128) e = 0;
                    e = min(max(e, -126), 126);
                    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    row_mul[i] *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k)
#pragma unroll
                        for (int x = 0; x < 4; ++x) f[i][k][x] *= down;
                }
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    q[k][i] = pack2(f[i & 1][k][2 * (i >> 1)], f[i & 1][k][2 * (i >> 1) + 1], __half{});
        }
    }

    float o[kTiles][4];
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float v_ref = 0.0f;  // 8 bits: O is in units of this value scale

    for (uint32_t base = 0; base < count; base += S::kStages) {
#pragma unroll
        for (int slot = 0; slot < S::kStages; ++slot) {
            const uint32_t i = base + slot;
            if (i >= count) break;
            cp_wait<S::kStages - 2>();
            __syncwarp();
            const int page = unit_pages[slot];
            const uint32_t key = key_of(i);
            const uint32_t k_at = ring_a + slot * 2 * S::kUnitBytes, v_at = k_at + S::kUnitBytes;
            float k_scale = 1.0f, v_scale = 1.0f;
            if constexpr (kCodes) {
                if (page >= 0) {
                    const size_t at = static_cast<size_t>(page) * a.c.kv_heads + h;
                    k_scale = a.c.k_scale[at];
                    v_scale = a.c.v_scale[at];
                    if (!isfinite(v_scale)) v_scale = __int_as_float(0x7fc00000);
                }
            }
            float sc[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
            if constexpr (!kCodes) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t b[4];  // keys 0-7 and 8-15, each channels 0-7 and 8-15 of the step
                    ldsm4(b, k_at + chunk_at<D, false>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                    mma<M>(sc[0], q[k], b[0], b[1]);
                    mma<M>(sc[1], q[k], b[2], b[3]);
                }
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    uint32_t w[kSteps];
                    if constexpr (D == 32) {
                        const uint32_t at = k_at + chunk_at<D, true>(g + 8 * n, t >> 1) + (t & 1) * 8;
                        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
                    } else {
#pragma unroll
                        for (int c = 0; c < D / 64; ++c) {
                            const uint32_t at = k_at + chunk_at<D, true>(g + 8 * n, 4 * c + t);
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(w[4 * c]), "=r"(w[4 * c + 1]), "=r"(w[4 * c + 2]), "=r"(w[4 * c + 3])
                                         : "r"(at)
                                         : "memory");
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kSteps; ++k)
                        mma<M>(sc[n], q[k], f16x2_from_e4m3x2(w[k]), f16x2_from_e4m3x2(w[k] >> 16));
                }
            }
            // scores in units of log2, masked where this row does not see the key
            const bool whole = page >= 0 && (key >= lo_max || key + kUnit <= sinks_end) &&
                               key + kUnit <= hi_min;
            bool seen[2][4];
            bool above = false;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i2 = e >> 1;
                    const uint32_t j = key + 8 * n + 2 * t + (e & 1);
                    seen[n][e] = whole || (page >= 0 && j < rr[i2].hi && (j >= rr[i2].lo || j < rr[i2].first));
                    sc[n][e] = seen[n][e] ? sc[n][e] * (k_scale * row_mul[i2]) : -INFINITY;
                    above |= sc[n][e] > m[i2] + kRaise;
                }
            // the maximum moves only when a score passes it by kRaise: until
            // then exp2(score - m) stays below 2^kRaise
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int i2 = 0; i2 < 2; ++i2) {
                    float x = fmaxf(fmaxf(sc[0][2 * i2], sc[0][2 * i2 + 1]), fmaxf(sc[1][2 * i2], sc[1][2 * i2 + 1]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    x = fmaxf(x, m[i2]);
                    const float down = m[i2] == -INFINITY ? 0.0f : exp2_fast(m[i2] - x);
                    m[i2] = x;
                    l[i2] *= down;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        o[n][2 * i2] *= down;
                        o[n][2 * i2 + 1] *= down;
                    }
                }
            }
            float v_mul = 1.0f;
            if constexpr (kCodes) {
                if (v_scale > v_ref) {
                    const float down = v_ref / v_scale;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][e] *= down;
                    v_ref = v_scale;
                }
                v_mul = v_scale == 0.0f ? 0.0f : v_scale / v_ref;
            }
            float p[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float top = m[e >> 1] == -INFINITY ? 0.0f : m[e >> 1];
                    p[n][e] = exp2_fast(sc[n][e] - top);
                    l[e >> 1] += p[n][e];
                    p[n][e] *= v_mul;
                }
            // P in the operands' type: 2^-9 (bf16) or 2^-12 (fp16) of itself,
            // no more than rounding the output costs
            const uint32_t pa[4] = {pack2(p[0][0], p[0][1], M{}), pack2(p[0][2], p[0][3], M{}),
                                    pack2(p[1][0], p[1][1], M{}), pack2(p[1][2], p[1][3], M{})};
            // a key that some rows of the tile see and others do not: zero
            // times an infinity or NaN would reach the others
            bool poison = false;
            if (!whole) {
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
                poison |= kCodes && v_scale != v_scale;
                poison = __any_sync(0xffffffffu, poison);
            }
            if (!poison) {
                if constexpr (!kCodes) {
#pragma unroll
                    for (int n = 0; n < kTiles; n += 2) {
                        uint32_t b[4];  // channels 8n.. and 8n + 8.., each keys 0-7 and 8-15
                        ldsm4t(b, v_at + chunk_at<D, false>((lane & 7) + (((lane >> 3) & 1) << 3), n + (lane >> 4)));
                        mma<M>(o[n], pa, b[0], b[1]);
                        mma<M>(o[n + 1], pa, b[2], b[3]);
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
                        for (int j = 0; j < 4; j += 2) {
                            const uint32_t sel = j == 0 ? 0x5140 : 0x7362;
                            const uint32_t lo2 = __byte_perm(w[0], w[1], sel), hi2 = __byte_perm(w[2], w[3], sel);
                            mma<M>(o[4 * c + j], pa, f16x2_from_e4m3x2(lo2), f16x2_from_e4m3x2(hi2));
                            mma<M>(o[4 * c + j + 1], pa, f16x2_from_e4m3x2(lo2 >> 16), f16x2_from_e4m3x2(hi2 >> 16));
                        }
                    }
                }
            } else {
                // one key after another, for the rows that see it
#pragma unroll 1
                for (int key_i = 0; key_i < kUnit; ++key_i) {
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        const int from = g * 4 + (key_i & 7) / 2;
                        float pk = 0.0f;
                        bool sk = false;
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float x = __shfl_sync(0xffffffffu, p[n][2 * i2 + e], from);
                                const bool y = __shfl_sync(0xffffffffu, seen[n][2 * i2 + e], from);
                                if (n == key_i >> 3 && e == (key_i & 1)) {
                                    pk = x;
                                    sk = y;
                                }
                            }
                        if (!sk) continue;
#pragma unroll
                        for (int n = 0; n < kTiles; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int ch = kCodes ? 32 * (n >> 2) + 8 * t + 4 * e + (n & 3) : 8 * n + 2 * t + e;
                                o[n][2 * i2 + e] += pk * value_at<T, D, kCodes>(ring + slot * 2 * S::kUnitBytes +
                                                                                     S::kUnitBytes, key_i, ch);
                            }
                    }
                }
            }
            __syncwarp();
            // refill: this slot's unit is done, the one kStages - 1 ahead goes to the slot before
            const uint32_t next = i + S::kStages - 1;
            const int to = (slot + S::kStages - 1) % S::kStages;
            if (next < count) unit_pages[to] = load(next, to);
            cp_commit();
        }
    }
    cp_wait<0>();
    if constexpr (kCodes) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= v_ref;
    }
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2) {
        l[i2] += __shfl_xor_sync(0xffffffffu, l[i2], 1);
        l[i2] += __shfl_xor_sync(0xffffffffu, l[i2], 2);
    }
    auto channel = [&](int n, int e) { return kCodes ? 32 * (n >> 2) + 8 * t + 4 * e + (n & 3) : 8 * n + 2 * t + e; };

    if constexpr (!kShared) {
        // the warp's own rows: through its ring to whole 16-byte stores
        __syncwarp();
        T* part = reinterpret_cast<T*>(ring);
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
            const float inv = l[i2] == 0.0f ? 0.0f : 1.0f / l[i2];
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    part[(g + 8 * i2) * D + channel(n, e)] = static_cast<T>(o[n][2 * i2 + e] * inv);
        }
        __syncwarp();
        for (int x = lane; x < 16 * D / 8; x += 32) {
            const uint32_t R = row0 + x / (D / 8), c8 = 8 * (x % (D / 8));
            if (R >= rows) continue;
            const uint32_t tok = a.group_div.div(R), head = h * a.group + (R - tok * a.group);
            store8(static_cast<T*>(a.out) + (v.start + tok) * a.o_ts + head * a.o_hs + c8,
                   *reinterpret_cast<const Vec8<T>*>(part + x * 8));
        }
    } else {
        // join the warps, then the blocks of the cluster
        __syncthreads();  // every ring is done with
        float* parts = reinterpret_cast<float*>(smem);
        float* mine = parts + warp * (S::kPartFloats + 32);
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) mine[(g + 8 * i2) * D + channel(n, e)] = o[n][2 * i2 + e];
            if (t == 0) {
                mine[S::kPartFloats + g + 8 * i2] = m[i2];
                mine[S::kPartFloats + 16 + g + 8 * i2] = l[i2];
            }
        }
        if (split > 1) cg::this_cluster().sync();
        else __syncthreads();
        if (live) {
            // this block finishes every split-th vector of 4 channels
            const uint32_t stride = split * kThreads;
            for (uint32_t x = rank * kThreads + threadIdx.x; x < 16 * D / 4; x += stride) {
                const uint32_t r = x / (D / 4), c4 = 4 * (x % (D / 4)), R = row0 + r;
                if (R >= rows) continue;
                float top = -INFINITY;
                for (uint32_t b = 0; b < split; ++b) {
                    const float* p = split > 1 ? cg::this_cluster().map_shared_rank(parts, b) : parts;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w)
                        top = fmaxf(top, p[w * (S::kPartFloats + 32) + S::kPartFloats + r]);
                }
                float sum = 0.0f;
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (uint32_t b = 0; b < split; ++b) {
                    const float* p = split > 1 ? cg::this_cluster().map_shared_rank(parts, b) : parts;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float* pw = p + w * (S::kPartFloats + 32);
                        const float mw = pw[S::kPartFloats + r];
                        const float lw = pw[S::kPartFloats + 16 + r];
                        if (lw == 0.0f) continue;  // saw nothing
                        const float f = exp2_fast(mw - top);
                        const float4 ov = *reinterpret_cast<const float4*>(pw + r * D + c4);
                        sum += lw * f;
                        acc.x += ov.x * f;
                        acc.y += ov.y * f;
                        acc.z += ov.z * f;
                        acc.w += ov.w * f;
                    }
                }
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const uint32_t tok = a.group_div.div(R), head = h * a.group + (R - tok * a.group);
                uint2 w2 = make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}));
                *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (v.start + tok) * a.o_ts + head * a.o_hs + c4) = w2;
            }
        }
        if (split > 1) cg::this_cluster().sync();  // a block's parts stay until all have read them
    }
}

template <typename T, int D, bool kCodes> cudaError_t launch(const CacheAttnArgs& a, cudaStream_t s) {
    using S = Shape<D, kCodes>;
    const uint32_t tiles = (a.c.max_new * a.group + 15) / 16;
    const uint64_t jobs = static_cast<uint64_t>(a.c.sequences) * a.c.kv_heads * tiles;
    // keys a row can see
    uint64_t span = a.c.max_length ? a.c.max_length : static_cast<uint64_t>(a.c.table_stride) << a.c.page_shift;
    if (a.window) span = min(span, static_cast<uint64_t>(a.window) * a.frame + a.sinks + a.c.max_new);
    const uint64_t units = (span + kUnit - 1) / kUnit;
    auto set = [](auto* kernel) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return e;
    };
    if (units <= 8 && jobs >= 148 * 4) {
        const cudaError_t e = set(cache_attn_kernel<T, D, kCodes, false>);
        if (e != cudaSuccess) return e;
        cache_attn_kernel<T, D, kCodes, false>
            <<<static_cast<uint32_t>((jobs + kWarps - 1) / kWarps), kThreads, S::kBytes, s>>>(a, tiles, 1);
        return cudaGetLastError();
    }
    // blocks for two a SM, at least four units a warp
    uint32_t split = 1;
    while (split < kMaxSplit && jobs * split < 148 * 2 && units >= static_cast<uint64_t>(split) * 2 * kWarps * 4)
        split *= 2;
    cudaError_t e = set(cache_attn_kernel<T, D, kCodes, true>);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<uint32_t>(jobs * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, cache_attn_kernel<T, D, kCodes, true>, a, tiles, split);
}

template <typename T, bool kCodes> cudaError_t by_dim(const CacheAttnArgs& a, cudaStream_t s) {
    switch (a.c.head_dim) {
        case 32: return launch<T, 32, kCodes>(a, s);
        case 64: return launch<T, 64, kCodes>(a, s);
        default: return launch<T, 128, kCodes>(a, s);
    }
}

}  // namespace

cudaError_t launch_cache_attention(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? by_dim<bf16, true>(a, s) : by_dim<__half, true>(a, s);
    return dtype == LWM_DTYPE_BF16 ? by_dim<bf16, false>(a, s) : by_dim<__half, false>(a, s);
}

}  // namespace lwm
