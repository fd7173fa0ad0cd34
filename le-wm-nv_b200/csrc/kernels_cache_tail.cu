// kernels_cache_tail.cu — what follows a shared prefix, for few query rows and
// short tails (lwm_cache_attention_shared_device): the candidates of a rollout
// with a handful of tokens of their own.
//
// A warp takes some kv heads of a sequence with up to 2 rows each, one after
// another: the lengths and pages of a sequence are looked up once.  16 bytes of a key a
// lane (8 of codes), so D / 8 lanes have a key and a warp 4 keys at 64
// channels; everything is in 32 bits on CUDA cores: the products of one row
// with a dozen keys are too few for the tensor cores' 16 x 8 tiles, of which
// they would fill one row.  The prefix's parts are asked for together with the
// keys, and joined at the end.  The grid may start beside the prefix's, but a
// warp waits for that before the join of its first head, so one head a warp runs
// ahead at most: with four heads a warp nearly nothing overlaps.
//
// What bounds it (one B200): instructions, and each head's chain of keys, scores
// and join.  1024 candidates of 16 heads of 64 with up to 16 tokens of their own
// (bf16): 18 us behind the prefix's 26, where their 35 MB of keys, values and
// rows and the parts' 8 would take 7 (the tensor-core kernel for few rows: 42;
// the whole call 57.8 us with that, 43.0 with this).  The next head's keys asked
// for ahead: 48.9 and 59.8, the registers cost a block or two of the SM's six.  4
// rows a warp: slower than tensor cores (16 vehicles' 64 candidates, 4 rows,
// 8-bit codes: 118 instead of 91), so up to 2, and tails up to 128 tokens.
#include "lwm_blocks.cuh"
#include "lwm_cache_attn.cuh"

namespace lwm {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;

template <typename T, bool kCodes> struct Chunk8 { uint4 w; };
template <typename T> struct Chunk8<T, true> { uint2 w; };

template <typename T, bool kCodes> __device__ __forceinline__ void values(const Chunk8<T, kCodes>& c, float (&f)[8]) {
    if constexpr (kCodes) from_e4m3(c.w, f);
    else unpack(Vec8<T>{c.w}, f);
}

// The larger one, NaN where either is (fmaxf leaves NaN out: a row that sees
// nothing but NaN would look like one that sees nothing).
__device__ __forceinline__ float max_or_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

template <typename T, int D, bool kCodes, int kRows>
__global__ void __launch_bounds__(kThreads, kRows == 1 ? 6 : 5) cache_tail_kernel(const __grid_constant__ CacheAttnArgs a, uint32_t heads) {
    using C = Chunk8<T, kCodes>;
    constexpr int kLanes = D / 8, kKeys = 32 / kLanes;  // lanes of a key, keys at once
    constexpr int kSteps = 4, kRun = kKeys * kSteps;    // keys in flight
    constexpr size_t kElem = kCodes ? 1 : 2;
    const int lane = threadIdx.x & 31, c = lane % kLanes, mine = lane / kLanes;
    const uint32_t job = blockIdx.x * kWarps + (threadIdx.x >> 5), s = a.kv_div.div(job), h0 = (job - s * a.kv_div.d) * heads;
    const uint32_t h_end = min(h0 + heads, a.c.kv_heads);
    // (every path below this line waits for the prefix's kernel, so that this grid is not done before that one)
    bool live = s < a.c.sequences;
    SeqView v;
    uint32_t shared = 0;
    bool joined = false;
    if (live) {
        v = sequence(a.c, s, false, h0 == 0 && lane == 0);
        if (v.ok && a.group_count && static_cast<int>(s) >= a.groups[0]) {
            const uint32_t g = last_at_most(a.groups, 0, a.group_count, static_cast<int>(s));
            if (static_cast<int>(s) < a.groups[g + 1]) {
                const GroupView group = group_view(a, g, false);
                joined = group.ok && v.start >= group.start && v.start + v.n <= group.start + group.n;  // (the prefix's rows)
                shared = group.shared;
                const bool reaches = joined && shared && v.n && static_cast<uint64_t>(v.n) + shared > v.length;
                if (reaches && h0 == 0 && lane == 0) cache_report(a.c.err, kCacheErrShared, s, shared);
                if (!joined || reaches) v.n = 0;
            }
        }
        live = v.n != 0;
    }
    if (!live) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const uint32_t rows = v.n * a.group;

    // what the rows see of the tail
    VisibleRange rr[kRows];
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        rr[r] = {0, 0, 0};
        if (static_cast<uint32_t>(r) >= rows) continue;
        rr[r] = visible(a, v, a.group_div.div(r));
        rr[r].lo = max(rr[r].lo, shared);
        lo = min(lo, rr[r].first > shared ? shared : rr[r].lo);
        hi = max(hi, rr[r].hi);
    }
    const uint32_t begin = lo / kKeys * kKeys, runs = hi > begin ? (hi - begin + kRun - 1) / kRun : 1;

    // a run of a head's keys and values, and at its first run the queries, 8 channels a lane
    struct Run {
        C k[kSteps], w[kSteps];
        float k_scale[kCodes ? kSteps : 1], v_scale[kCodes ? kSteps : 1];
        Vec8<T> q[kRows];
        uint32_t here;  // bit x: step x has a key
    };
    int pages[kSteps];
    auto fetch = [&](Run& run, uint32_t h, uint32_t i) {
        const uint32_t key0 = begin + i * kRun;
        if (runs > 1 || h == h0) {
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {  // (all of them asked for before any is used)
                const uint32_t j = key0 + x * kKeys + mine;
                pages[x] = j >= lo && j < hi ? a.c.table[static_cast<size_t>(s) * a.c.table_stride + (j >> a.c.page_shift)] : -1;
            }
        }
        if (i == 0) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                run.q[r].a = make_uint4(0, 0, 0, 0);
                if (static_cast<uint32_t>(r) >= rows) continue;
                const uint32_t tok = a.group_div.div(r);
                run.q[r] = load8(static_cast<const T*>(a.q) + (v.start + tok) * a.q_ts + (h * a.group + (r - tok * a.group)) * a.q_hs + 8 * c);
            }
        }
        run.here = 0;
#pragma unroll
        for (int x = 0; x < kSteps; ++x) {
            const uint32_t j = key0 + x * kKeys + mine;
            const bool wanted = j >= lo && j < hi, in_pool = static_cast<uint32_t>(pages[x]) < a.c.pages;
            if (wanted && !in_pool && c == 0) cache_report(a.c.err, kCacheErrPage, s, pages[x]);
            run.k[x].w = {}, run.w[x].w = {};
            if constexpr (kCodes) run.k_scale[x] = run.v_scale[x] = 1.0f;
            if (!wanted || !in_pool) continue;
            run.here |= 1u << x;
            const size_t from = pool_at(a.c, pages[x], h, j & (a.c.page_tokens - 1)) + 8 * c;
            run.k[x].w = *reinterpret_cast<const decltype(run.k[x].w)*>(static_cast<const uint8_t*>(a.c.k) + from * kElem);
            run.w[x].w = *reinterpret_cast<const decltype(run.k[x].w)*>(static_cast<const uint8_t*>(a.c.v) + from * kElem);
            if constexpr (kCodes) {
                const size_t sc = static_cast<size_t>(pages[x]) * a.c.kv_heads + h;
                run.k_scale[x] = a.c.k_scale[sc], run.v_scale[x] = a.c.v_scale[sc];
            }
        }
    };
    const size_t part_rows = static_cast<size_t>(a.c.tokens) * a.heads;
    auto row_of = [&](uint32_t R, uint32_t h) {
        const uint32_t tok = a.group_div.div(R);
        return (static_cast<size_t>(v.start) + tok) * a.heads + h * a.group + (R - tok * a.group);
    };
    // row `mine` is this lane's to join and write
    const uint32_t R = mine;
    const bool owns = R < rows && R < kRows;
    bool ready = false;

#pragma unroll 1
    for (uint32_t h = h0; h < h_end; ++h) {
        Run cur;
        fetch(cur, h, 0);
        float m[kRows], l[kRows], out[kRows][8];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) out[r][e] = 0.0f;
        }
        // the prefix's first part (before the first head is done it may not be there yet)
        const size_t row = owns ? row_of(R, h) : 0;
        float first_log = -INFINITY;
        Vec8<float> first_out = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
        auto ask = [&] {
            if (!joined || !owns) return;
            first_log = a.part_log[row];
            first_out = load8(a.part_out + row * D + 8 * c);
        };
        if (ready) ask();
#pragma unroll 1
        for (uint32_t i = 0; i < runs; ++i) {
            if (i) fetch(cur, h, i);
            const uint32_t key0 = begin + i * kRun;
            float sc[kRows][kSteps];
            uint32_t seen[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                seen[r] = 0;
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const uint32_t j = key0 + x * kKeys + mine;
                    if (j < rr[r].hi && (j >= rr[r].lo || (j < rr[r].first && j >= shared))) seen[r] |= 1u << x;
                }
                seen[r] &= cur.here;
            }
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
                float f[8];
                values(cur.k[x], f);
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    float dot = 0.0f, q[8];
                    unpack(cur.q[r], q);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot = fmaf(q[e], f[e], dot);
#pragma unroll
                    for (int o = kLanes / 2; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                    sc[r][x] = (seen[r] >> x) & 1 ? dot * (kCodes ? cur.k_scale[kCodes ? x : 0] * a.scale_log2 : a.scale_log2) : -INFINITY;
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                float top = max_or_nan(max_or_nan(sc[r][0], sc[r][1]), max_or_nan(sc[r][2], sc[r][3]));
#pragma unroll
                for (int o = kLanes; o < 32; o *= 2) top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = max_or_nan(top, m[r]);
                const float down = m[r] == -INFINITY ? 0.0f : exp2_fast(m[r] - top);
                m[r] = top;
                if (i == 0) continue;
                l[r] *= down;
#pragma unroll
                for (int e = 0; e < 8; ++e) out[r][e] *= down;
            }
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
                float f[8];
                values(cur.w[x], f);
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    // (a value that a row does not see is left out, not multiplied by zero)
                    if (!((seen[r] >> x) & 1) || m[r] == -INFINITY) continue;
                    const float p = exp2_fast(sc[r][x] - m[r]);
                    l[r] += p;
                    float pv = p;
                    if constexpr (kCodes) pv *= isfinite(cur.v_scale[x]) ? cur.v_scale[x] : __int_as_float(0x7fc00000);
#pragma unroll
                    for (int e = 0; e < 8; ++e) out[r][e] = fmaf(pv, f[e], out[r][e]);
                }
            }
        }
        if (!ready) {
            asm volatile("griddepcontrol.wait;" ::: "memory");  // the prefix's parts are there
            ready = true;
            ask();
        }
        // sums over the lanes that had other keys
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int o = kLanes; o < 32; o *= 2) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
#pragma unroll
                for (int e = 0; e < 8; ++e) out[r][e] += __shfl_xor_sync(0xffffffffu, out[r][e], o);
            }
        float y[8], ml = m[0], ll = l[0];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = out[0][e];
#pragma unroll
        for (int r = 1; r < kRows; ++r)
            if (static_cast<uint32_t>(r) == R) {
                ml = m[r], ll = l[r];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = out[r][e];
            }
        if (!owns) continue;
        // the tail's sum is ll 2^ml; a part's, its logarithm with its values already divided by it
        float top = ll == 0.0f ? -INFINITY : ml;
        bool nan = ll != ll;
        auto part_at = [&](uint32_t x) { return x == 0 ? first_log : a.part_log[x * part_rows + row]; };
        if (joined)
            for (uint32_t x = 0; x < a.splits; ++x) {
                const float log = part_at(x);
                top = fmaxf(top, log);
                nan |= log != log;
            }
        if (nan) top = __int_as_float(0x7fc00000);
        const float tail = ll == 0.0f ? 0.0f : exp2_fast(ml - top);
        float sum = ll * tail;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = ll == 0.0f ? 0.0f : y[e] * tail;
        if (joined && top != -INFINITY)
            for (uint32_t x = 0; x < a.splits; ++x) {
                const float p = exp2_fast(part_at(x) - top);
                if (p == 0.0f) continue;
                float f[8];
                if (x == 0) unpack(first_out, f);
                else unpack(load8(a.part_out + (x * part_rows + row) * D + 8 * c), f);
                sum += p;
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fmaf(p, f[e], y[e]);
            }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= inv;
        const uint32_t tok = a.group_div.div(R);
        store8(static_cast<T*>(a.out) + (v.start + tok) * a.o_ts + (h * a.group + (R - tok * a.group)) * a.o_hs + 8 * c, pack<T>(y));
    }
}

template <typename T, int D, bool kCodes, int kRows> cudaError_t launch(CacheAttnArgs a, cudaStream_t s) {
    // heads a warp: as few as fill the GPU with warps (24 a SM)
    const uint64_t jobs = static_cast<uint64_t>(a.c.sequences) * a.c.kv_heads;
    uint32_t heads = static_cast<uint32_t>(min(uint64_t{a.c.kv_heads}, max(uint64_t{1}, jobs / (148 * 24))));
    const uint32_t parts = (a.c.kv_heads + heads - 1) / heads;
    a.kv_div = FastDiv(parts);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<uint32_t>((static_cast<uint64_t>(a.c.sequences) * parts + kWarps - 1) / kWarps));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute early{};  // beside the prefix's kernel
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cache_tail_kernel<T, D, kCodes, kRows>, a, heads);
}
template <typename T, int D, bool kCodes> cudaError_t by_rows(const CacheAttnArgs& a, cudaStream_t s) {
    const uint32_t rows = a.c.max_new * a.group;
    return rows <= 1 ? launch<T, D, kCodes, 1>(a, s) : launch<T, D, kCodes, 2>(a, s);
}
template <typename T, bool kCodes> cudaError_t by_dim(const CacheAttnArgs& a, cudaStream_t s) {
    switch (a.c.head_dim) {
        case 32: return by_rows<T, 32, kCodes>(a, s);
        case 64: return by_rows<T, 64, kCodes>(a, s);
        default: return by_rows<T, 128, kCodes>(a, s);
    }
}

}  // namespace

bool short_tails(const CacheAttnArgs& a) {
    return a.c.max_new * a.group <= 2 && a.max_tail && a.max_tail <= 128;
}

cudaError_t launch_cache_attention_short_tail(const CacheAttnArgs& a, int dtype, int storage, cudaStream_t s) {
    if (storage == LWM_CACHE_E4M3)
        return dtype == LWM_DTYPE_BF16 ? by_dim<bf16, true>(a, s) : by_dim<__half, true>(a, s);
    return dtype == LWM_DTYPE_BF16 ? by_dim<bf16, false>(a, s) : by_dim<__half, false>(a, s);
}

}  // namespace lwm
