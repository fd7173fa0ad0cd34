// kernels_sample.cu — tokens drawn from logits with given random numbers
// (lwm_sample_tokens_device).
//
// A row lives in the shared memory of one block (up to 32768 logits) or of a
// cluster, a slice of it in each block; every pass over the row (largest
// logit, the thresholds of top_k and top_p, the draw) reads it there, and the
// logits are read from memory once.
//
// Which token a random number falls on depends on sums over the whole row, so
// those are exact: a weight exp((x - max) / temperature) is computed in 64 bits
// (relative error below 1e-13) and rounded to a multiple of 2^-43, and sums are
// integers, which have no order.  A threshold (the last token that top_k or
// top_p keeps) is found by a histogram over the logits, in 512 bins that span 45
// powers of two of the weight: counts, or masses in 13 bits of each bin's
// own scale.  The bin that a rough sum points at is proved, or changed, by
// exact sums; its tokens are sorted and walked, or, where they are more than
// the list takes, binned again by their keys, down to one logit if need be.
// With top_k up to the list's length all that is kept is in the list, and the
// rest of the call works on that alone.
//
// What bounds it (one B200): instructions.  256 rows of 32000 f32 logits with
// top_p 0.95 take 104 us, of which their 33 MB from memory would be 5: two
// passes that compute weights of 64 bits (28000 cycles of a block, the double
// precision units of its SM the limit), a histogram of 32000 shared atomics, a
// sort (11000 cycles) and about twenty barriers, for two blocks a SM one after
// another.  Rows kept in registers (65 a thread) spilled: 439 us.  With top_k
// no pass but the list's computes weights: 16 rows of 131072 bf16, top 50,
// 16.5 us, eight blocks each.  1024 rows of 1024 bf16 without filters: 6 to 7
// us, a launch and one pass, a warp a row.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "lwm_blocks.cuh"

namespace lwm {

namespace {

namespace cg = cooperative_groups;

constexpr int kList = 1024;     // candidates that are sorted
constexpr uint32_t kMaxSplit = 8;      // blocks of a row
constexpr int kBins = 512;
constexpr uint32_t kMaxSlice = 32768;  // logits of a block
static_assert(kMaxSplit * kMaxSlice >= kSampleVocab, "a row fits its blocks");
constexpr float kSpan = 45.0f;  // powers of two that the bins span: weights end there
constexpr float kUnits = 8192.0f;
static_assert(kUnits * kSampleVocab < 4294967296.0f, "a bin's mass");

// Order of logits: larger ones have larger keys; 0 for what is never drawn
// (minus infinity, NaN).
__device__ __forceinline__ uint32_t key_of(float x) {
    x += 0.0f;  // (minus zero is zero)
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The weights of a row.
struct Weights {
    double top, rate;  // largest logit, 64 log2(e) / temperature
    float top32, rate32;
};
constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number in the low bits
// A float as a double, without the conversion unit (subnormals may become any tiny number).
__device__ __forceinline__ double widen(float x) {
    const uint32_t b = __float_as_uint(x), m = b & 0x7fffffffu;
    return __hiloint2double(static_cast<int>((b & 0x80000000u) | (m == 0 ? 0u : (m >> 3) + 0x38000000u)), static_cast<int>(b << 29));
}
// 2^43 exp((x - top) / temperature), rounded to a whole number (a thread's sums of them stay below 2^53, so
// they are exact).  2^(n / 64) comes from a table, the rest, below 2^-7, from five terms of the series.
__device__ __forceinline__ double weight(const Weights& w, const double* table, float x) {
    const double y = (widen(x) - w.top) * w.rate;  // 64ths of a power of two
    const double t = y + kMagic, n = t - kMagic;
    const int i = __double2loint(t);
    const double r = (y - n) * 0.010830424696249145;  // ln 2 / 64
    const double r2 = r * r;
    const double p = fma(fma(1.0 / 24.0, r2, 0.5), r2, 1.0) + fma(1.0 / 6.0, r2, 1.0) * r;  // the series to r^4
    const double f = table[i & 63] * p;  // [2^-1/128, 2)
    const int up = static_cast<uint32_t>(__double2hiint(y)) < 0xc0a6a800u ? (((i >> 6) + 43) << 20) : -(1 << 30);  // (y <= -2900: 2^-45 and less)
    const double scaled = __hiloint2double(max(__double2hiint(f) + up, 0), __double2loint(f));
    return (scaled + kMagic) - kMagic;
}

struct Params {
    double temperature, top_p, min_p;
    uint32_t top_k;
};
__device__ __forceinline__ Params params_of(const TokenArgs& a, uint32_t row) {
    Params p{a.temperature, a.top_p, a.min_p, a.top_k};
    if (a.temperatures) p.temperature = a.temperatures[row];
    if (a.top_ps) p.top_p = a.top_ps[row];
    if (a.min_ps) p.min_p = a.min_ps[row];
    if (a.top_ks) p.top_k = static_cast<uint32_t>(max(a.top_ks[row], 0));
    if (!(p.temperature > 0.0)) p.top_k = 1, p.temperature = 1.0;  // the largest
    p.temperature = fmin(fmax(p.temperature, 1e-30), 1e30);
    if (!(p.top_p < 1.0)) p.top_p = 1.0;
    if (!(p.min_p > 0.0)) p.min_p = 0.0;
    p.min_p = fmin(p.min_p, 1.0);
    return p;
}

template <int kThreads> struct Shared {
    static constexpr int kWarps = kThreads / 32;
    double table[64];
    uint64_t sums[2][kMaxSplit * kWarps];
    uint32_t counts[2][kMaxSplit * kWarps];
};
struct Filter {  // of a kernel with thresholds
    uint32_t bins[kBins];  // of the row, in every block
    uint32_t mine[kBins];  // of this block
    uint64_t list[kList];
    uint64_t mass[kList];
    uint64_t found, most;
    uint32_t listed, picked;
};

// kFilter: top_k or top_p may be on.
template <typename T, int kThreads, bool kFilter>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ TokenArgs a, uint32_t split, uint32_t slice, int vectors) {
    constexpr int kWarps = kThreads / 32;
    extern __shared__ __align__(16) float x[];  // the slice's logits; minus infinity: never drawn
    using S = Shared<kThreads>;
    __shared__ S sh;
    __shared__ std::conditional_t<kFilter, Filter, char> filter_s;
    const uint32_t rank = blockIdx.x % split, row = blockIdx.x / split;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Params par = params_of(a, row);
    const uint32_t base = rank * slice, count = base < a.vocab ? min(slice, a.vocab - base) : 0;
    // A thread's logits: a run of odd length, so that the threads of a warp read different banks, in order of index.
    const uint32_t each = ((count + kThreads - 1) / kThreads) | 1u;
    const uint32_t run0 = min(threadIdx.x * each, count), run1 = min(run0 + each, count);
    float top = -INFINITY;  // of the logits that this thread loads
    {
        const T* src = static_cast<const T*>(a.logits) + row * a.stride + base;
        auto clean = [&](float v) {
            v = v == v ? v + 0.0f : -INFINITY;  // (minus zero is zero)
            top = fmaxf(top, v);
            return v;
        };
        const uint32_t whole = vectors ? count / 8 : 0;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < whole; i += kThreads) {
            float f[8];
            unpack(load8(src + 8 * i), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = clean(f[e]);
            store8(x + 8 * i, pack<float>(f));
        }
#pragma unroll 4
        for (uint32_t i = 8 * whole + threadIdx.x; i < count; i += kThreads) x[i] = clean(static_cast<float>(src[i]));
    }
    for (int i = threadIdx.x; i < 64; i += kThreads) sh.table[i] = exp2(i / 64.0);
    if constexpr (kFilter)
        for (int i = threadIdx.x; i < kBins; i += kThreads) filter_s.bins[i] = filter_s.mine[i] = 0;

    if (split > 1) cg::this_cluster().sync();  // every block runs before another writes to it
    int turn = 0;
    auto meet = [&] {
        if (split > 1) cg::this_cluster().sync();
        else __syncthreads();
    };
    auto block_of = [&](auto* p, uint32_t b) { return split > 1 ? cg::this_cluster().map_shared_rank(p, b) : p; };
    // Sums of a warp's values to every block: one barrier, the buffers alternate.
    auto share = [&](uint64_t v, uint32_t c) {
        const uint32_t slot = rank * kWarps + warp;
        if (lane < split) {
            S* to = block_of(&sh, lane);
            to->sums[turn][slot] = v, to->counts[turn][slot] = c;
        }
        meet();
    };
    auto warp_sum = [&](uint64_t v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    auto sum_all = [&](uint64_t v, uint32_t c, uint64_t& v_all, uint32_t& c_all) {
        share(warp_sum(v), __reduce_add_sync(0xffffffffu, c));
        v = 0, c = 0;
        for (uint32_t i = lane; i < split * kWarps; i += 32) v += sh.sums[turn][i], c += sh.counts[turn][i];
        v_all = warp_sum(v), c_all = __reduce_add_sync(0xffffffffu, c);
        turn ^= 1;
    };

    // The thread's logits four at a time, so that their chains run side by side.
    auto by_four = [&](auto what) {
        for (uint32_t i = run0; i < run1; i += 4) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i + e < run1 ? x[i + e] : -INFINITY;
            what(v, base + i);
        }
    };
    // the largest logit
    Weights w;
    {
        uint32_t k = __reduce_max_sync(0xffffffffu, key_of(top));
        share(0, k);
        for (uint32_t i = lane; i < split * kWarps; i += 32) k = max(k, sh.counts[turn][i]);
        k = __reduce_max_sync(0xffffffffu, k);
        turn ^= 1;
        if (k == 0) {  // nothing can be drawn
            if (rank == 0 && threadIdx.x == 0) {
                a.tokens[row] = -1;
                if (a.log_probs) a.log_probs[row] = -INFINITY;
            }
            if (split > 1) cg::this_cluster().sync();
            return;
        }
        w.top32 = value_of(k);
        if (w.top32 == INFINITY) {  // infinities share the row: as if they were zero, and nothing else there
            for (uint32_t i = run0; i < run1; ++i) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
            top = top == INFINITY ? 0.0f : -INFINITY;
            w.top32 = 0.0f;
            __syncthreads();
        }
        w.top = widen(w.top32);
        w.rate = 92.332482616893657 / par.temperature;  // 64 log2(e)
        w.rate32 = static_cast<float>(1.4426950408889634 / par.temperature);
    }
    const double least = par.min_p > 0.0 ? ceil(par.min_p * 8796093022208.0) : 1.0;  // 2^43 min_p
    const bool by_min = least > 1.0;
    const float u = a.uniform[row];
    // the point on the sum `all` of kept weights that the random number stands for: the first sum above it is drawn
    auto point_of = [&](uint64_t all) {
        const double at = (u > 0.0f ? static_cast<double>(fminf(u, 1.0f)) : 0.0) * static_cast<double>(all);
        return min(static_cast<uint64_t>(at), all - 1);
    };
    auto answer = [&](uint32_t token, uint64_t mass, uint64_t all) {
        a.tokens[row] = static_cast<int32_t>(token);
        if (a.log_probs) a.log_probs[row] = static_cast<float>(log(static_cast<double>(mass) / static_cast<double>(all)));
    };

    // Tokens in order: larger logits first, then smaller indices; those up to (edge, edge_index) are kept.
    float edge = -FLT_MAX;
    uint32_t edge_index = 0xffffffffu;
    // Of the kept ones above `settled` the thread's sum is `known` already.
    float settled = INFINITY;
    uint64_t known = 0;
    auto kept = [&](float v, uint32_t i) { return v > edge || (v == edge && i <= edge_index); };

    if constexpr (kFilter) {
        Filter& f = filter_s;
        auto place = [&](float v, uint32_t i) { return static_cast<uint64_t>(key_of(v)) << 32 | (0xffffffffu - i); };
        auto index_at = [](uint64_t p) { return 0xffffffffu - static_cast<uint32_t>(p); };
        // The tokens for which `which` holds, sorted, in block 0 (where the number of them is at most kList); the
        // other blocks pass through.
        auto sorted = [&](auto which) {
            if (threadIdx.x == 0) f.listed = 0;
            meet();
            Filter* to = block_of(&f, 0);
#pragma unroll 4
            for (uint32_t i = run0; i < run1; ++i)
                    if (which(x[i], base + i)) {
                        const uint32_t at = atomicAdd(&to->listed, 1u);
                        if (at < kList) to->list[at] = place(x[i], base + i);
                    }
            meet();
            if (rank) return 0;
            const int n = min(f.listed, static_cast<uint32_t>(kList));
            int size = 2;
            while (size < n) size *= 2;
            for (int i = n + threadIdx.x; i < size; i += kThreads) f.list[i] = 0;
            __syncthreads();
            // a warp keeps 32 neighbours in registers: steps within them need no barrier
            for (int k = 2; k <= size; k *= 2) {
                int j = k / 2;
                for (; j >= 32; j /= 2) {
                    for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                        const uint64_t p = f.list[lo], q = f.list[hi];
                        if ((p < q) == ((lo & k) == 0)) f.list[lo] = q, f.list[hi] = p;  // descending
                    }
                    __syncthreads();
                }
                if (k < 32 && k * 2 <= min(size, 32)) continue;  // (the first ones all at once, below)
                for (int i = threadIdx.x; i < ((size + 31) & ~31); i += kThreads) {
                    uint64_t p = i < size ? f.list[i] : 0;
                    for (int kk = k <= 32 ? 2 : k; kk <= k; kk *= 2)
                        for (int jj = min(j, kk / 2); jj > 0; jj /= 2) {
                            const uint64_t q = __shfl_xor_sync(0xffffffffu, p, jj);
                            const bool larger_first = (i & kk) == 0, is_low = (i & jj) == 0;
                            if ((p < q) == (larger_first == is_low)) p = q;
                        }
                    if (i < size) f.list[i] = p;
                }
                __syncthreads();
            }
            return n;
        };
        auto weight_at = [&](int i) { return static_cast<uint64_t>(weight(w, sh.table, value_of(static_cast<uint32_t>(f.list[i] >> 32)))); };

        // A logit's place in bins, 0 for the largest; the last bin takes all that is left.
        const float per_bin = kBins / kSpan * w.rate32;
        auto place0 = [&](float v) { return fminf((w.top32 - v) * per_bin, kBins - 1.0f); };
        // The counts of all blocks' bins in every block (the caller's are in f.mine), and the bin with which the sum
        // from the first one on reaches `goal`: each bin counts `unit` times its own weight.
        auto pick = [&](auto weigh, auto goal_of) {
            __syncthreads();
            if (split > 1) {
                for (int i = threadIdx.x; i < kBins; i += kThreads)
                    if (f.mine[i])
                        for (uint32_t b = 0; b < split; ++b) atomicAdd(&block_of(&f, b)->bins[i], f.mine[i]);
                meet();
            }
            const uint32_t* bins = split > 1 ? f.bins : f.mine;
            if (warp == 0) {
                auto here = [&](int i) {
                    const int b = lane * (kBins / 32) + i;
                    return bins[b] ? bins[b] * weigh(b) : 0.0;
                };
                double sum = 0.0;
#pragma unroll 1
                for (int i = 0; i < kBins / 32; ++i) sum += here(i);
                double upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const double y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                const double goal = goal_of(__shfl_sync(0xffffffffu, upto, 31));
                double before = upto - sum;
                int mine = -1, any = -1;
#pragma unroll 1
                for (int i = 0; i < kBins / 32; ++i) {
                    const double mass = here(i);
                    if (mass > 0.0) {
                        any = lane * (kBins / 32) + i;
                        if (mine < 0 && before + mass >= goal) mine = any;
                    }
                    before += mass;
                }
                const uint32_t has = __ballot_sync(0xffffffffu, mine >= 0), some = __ballot_sync(0xffffffffu, any >= 0);
                const int b = has ? __shfl_sync(0xffffffffu, mine, __ffs(has) - 1)
                                  : some ? __shfl_sync(0xffffffffu, any, 31 - __clz(some)) : 0;
                if (lane == 0) f.picked = b;
            }
            __syncthreads();
            return static_cast<int>(f.picked);
        };
        auto clear_bins = [&] {
            meet();
            for (int i = threadIdx.x; i < kBins; i += kThreads) f.bins[i] = f.mine[i] = 0;
            meet();
        };
        // The last token of the first `want_count`, or of the first whose mass is at least `share_of` of the kept ones'.
        auto threshold = [&](auto by_mass, double share_of, uint32_t want_count) {
            constexpr bool kByMass = decltype(by_mass)::value;
            uint32_t lo = 0, hi = 0, shift = 0;  // keys (lo, hi] after the first time round
            uint64_t above = 0;                  // exact mass, or count, of what lies above the bins
            double want = kByMass ? 0.0 : want_count;
            // one level of bins; true when the threshold is found
            auto level = [&](auto is_first) {
                constexpr bool kFirst = decltype(is_first)::value;
                auto inside = [&](float v, uint32_t i) {
                    if (v == -INFINITY || !kept(v, i)) return false;
                    if constexpr (kFirst) return true;
                    const uint32_t k = key_of(v);
                    return k > lo && k <= hi;
                };
                // (a whole number; the first time with a fraction behind it)
                auto bin = [&](float v) {
                    if constexpr (kFirst) return place0(v);
                    else return static_cast<float>((hi - key_of(v)) >> shift);
                };
                const float high = kFirst ? 0.0f : value_of(hi);
#pragma unroll 4
                for (uint32_t i = run0; i < run1; ++i) {
                    const float v = x[i];
                    if (!inside(v, base + i)) continue;
                    const float c = bin(v);
                    uint32_t m = 1;
                    if constexpr (kByMass) {
                        if (kFirst && c >= kBins - 1.0f) continue;  // (no weight, or next to none)
                        // weights in units of 2^-13 of the largest that the bin can hold: 2^18 of them fit 32 bits, so
                        // no bin with a token looks empty
                        float y;
                        asm("ex2.approx.ftz.f32 %0, %1;"
                            : "=f"(y)
                            : "f"(kFirst ? (truncf(c) - c) * (kSpan / kBins) : (v - high) * w.rate32));
                        m = __float2uint_rn(fminf(y, 1.0f) * kUnits);
                    }
                    atomicAdd(&f.mine[static_cast<int>(c)], m);
                }
                int b = pick([&](int c) { return kByMass && kFirst ? static_cast<double>(exp2f(-c * (kSpan / kBins))) : 1.0; },
                             [&](double total) {
                                 if (!kByMass) return want - static_cast<double>(above);
                                 if (kFirst) return share_of * total;
                                 return (want - static_cast<double>(above)) * (kUnits / 8796093022208.0) *
                                        exp2f((w.top32 - high) * w.rate32);
                             });
                const uint32_t* bins = split > 1 ? f.bins : f.mine;
                // exact sums: all of them the first time, those above the bin, those in it
                uint64_t over;
                uint32_t n;
                if constexpr (kByMass) {
                    uint64_t sure, in;  // sure: the thread's part of what is above the bin and passes min_p
                    while (true) {
                        double s_all = 0.0, s_over = 0.0, s_in = 0.0, s_sure = 0.0;
                        uint32_t c_in = 0;
                        const float b0 = static_cast<float>(b), b1 = static_cast<float>(b + 1);
                        by_four([&](const float(&v)[4], uint32_t i) {
                            bool need[4], some = false;
                            float c[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                need[e] = inside(v[e], i + e);
                                c[e] = bin(v[e]);
                                need[e] &= c[e] < (kFirst ? kBins - 1.0f : b1);
                                some |= need[e];
                            }
                            if (!some) return;
                            double m[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) m[e] = weight(w, sh.table, v[e]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (!need[e]) continue;
                                if (kFirst) s_all += m[e];
                                if (c[e] < b0) s_over += m[e];
                                if (by_min && c[e] < b0 && m[e] >= least) s_sure += m[e];
                                if (c[e] >= b0 && c[e] < b1) s_in += m[e], ++c_in;
                            }
                        });
                        sure = static_cast<uint64_t>(by_min ? s_sure : s_over);
                        uint64_t all;
                        uint32_t none;
                        if constexpr (kFirst) {
                            sum_all(static_cast<uint64_t>(s_all), 0, all, none);
                            want = share_of * static_cast<double>(all);
                        }
                        sum_all(static_cast<uint64_t>(s_over), 0, over, none);
                        sum_all(static_cast<uint64_t>(s_in), c_in, in, n);
                        // (a rough sum may have missed by a bin that holds next to nothing)
                        int next = b;
                        if (static_cast<double>(above + over) >= want) {
                            for (next = b - 1; next > 0 && !bins[next]; --next) {}
                            if (next < 0) next = b;
                        } else if (static_cast<double>(above + over + in) < want) {
                            for (next = b + 1; next < kBins && !bins[next] && !(kFirst && next == kBins - 1); ++next) {}
                            if (next == kBins) next = b;
                        }
                        if (next == b) break;
                        b = next;
                    }
                    known += sure;
                } else {
                    uint64_t c_over = 0;
                    for (int i = lane; i < b; i += 32) c_over += bins[i];
                    over = warp_sum(c_over);
                    n = bins[b];
                }
                above += over;
                if (n <= kList) {
                    const int found = sorted([&](float v, uint32_t i) { return inside(v, i) && static_cast<int>(bin(v)) == b; });
                    if (rank == 0) {
                        if constexpr (kByMass) {
                            for (int i = threadIdx.x; i < found; i += kThreads) f.mass[i] = weight_at(i);
                            __syncthreads();
                            if (warp == 0) {
                                uint64_t before = above;
                                for (int i = 0; i < found; i += 32) {
                                    uint64_t y = i + lane < found ? f.mass[i + lane] : 0;
#pragma unroll
                                    for (int o = 1; o < 32; o *= 2) {
                                        const uint64_t z = __shfl_up_sync(0xffffffffu, y, o);
                                        if (lane >= o) y += z;
                                    }
                                    const bool there = i + lane < found && (static_cast<double>(before + y) >= want || i + lane == found - 1);
                                    const uint32_t who = __ballot_sync(0xffffffffu, there);
                                    if (who) {
                                        if (lane < split) {
                                            Filter* to = block_of(&f, lane);
                                            to->found = f.list[i + __ffs(who) - 1], to->most = f.list[0];
                                        }
                                        break;
                                    }
                                    before += __shfl_sync(0xffffffffu, y, 31);
                                }
                            }
                        } else if (threadIdx.x < split) {
                            block_of(&f, threadIdx.x)->found = f.list[max(1, min(static_cast<int>(want_count - above), found)) - 1];
                        }
                    }
                    meet();
                    edge = value_of(static_cast<uint32_t>(f.found >> 32));
                    edge_index = index_at(f.found);
                    if (kByMass) settled = value_of(static_cast<uint32_t>(f.most >> 32));
                    return true;
                }
                // too many: their keys
                uint32_t least_key = 0xffffffffu, most_key = 0;
                for (uint32_t i = run0; i < run1; ++i)
                    if (inside(x[i], base + i) && static_cast<int>(bin(x[i])) == b) {
                        const uint32_t k = key_of(x[i]);
                        least_key = min(least_key, k), most_key = max(most_key, k);
                    }
                share(__reduce_min_sync(0xffffffffu, least_key), __reduce_max_sync(0xffffffffu, most_key));
                for (uint32_t i = 0; i < split * kWarps; ++i) {
                    least_key = min(least_key, static_cast<uint32_t>(sh.sums[turn][i]));
                    most_key = max(most_key, sh.counts[turn][i]);
                }
                turn ^= 1;
                if (least_key == most_key) {
                    // many tokens of one logit: the first so many of them, in order of index
                    const float v = value_of(least_key);
                    uint32_t need = want_count - static_cast<uint32_t>(above);
                    if constexpr (kByMass) {
                        const double one = weight(w, sh.table, v);
                        need = static_cast<uint32_t>(fmin(fmax(ceil((want - static_cast<double>(above)) / fmax(one, 1.0)), 1.0), 4e9));
                    }
                    need = min(need, n);
                    uint32_t mine = 0;
                    for (uint32_t i = run0; i < run1; ++i) mine += x[i] == v && kept(v, base + i);
                    uint32_t y = mine;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
                        if (lane >= o) y += z;
                    }
                    share(0, __shfl_sync(0xffffffffu, y, 31));
                    uint32_t before = y - mine;
                    for (uint32_t i = 0; i < rank * kWarps + warp; ++i) before += sh.counts[turn][i];
                    turn ^= 1;
                    if (before < need && before + mine >= need) {
                        uint32_t left = need - before;
                        for (uint32_t i = run0; left; ++i)
                            if (x[i] == v && kept(v, base + i) && --left == 0)
                                for (uint32_t o = 0; o < split; ++o) block_of(&f, o)->found = place(v, base + i);
                    }
                    meet();
                    edge = v;
                    edge_index = index_at(f.found);
                    if (kByMass) settled = v;
                    return true;
                }
                lo = least_key - 1, hi = most_key;
                shift = 0;
                while ((most_key - least_key) >> shift >= kBins) ++shift;
                clear_bins();
                return false;
            };
            if (!level(std::true_type{}))
                while (!level(std::false_type{})) {}
        };

        bool count_on = par.top_k && par.top_k < a.vocab, few = false;
        int n = 0;
        if (count_on && par.top_k <= min(kList / 2, kThreads * static_cast<int>(split) / 2)) {
            // As many threads' largest logits are at least the top_k-th of all: with their bins the first top_k tokens
            // are among few.
            if (top != -INFINITY) atomicAdd(&f.mine[static_cast<int>(place0(top))], 1u);
            const uint32_t want = par.top_k;
            const float last = static_cast<float>(pick([](int) { return 1.0; }, [&](double) { return static_cast<double>(want); }) + 1);
            const uint32_t* bins = split > 1 ? f.bins : f.mine;
            uint32_t tops = 0;
            for (int i = lane; i < kBins; i += 32) tops += bins[i];
            tops = __reduce_add_sync(0xffffffffu, tops);
            if (tops >= want && last < kBins) {
                n = sorted([&](float v, uint32_t) { return v != -INFINITY && place0(v) < last; });
                few = block_of(&f, 0)->listed <= kList;
                n = min(n, static_cast<int>(want));
            }
            if (!few) clear_bins();
            else if (split > 1) meet();  // (block 0's count has been read)
        }
        if (count_on && !few) {
            uint32_t c = 0, c_all;
            uint64_t none;
#pragma unroll 4
            for (uint32_t i = run0; i < run1; ++i) c += x[i] != -INFINITY;
            sum_all(0, c, none, c_all);
            count_on = c_all > par.top_k;
        }
        if (count_on && !few) {
            threshold(std::false_type{}, 0.0, par.top_k);
            if (par.top_k <= kList) {
                n = sorted([&](float v, uint32_t i) { return v != -INFINITY && kept(v, i); });
                few = true;
            }
        }
        if (few) {
            // all that is kept: a list
            if (rank) return;  // (no other block writes to this one any more)
            for (int i = threadIdx.x; i < n; i += kThreads) f.mass[i] = weight_at(i);
            __syncthreads();
            // how many top_p and min_p keep, and their mass
            if (warp == 0) {
                uint64_t all = 0;
                for (int i = lane; i < n; i += 32) all += f.mass[i];
                all = warp_sum(all);
                const double want = par.top_p < 1.0 ? fmax(par.top_p, 0.0) * static_cast<double>(all) : INFINITY;
                uint64_t before = 0;
                int m = 0;
                for (int i = 0; i < n; i += 32) {
                    const uint64_t own = i + lane < n ? f.mass[i + lane] : 0;
                    uint64_t y = own;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const uint64_t z = __shfl_up_sync(0xffffffffu, y, o);
                        if (lane >= o) y += z;
                    }
                    const bool keep = i + lane < n && static_cast<double>(own) >= least && (i + lane == 0 || static_cast<double>(before + y - own) < want);
                    const uint32_t who = __ballot_sync(0xffffffffu, keep);
                    m += __popc(who);
                    if (who != 0xffffffffu) {
                        before += who ? __shfl_sync(0xffffffffu, y, 31 - __clz(who)) : 0;
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, y, 31);
                }
                if (lane == 0) f.listed = m, f.found = before;
            }
            __syncthreads();
            const int m = f.listed;
            const uint64_t all = f.found, point = point_of(all);
            // each kept token: the sum of those of lower index
            for (int i = threadIdx.x; i < m; i += kThreads) {
                const uint32_t mine = index_at(f.list[i]);
                uint64_t sum = 0;
                for (int j = 0; j < m; ++j) sum += index_at(f.list[j]) < mine ? f.mass[j] : 0;
                if (sum <= point && point < sum + f.mass[i]) answer(mine, f.mass[i], all);
            }
            return;
        }
        if (par.top_p < 1.0) {
            if (count_on) clear_bins();
            threshold(std::true_type{}, fmax(par.top_p, 0.0), 0);
        }
    }

    // the draw: sums of the kept tokens, thread by thread
    uint64_t all = 0;
    double rest = 0.0;
    by_four([&](const float(&v)[4], uint32_t i) {
        bool need[4], some = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) some |= need[e] = kept(v[e], i + e) && v[e] <= settled;
        if (!some) return;
        double m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = weight(w, sh.table, v[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (need[e] && m[e] >= least) rest += m[e];
    });
    const uint64_t mine = known + static_cast<uint64_t>(rest);
    uint64_t y = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint64_t z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    share(__shfl_sync(0xffffffffu, y, 31), 0);
    uint64_t sum = y - mine;
    for (uint32_t i = 0; i < split * kWarps; ++i) {
        if (i < rank * kWarps + warp) sum += sh.sums[turn][i];
        all += sh.sums[turn][i];
    }
    turn ^= 1;
    const uint64_t point = point_of(all);
    // the thread whose run it falls into, and with its warp's help the token
    const uint32_t who = __ballot_sync(0xffffffffu, sum <= point && point < sum + mine);
    if (who) {
        const int owner = __ffs(who) - 1;
        const uint32_t from = __shfl_sync(0xffffffffu, run0, owner), to = __shfl_sync(0xffffffffu, run1, owner);
        sum = __shfl_sync(0xffffffffu, sum, owner);
        for (uint32_t i = from; i < to; i += 32) {
            const float v = i + lane < to ? x[i + lane] : -INFINITY;
            const double own = kept(v, base + i + lane) ? weight(w, sh.table, v) : 0.0;
            const uint64_t m = own >= least ? static_cast<uint64_t>(own) : 0;
            uint64_t z = m;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint64_t q = __shfl_up_sync(0xffffffffu, z, o);
                if (lane >= o) z += q;
            }
            if (sum + z - m <= point && point < sum + z) answer(base + i + lane, m, all);
            sum += __shfl_sync(0xffffffffu, z, 31);
        }
    }
    if (split > 1) cg::this_cluster().sync();  // (no block ends while another writes to it)
}

template <typename T, int kThreads, bool kFilter> cudaError_t launch(const TokenArgs& a, uint32_t split, cudaStream_t s) {
    auto* kernel = sample_kernel<T, kThreads, kFilter>;
    const int vectors = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.stride * sizeof(T) % 16 == 0;
    const uint32_t slice = ((a.vocab + split - 1) / split + 7) / 8 * 8;
    cudaError_t e = cudaSuccess;
    if (slice * 4 > 16384) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice * 4);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.rows * split);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = slice * 4;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, split, slice, vectors);
}

template <typename T, bool kFilter> cudaError_t by_vocab(const TokenArgs& a, cudaStream_t s) {
    if (a.vocab <= 1024) return launch<T, 32, kFilter>(a, 1, s);
    if (a.vocab <= 8192) return launch<T, 128, kFilter>(a, 1, s);
    uint32_t split = 1;
    while (split * kMaxSlice < a.vocab) split *= 2;
    // few rows: more blocks each, down to 8192 logits
    while (a.rows * split * 2 <= 148 && split < kMaxSplit && split * 2 * 8192 <= a.vocab) split *= 2;
    return a.vocab > 16384 * split ? launch<T, 1024, kFilter>(a, split, s) : launch<T, 512, kFilter>(a, split, s);
}

template <typename T> cudaError_t by_filter(const TokenArgs& a, cudaStream_t s) {
    const bool filter = a.top_ks || a.top_ps || a.temperatures || a.top_k || a.top_p < 1.0 || !(a.temperature > 0.0);
    return filter ? by_vocab<T, true>(a, s) : by_vocab<T, false>(a, s);
}

}  // namespace

cudaError_t launch_sample_tokens(const TokenArgs& a, int dtype, cudaStream_t s) {
    if (dtype == LWM_DTYPE_F32) return by_filter<float>(a, s);
    return dtype == LWM_DTYPE_BF16 ? by_filter<bf16>(a, s) : by_filter<__half>(a, s);
}

}  // namespace lwm
