// kernels_sample.cu — tokens drawn from logits with given random numbers
// (lwm_sample_tokens_device).
//
// A row lives in the registers of one block (up to 16384 logits) or of a
// cluster, a slice of it in each block; every pass over the row (largest
// logit, the thresholds of top_k and top_p, the draw) reads registers, and the
// logits are read from memory once.
//
// Which token a random number falls on depends on sums over the whole row, so
// those are exact: a weight exp((x - max) / temperature) is computed in 64 bits
// (relative error below 1e-13) and rounded to a multiple of 2^-43, and sums are
// integers, which have no order.  Thresholds are found by bisection on the
// logit with 32-bit sums, decided by exact ones where those are too near; the
// last few hundred candidates of a threshold are sorted.
#include <cooperative_groups.h>

#include <algorithm>

#include "lwm_blocks.cuh"

namespace lwm {

namespace {

namespace cg = cooperative_groups;

constexpr int kList = 1024;     // candidates that are sorted
constexpr int kMaxSplit = 16;   // blocks of a row
constexpr float kNear = 1e-5f;  // more than a 32-bit sum of weights can be off

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
    bool infinite;     // the largest logit is plus infinity: all such tokens weigh the same
};
constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number in the low bits
// A float as a double, without the conversion unit (subnormals may become any tiny number).
__device__ __forceinline__ double widen(float x) {
    const uint32_t b = __float_as_uint(x), m = b & 0x7fffffffu;
    return __hiloint2double(static_cast<int>((b & 0x80000000u) | (m == 0 ? 0u : (m >> 3) + 0x38000000u)), static_cast<int>(b << 29));
}
// round(2^43 exp((x - top) / temperature)).  2^(n / 64) comes from a table,
// the rest, below 2^-7, from five terms of the series.
__device__ __forceinline__ uint64_t weight(const Weights& w, const double* table, uint32_t key) {
    if (key == 0) return 0;
    const float x = value_of(key);
    if (w.infinite) return x == INFINITY ? 1ull << 43 : 0;
    const double y = (widen(x) - w.top) * w.rate;  // 64ths of a power of two
    if (y < -2900.0) return 0;                     // below 2^-45
    const double t = y + kMagic, n = t - kMagic;
    const int i = __double2loint(t);
    const double r = (y - n) * 0.010830424696249145;  // ln 2 / 64
    const double p = fma(fma(fma(fma(1.0 / 24.0, r, 1.0 / 6.0), r, 0.5), r, 1.0), r, 1.0);
    const double f = table[i & 63] * p;  // [2^-1/128, 2)
    const double scaled = __hiloint2double(__double2hiint(f) + (((i >> 6) + 43) << 20), __double2loint(f));
    return __double_as_longlong(scaled + kMagic) - __double_as_longlong(kMagic);
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
    uint64_t list[kList];
    uint64_t mass[kList];
    uint64_t found;
    uint32_t listed;
};

template <typename T, int kThreads, int kVals>
__global__ void __launch_bounds__(kThreads, kThreads == 512 ? 2 : 1)
    sample_kernel(const __grid_constant__ TokenArgs a, uint32_t split, int vectors) {
    constexpr int kWarps = kThreads / 32, kRounds = kVals / 8;
    using S = Shared<kThreads>;
    __shared__ S sh;
    const uint32_t rank = blockIdx.x % split, row = blockIdx.x / split;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Params par = params_of(a, row);
    // elements 8 threadIdx.x + e of run j
    const uint32_t base = rank * kThreads * kVals + threadIdx.x * 8;
    auto index_of = [&](int j, int e) { return base + j * kThreads * 8 + e; };
    uint32_t key[kVals];
    {
        const T* src = static_cast<const T*>(a.logits) + row * a.stride;
#pragma unroll
        for (int j = 0; j < kRounds; ++j) {
            const uint32_t i = index_of(j, 0);
            float f[8];
            if (vectors && i + 8 <= a.vocab) {
                unpack(load8(src + i), f);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = i + e < a.vocab ? static_cast<float>(src[i + e]) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) key[8 * j + e] = key_of(f[e]);
        }
    }
    for (int i = threadIdx.x; i < 64; i += kThreads) sh.table[i] = exp2(i / 64.0);

    if (split > 1) cg::this_cluster().sync();  // every block runs before another writes to it
    int turn = 0;
    auto meet = [&] {
        if (split > 1) cg::this_cluster().sync();
        else __syncthreads();
    };
    // Sums over the row, the same in every thread: one barrier each, the buffers alternate.
    auto share = [&](uint64_t x, uint32_t c) {
        const uint32_t slot = rank * kWarps + warp;
        if (split == 1) {
            if (lane == 0) sh.sums[turn][slot] = x, sh.counts[turn][slot] = c;
        } else if (lane < split) {
            S* to = cg::this_cluster().map_shared_rank(&sh, lane);
            to->sums[turn][slot] = x, to->counts[turn][slot] = c;
        }
        meet();
    };
    auto sum_all = [&](uint64_t x, uint32_t c, uint64_t& x_all, uint32_t& c_all) {
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        c = __reduce_add_sync(0xffffffffu, c);
        share(x, c);
        x = 0, c = 0;
        for (uint32_t i = lane; i < split * kWarps; i += 32) x += sh.sums[turn][i], c += sh.counts[turn][i];
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x_all = x, c_all = __reduce_add_sync(0xffffffffu, c);
        turn ^= 1;
    };
    // the same with a 32-bit float sum
    auto sum_rough = [&](float x, uint32_t c, float& x_all, uint32_t& c_all) {
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        c = __reduce_add_sync(0xffffffffu, c);
        share(__float_as_uint(x), c);
        x = 0.0f, c = 0;
        for (uint32_t i = lane; i < split * kWarps; i += 32)
            x += __uint_as_float(static_cast<uint32_t>(sh.sums[turn][i])), c += sh.counts[turn][i];
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x_all = x, c_all = __reduce_add_sync(0xffffffffu, c);
        turn ^= 1;
    };

    // the largest logit
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVals; ++i) top = max(top, key[i]);
    top = __reduce_max_sync(0xffffffffu, top);
    share(0, top);
    for (uint32_t i = lane; i < split * kWarps; i += 32) top = max(top, sh.counts[turn][i]);
    top = __reduce_max_sync(0xffffffffu, top);
    turn ^= 1;
    if (top == 0) {  // nothing can be drawn
        if (rank == 0 && threadIdx.x == 0) {
            a.tokens[row] = -1;
            if (a.log_probs) a.log_probs[row] = -INFINITY;
        }
        if (split > 1) cg::this_cluster().sync();
        return;
    }
    Weights w;
    w.top32 = value_of(top);
    w.infinite = w.top32 == INFINITY;
    w.top = widen(w.top32);
    w.rate = 92.332482616893657 / par.temperature;  // 64 log2(e)
    w.rate32 = static_cast<float>(1.4426950408889634 / par.temperature);
    auto rough = [&](uint32_t k) {
        float r;
        const float x = value_of(k);
        const float y = w.infinite ? (x == INFINITY ? 0.0f : -INFINITY) : (x - w.top32) * w.rate32;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
        return r;
    };
    // Tokens in order: larger logits first, then smaller indices.  A threshold is the last token kept, as
    // key << 32 | ~index; those not below it are kept.
    auto place = [&](uint32_t k, uint32_t i) { return static_cast<uint64_t>(k) << 32 | (0xffffffffu - i); };
    uint64_t border = static_cast<uint64_t>(1) << 32;  // every key but 0

    // The threshold of a filter: kByMass, the first token with which the mass of the kept ones (those not below
    // `border`) reaches `want`; else the want-th.
    auto threshold = [&](auto by_mass, double want_mass, uint32_t want_count) {
        constexpr bool kByMass = decltype(by_mass)::value;
        uint32_t lo = max(static_cast<uint32_t>(border >> 32), 1u), hi = top + 1, above_count = 0;  // keys [lo, hi) hold it
        if (kByMass && !w.infinite) lo = max(lo, key_of(w.top32 - 32.0f / w.rate32));  // (weights end at 2^-45)
        uint64_t above = 0;  // mass and count of the keys from hi on
        uint32_t inside = 0xffffffffu;
        bool exact = true;   // `above` is
        for (int step = 0; hi - lo > 1; ++step) {
            uint32_t mid = lo + (hi - lo) / 2;
            if (!(step & 1)) {  // halfway between the logits, then between the keys: one of them soon gets there
                const float x = 0.5f * value_of(lo) + 0.5f * value_of(hi - 1);
                const uint32_t k = key_of(x);
                if (k > lo && k < hi) mid = k;
            }
            float m = 0.0f;
            uint32_t n = 0, below = 0;
#pragma unroll
            for (int i = 0; i < kVals; ++i) {
                const bool kept = place(key[i], index_of(i >> 3, i & 7)) >= border;
                if (kept && key[i] >= mid) {
                    ++n;
                    if (kByMass) m += rough(key[i]);
                } else if (kept && key[i] >= lo) {
                    ++below;
                }
            }
            float m_all;
            uint32_t both;
            uint32_t n_all, below_all;
            sum_rough(m, n, m_all, n_all);
            sum_rough(0.0f, below, m, both);
            below_all = both;
            bool up;  // the threshold is at or above mid
            if constexpr (kByMass) {
                const double rough_mass = static_cast<double>(m_all) * 8796093022208.0;  // 2^43
                if (rough_mass > want_mass * (1.0 + kNear)) {
                    up = true;
                } else if (rough_mass < want_mass * (1.0 - kNear)) {
                    up = false;
                    exact = false;
                } else {
                    uint64_t x = 0, x_all;
                    uint32_t c;
#pragma unroll
                    for (int i = 0; i < kVals; ++i)
                        if (key[i] >= mid && place(key[i], index_of(i >> 3, i & 7)) >= border) x += weight(w, sh.table, key[i]);
                    sum_all(x, 0, x_all, c);
                    up = static_cast<double>(x_all) >= want_mass;
                    if (!up) above = x_all, exact = true;
                }
            } else {
                up = n_all >= want_count;
            }
            if (up) {
                lo = mid;
                inside = n_all - above_count;
            } else {
                hi = mid;
                above_count = n_all;
                inside = below_all;
            }
            if (inside <= kList) break;
        }
        if (kByMass && !exact) {
            uint64_t x = 0;
            uint32_t c;
#pragma unroll
            for (int i = 0; i < kVals; ++i)
                if (key[i] >= hi && place(key[i], index_of(i >> 3, i & 7)) >= border) x += weight(w, sh.table, key[i]);
            sum_all(x, 0, above, c);
        }
        if (hi - lo > 1 || inside <= kList) {
            // few: listed in every block, sorted, and walked
            if (threadIdx.x == 0) sh.listed = 0;
            for (int i = threadIdx.x; i < kList; i += kThreads) sh.list[i] = 0;
            meet();
#pragma unroll
            for (int i = 0; i < kVals; ++i) {
                const uint64_t p = place(key[i], index_of(i >> 3, i & 7));
                if (key[i] >= lo && key[i] < hi && p >= border) {
                    for (uint32_t b = 0; b < split; ++b) {
                        S* to = split > 1 ? cg::this_cluster().map_shared_rank(&sh, b) : &sh;
                        const uint32_t at = atomicAdd(&to->listed, 1u);
                        if (at < kList) to->list[at] = p;
                    }
                }
            }
            meet();
            const int n = min(sh.listed, static_cast<uint32_t>(kList));
            int size = 2;
            while (size < n) size *= 2;
            for (int k = 2; k <= size; k *= 2)
                for (int j = k / 2; j > 0; j /= 2) {
                    for (int i = threadIdx.x; i < size; i += kThreads) {
                        const int o = i ^ j;
                        if (o > i) {
                            const uint64_t x = sh.list[i], y = sh.list[o];
                            if ((x < y) == ((i & k) == 0)) sh.list[i] = y, sh.list[o] = x;  // descending
                        }
                    }
                    __syncthreads();
                }
            if constexpr (kByMass) {
                for (int i = threadIdx.x; i < size; i += kThreads) sh.mass[i] = i < n ? weight(w, sh.table, static_cast<uint32_t>(sh.list[i] >> 32)) : 0;
                __syncthreads();
                if (warp == 0) {
                    uint64_t before = above;
                    for (int i = 0; i < n; i += 32) {
                        uint64_t x = i + lane < n ? sh.mass[i + lane] : 0;
#pragma unroll
                        for (int o = 1; o < 32; o *= 2) {
                            const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
                            if (lane >= o) x += y;
                        }
                        const bool there = i + lane < n && (static_cast<double>(before + x) >= want_mass || i + lane == n - 1);
                        const uint32_t who = __ballot_sync(0xffffffffu, there);
                        if (who) {
                            if (lane == 0) sh.found = sh.list[i + __ffs(who) - 1];
                            break;
                        }
                        before += __shfl_sync(0xffffffffu, x, 31);
                    }
                }
                __syncthreads();
                border = sh.found;
            } else {
                border = sh.list[min(want_count - above_count, static_cast<uint32_t>(n)) - 1];
            }
            meet();
        } else {
            // many tokens of one logit: the first so many of them
            uint32_t need;
            if constexpr (kByMass) {
                const double each = static_cast<double>(weight(w, sh.table, lo));
                const double c = ceil((want_mass - static_cast<double>(above)) / fmax(each, 1.0));
                need = static_cast<uint32_t>(fmin(fmax(c, 1.0), 4e9));
            } else {
                need = want_count - above_count;
            }
            // the need-th in order of index: by runs of every block, then by threads
            uint32_t mine[kRounds];
            bool done = false;
            uint32_t seen = 0;
            if (threadIdx.x == 0) sh.found = 0;
#pragma unroll
            for (int j = 0; j < kRounds; ++j) {
                mine[j] = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    mine[j] += key[8 * j + e] == lo && place(lo, index_of(j, e)) >= border;
            }
            // (runs of a block are in order, and blocks are)
            uint32_t of_block = 0;
#pragma unroll
            for (int j = 0; j < kRounds; ++j) of_block += mine[j];
            of_block = __reduce_add_sync(0xffffffffu, of_block);
            share(0, of_block);
            uint32_t total = 0;
            for (uint32_t i = 0; i < split * kWarps; ++i) {
                if (i / kWarps < rank) seen += sh.counts[turn][i];
                total += sh.counts[turn][i];
            }
            turn ^= 1;
            need = min(need, total);
#pragma unroll
            for (int j = 0; j < kRounds; ++j) {
                // prefix over the block's threads
                uint32_t x = mine[j];
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                if (lane == 31) sh.mass[j * kWarps + warp] = x;
                __syncthreads();
                uint32_t run = 0, prefix = 0;
                for (int i = 0; i < kWarps; ++i) {
                    if (i < warp) prefix += static_cast<uint32_t>(sh.mass[j * kWarps + i]);
                    run += static_cast<uint32_t>(sh.mass[j * kWarps + i]);
                }
                const uint32_t before = seen + prefix + x - mine[j];
                if (!done && before < need && before + mine[j] >= need) {
                    uint32_t left = need - before;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (left && key[8 * j + e] == lo && place(lo, index_of(j, e)) >= border && --left == 0) {
                            for (uint32_t b = 0; b < split; ++b)
                                (split > 1 ? cg::this_cluster().map_shared_rank(&sh, b) : &sh)->found = place(lo, index_of(j, e));
                        }
                    done = true;
                }
                seen += run;
            }
            meet();
            border = sh.found;
            meet();
        }
    };

    if (par.top_k && par.top_k < a.vocab) {
        uint32_t n = 0, n_all;
        float none;
#pragma unroll
        for (int i = 0; i < kVals; ++i) n += key[i] != 0;
        sum_rough(0.0f, n, none, n_all);
        if (n_all > par.top_k) threshold(std::false_type{}, 0.0, par.top_k);
    }
    if (par.top_p < 1.0) {
        uint64_t x = 0, all;
        uint32_t c;
#pragma unroll
        for (int i = 0; i < kVals; ++i)
            if (key[i] && place(key[i], index_of(i >> 3, i & 7)) >= border) x += weight(w, sh.table, key[i]);
        sum_all(x, 0, all, c);
        threshold(std::true_type{}, fmax(par.top_p, 0.0) * static_cast<double>(all), 0);
    }
    // the draw: sums of the kept tokens by runs of 8
    const uint64_t least = par.min_p > 0.0 ? static_cast<uint64_t>(ceil(par.min_p * 8796093022208.0)) : 1;
    uint64_t run[kRounds];
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
        run[j] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t k = key[8 * j + e];
            if (k == 0 || place(k, index_of(j, e)) < border) continue;
            const uint64_t x = weight(w, sh.table, k);
            if (x >= least) run[j] += x;
        }
    }
    uint64_t mine = 0, all;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) mine += run[j];
    uint64_t in_block = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) in_block += __shfl_xor_sync(0xffffffffu, in_block, o);
    share(in_block, 0);
    uint64_t before = 0;  // of the blocks before this one
    all = 0;
    for (uint32_t i = 0; i < split * kWarps; ++i) {
        if (i / kWarps < rank) before += sh.sums[turn][i];
        all += sh.sums[turn][i];
    }
    turn ^= 1;
    const float u = a.uniform[row];
    const double at = (u > 0.0f ? static_cast<double>(fminf(u, 1.0f)) : 0.0) * static_cast<double>(all);
    const uint64_t point = min(static_cast<uint64_t>(at), all - 1);  // the first token whose sum passes it
    uint64_t* const parts = sh.mass;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
        uint64_t x = run[j];
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) parts[j * kWarps + warp] = x;
        __syncthreads();
        uint64_t total = 0, prefix = 0;
        for (int i = 0; i < kWarps; ++i) {
            if (i < warp) prefix += parts[j * kWarps + i];
            total += parts[j * kWarps + i];
        }
        uint64_t sum = before + prefix + x - run[j];
        if (sum <= point && point < sum + run[j]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t k = key[8 * j + e];
                if (k == 0 || place(k, index_of(j, e)) < border) continue;
                const uint64_t y = weight(w, sh.table, k);
                if (y < least) continue;
                if (sum <= point && point < sum + y) {
                    a.tokens[row] = static_cast<int32_t>(index_of(j, e));
                    if (a.log_probs) a.log_probs[row] = static_cast<float>(log(static_cast<double>(y) / static_cast<double>(all)));
                }
                sum += y;
            }
        }
        before += total;
    }
    if (split > 1) cg::this_cluster().sync();  // (no block ends while another writes to it)
}

template <typename T, int kThreads, int kVals> cudaError_t launch(const TokenArgs& a, uint32_t split, cudaStream_t s) {
    auto* kernel = sample_kernel<T, kThreads, kVals>;
    const int vectors = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.stride * sizeof(T) % 16 == 0;
    if (split > 8) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.rows * split);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, split, vectors);
}

template <typename T> cudaError_t by_vocab(const TokenArgs& a, cudaStream_t s) {
    if (a.vocab <= 1024) return launch<T, 128, 8>(a, 1, s);
    if (a.vocab <= 4096) return launch<T, 128, 32>(a, 1, s);
    const uint32_t slices = (a.vocab + 16383) / 16384;
    uint32_t split = 1;
    while (split < slices) split *= 2;
    return launch<T, 512, 32>(a, split, s);
}

}  // namespace

cudaError_t launch_sample_tokens(const TokenArgs& a, int dtype, cudaStream_t s) {
    if (dtype == LWM_DTYPE_F32) return by_vocab<float>(a, s);
    return dtype == LWM_DTYPE_BF16 ? by_vocab<bf16>(a, s) : by_vocab<__half>(a, s);
}

}  // namespace lwm
