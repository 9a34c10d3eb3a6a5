// The next token of every row with settings of its own: temperature, top-k, top-p, min-p, and the draw by the inverse CDF in
// token order (include/gq.h, gq_sample_rows). Beside gq_sample (sample.cu), which has one setting for all rows.
//
// w_i = exp((x_i - M) / T), M the row's maximum, in float64, and so the draw's sums; what top-p compares is added by atomics, as whole
// numbers w 2^40, so that no result depends on their order. A row is a cluster of up to eight CTAs that keep its logits in shared memory: they
// are read from memory once, and a row's work is spread where there are few rows. "Bins" are 2048 steps linear in x over
// the top 64 T nats, or over the row's range where that is less; what lies below weighs under e^-64 and is dropped.
//   1 every thread's maximum, the row's maximum
//   2 top-k, as long as there are k threads: the threads' maxima alone go into a histogram; at least k tokens lie in or above the
//     bin where it reaches k. Those are listed in the first CTA's shared memory, and it finishes the row alone: it
//     counts for every listed token how many and how much lie above, and lays the kept ones' weights out in token order.
//   3 otherwise, for top-k and then top-p: a histogram of all tokens (counts or masses), its crossing bin, and that bin's
//     tokens as a list that is ranked the same way, or bisected where it is long
//   4 every thread's kept mass, a thread owning consecutive tokens; the thread that holds the target walks its own
// A bin of more tokens than the list holds (ties, a flat row) falls back to bisecting the float's bits with a pass over the
// row per step.
//
// Bound: latency and instruction issue, not memory: one row of 151936 (0.6 MB) takes 13.4 us, 64 rows (39 MB, 5.9 us at the rate
// of a copy) 73, 200 rows of 32003 (26 MB, 3.9 us) 40.5. 15 us of the 73 go into reading the rows into shared memory, 30 into
// the masses' histogram (a float64 exponential a token, 33 instructions, and an atomic addition), 18 into listing and ranking
// its crossing bin, 10 into the draw; 64 rows of eight CTAs run as two waves, since 39 MB do not fit the SMs at once.
#include <cooperative_groups.h>

#include "gq_internal.h"

namespace cg = cooperative_groups;

namespace gq {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kBins = 2048, kList = 2048, kMostCtas = 8;
constexpr int kFixedBits = 40;
constexpr double kFixed = 1099511627776.0;  // 2^40
constexpr uint32_t kRanked = 96;            // tokens that are ranked by comparing all with all; more are bisected (see select)
constexpr uint32_t kStaged = 19 * 1024;     // logits of a row that a CTA keeps at most: two CTAs an SM

__device__ __forceinline__ uint32_t key_of(float f) {  // a < b as floats <=> key_of(a) < key_of(b)
    const uint32_t b = __float_as_uint(f);
    return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }
// a logit as it is compared: NaN counts as -inf, -0 is 0
__device__ __forceinline__ float clean(float v) { return v == v ? v + 0.0f : -INFINITY; }

// A float as a double without the conversion pipe: the exponent moved over, the mantissa shifted. (A zero or a denormal becomes
// a number of 2^-127, which is as good beside a logit.)
__device__ __forceinline__ double widen(float v) {
    const uint32_t b = __float_as_uint(v);
    return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
}

struct Control {
    uint32_t top[2];             // this CTA's largest key, smallest above -inf
    uint32_t border, listed, low, range_lo, range_hi, owner_warp, pick;
    unsigned long long above, target, part[2];
    double before, goal, total;
    double warp_sum[kWarps];
    unsigned long long scan[kWarps];
};
struct alignas(16) Shared {  // the logits behind it are stored four at a time
    double pow2[16];  // 2^(i / 16)
    Control ctl;
    union {
        struct {
            uint32_t lo[kBins], hi[kBins];
        } hist;
        struct {
            unsigned long long mass[kList];
            uint32_t key[kList], at[kList];  // the token's index
        } list;
    };
};

// exp(d ln 2 / 16 step) 2^PLUS + add for d <= 0, step = 16 / (T ln 2): 2^(n / 16) from a table of sixteen (as many as give the
// lanes' loads no bank conflicts) with n's whole part in its exponent, times the Taylor polynomial of 2^(f / 16), |f| <= 1/2,
// whose next term is below 2e-13. The exponent stays above 2^-1022 for all that weighs more than e^-64.
template <int PLUS>
__device__ __forceinline__ double exp_of(double d, double step, const double* pow2, double add) {
    const double t = __fma_rn(d, step, 6755399441055744.0);  // 1.5 * 2^52 rounds to a whole number
    const int n = __double2loint(t);
    const double f = __fma_rn(d, step, -(t - 6755399441055744.0));
    double p = __fma_rn(f, 1.271587195055813e-09, 1.467610032291943e-07);  // (ln 2 / 16)^k / k!
    p = __fma_rn(p, f, 1.3550807779497455e-05);
    p = __fma_rn(p, f, 0.0009383847928089871);
    p = __fma_rn(p, f, 0.04332169878499658);
    p = __fma_rn(p, f, 1.0);
    const double v = pow2[n & 15];
    return __fma_rn(p, __hiloint2double(__double2hiint(v) + (n & ~15) * 65536 + PLUS * 1048576, __double2loint(v)), add);
}

// STAGED: a CTA's logits fit its shared memory.
template <bool STAGED>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const float* __restrict__ logits, uint32_t vocab, uint32_t slice,
                                                                 const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
                                                                 const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                                 const float* __restrict__ uniforms, uint32_t uniform_rows, uint32_t* draws, int32_t* tokens,
                                                                 float* probs, uint32_t* ticket) {
    GQ_GRID_DEP_SYNC();
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    float* stage = reinterpret_cast<float*>(smem + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / ctas, rows = gridDim.x / ctas;
    const uint32_t first = min(rank * slice, vocab), n = min(slice, vocab - first);
    const float* x = logits + (size_t)row * vocab + first;
    Shared* lead = cluster.map_shared_rank(&sh, 0);

    if (tid < 16) sh.pow2[tid] = exp2((double)tid / 16.0);
    for (uint32_t i = tid; i < kBins; i += kThreads) sh.hist.lo[i] = sh.hist.hi[i] = 0;
    const float u = uniforms[(size_t)(draws ? *draws % uniform_rows : 0u) * rows + row];
    if (tid == 0) sh.ctl.top[0] = 0, sh.ctl.top[1] = 0xffffffffu, sh.ctl.listed = 0, sh.ctl.range_lo = 0xffffffffu, sh.ctl.range_hi = 0;
    __syncthreads();
    if (draws && tid == 0) {  // the last CTA to have read the counter advances it
        __threadfence();
        if (atomicAdd(ticket, 1u) == gridDim.x - 1) *ticket = 0, *draws += 1;
    }

    // 1: the row into shared memory, its largest and smallest values
    float most = -INFINITY, least_seen = INFINITY;
    auto see = [&](float v) {
        most = fmaxf(most, v);
        if (v != -INFINITY) least_seen = fminf(least_seen, v);
    };
    const uint32_t lead_in = min(n, (uint32_t)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 4), quads = (n - lead_in) / 4;
    if (STAGED) {
        // (the part on 16-byte boundaries four at a time; in shared memory the logits lie one behind the other from 0 on)
        const float4* x4 = reinterpret_cast<const float4*>(x + lead_in);
#pragma unroll 4
        for (uint32_t i = tid; i < quads; i += kThreads) {
            float4 v = __ldcs(x4 + i);
            v = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
            float* at = stage + lead_in + 4 * i;
            if (lead_in == 0) *reinterpret_cast<float4*>(at) = v;
            else at[0] = v.x, at[1] = v.y, at[2] = v.z, at[3] = v.w;
            see(v.x), see(v.y), see(v.z), see(v.w);
        }
        for (uint32_t i = tid; i < n - 4 * quads; i += kThreads) {  // the few before and behind
            const uint32_t at = i < lead_in ? i : 4 * quads + i;
            const float v = clean(x[at]);
            stage[at] = v;
            see(v);
        }
    } else {
        for (uint32_t i = tid; i < n; i += kThreads) see(clean(x[i]));
    }
    auto logit = [&](uint32_t i) { return STAGED ? stage[i] : clean(x[i]); };
    {
        const uint32_t mk = __reduce_max_sync(0xffffffffu, key_of(most)), lk = __reduce_min_sync(0xffffffffu, key_of(least_seen));
        if (lane == 0) atomicMax(&sh.ctl.top[0], mk), atomicMin(&sh.ctl.top[1], lk);
    }
    cluster.sync();
    uint32_t mk = 0, lk = 0xffffffffu;
    for (uint32_t c = 0; c < ctas; ++c) {
        const Control& o = cluster.map_shared_rank(&sh, c)->ctl;
        mk = max(mk, o.top[0]), lk = min(lk, o.top[1]);
    }
    const float M = value_of(mk), tf = temperature[row];
    if (M == -INFINITY) {  // every logit is -inf
        if (rank == 0 && tid == 0) {
            tokens[row] = -1;
            if (probs) probs[row] = 0.0f;
        }
        cluster.sync();  // nobody leaves while its shared memory may be read
        return;
    }
    const bool greedy = !(tf > 0.0f);
    const double Md = widen(M), step = greedy ? 0.0 : 23.083120654223414 / (double)tf;  // 16 / ln 2
    const float per_x = fminf(fmaxf(32.0f / tf, (float)(kBins - 1) / (M - value_of(lk))), 3e38f), top = fminf(M, 3.402823466e+38f);
    auto weight = [&](float v) { return exp_of<0>(widen(v) - Md, step, sh.pow2, 0.0); };  // of what is not below `low`; the largest's is 1
    auto fixed = [&](float v) {  // w 2^40 as a whole number, by the last place of 2^52
        return (unsigned long long)__double_as_longlong(exp_of<kFixedBits>(widen(v) - Md, step, sh.pow2, 4503599627370496.0)) & 0xfffffffffffffull;
    };
    // falls as v rises; rounded by the last place of 2^23 (+inf, where that is the largest: -inf, whose last bits are 0)
    auto bin_of = [&](float v) { return (int)(__float_as_uint(fminf((top - v) * per_x, (float)(kBins - 1)) + 8388608.0f) & (kBins - 1)); };
    // tokens below are dropped: at first what weighs less than e^-64 (in a bin behind the last, too)
    float low = greedy ? M : fmaxf(M - 64.0f * tf, -3.402823466e+38f);

    // adds the other CTAs' histograms to the first one's
    auto gather = [&]() {
        __syncthreads();
        if (rank != 0)
            for (uint32_t b = tid; b < kBins; b += kThreads) {
                const uint32_t l = sh.hist.lo[b];
                uint32_t h = sh.hist.hi[b];
                if (l) {
                    const uint32_t was = atomicAdd(&lead->hist.lo[b], l);
                    h += was + l < was;
                }
                if (h) atomicAdd(&lead->hist.hi[b], h);
            }
        cluster.sync();
    };
    // The bin where the first CTA's histogram reaches the target (the count, or a share of the whole); kBins: nowhere.
    auto cross = [&](bool by_mass, double share, unsigned long long count) {
        if (rank == 0) {  // a scan, some bins a thread
            constexpr uint32_t kPer = kBins / kThreads;
            unsigned long long m[kPer], mine = 0;
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                const uint32_t b = tid * kPer + j;
                m[j] = (unsigned long long)sh.hist.hi[b] << 32 | sh.hist.lo[b];
                mine += m[j];
            }
            unsigned long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += y;
            }
            if (lane == 31) sh.ctl.scan[warp] = upto;
            if (tid == 0) sh.ctl.border = kBins;
            __syncthreads();
            unsigned long long sums = lane < kWarps ? sh.ctl.scan[lane] : 0ull, upto_warp = sums;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, upto_warp, o);
                if (lane >= (uint32_t)o) upto_warp += y;
            }
            const unsigned long long all = __shfl_sync(0xffffffffu, upto_warp, 31);
            unsigned long long above = upto - mine + __shfl_sync(0xffffffffu, upto_warp - sums, warp);
            // less than the target <=> below this whole number; the largest token always stays
            const unsigned long long target = by_mass ? (unsigned long long)fmax(ceil(share * (double)all), 1.0) : count;
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                if (above < target && above + m[j] >= target) sh.ctl.border = tid * kPer + j, sh.ctl.above = above, sh.ctl.target = target;
                above += m[j];
            }
        }
        cluster.sync();
        return (int)lead->ctl.border;
    };
    // Over the list of the first CTA, for a token each: the sum of what `other(i, j)` gives over all j. A token is shared by a
    // few lanes of a warp, so that each has some eight others to look at and few warps take part.
    auto each_listed = [&](uint32_t listed, auto other, auto done) {
        uint32_t bits = 0;
        while (bits < 5 && (16u << bits) <= listed && (listed << (bits + 1)) <= (uint32_t)kThreads) ++bits;
        const uint32_t part = tid & ((1u << bits) - 1);
        for (uint32_t i0 = 0; i0 < listed; i0 += kThreads >> bits) {
            const uint32_t i = i0 + (tid >> bits);
            if (i - lane / (1u << bits) >= listed) break;  // the whole warp is behind the list
            unsigned long long sum = 0;
            if (i < listed) {
#pragma unroll 4
                for (uint32_t j = part; j < listed; j += 1u << bits) sum += other(i, j);
            }
            for (uint32_t o = 1u << bits >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (i < listed && part == 0) done(i, sum);
        }
    };
    auto warp_sum = [](unsigned long long v) {  // in pieces of 22 bits
        const uint32_t lo = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3fffffu), mid = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 22) & 0x3fffffu);
        return lo + ((unsigned long long)mid << 22) + ((unsigned long long)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 44)) << 44);
    };
    auto block_sum = [&](unsigned long long v) {  // of the CTA's threads, the same for all
        v = warp_sum(v);
        if (lane == 0) sh.ctl.scan[warp] = v;
        __syncthreads();
        v = warp_sum(lane < kWarps ? sh.ctl.scan[lane] : 0ull);
        __syncthreads();
        return v;
    };
    auto clear_lists = [&]() {  // the histogram and the list share their memory
        cluster.sync();
        for (uint32_t i = tid; i < kBins; i += kThreads) sh.hist.lo[i] = sh.hist.hi[i] = 0;
        if (tid == 0) sh.ctl.listed = 0, sh.ctl.range_lo = 0xffffffffu, sh.ctl.range_hi = 0;
        cluster.sync();
    };
    // calls `take` with every logit of at least `bound`, eight loads in flight
    auto every = [&](float bound, auto take) {
        constexpr uint32_t kAtOnce = 8;
        for (uint32_t i = tid; i < n; i += kAtOnce * kThreads) {
            float v[kAtOnce];
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j) v[j] = i + j * kThreads < n ? logit(i + j * kThreads) : -INFINITY;
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j)
                if (v[j] >= bound) take(v[j], i + j * kThreads);
        }
    };

    // raises `low` to the smallest value above which there is less than the target: of tokens (by_mass false) or of mass
    auto select = [&](bool by_mass, double share, unsigned long long count) {
        if (!by_mass) {
            every(low, [&](float v, uint32_t) { atomicAdd(&sh.hist.lo[bin_of(v)], 1u); });
        } else {
            // (the exponentials of four tokens side by side: one is a chain of fourteen float64 operations)
            constexpr uint32_t kAtOnce = 4;
            for (uint32_t i = tid; i < n; i += kAtOnce * kThreads) {
                float v[kAtOnce];
                unsigned long long m[kAtOnce];
#pragma unroll
                for (uint32_t j = 0; j < kAtOnce; ++j) v[j] = i + j * kThreads < n ? logit(i + j * kThreads) : -INFINITY;
#pragma unroll
                for (uint32_t j = 0; j < kAtOnce; ++j) m[j] = fixed(v[j]);
#pragma unroll
                for (uint32_t j = 0; j < kAtOnce; ++j) {
                    if (v[j] < low) continue;
                    const int b = bin_of(v[j]);
                    const uint32_t l = (uint32_t)m[j], was = atomicAdd(&sh.hist.lo[b], l);
                    const uint32_t h = (uint32_t)(m[j] >> 32) + (was + l < was);
                    if (h) atomicAdd(&sh.hist.hi[b], h);
                }
            }
        }
        gather();
        const int border = cross(by_mass, share, count);
        if (border == (int)kBins) return;  // everything stays
        const unsigned long long above = lead->ctl.above, target = lead->ctl.target;
        uint32_t lo = 0xffffffffu, hi = 0;
        every(fmaxf(low, M - ((float)border + 1.0f) / per_x), [&](float v, uint32_t) {
            if (bin_of(v) != border) return;
            const uint32_t key = key_of(v), at = atomicAdd(&lead->ctl.listed, 1u);
            lo = min(lo, key), hi = max(hi, key);
            if (at < kList) lead->list.key[at] = key, lead->list.mass[at] = by_mass ? fixed(v) : 1ull;
        });
        lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0 && lo <= hi) atomicMin(&lead->ctl.range_lo, lo), atomicMax(&lead->ctl.range_hi, hi);
        cluster.sync();
        const uint32_t listed = lead->ctl.listed;
        lo = lead->ctl.range_lo, hi = lead->ctl.range_hi;
        if (listed <= kList) {
            if (rank == 0) {
                if (listed <= kRanked) {
                    if (tid == 0) sh.ctl.low = hi;
                    __syncthreads();
                    each_listed(
                        listed,
                        [&](uint32_t i, uint32_t j) { return sh.list.key[j] > sh.list.key[i] ? sh.list.mass[j] : 0ull; },
                        [&](uint32_t i, unsigned long long mass) {
                            if (above + mass < target) atomicMin(&sh.ctl.low, sh.list.key[i]);
                        });
                } else {
                    // The floats' bits bisected, every thread with its tokens in registers: 3.3k cycles however many they are, where
                    // comparing all with all takes 2k for 60 tokens and 12k for 250. (64 rows of 151936: 74.6 us with the bisection
                    // alone, 78.3 without it, 72.9 from 96 tokens on; 200 rows of 32003: 43.9, 40.0, 40.0.)
                    constexpr uint32_t kPer = kList / kThreads;
                    uint32_t key[kPer];
                    unsigned long long mass[kPer];
#pragma unroll
                    for (uint32_t j = 0; j < kPer; ++j) {
                        const uint32_t i = tid + j * kThreads;
                        key[j] = i < listed ? sh.list.key[i] : 0u, mass[j] = i < listed ? sh.list.mass[i] : 0ull;
                    }
                    while (lo < hi) {
                        const uint32_t mid = lo + (hi - lo) / 2;
                        unsigned long long over = 0;
#pragma unroll
                        for (uint32_t j = 0; j < kPer; ++j) over += key[j] > mid ? mass[j] : 0ull;
                        if (above + block_sum(over) < target) hi = mid;
                        else lo = mid + 1;
                    }
                    if (tid == 0) sh.ctl.low = lo;
                }
            }
            cluster.sync();
            low = value_of(lead->ctl.low);
        } else {
            for (uint32_t round = 0; lo < hi; ++round) {  // the same bounds in every thread of the cluster
                const uint32_t mid = lo + (hi - lo) / 2;
                unsigned long long over = 0;
                every(low, [&](float v, uint32_t) {
                    if (key_of(v) > mid && bin_of(v) == border) over += by_mass ? fixed(v) : 1ull;
                });
                over = block_sum(over);
                if (tid == 0) sh.ctl.part[round & 1] = over;
                cluster.sync();
                unsigned long long sum = above;
                for (uint32_t c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(&sh, c)->ctl.part[round & 1];
                if (sum < target) hi = mid;
                else lo = mid + 1;
            }
            cluster.sync();  // the sums may still be read
            low = value_of(lo);
        }
    };
    const double least = greedy ? 0.0 : (double)min_p[row];
    const float p = greedy ? 1.0f : top_p[row];
    const int32_t k = greedy ? 0 : top_k[row];
    const bool by_k = k > 0 && (uint32_t)k < vocab, by_p = p < 1.0f;
    if (by_k) {
        // 2: at least k tokens lie in or above the bin where the threads' maxima reach k
        if (most >= low) atomicAdd(&sh.hist.lo[bin_of(most)], 1u);
        gather();
        const int border = cross(false, 0.0, (unsigned long long)k);
        if (border != (int)kBins) {
            // (no value below this is in such a bin, whatever its rounding)
            every(fmaxf(low, M - ((float)border + 1.0f) / per_x), [&](float v, uint32_t i) {
                if (bin_of(v) > border) return;
                const uint32_t at = atomicAdd(&lead->ctl.listed, 1u);
                if (at < kList) lead->list.key[at] = key_of(v), lead->list.at[at] = first + i, lead->list.mass[at] = fixed(v);
            });
            cluster.sync();
            const uint32_t listed = lead->ctl.listed;
            if (listed <= kList) {
                if (rank == 0) {
                    // what lies above a token, of all (counted) and of those top-k keeps
                    if (tid == 0) sh.ctl.low = mk, sh.ctl.pick = 0xffffffffu;
                    __syncthreads();
                    unsigned long long kept_mass = 0;  // of this thread's tokens
                    each_listed(
                        listed, [&](uint32_t i, uint32_t j) { return sh.list.key[j] > sh.list.key[i] ? 1ull : 0ull; },
                        [&](uint32_t i, unsigned long long count) {
                            if (count < (unsigned long long)k) atomicMin(&sh.ctl.low, sh.list.key[i]), kept_mass += sh.list.mass[i];
                        });
                    const unsigned long long of_k = block_sum(kept_mass);
                    const uint32_t kth = sh.ctl.low;
                    const unsigned long long target = by_p ? (unsigned long long)fmax(ceil((double)p * (double)of_k), 1.0) : ~0ull;
                    unsigned long long kept = 0;
                    // out of the list goes what top-k, top-p or min-p drop: its index becomes one beyond all
                    each_listed(
                        listed,
                        [&](uint32_t i, uint32_t j) { return sh.list.key[j] > sh.list.key[i] ? sh.list.mass[j] : 0ull; },
                        [&](uint32_t i, unsigned long long mass) {
                            const uint32_t key = sh.list.key[i];
                            const bool keep = key == mk || (key >= kth && mass < target && weight(value_of(key)) >= least);
                            if (keep) ++kept;
                            else sh.list.at[i] |= 0x80000000u;
                        });
                    kept = block_sum(kept);
                    // the draw, in float64 as below: the kept weights in token order (in the masses' place; a token's place in its key's)
                    double* const w = reinterpret_cast<double*>(sh.list.mass);
                    each_listed(
                        listed, [&](uint32_t i, uint32_t j) { return sh.list.at[j] < sh.list.at[i] ? 1ull : 0ull; },
                        [&](uint32_t i, unsigned long long place) {
                            const uint32_t key = sh.list.key[i];
                            const bool in = sh.list.at[i] >> 31 == 0;
                            if (in) w[place] = weight(value_of(key));
                            sh.list.key[i] = in ? (uint32_t)place : 0xffffffffu;
                        });
                    __syncthreads();
                    const uint32_t each = ((uint32_t)kept + kThreads - 1) / kThreads, t0 = min(tid * each, (uint32_t)kept), t1 = min(t0 + each, (uint32_t)kept);
                    double sum = 0.0;
                    for (uint32_t t = t0; t < t1; ++t) sum += w[t];
                    double upto = sum;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double y = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= (uint32_t)o) upto += y;
                    }
                    if (lane == 31) sh.ctl.warp_sum[warp] = upto;
                    __syncthreads();
                    double total = 0.0, run = 0.0;
                    for (uint32_t i = 0; i < kWarps; ++i) {
                        if (i == warp) run = total;
                        total += sh.ctl.warp_sum[i];
                    }
                    run += upto - sum;
                    const double goal = (double)u * total;
                    for (uint32_t t = t0; t < t1; ++t) {
                        run += w[t];
                        if (run > goal) {
                            atomicMin(&sh.ctl.pick, t);
                            break;
                        }
                    }
                    __syncthreads();
                    const uint32_t chosen = min(sh.ctl.pick, (uint32_t)kept - 1);  // the target at the very end: the last kept token
                    for (uint32_t i = tid; i < listed; i += kThreads)
                        if (sh.list.key[i] == chosen) {
                            tokens[row] = (int32_t)sh.list.at[i];
                            if (probs) probs[row] = (float)(w[chosen] / total);
                        }
                }
                cluster.sync();  // nobody leaves while its shared memory may be read
                return;
            }
        }
        // 3: more than k threads' worth, or more tokens beside the k-th than the list holds
        clear_lists();
        select(false, 0.0, (unsigned long long)k);
        if (by_p) clear_lists();
    }
    if (by_p) select(true, (double)p, 0);

    // 4: the draw. A thread owns `per` consecutive tokens, an odd number so that its warp's loads meet no bank conflicts.
    // (min_p's own test is in float64; below `near` the weight is under it for certain)
    const float near = least > 0.0 ? fmaxf(low, fminf(M + tf * (__logf((float)least) * 1.0001f - 0.001f) - fabsf(M) * 1e-6f, M)) : low;
    auto kept = [&](float v) -> double {
        const double w = weight(v);
        return w >= least || v == M ? w : 0.0;
    };
    const uint32_t per = ((n + kThreads - 1) / kThreads) | 1, t0 = min(tid * per, n), t1 = min(t0 + per, n);
    double sum = 0.0;
    for (uint32_t i = t0; i < t1; i += 8) {
        float v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = i + j < t1 ? logit(i + j) : -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (v[j] >= near) sum += kept(v[j]);
    }
    double upto = sum;  // of the warp's threads, in order
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= (uint32_t)o) upto += y;
    }
    if (lane == 31) sh.ctl.warp_sum[warp] = upto;
    cluster.sync();
    if (warp == 0) {  // every CTA finds the warp that holds the target: lane = some of the cluster's warps, in order
        constexpr uint32_t kPer = kMostCtas * kWarps / 32;
        double s[kPer], mine = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) {
            const uint32_t w = lane * kPer + j;
            s[j] = w < ctas * kWarps ? cluster.map_shared_rank(&sh, w / kWarps)->ctl.warp_sum[w % kWarps] : 0.0;
            mine += s[j];
        }
        double through = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, through, o);
            if (lane >= (uint32_t)o) through += y;
        }
        const double total = __shfl_sync(0xffffffffu, through, 31), goal = greedy ? 0.0 : (double)u * total;
        double before = __shfl_up_sync(0xffffffffu, through, 1);
        if (lane == 0) before = 0.0;
        uint32_t hit = 0xffffffffu, last = 0;
        double hit_before = 0.0, last_before = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) {
            if (s[j] > 0.0) {
                last = lane * kPer + j + 1, last_before = before;
                if (hit == 0xffffffffu && before + s[j] > goal) hit = lane * kPer + j, hit_before = before;
            }
            before += s[j];
        }
        const uint32_t owner = __reduce_min_sync(0xffffffffu, hit), end = __reduce_max_sync(0xffffffffu, last) - 1;
        const uint32_t at = owner != 0xffffffffu ? owner : end;  // the target at the very end: the last kept token
        const double own_before = __shfl_sync(0xffffffffu, owner != 0xffffffffu ? hit_before : last_before, at / kPer);
        if (lane == 0) sh.ctl.owner_warp = at, sh.ctl.before = own_before, sh.ctl.goal = goal, sh.ctl.total = total;
    }
    __syncthreads();
    if (sh.ctl.owner_warp == rank * kWarps + warp) {
        // the first thread that passes the target, else the last that keeps anything; it walks its tokens
        const double goal = sh.ctl.goal, before = sh.ctl.before;
        const uint32_t over = __ballot_sync(0xffffffffu, sum > 0.0 && before + upto > goal), some = __ballot_sync(0xffffffffu, sum > 0.0);
        const uint32_t owner = over ? __ffs(over) - 1 : 31 - __clz(some);
        if (lane == owner) {
            double run = before + (upto - sum), share = 0.0;
            uint32_t chosen = 0;
            for (uint32_t i = t0; i < t1; ++i) {
                const float v = logit(i);
                if (v < near) continue;
                const double w = kept(v);
                if (w == 0.0) continue;
                chosen = i, share = w, run += w;  // the last one, should no more come
                if (run > goal) break;
            }
            tokens[row] = (int32_t)(first + chosen);
            if (probs) probs[row] = (float)(share / sh.ctl.total);
        }
    }
    cluster.sync();  // nobody leaves while its shared memory may be read
}

}  // namespace

void launch_sample_rows(cudaStream_t s, int sm_count, const float* logits, uint32_t rows, uint32_t vocab, const float* temperature, const int32_t* top_k,
                        const float* top_p, const float* min_p, const float* uniforms, uint32_t uniform_rows, uint32_t* draws, int32_t* tokens, float* probs,
                        uint32_t* ticket) {
    // CTAs of a row: as many as leave each some thousands of tokens while the CTAs an SM holds (two) hold all rows, and as
    // many as keep the row in shared memory. (1024 threads and one CTA an SM, before the exponential and the ranking were made
    // shorter: 14.6 us for one row of 151936 against 13.6, 49 for 200 rows of 32003 against 43, 77 for 64 rows of 151936 against 84.)
    uint32_t ctas = 1;
    while (ctas < kMostCtas && ((vocab / ctas >= 8192 && rows * ctas <= (uint32_t)sm_count) || (vocab + ctas - 1) / ctas > kStaged)) ctas *= 2;
    const uint32_t slice = ((vocab + ctas - 1) / ctas + 3) / 4 * 4, staged = slice <= kStaged;
    const size_t smem = sizeof(Shared) + (staged ? slice * 4 : 0);
    auto kernel = staged ? sample_rows_kernel<true> : sample_rows_kernel<false>;
    GQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * ctas), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    GQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, logits, vocab, slice, temperature, top_k, top_p, min_p, uniforms, uniform_rows, draws,
                               tokens, probs, ticket));
}

}  // namespace gq
