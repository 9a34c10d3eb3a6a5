// The next token of every row with settings of its own: temperature, top-k, top-p, min-p, and the draw by the inverse CDF in
// token order (include/gq.h, gq_sample_rows). Beside gq_sample (sample.cu), which has one setting for all rows.
//
// w_i = exp((x_i - M) / T), M the row's maximum, in float64; top-p's masses as 64-bit integers w 2^40, so that
// histograms do not depend on the order of their additions. A row is a cluster of up to eight CTAs that keep its logits in
// shared memory: they are read from memory once, and a row's work is spread where there are few rows.
//   1 the maximum
//   2 top-k: a histogram of counts over 2048 bins that are linear in x (the top 64 T nats, or the row's range where
//     that is less: what lies below weighs under e^-64 and is dropped), its crossing bin, and that bin's tokens as a list
//     that the cluster's first CTA ranks by comparing all pairs
//   3 top-p: the same with masses
//   4 every warp's kept mass, in token order; the warp that holds the target walks its tokens
// A bin of more tokens than the list holds (ties, a flat row) falls back to bisecting the float's bits with a pass over the
// row per step. Bound: latency (some ten cluster barriers); of large batches the float64 pipe, ~14 operations a token.
#include <cooperative_groups.h>

#include "gq_internal.h"

namespace cg = cooperative_groups;

namespace gq {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kBins = 2048, kList = 2048, kMostCtas = 8;
constexpr double kFixed = 1099511627776.0;  // 2^40
constexpr uint32_t kStaged = 44 * 1024;     // logits of a row that a CTA keeps at most

__device__ __forceinline__ uint32_t key_of(float f) {  // a < b as floats <=> key_of(a) < key_of(b); NaN as -inf
    const uint32_t b = f == f ? __float_as_uint(f) : 0xff800000u;
    return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }

struct Control {
    uint32_t top[2];             // this CTA's largest key, smallest above -inf
    uint32_t border, listed, low, range_lo, range_hi, owner_warp;
    unsigned long long above, target, part[2];
    double before, goal, total;
    double warp_sum[kWarps];
    unsigned long long scan[kWarps];
};
struct alignas(16) Shared {  // the logits behind it are stored four at a time
    double pow2[64];  // 2^(i / 64)
    Control ctl;
    union {
        struct {
            uint32_t lo[kBins], hi[kBins];
        } hist;
        struct {
            unsigned long long mass[kList];
            uint32_t key[kList];
        } list;
    };
};

// exp(y) for y <= 0: 2^(n / 64) from a table times the Taylor polynomial of the rest, |r| <= ln 2 / 128: r^6 / 720 < 2^-54
__device__ __forceinline__ double exp_of(double y, const double* pow2) {
    if (!(y > -700.0)) return 0.0;
    const double t = __fma_rn(y, 92.332482616893656, 6755399441055744.0);  // 64 / ln 2; 1.5 * 2^52 rounds to a whole number
    const int n = __double2loint(t);
    const double nf = t - 6755399441055744.0;
    // ln 2 / 64 in two parts, the first of 32 bits so that its product with n is exact
    double r = __fma_rn(nf, -0x1.62e42feep-7, y);
    r = __fma_rn(nf, -0x1.a39ef35793c76p-39, r);
    double p = __fma_rn(r, 1.0 / 120.0, 1.0 / 24.0);
    p = __fma_rn(p, r, 1.0 / 6.0);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    p = __fma_rn(p, r, 1.0);
    const double v = p * pow2[n & 63];
    return __hiloint2double(__double2hiint(v) + ((n >> 6) << 20), __double2loint(v));
}

__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const float* __restrict__ logits, uint32_t vocab, uint32_t slice, uint32_t staged,
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

    if (tid < 64) sh.pow2[tid] = exp2((double)tid / 64.0);
    for (uint32_t i = tid; i < kBins; i += kThreads) sh.hist.lo[i] = sh.hist.hi[i] = 0;
    const float u = uniforms[(size_t)(draws ? *draws % uniform_rows : 0u) * rows + row];
    if (tid == 0) sh.ctl.top[0] = 0, sh.ctl.top[1] = 0xffffffffu, sh.ctl.listed = 0, sh.ctl.range_lo = 0xffffffffu, sh.ctl.range_hi = 0;
    __syncthreads();
    if (draws && tid == 0) {  // the last CTA to have read the counter advances it
        __threadfence();
        if (atomicAdd(ticket, 1u) == gridDim.x - 1) *ticket = 0, *draws += 1;
    }

    // 1: the row into shared memory, its largest and smallest values
    const uint32_t none = key_of(__uint_as_float(0xff800000u));
    uint32_t mk = 0, lk = 0xffffffffu;
    auto see = [&](float v) {
        const uint32_t k = key_of(v);
        mk = max(mk, k);
        if (k != none) lk = min(lk, k);
    };
    uint32_t i0 = 0;
    if (staged && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
        i0 = n & ~3u;
#pragma unroll 4
        for (uint32_t i = 4 * tid; i < i0; i += 4 * kThreads) {
            const float4 v = __ldcs(reinterpret_cast<const float4*>(x + i));
            *reinterpret_cast<float4*>(stage + i) = v;
            see(v.x), see(v.y), see(v.z), see(v.w);
        }
    }
#pragma unroll 4
    for (uint32_t i = i0 + tid; i < n; i += kThreads) {
        const float v = x[i];
        if (staged) stage[i] = v;
        see(v);
    }
    const float* xs = staged ? stage : x;
    mk = __reduce_max_sync(0xffffffffu, mk), lk = __reduce_min_sync(0xffffffffu, lk);
    if (lane == 0) atomicMax(&sh.ctl.top[0], mk), atomicMin(&sh.ctl.top[1], lk);
    cluster.sync();
    for (uint32_t c = 0; c < ctas; ++c) {
        const Control& o = cluster.map_shared_rank(&sh, c)->ctl;
        mk = max(mk, o.top[0]), lk = min(lk, o.top[1]);
    }

    if (mk == none) {  // every logit is -inf
        if (rank == 0 && tid == 0) {
            tokens[row] = -1;
            if (probs) probs[row] = 0.0f;
        }
        cluster.sync();  // nobody leaves while its shared memory may be read
        return;
    }
    const float M = value_of(mk), tf = temperature[row];
    const bool greedy = !(tf > 0.0f);
    const double Md = (double)M, inv_t = greedy ? 0.0 : 1.0 / (double)tf;
    const float per_x = fmaxf(32.0f / tf, (float)(kBins - 1) / (M - value_of(lk)));
    auto weight = [&](uint32_t key, float v) { return key == mk ? 1.0 : exp_of(((double)v - Md) * inv_t, sh.pow2); };
    auto fixed = [&](uint32_t key) { return (unsigned long long)(weight(key, value_of(key)) * kFixed + 0.5); };
    auto bin_of = [&](uint32_t key, float v) {  // monotone in the key
        const float f = key == mk ? 0.0f : (M - v) * per_x;
        return f < (float)kBins ? (int)f : -1;
    };
    uint32_t low = greedy ? mk : none + 1;  // keys below are dropped

    // the smallest key above which there is less than the target: of tokens (by_mass false) or of mass
    auto select = [&](bool by_mass, double share, unsigned long long count) {
        for (uint32_t i = tid; i < n; i += kThreads) {
            const float v = xs[i];
            const uint32_t key = key_of(v);
            const int b = bin_of(key, v);
            if (b < 0 || key < low) continue;
            if (!by_mass) {
                atomicAdd(&sh.hist.lo[b], 1u);
            } else {
                const unsigned long long m = fixed(key);
                const uint32_t l = (uint32_t)m, was = atomicAdd(&sh.hist.lo[b], l);
                const uint32_t h = (uint32_t)(m >> 32) + (was + l < was);
                if (h) atomicAdd(&sh.hist.hi[b], h);
            }
        }
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
        if (rank == 0) {  // the crossing bin: a scan, four bins a thread
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
            unsigned long long above = upto - mine, all = 0;
            for (uint32_t w = 0; w < (uint32_t)kWarps; ++w) {
                if (w < warp) above += sh.ctl.scan[w];
                all += sh.ctl.scan[w];
            }
            // less than the target <=> below this whole number; the largest token always stays
            const unsigned long long target = by_mass ? (unsigned long long)fmax(ceil(share * (double)all), 1.0) : count;
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                if (above < target && above + m[j] >= target) sh.ctl.border = tid * kPer + j, sh.ctl.above = above, sh.ctl.target = target;
                above += m[j];
            }
        }
        cluster.sync();
        const int border = (int)lead->ctl.border;
        if (border == (int)kBins) return;  // everything stays
        const unsigned long long above = lead->ctl.above, target = lead->ctl.target;
        uint32_t lo = 0xffffffffu, hi = 0;
        for (uint32_t i = tid; i < n; i += kThreads) {
            const float v = xs[i];
            const uint32_t key = key_of(v);
            if (key < low || bin_of(key, v) != border) continue;
            lo = min(lo, key), hi = max(hi, key);
            const uint32_t at = atomicAdd(&lead->ctl.listed, 1u);
            if (at < kList) lead->list.key[at] = key, lead->list.mass[at] = by_mass ? fixed(key) : 1ull;
        }
        lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) atomicMin(&lead->ctl.range_lo, lo), atomicMax(&lead->ctl.range_hi, hi);
        cluster.sync();
        const uint32_t listed = lead->ctl.listed;
        lo = lead->ctl.range_lo, hi = lead->ctl.range_hi;
        if (listed <= kList) {
            if (rank == 0) {
                uint32_t least = hi;
                for (uint32_t i = tid; i < listed; i += kThreads) {
                    const uint32_t key = sh.list.key[i];
                    unsigned long long over = above;
                    for (uint32_t j = 0; j < listed; ++j)
                        if (sh.list.key[j] > key) over += sh.list.mass[j];
                    if (over < target) least = min(least, key);
                }
                least = __reduce_min_sync(0xffffffffu, least);
                if (tid == 0) sh.ctl.low = hi;
                __syncthreads();
                if (lane == 0) atomicMin(&sh.ctl.low, least);
            }
            cluster.sync();
            low = lead->ctl.low;
        } else {
            for (uint32_t round = 0; lo < hi; ++round) {  // the same bounds in every thread of the cluster
                const uint32_t mid = lo + (hi - lo) / 2;
                unsigned long long over = 0;
                for (uint32_t i = tid; i < n; i += kThreads) {
                    const float v = xs[i];
                    const uint32_t key = key_of(v);
                    if (key > mid && key >= low && bin_of(key, v) == border) over += by_mass ? fixed(key) : 1ull;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) over += __shfl_xor_sync(0xffffffffu, over, o);
                if (lane == 0) sh.ctl.scan[warp] = over;
                __syncthreads();
                if (tid == 0) {
                    unsigned long long sum = 0;
                    for (int w = 0; w < kWarps; ++w) sum += sh.ctl.scan[w];
                    sh.ctl.part[round & 1] = sum;
                }
                cluster.sync();
                unsigned long long sum = above;
                for (uint32_t c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(&sh, c)->ctl.part[round & 1];
                if (sum < target) hi = mid;
                else lo = mid + 1;
            }
            cluster.sync();  // the sums may still be read
            low = lo;
        }
    };
    if (!greedy) {
        const int32_t k = top_k[row];
        const float p = top_p[row];
        const bool by_k = k > 0 && (uint32_t)k < vocab, by_p = p < 1.0f;
        if (by_k) select(false, 0.0, (unsigned long long)k);
        if (by_k && by_p) {  // the histogram and the list share their memory
            cluster.sync();
            for (uint32_t i = tid; i < kBins; i += kThreads) sh.hist.lo[i] = sh.hist.hi[i] = 0;
            if (tid == 0) sh.ctl.listed = 0, sh.ctl.range_lo = 0xffffffffu, sh.ctl.range_hi = 0;
            cluster.sync();
        }
        if (by_p) select(true, (double)p, 0);
    }

    // 4: the draw. A warp owns consecutive tokens.
    const double least = greedy ? 0.0 : (double)min_p[row];
    auto kept = [&](float v) -> double {
        const uint32_t key = key_of(v);
        if (key < low || bin_of(key, v) < 0) return 0.0;
        const double w = weight(key, v);
        return w >= least || key == mk ? w : 0.0;
    };
    const uint32_t span = (n + kThreads - 1) / kThreads * 32, w0 = min(warp * span, n), w1 = min(w0 + span, n);
    double sum = 0.0;
    for (uint32_t i = w0 + lane; i < w1; i += 32) sum += kept(xs[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.ctl.warp_sum[warp] = sum;
    cluster.sync();
    if (warp == 0) {  // every CTA finds the warp that holds the target: lane = four of the cluster's warps, in order
        constexpr uint32_t kPer = kMostCtas * kWarps / 32;
        double s[kPer], mine = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) {
            const uint32_t w = lane * kPer + j;
            s[j] = w < ctas * kWarps ? cluster.map_shared_rank(&sh, w / kWarps)->ctl.warp_sum[w % kWarps] : 0.0;
            mine += s[j];
        }
        double upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += y;
        }
        const double total = __shfl_sync(0xffffffffu, upto, 31), goal = greedy ? 0.0 : (double)u * total;
        double before = __shfl_up_sync(0xffffffffu, upto, 1);
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
        const double goal = sh.ctl.goal;
        double run = sh.ctl.before;
        uint32_t chosen = 0;
        double share = 0.0;
        for (uint32_t i = w0; i < w1; i += 32) {
            const double w = i + lane < w1 ? kept(xs[i + lane]) : 0.0;
            const uint32_t some = __ballot_sync(0xffffffffu, w > 0.0);
            if (!some) continue;
            double upto = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += y;
            }
            const uint32_t over = __ballot_sync(0xffffffffu, w > 0.0 && run + upto > goal);
            const int pick = over ? __ffs(over) - 1 : 31 - __clz(some);  // else the last one, should no more come
            chosen = i + pick, share = __shfl_sync(0xffffffffu, w, pick);
            if (over) break;
            run += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) {
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
    // CTAs of a row: as many as give each 4096 tokens while two CTAs an SM hold all rows, and what its shared memory needs
    uint32_t ctas = 1;
    while (ctas < kMostCtas && ((vocab / ctas >= 8192 && rows * ctas * 2 <= 2u * (uint32_t)sm_count) || (vocab + ctas - 1) / ctas > kStaged)) ctas *= 2;
    const uint32_t slice = ((vocab + ctas - 1) / ctas + 3) / 4 * 4, staged = slice <= kStaged;
    const size_t smem = sizeof(Shared) + (staged ? slice * 4 : 0);
    GQ_CUDA(cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * ctas), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    GQ_CUDA(cudaLaunchKernelEx(&cfg, sample_rows_kernel, logits, vocab, slice, staged, temperature, top_k, top_p, min_p, uniforms, uniform_rows, draws,
                               tokens, probs, ticket));
}

}  // namespace gq
