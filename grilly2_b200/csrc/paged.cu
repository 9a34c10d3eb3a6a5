// The paged int8 KV cache's bookkeeping and writes (no counterpart in the reference, whose cache is contiguous and of batch
// 1: crates/grilly-infer/src/kv_cache.rs:1-33).
//
// plan: the new tokens of every request get positions, rows, blocks and slots. With c_b = counts[b] and n_b = lens[b]:
//   starts = exclusive sum of c; request b touches the table entries n_b / bs .. (n_b + c_b - 1) / bs, one RUN of rows each;
//   the r-th touched entry without a block, in order of (b, entry), takes free[free_count - 1 - r];
//   slot = table[b][p / bs] * bs + p % bs for p = n_b + (row - starts[b]).
// Both sums are block scans over the requests; runs and rows find their request by a binary search in shared memory. Few
// rows run as one CTA; many as a cluster of eight, whose first CTA hands out the blocks while the cluster barrier holds
// the others back from the table. Bound: latency (three scans); the maps are a few bytes per row.
//
// append: one CTA per run of rows that share a block, KV head and K or V (further CTAs rotate q): the largest |value| of the
// run gives the scale, the block's older codes are rounded again if it grew, the run's values are rounded and stored in
// the core-matrix order of the pool. A 32-bit word of codes has one owner, so a word that holds old and new codes is
// read and written by one thread. Bound: bytes (q | k | v read once, the k and v part twice through L1).
#include "gq_internal.h"
#include "paged.cuh"

namespace gq {

namespace {

constexpr int kPlanThreads = 1024;
constexpr uint32_t kPlanCluster = 8;

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive scan of one value per thread of the CTA, sums saturating at `cap` (which keeps them in 32 bits); *total is the sum.
__device__ uint32_t block_scan(uint32_t v, uint32_t cap, uint32_t* warp_sums, uint32_t* total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x = min(x + y, cap);
    }
    __syncthreads();  // warp_sums may still be read from the scan before
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = lane < kPlanThreads / 32 ? warp_sums[lane] : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= (uint32_t)o) s = min(s + y, cap);
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    *total = warp_sums[kPlanThreads / 32 - 1];
    const uint32_t before = warp ? warp_sums[warp - 1] : 0u;
    const uint32_t left = __shfl_up_sync(0xffffffffu, x, 1);
    return lane ? min(before + left, cap) : before;
}

// the request that owns item i: the last b with at[b] <= i, at ascending
__device__ __forceinline__ uint32_t owner_of(const uint32_t* at, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n;  // at[lo] <= i < at[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (at[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedView c, StepView s, const int32_t* __restrict__ counts,
                                                                 const int32_t* __restrict__ free_list, int32_t* free_count) {
    GQ_GRID_DEP_SYNC();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t warp_sums[32];
    uint32_t* start = smem;                  // [seqs + 1]
    uint32_t* run = start + c.seqs + 1;      // [seqs + 1]
    uint32_t* len = run + c.seqs + 1;        // [seqs]
    const uint32_t tid = threadIdx.x, per = (c.seqs + kPlanThreads - 1) / kPlanThreads, b0 = tid * per, b1 = min(b0 + per, c.seqs);
    uint32_t total, runs, sum = 0;
    for (uint32_t b = b0; b < b1; ++b) sum = min(sum + min((uint32_t)max(counts[b], 0), s.tokens), s.tokens);
    uint32_t at = block_scan(sum, s.tokens, warp_sums, &total);
    sum = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t next = min(at + min((uint32_t)max(counts[b], 0), s.tokens), s.tokens), n = paged_len(c, b);
        start[b] = at, len[b] = n;
        if (next > at) sum += ((n + (next - at) - 1) >> c.shift) - (n >> c.shift) + 1;
        at = next;
    }
    if (tid == 0) start[c.seqs] = total;
    at = block_scan(sum, s.runs_cap, warp_sums, &runs);  // (its barriers publish start and len)
    for (uint32_t b = b0; b < b1; ++b) {
        run[b] = at;
        const uint32_t rows = start[b + 1] - start[b];
        if (rows) at += ((len[b] + rows - 1) >> c.shift) - (len[b] >> c.shift) + 1;
    }
    if (tid == 0) run[c.seqs] = runs;
    __syncthreads();

    if (blockIdx.x == 0) {
        // the runs, and a block for every touched entry that has none
        const uint32_t have = (uint32_t)min(max(*free_count, 0), (int32_t)c.blocks);
        uint32_t wanted = 0;
        for (uint32_t r0 = 0; r0 < runs; r0 += kPlanThreads) {
            const uint32_t r = r0 + tid;
            int32_t* entry = nullptr;
            bool need = false;
            if (r < runs) {
                const uint32_t b = owner_of(run, c.seqs, r), j = (len[b] >> c.shift) + (r - run[b]);
                s.runs[r] = (int32_t)(r == run[b] ? start[b] : start[b] + ((j << c.shift) - len[b]));
                if (j < c.max_blocks) entry = c.table + (size_t)b * c.max_blocks + j, need = *entry < 0;
            }
            uint32_t here;
            const uint32_t rank = wanted + block_scan(need ? 1u : 0u, 0x7fffffffu, warp_sums, &here);
            if (need && rank < have) *entry = free_list[have - 1 - rank];
            wanted += here;
        }
        for (uint32_t r = runs + tid; r <= s.runs_cap; r += kPlanThreads) s.runs[r] = (int32_t)total;
        for (uint32_t b = tid; b <= c.seqs; b += kPlanThreads) {
            s.starts[b] = (int32_t)start[b];
            if (b < c.seqs) s.last[b] = start[b + 1] > start[b] ? (int32_t)start[b + 1] - 1 : -1;
        }
        if (tid == 0) {  // every thread read *free_count before the scans' barriers (or nothing was wanted)
            if (wanted) *free_count = (int32_t)(have - min(wanted, have));
            s.info[0] = (int32_t)total, s.info[1] = (int32_t)(wanted - min(wanted, have));
        }
    }
    if (gridDim.x > 1) cluster_barrier();
    else __syncthreads();
    for (uint32_t t = blockIdx.x * kPlanThreads + tid; t < s.tokens; t += gridDim.x * kPlanThreads) {
        int32_t slot = -1, pos = -1;
        if (t < total) {
            const uint32_t b = owner_of(start, c.seqs, t), p = len[b] + (t - start[b]), j = p >> c.shift;
            pos = (int32_t)p;
            if (j < c.max_blocks) {
                const int32_t e = __ldcg(c.table + (size_t)b * c.max_blocks + j);
                if (e >= 0 && (uint32_t)e < c.blocks) slot = (int32_t)(((uint32_t)e << c.shift) + (p & (c.block - 1)));
            }
        }
        s.slots[t] = slot, s.positions[t] = pos;
    }
}

__global__ void __launch_bounds__(256) paged_advance_kernel(PagedView c, StepView s) {
    GQ_GRID_DEP_SYNC();
    const uint32_t b = blockIdx.x * 256 + threadIdx.x;
    if (b >= c.seqs) return;
    const uint32_t from = paged_start(s, b), to = paged_start(s, b + 1);
    if (to > from) c.lens[b] = (int32_t)min(paged_len(c, b) + (to - from), c.max_blocks << c.shift);
}

__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(PagedView c, const int32_t* __restrict__ which, int32_t* free_list, int32_t* free_count) {
    GQ_GRID_DEP_SYNC();
    __shared__ uint32_t warp_sums[32];
    const uint32_t tid = threadIdx.x;
    uint32_t have = (uint32_t)min(max(*free_count, 0), (int32_t)c.blocks);
    for (uint32_t b = 0; b < c.seqs; ++b) {
        if (which[b] == 0) continue;  // the same for every thread
        for (uint32_t j0 = 0; j0 < c.max_blocks; j0 += kPlanThreads) {
            const uint32_t j = j0 + tid;
            int32_t e = -1;
            if (j < c.max_blocks) {
                int32_t* entry = c.table + (size_t)b * c.max_blocks + j;
                e = *entry;
                *entry = -1;
            }
            const bool held = e >= 0 && (uint32_t)e < c.blocks;
            uint32_t here;
            const uint32_t rank = have + block_scan(held ? 1u : 0u, 0x7fffffffu, warp_sums, &here);
            if (held && rank < c.blocks) free_list[rank] = e;
            have = min(have + here, c.blocks);
        }
        if (tid == 0) c.lens[b] = 0;
    }
    __syncthreads();  // every thread has read *free_count
    if (tid == 0) *free_count = (int32_t)have;
}

constexpr int kAppendThreads = 256;
constexpr uint32_t kQHeads = 4;  // heads of q a CTA rotates

// four values of a rotated row and the four half a head further: x cos + rot(x) sin, each operation rounded on its own
__device__ __forceinline__ void rotate4(const float4& lo, const float4& hi, const float* cosv, const float* sinv, uint32_t d, uint32_t half, float4& out_lo,
                                        float4& out_hi) {
    const float4 cl = *reinterpret_cast<const float4*>(cosv + d), ch = *reinterpret_cast<const float4*>(cosv + d + half);
    const float4 sl = *reinterpret_cast<const float4*>(sinv + d), sh = *reinterpret_cast<const float4*>(sinv + d + half);
    out_lo.x = __fadd_rn(__fmul_rn(lo.x, cl.x), __fmul_rn(-hi.x, sl.x)), out_lo.y = __fadd_rn(__fmul_rn(lo.y, cl.y), __fmul_rn(-hi.y, sl.y));
    out_lo.z = __fadd_rn(__fmul_rn(lo.z, cl.z), __fmul_rn(-hi.z, sl.z)), out_lo.w = __fadd_rn(__fmul_rn(lo.w, cl.w), __fmul_rn(-hi.w, sl.w));
    out_hi.x = __fadd_rn(__fmul_rn(hi.x, ch.x), __fmul_rn(lo.x, sh.x)), out_hi.y = __fadd_rn(__fmul_rn(hi.y, ch.y), __fmul_rn(lo.y, sh.y));
    out_hi.z = __fadd_rn(__fmul_rn(hi.z, ch.z), __fmul_rn(lo.z, sh.z)), out_hi.w = __fadd_rn(__fmul_rn(hi.w, ch.w), __fmul_rn(lo.w, sh.w));
}

// bits of |v|: as integers they order like the values, with infinity and NaN on top, so the maximum keeps them
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t mag4(const float4& v) { return max(max(mag(v.x), mag(v.y)), max(mag(v.z), mag(v.w))); }

// rint(v / s) in the codes' range; an empty scale (all zeros) and a value that is not a number give 0
__device__ __forceinline__ uint32_t code_of(float v, float s) {
    const float r = s == 0.0f ? 0.0f : __fdiv_rn(v, s);
    return (uint32_t)max(-127, min(127, __float2int_rn(r))) & 0xffu;
}
__device__ __forceinline__ uint32_t recode(uint32_t word, uint32_t byte, float ratio) {
    return (uint32_t)__float2int_rn(__fmul_rn((float)(int8_t)(word >> (8 * byte)), ratio)) & 0xffu;
}

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(PagedView c, StepView s, const float* __restrict__ qkv, uint32_t heads,
                                                                     const float* __restrict__ cosv, const float* __restrict__ sinv, uint32_t max_pos,
                                                                     float* __restrict__ q_out) {
    GQ_GRID_DEP_SYNC();
    __shared__ uint32_t most[kAppendThreads / 32];
    const uint32_t tid = threadIdx.x, dim = c.dim, half = dim / 2, quads = half / 4, pitch = (heads + 2 * c.kv_heads) * dim;
    const uint32_t total = paged_start(s, c.seqs);
    const uint32_t r = blockIdx.x;
    const uint32_t t0 = (uint32_t)max(s.runs[r], 0), t1 = min((uint32_t)max(s.runs[r + 1], 0), total);
    if (t0 >= t1) return;  // behind the last run
    if (blockIdx.y >= 2 * c.kv_heads) {  // q
        const uint32_t h0 = (blockIdx.y - 2 * c.kv_heads) * kQHeads, hn = min(kQHeads, heads - h0), per_row = hn * quads;
        for (uint32_t i = tid; i < (t1 - t0) * per_row; i += kAppendThreads) {
            const uint32_t row = i / per_row, e = i - row * per_row, t = t0 + row, d = (e % quads) * 4, h = h0 + e / quads;
            const uint32_t p = min((uint32_t)max(s.positions[t], 0), max_pos - 1);
            const float* src = qkv + (size_t)t * pitch + h * dim + d;
            float4 lo, hi;
            rotate4(*reinterpret_cast<const float4*>(src), *reinterpret_cast<const float4*>(src + half), cosv + (size_t)p * dim, sinv + (size_t)p * dim,
                    d, half, lo, hi);
            float* dst = q_out + ((size_t)t * heads + h) * dim + d;
            *reinterpret_cast<float4*>(dst) = lo;
            *reinterpret_cast<float4*>(dst + half) = hi;
        }
        return;
    }
    const uint32_t head = blockIdx.y >> 1, is_v = blockIdx.y & 1;
    const int32_t slot = s.slots[t0];
    if (slot < 0 || ((uint32_t)slot >> c.shift) >= c.blocks) return;  // no room for this run
    const uint32_t block = (uint32_t)slot >> c.shift, off0 = (uint32_t)slot & (c.block - 1), n = min(t1 - t0, c.block - off0);
    const float* src = qkv + (size_t)t0 * pitch + (size_t)(heads + (is_v ? c.kv_heads : 0) + head) * dim;
    auto key_quads = [&](uint32_t row, uint32_t d, float4& lo, float4& hi) {
        const uint32_t p = min((uint32_t)max(s.positions[t0 + row], 0), max_pos - 1);
        const float* x = src + (size_t)row * pitch + d;
        rotate4(*reinterpret_cast<const float4*>(x), *reinterpret_cast<const float4*>(x + half), cosv + (size_t)p * dim, sinv + (size_t)p * dim, d, half,
                lo, hi);
    };
    uint32_t m = 0;
    if (!is_v) {
        for (uint32_t i = tid; i < n * quads; i += kAppendThreads) {
            float4 lo, hi;
            key_quads(i / quads, (i % quads) * 4, lo, hi);
            m = max(m, max(mag4(lo), mag4(hi)));
        }
    } else {
        for (uint32_t i = tid; i < n * 2 * quads; i += kAppendThreads)
            m = max(m, mag4(*reinterpret_cast<const float4*>(src + (size_t)(i / (2 * quads)) * pitch + (i % (2 * quads)) * 4)));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) most[tid >> 5] = m;
    float* scale_at = (is_v ? c.vscale : c.kscale) + (size_t)block * c.kv_heads + head;
    const float old = off0 ? *scale_at : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) m = max(m, most[w]);
    const uint32_t fresh = mag(__fdiv_rn(__uint_as_float(m), 127.0f));
    const bool grows = fresh > mag(old);
    const float scale = grows ? __uint_as_float(fresh) : old, ratio = grows ? __fdiv_rn(old, scale) : 1.0f;
    if (tid == 0) *scale_at = scale;
    uint32_t* pool = reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + ((size_t)block * c.kv_heads + head) * c.block * dim);
    if (!is_v) {
        if (grows)  // the block's other tokens, a word = four components of one token
            for (uint32_t i = tid; i < (c.block - n) * 2 * quads; i += kAppendThreads) {
                uint32_t t = i / (2 * quads);
                t += t < off0 ? 0 : n;
                uint32_t* w = pool + key_at(dim, t, (i % (2 * quads)) * 4) / 4;
                const uint32_t was = off0 ? *w : 0u;  // a block that starts anew starts as zeros
                *w = recode(was, 0, ratio) | recode(was, 1, ratio) << 8 | recode(was, 2, ratio) << 16 | recode(was, 3, ratio) << 24;
            }
        for (uint32_t i = tid; i < n * quads; i += kAppendThreads) {
            const uint32_t row = i / quads, d = (i % quads) * 4;
            float4 lo, hi;
            key_quads(row, d, lo, hi);
            pool[key_at(dim, off0 + row, d) / 4] = code_of(lo.x, scale) | code_of(lo.y, scale) << 8 | code_of(lo.z, scale) << 16 | code_of(lo.w, scale) << 24;
            pool[key_at(dim, off0 + row, d + half) / 4] =
                code_of(hi.x, scale) | code_of(hi.y, scale) << 8 | code_of(hi.z, scale) << 16 | code_of(hi.w, scale) << 24;
        }
    } else {
        // a word = four tokens of one component: the run's first and last may hold others too
        const uint32_t w0 = grows ? 0 : off0 >> 2, w1 = grows ? c.block >> 2 : (off0 + n + 3) >> 2;
        for (uint32_t i = tid; i < (w1 - w0) * dim; i += kAppendThreads) {
            const uint32_t d = i % dim, t = (w0 + i / dim) * 4;
            uint32_t* at = pool + value_at(c.block, t, d) / 4;
            uint32_t word = (t < off0 || t + 4 > off0 + n) && (off0 || !grows) ? *at : 0u;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                uint32_t code = word >> (8 * j) & 0xffu;
                if (t + j >= off0 && t + j < off0 + n) code = code_of(src[(size_t)(t + j - off0) * pitch + d], scale);
                else if (grows) code = recode(word, j, ratio);
                word = (word & ~(0xffu << (8 * j))) | code << (8 * j);
            }
            *at = word;
        }
    }
}

}  // namespace

void launch_paged_plan(cudaStream_t s, const PagedView& c, const StepView& st, const int32_t* counts, const int32_t* free_list, int32_t* free_count) {
    // One CTA fills 8192 rows of the maps in the time that the cluster's barrier takes.
    const uint32_t ctas = st.tokens > 8192 ? kPlanCluster : 1;
    const size_t smem = (size_t)(3 * c.seqs + 2) * 4;
    if (smem + 256 > 48 * 1024) GQ_CUDA(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(kPlanThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    GQ_CUDA(cudaLaunchKernelEx(&cfg, paged_plan_kernel, c, st, counts, free_list, free_count));
}

void launch_paged_advance(cudaStream_t s, const PagedView& c, const StepView& st) {
    launch_after(paged_advance_kernel, dim3((c.seqs + 255) / 256), dim3(256), 0, s, c, st);
}

void launch_paged_release(cudaStream_t s, const PagedView& c, const int32_t* which, int32_t* free_list, int32_t* free_count) {
    launch_after(paged_release_kernel, dim3(1), dim3(kPlanThreads), 0, s, c, which, free_list, free_count);
}

void launch_paged_append(cudaStream_t s, const PagedView& c, const StepView& st, const float* qkv, uint32_t heads, const float* cosv, const float* sinv,
                         uint32_t max_pos, float* q_out) {
    const uint32_t parts = 2 * c.kv_heads + (heads + kQHeads - 1) / kQHeads;
    launch_after(paged_append_kernel, dim3(st.runs_cap, parts), dim3(kAppendThreads), 0, s, c, st, qkv, heads, cosv, sinv, max_pos, q_out);
}

}  // namespace gq
