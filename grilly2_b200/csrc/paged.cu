// The paged int8 KV cache's bookkeeping and writes (no counterpart in the reference, whose cache is contiguous and of batch
// 1: crates/grilly-infer/src/kv_cache.rs:1-33).
//
// plan: the new tokens of every request get positions, rows, blocks and slots. With c_b = counts[b] and n_b = lens[b]:
//   starts = exclusive sum of c; request b touches the table entries n_b / bs .. (n_b + c_b - 1) / bs, one RUN of rows each;
//   the r-th touched entry without a block, in order of (b, entry), takes free[free_count - 1 - r] — unless n_b lies inside it:
//   then its earlier tokens found no room, and a block given now would be read as if it held them;
//   slot = table[b][p / bs] * bs + p % bs for p = n_b + (row - starts[b]).
// Both sums are block scans over the requests; runs and rows find their request by a binary search in shared memory. Few
// rows run as one CTA; many as a cluster of eight, whose first CTA hands out the blocks while the cluster barrier holds
// the others back from the table. Bound: latency (three scans); the maps are a few bytes per row. 8 requests with a token each
// take 4.8 us, 1000 requests with 33 thousand rows 11.9 (a search for each of a thread's four rows, side by side: 13.4).
//
// append: one CTA per run of rows that share a block, KV head and K or V (further CTAs rotate q): the largest |value| of the
// run gives the scale, the block's older codes are rounded again if it grew, the run's values are rounded and stored in
// the core-matrix order of the pool. A 32-bit word of codes has one owner, so a word that holds old and new codes is
// read and written by one thread. Bound: bytes where there are many rows (8 prompts of 5568 rows in all, 32 heads over 8 of 128:
// 245 MB in 53.5 us = 4.6 TB/s; a chain of loads, a maximum over the CTA and stores for each run keeps it from the copy's 37),
// launch latency for single tokens (64 requests: 5.9 us).
#include "gq_internal.h"
#include "paged.cuh"

namespace gq {

namespace {

constexpr uint32_t kPlanThreads = 1024, kPlanFew = 256;  // of a CTA; where requests and rows are few (its barriers cost less)
constexpr uint32_t kPlanCluster = 8;
constexpr uint32_t kAtOnce = 4;  // runs of a thread whose loads are in flight together

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive scan of one value per thread of the CTA, sums saturating at `cap` (which keeps them in 32 bits); *total is the sum.
template <uint32_t NT>
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
        uint32_t s = lane < NT / 32 ? warp_sums[lane] : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= (uint32_t)o) s = min(s + y, cap);
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    *total = warp_sums[NT / 32 - 1];
    const uint32_t before = warp ? warp_sums[warp - 1] : 0u;
    const uint32_t left = __shfl_up_sync(0xffffffffu, x, 1);
    return lane ? min(before + left, cap) : before;
}

// The request that owns an item: the last b >= from with at[b] <= item, at ascending and at[from] <= item.
__device__ __forceinline__ uint32_t owner_of(const uint32_t* at, uint32_t n, uint32_t item, uint32_t from = 0) {
    uint32_t b = from;
    for (uint32_t step = n - from > 1 ? 1u << (31 - __clz(n - from - 1)) : 0; step > 0; step >>= 1)
        if (b + step < n && at[b + step] <= item) b += step;
    return b;
}

template <uint32_t NT>
__global__ void __launch_bounds__(NT) paged_plan_kernel(PagedView c, StepView s, const int32_t* __restrict__ counts,
                                                                 const int32_t* __restrict__ free_list, int32_t* free_count) {
    GQ_GRID_DEP_SYNC();
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t warp_sums[32], refused;
    uint32_t* start = smem;                  // [seqs + 1]
    uint32_t* run = start + c.seqs + 1;      // [seqs + 1]
    uint32_t* len = run + c.seqs + 1;        // [seqs]
    const uint32_t tid = threadIdx.x, per = (c.seqs + NT - 1) / NT, b0 = tid * per, b1 = min(b0 + per, c.seqs);
    uint32_t total, runs, sum = 0;
    if (tid == 0) refused = 0;
    for (uint32_t b = b0; b < b1; ++b) sum = min(sum + min((uint32_t)max(counts[b], 0), s.tokens), s.tokens);
    uint32_t at = block_scan<NT>(sum, s.tokens, warp_sums, &total);
    sum = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t next = min(at + min((uint32_t)max(counts[b], 0), s.tokens), s.tokens), n = paged_len(c, b);
        start[b] = at, len[b] = n;
        if (next > at) sum += ((n + (next - at) - 1) >> c.shift) - (n >> c.shift) + 1;
        at = next;
    }
    if (tid == 0) start[c.seqs] = total;
    at = block_scan<NT>(sum, s.runs_cap, warp_sums, &runs);  // (its barriers publish start and len)
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
        for (uint32_t r0 = 0; r0 < runs; r0 += kAtOnce * NT) {
            int32_t* entry[kAtOnce];
            uint32_t need = 0, inside = 0, packed_lo = 0, packed_hi = 0;  // four counts of 16 bits, one for each slab of NT runs
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                const uint32_t r = r0 + k * NT + tid;
                entry[k] = nullptr;
                if (r < runs) {
                    const uint32_t b = owner_of(run, c.seqs, r), j = (len[b] >> c.shift) + (r - run[b]);
                    s.runs[r] = (int32_t)(r == run[b] ? start[b] : start[b] + ((j << c.shift) - len[b]));
                    if (j < c.max_blocks) entry[k] = c.table + (size_t)b * c.max_blocks + j;
                    if ((j << c.shift) < len[b]) inside |= 1u << k;
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k)
                if (entry[k] && *entry[k] < 0) {
                    if (inside >> k & 1) atomicAdd(&refused, 1u);  // (rare; the scan's barriers publish it)
                    else need |= 1u << k;
                }
            packed_lo = (need & 1) | (need & 2) << 15, packed_hi = (need >> 2 & 1) | (need & 8) << 13;
            uint32_t all_lo, all_hi = 0, before_hi = 0;
            const uint32_t before_lo = block_scan<NT>(packed_lo, 0xffffffffu, warp_sums, &all_lo);
            if (r0 + 2 * NT < runs) before_hi = block_scan<NT>(packed_hi, 0xffffffffu, warp_sums, &all_hi);
            const uint32_t before[kAtOnce] = {before_lo & 0xffffu, before_lo >> 16, before_hi & 0xffffu, before_hi >> 16};
            const uint32_t all[kAtOnce] = {all_lo & 0xffffu, all_lo >> 16, all_hi & 0xffffu, all_hi >> 16};
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                const uint32_t rank = wanted + before[k];
                if ((need >> k & 1) && rank < have) *entry[k] = free_list[have - 1 - rank];
                wanted += all[k];
            }
        }
        for (uint32_t r = runs + tid; r <= s.runs_cap; r += NT) s.runs[r] = (int32_t)total;
        for (uint32_t b = tid; b <= c.seqs; b += NT) {
            s.starts[b] = (int32_t)start[b];
            if (b < c.seqs) s.last[b] = start[b + 1] > start[b] ? (int32_t)start[b + 1] - 1 : -1;
        }
        if (tid == 0) {  // every thread read *free_count before the scans' barriers (or nothing was wanted)
            if (wanted) *free_count = (int32_t)(have - min(wanted, have));
            s.info[0] = (int32_t)total, s.info[1] = (int32_t)(wanted - min(wanted, have) + refused);
        }
    }
    if (gridDim.x > 1) cluster_barrier();
    else __syncthreads();
    // four rows a thread, one behind the other: one search, and another only where a request ends among them
    const bool wide = ((reinterpret_cast<uintptr_t>(s.slots) | reinterpret_cast<uintptr_t>(s.positions)) & 15) == 0;
    for (uint32_t t0 = 4 * (blockIdx.x * NT + tid); t0 < s.tokens; t0 += 4 * gridDim.x * NT) {
        int32_t pos[4], slot[4];
        uint32_t entry[4], b = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t t = t0 + k;
            pos[k] = slot[k] = -1, entry[k] = 0xffffffffu;
            if (t >= total) continue;
            if (k == 0 || start[b + 1] <= t) b = owner_of(start, c.seqs, t, b);
            const uint32_t p = len[b] + (t - start[b]), j = p >> c.shift;
            pos[k] = (int32_t)p;
            if (j < c.max_blocks) entry[k] = b * c.max_blocks + j;
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (entry[k] != 0xffffffffu) slot[k] = __ldcg(c.table + entry[k]);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            slot[k] = slot[k] >= 0 && (uint32_t)slot[k] < c.blocks ? (int32_t)(((uint32_t)slot[k] << c.shift) + ((uint32_t)pos[k] & (c.block - 1))) : -1;
        if (wide && t0 + 4 <= s.tokens) {
            *reinterpret_cast<int4*>(s.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4*>(s.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (t0 + k < s.tokens) s.slots[t0 + k] = slot[k], s.positions[t0 + k] = pos[k];
        }
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
            const uint32_t rank = have + block_scan<kPlanThreads>(held ? 1u : 0u, 0x7fffffffu, warp_sums, &here);
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

// rint(v / s) in the codes' range, the quotient rounded as IEEE division does; an empty scale (all zeros) and a value that is not a
// number give 0. The product with the reciprocal differs from the quotient by two roundings, 127 * 2^-23 = 1.5e-5 at most, so only
// next to a half does it take the division to tell.
__device__ __forceinline__ uint32_t code_of(float v, float s, float inverse) {
    float r = v * inverse;
    const float whole = rintf(r);
    if (!(fabsf(r - whole) <= 0.4998f)) r = __fdiv_rn(v, s);
    return (uint32_t)max(-127, min(127, __float2int_rn(r))) & 0xffu;
}
__device__ __forceinline__ uint32_t recode(uint32_t word, uint32_t byte, float ratio) {
    return (uint32_t)__float2int_rn(__fmul_rn((float)(int8_t)(word >> (8 * byte)), ratio)) & 0xffu;
}

template <int DIM>
__global__ void __launch_bounds__(kAppendThreads, 4) paged_append_kernel(PagedView c, StepView s, const float* __restrict__ qkv, uint32_t heads,
                                                                     const float* __restrict__ cosv, const float* __restrict__ sinv, uint32_t max_pos,
                                                                     float* __restrict__ q_out) {
    GQ_GRID_DEP_SYNC();
    // A thread has four components and the four half a head further, of every kRows-th row; kHeld of its rows stay in
    // registers between the two passes, the others are read again.
    constexpr uint32_t kHalf = DIM / 2, kQuads = kHalf / 4, kRows = kAppendThreads / kQuads, kHeld = 4;
    __shared__ uint32_t most[kAppendThreads / 32];
    const uint32_t tid = threadIdx.x, d = tid % kQuads * 4, row0 = tid / kQuads, pitch = (heads + 2 * c.kv_heads) * DIM;
    const uint32_t r = blockIdx.x;
    const uint32_t t0 = (uint32_t)max(s.runs[r], 0), t1 = min((uint32_t)max(s.runs[r + 1], 0), paged_start(s, c.seqs));
    if (t0 >= t1) return;  // behind the last run
    const uint32_t pos0 = (uint32_t)max(s.positions[t0], 0);  // a run's positions follow one another
    auto position = [&](uint32_t t) { return min(pos0 + (t - t0), max_pos - 1); };
    if (blockIdx.y >= 2 * c.kv_heads) {  // q: kQHeads heads of every row
        const uint32_t h0 = (blockIdx.y - 2 * c.kv_heads) * kQHeads, items = (t1 - t0) * kQHeads;
        constexpr uint32_t kAtOnce = 4;
        for (uint32_t i0 = row0; i0 < items; i0 += kAtOnce * kRows) {
            float4 lo[kAtOnce], hi[kAtOnce];
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j) {
                const uint32_t i = i0 + j * kRows, t = t0 + i / kQHeads, h = h0 + i % kQHeads;
                if (i >= items || h >= heads) continue;
                const float* src = qkv + (size_t)t * pitch + h * DIM + d;
                lo[j] = __ldcs(reinterpret_cast<const float4*>(src)), hi[j] = __ldcs(reinterpret_cast<const float4*>(src + kHalf));
            }
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j) {
                const uint32_t i = i0 + j * kRows, t = t0 + i / kQHeads, h = h0 + i % kQHeads;
                if (i >= items || h >= heads) continue;
                const size_t p = (size_t)position(t) * DIM;
                float4 a, b;
                rotate4(lo[j], hi[j], cosv + p, sinv + p, d, kHalf, a, b);
                float* dst = q_out + ((size_t)t * heads + h) * DIM + d;
                *reinterpret_cast<float4*>(dst) = a;
                *reinterpret_cast<float4*>(dst + kHalf) = b;
            }
        }
        return;
    }
    const uint32_t head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const int32_t slot = s.slots[t0];
    if (slot < 0 || ((uint32_t)slot >> c.shift) >= c.blocks) return;  // no room for this run
    const uint32_t block = (uint32_t)slot >> c.shift, off0 = (uint32_t)slot & (c.block - 1), n = min(t1 - t0, c.block - off0);
    const float* src = qkv + (size_t)t0 * pitch + (size_t)(heads + (is_v ? c.kv_heads : 0) + head) * DIM;
    float* scale_at = (is_v ? c.vscale : c.kscale) + (size_t)block * c.kv_heads + head;
    const float old = off0 ? *scale_at : 0.0f;
    auto load = [&](uint32_t row, float4& lo, float4& hi) {
        const float* x = src + (size_t)row * pitch + d;
        lo = *reinterpret_cast<const float4*>(x), hi = *reinterpret_cast<const float4*>(x + kHalf);
    };
    auto turn = [&](uint32_t row, float4& lo, float4& hi) {
        const size_t p = (size_t)position(t0 + row) * DIM;
        float4 a, b;
        rotate4(lo, hi, cosv + p, sinv + p, d, kHalf, a, b);
        lo = a, hi = b;
    };
    uint32_t m = 0;
    float4 lo[kHeld], hi[kHeld];
#pragma unroll
    for (uint32_t j = 0; j < kHeld; ++j)
        if (row0 + j * kRows < n) load(row0 + j * kRows, lo[j], hi[j]);
#pragma unroll
    for (uint32_t j = 0; j < kHeld; ++j)
        if (row0 + j * kRows < n) {
            if (!is_v) turn(row0 + j * kRows, lo[j], hi[j]);
            m = max(m, max(mag4(lo[j]), mag4(hi[j])));
        }
    for (uint32_t row = row0 + kHeld * kRows; row < n; row += kRows) {
        float4 a, b;
        load(row, a, b);
        if (!is_v) turn(row, a, b);
        m = max(m, max(mag4(a), mag4(b)));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) most[tid >> 5] = m;
    __syncthreads();  // (and every thread has read the old scale)
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) m = max(m, most[w]);
    const uint32_t fresh = mag(__fdiv_rn(__uint_as_float(m), 127.0f));
    const bool grows = fresh > mag(old);
    const float scale = grows ? __uint_as_float(fresh) : old, ratio = grows ? __fdiv_rn(old, scale) : 1.0f;
    // a scale whose reciprocal may not be a normal number has none: every code of it is divided for
    const float inverse = scale == 0.0f ? 0.0f : scale > 0x1p-100f && scale < 0x1p100f ? __fdiv_rn(1.0f, scale) : __int_as_float(0x7fc00000);
    if (tid == 0) *scale_at = scale;
    uint32_t* pool = reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + ((size_t)block * c.kv_heads + head) * c.block * DIM);
    if (!is_v) {
        if (grows)  // the block's other tokens, a word = four components of one token
            for (uint32_t i = tid; i < (c.block - n) * 2 * kQuads; i += kAppendThreads) {
                uint32_t t = i / (2 * kQuads);
                t += t < off0 ? 0 : n;
                uint32_t* w = pool + key_at(DIM, t, i % (2 * kQuads) * 4) / 4;
                const uint32_t was = off0 ? *w : 0u;  // a block that starts anew starts as zeros
                *w = recode(was, 0, ratio) | recode(was, 1, ratio) << 8 | recode(was, 2, ratio) << 16 | recode(was, 3, ratio) << 24;
            }
        auto store = [&](uint32_t row, const float4& a, const float4& b) {
            pool[key_at(DIM, off0 + row, d) / 4] = code_of(a.x, scale, inverse) | code_of(a.y, scale, inverse) << 8 | code_of(a.z, scale, inverse) << 16 | code_of(a.w, scale, inverse) << 24;
            pool[key_at(DIM, off0 + row, d + kHalf) / 4] = code_of(b.x, scale, inverse) | code_of(b.y, scale, inverse) << 8 | code_of(b.z, scale, inverse) << 16 | code_of(b.w, scale, inverse) << 24;
        };
#pragma unroll
        for (uint32_t j = 0; j < kHeld; ++j)
            if (row0 + j * kRows < n) store(row0 + j * kRows, lo[j], hi[j]);
        for (uint32_t row = row0 + kHeld * kRows; row < n; row += kRows) {
            float4 a, b;
            load(row, a, b);
            turn(row, a, b);
            store(row, a, b);
        }
    } else {
        // a word = four tokens of one component: the run's first and last may hold others too
        const uint32_t w0 = grows ? 0 : off0 >> 2, w1 = grows ? c.block >> 2 : (off0 + n + 3) >> 2;
#pragma unroll 2
        for (uint32_t i = tid; i < (w1 - w0) * DIM; i += kAppendThreads) {
            const uint32_t comp = i % DIM, t = (w0 + i / DIM) * 4;
            uint32_t* at = pool + value_at(c.block, t, comp) / 4;
            uint32_t word = (t < off0 || t + 4 > off0 + n) && (off0 || !grows) ? *at : 0u;
            float x[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) x[j] = t + j >= off0 && t + j < off0 + n ? src[(size_t)(t + j - off0) * pitch + comp] : 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                uint32_t code = word >> (8 * j) & 0xffu;
                if (t + j >= off0 && t + j < off0 + n) code = code_of(x[j], scale, inverse);
                else if (grows) code = recode(word, j, ratio);
                word = (word & ~(0xffu << (8 * j))) | code << (8 * j);
            }
            *at = word;
        }
    }
}

}  // namespace

void launch_paged_plan(cudaStream_t s, const PagedView& c, const StepView& st, const int32_t* counts, const int32_t* free_list, int32_t* free_count) {
    // One CTA fills 8192 rows of the maps in about the time that the cluster's start and barrier take.
    const uint32_t ctas = st.tokens > 8192 ? kPlanCluster : 1;
    const bool few = c.seqs <= kPlanFew && st.tokens <= 4 * kPlanFew;
    const size_t smem = (size_t)(3 * c.seqs + 2) * 4;
    auto kernel = few ? paged_plan_kernel<kPlanFew> : paged_plan_kernel<kPlanThreads>;
    if (smem + 256 > 48 * 1024) GQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(few ? kPlanFew : kPlanThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    GQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, c, st, counts, free_list, free_count));
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
    auto kernel = c.dim == 128 ? paged_append_kernel<128> : c.dim == 64 ? paged_append_kernel<64> : paged_append_kernel<32>;
    launch_after(kernel, dim3(st.runs_cap, parts), dim3(kAppendThreads), 0, s, c, st, qkv, heads, cosv, sinv, max_pos, q_out);
}

}  // namespace gq
