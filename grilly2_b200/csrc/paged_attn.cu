// Causal grouped-query attention of a step's rows over the paged int8 KV cache, in exact integer products on the fifth-
// generation tensor cores (tcgen05.mma kind::i8), softmax in float32. No counterpart in the reference.
//
//   s[r][j] = scale (q_r . k_j),  w[r][j] = exp(s[r][j] - max),  out[r] = sum_j w[r][j] v_j / sum_j w[r][j]
//
// The cached codes are the A operand exactly as they lie in the pool (its blocks are core matrices of 8 x 16 bytes):
// k_j = kscale_j K_j with 128 keys on the lanes of tensor memory, v_j = vscale_j V_j with the components on the lanes. What
// meets them is held as an exact fixed-point integer in three base-256 digits, so three products in int32 and one join
// give a float32 result:
//   q_r = 2^(e_r - 22) Q, Q in signed digits; kscale_j is a factor of a lane;
//   w vscale = 2^(n - 24) P, P in unsigned digits, where 2^n bounds the tile's largest w vscale of that row. The value scales are
//   folded into P because the sum over j runs across blocks; n follows the tile's own largest product, so a block with large
//   values and no weight does not coarsen the others' steps.
//
// A CTA takes a contiguous range of all (request, row tile, KV head, 128-key tile) units, equal ranges for all CTAs: with ragged
// lengths no CTA waits for a long request, and a single request fills the GPU. A row tile is RP rows of (token, head of the
// group), N = 3 RP digit rows. An (item = request, row tile, KV head) that ends inside one range is written out; the
// others leave (max, sum, weighted V) per CTA and the last CTA of an item to arrive adds them in order (deterministic).
//   warp 5  copies the tile's K and V blocks into a ring of stages (bulk copies; the table gives the addresses)
//   warp 4  issues the products: S = K Q (128 x N), then D = V P (dim x N) when P is written
//   warps 0-3  a thread owns a key of S: joins the digits, one maximum over the 128 keys per row (warp reductions and one
//           exchange), P's digits to shared memory; then it owns a component of D and adds it to its float32 sums
// Bound: the codes' bytes.
#include "gq_internal.h"
#include "paged.cuh"
#include "tc_common.cuh"

namespace gq {

namespace {

constexpr uint32_t kKeys = 128;    // keys of a tile
constexpr int kThreads = 192;
constexpr float kNone = -INFINITY;
constexpr uint32_t kMostPerSm = 4;  // CTAs of an SM

template <int RP, int DIM>
struct Split {
    static constexpr uint32_t kN = RP == 8 ? 32 : 3 * RP;                        // columns: a multiple of 16; digit d of row r in column d RP + r
    static constexpr uint32_t kCols = RP == 8 ? 32 : RP == 16 ? 64 : 128;        // S at column 0, D at kCols
    static constexpr uint32_t kM = DIM == 128 ? 128 : 64;                        // lanes of D: dim, at least 64
    static constexpr uint32_t kTileBytes = kKeys * DIM, kStageBytes = 2 * kTileBytes;
    static constexpr uint32_t kStages = DIM == 128 ? 2 : DIM == 64 ? 3 : 4;
    // (dim 32: the 64 lanes of D read 32 rows that are not there, up to 4 KB behind the last stage; nobody reads the sums)
    static constexpr uint32_t kQAt = kStages * kStageBytes + (DIM == 32 ? 4096 : 0);
    static constexpr uint32_t kPAt = kQAt + kN * DIM, kMiscAt = kPAt + kN * kKeys;
    static constexpr uint32_t kSmem = kMiscAt + 1024 + 4 * RP * 16 + 2 * 4 * RP * 8 + RP * 8 + 4 * RP * 4;
};

__device__ __forceinline__ float warp_max(float v) {  // the largest that is a number
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
template <int R>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t (&r)[R]) {
    if constexpr (R == 8) tmem_ld8(addr, r);
    else tmem_ld16(addr, r);
}
// three digit sums of up to 22 bits, joined with two roundings
__device__ __forceinline__ float join(uint32_t d0, uint32_t d1, uint32_t d2) {
    return __fmaf_rn((float)(int)d2, 65536.0f, (float)((int)d0 + ((int)d1 << 8)));
}

// One request's share of the units.
struct Request {
    uint32_t start, rows, len, keys, tiles, items;  // keys = cached and new ones, inside the table
    __device__ uint64_t units() const { return (uint64_t)items * tiles; }
};
__device__ __forceinline__ Request request_of(const PagedView& c, const StepView& s, uint32_t b, uint32_t group, uint32_t rp) {
    Request r;
    r.start = paged_start(s, b);
    const uint32_t end = paged_start(s, b + 1), count = end > r.start ? end - r.start : 0;
    r.rows = count * group, r.len = paged_len(c, b);
    r.keys = min(r.len + count, c.max_blocks << c.shift);
    r.tiles = (r.keys + kKeys - 1) / kKeys, r.items = (r.rows + rp - 1) / rp * c.kv_heads;
    return r;
}

// What a stretch of one item's tiles is.
struct Segment {
    uint32_t b, item, t0, t1;      // tiles [t0, t1): those with a key that some row of the item sees
    uint32_t row0, rows, head;     // rows of the request's count * group, KV head
    uint64_t first, last;          // the item's units [first, last)
    bool whole;
};

// Walks the units [lo, hi) of this CTA, segment by segment; every role runs the same walk.
struct Walk {
    uint64_t u, hi, base;  // base = the units before request b
    uint32_t b;
    Request r;
    __device__ bool next(const PagedView& c, const StepView& s, uint32_t group, uint32_t rp, Segment& g) {
        if (u >= hi) return false;
        while (u >= base + r.units()) base += r.units(), r = request_of(c, s, ++b, group, rp);
        const uint64_t v = u - base;
        g.b = b, g.item = (uint32_t)(v / r.tiles), g.t0 = (uint32_t)(v - (uint64_t)g.item * r.tiles);
        g.first = base + (uint64_t)g.item * r.tiles, g.last = g.first + r.tiles;
        const uint64_t end = min(hi, g.last);
        g.whole = u == g.first && end == g.last;
        g.head = g.item % c.kv_heads, g.row0 = g.item / c.kv_heads * rp, g.rows = min(rp, r.rows - g.row0);
        const uint32_t seen = min(r.len + (g.row0 + g.rows - 1) / group + 1, r.keys);  // keys of the tile's last token
        g.t1 = max(g.t0, min(g.t0 + (uint32_t)(end - u), (seen + kKeys - 1) / kKeys));
        u = end;
        return true;
    }
};

template <int RP, int DIM>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(PagedView c, StepView s, const float* __restrict__ q, uint32_t heads, float scale,
                                                             float* __restrict__ out, float* __restrict__ partials, uint32_t* counters, uint32_t* status) {
    using T = Split<RP, DIM>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* misc = smem + T::kMiscAt;
    uint64_t* full = reinterpret_cast<uint64_t*>(misc);  // [kStages] a stage's blocks have landed
    uint64_t* empty = full + 4;                          // [kStages] its products are complete
    uint64_t* s_full = empty + 4;                        // S is complete
    uint64_t* p_full = s_full + 1;                       // P is written, S and the D before are read
    uint64_t* d_full = p_full + 1;                       // D is complete
    uint64_t* q_full = d_full + 1;                       // Q is written
    uint64_t* scan = q_full + 1;                         // [8]
    uint64_t* found = scan + 8;                          // the units before the request that the range starts in
    uint32_t* found_b = reinterpret_cast<uint32_t*>(found + 1);
    uint32_t* tmem_slot = found_b + 1;
    uint32_t* arrived = tmem_slot + 1;
    volatile uint32_t* failed = arrived + 1;
    float4* rowbuf = reinterpret_cast<float4*>(misc + 1024);             // [4 warps][RP] max, correction, digits' factor, sums' factor
    float2* exchange = reinterpret_cast<float2*>(rowbuf + 4 * RP);       // [2][4][RP] warps' maxima
    float2* row_in = exchange + 2 * 4 * RP;                              // [RP] scale of a row of q, last position it sees
    float* lsum = reinterpret_cast<float*>(row_in + RP);                 // [4][RP]

    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = heads / c.kv_heads;
    if (tid == 0) {
        for (uint32_t i = 0; i < T::kStages; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        mbar_init(s_full, 1), mbar_init(p_full, kKeys), mbar_init(d_full, 1), mbar_init(q_full, kKeys);
        *failed = 0;
        mbar_fence_init();
    }
    if (warp == 4) tmem_alloc(tmem_slot, 2 * T::kCols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    GQ_GRID_DEP_SYNC();

    // the units of all requests, and the request that this CTA's range starts in
    const uint32_t per = (c.seqs + kThreads - 1) / kThreads, b0 = min(tid * per, c.seqs), b1 = min(b0 + per, c.seqs);
    uint64_t mine = 0;
    for (uint32_t b = b0; b < b1; ++b) mine += request_of(c, s, b, group, RP).units();
    uint64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= (uint32_t)o) upto += y;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    uint64_t total = 0, before = upto - mine;
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    const uint64_t ctas = min((uint64_t)gridDim.x, total);
    auto range_at = [&](uint64_t i) { return total * i / ctas; };
    Walk walk;
    if (blockIdx.x < ctas) {
        walk.u = range_at(blockIdx.x), walk.hi = range_at(blockIdx.x + 1);
        if (walk.u >= before && walk.u < before + mine) {
            uint32_t b = b0;
            uint64_t base = before, units;
            while (walk.u >= base + (units = request_of(c, s, b, group, RP).units())) base += units, ++b;
            *found = base, *found_b = b;
        }
    } else {
        walk.u = walk.hi = 0;
    }
    __syncthreads();
    walk.base = *found, walk.b = *found_b;
    if (walk.u < walk.hi) walk.r = request_of(c, s, walk.b, group, RP);
    Segment g;
    bool ok = true;

    if (warp == 5) {
        uint32_t st = 0, round = 0;
        const uint32_t per_tile = kKeys >> c.shift, bytes = c.block * DIM;
        while (walk.next(c, s, group, RP, g)) {
            const int32_t* table = c.table + (size_t)g.b * c.max_blocks;
            for (uint32_t t = g.t0; t < g.t1; ++t) {
                const uint32_t j = t * per_tile + lane;  // one lane per block
                int32_t e = lane < per_tile && j < c.max_blocks && (j << c.shift) < walk.r.keys ? table[j] : -1;
                if (e < 0 || (uint32_t)e >= c.blocks) e = -1;
                if (round) ok = ok && mbar_wait(empty + st, (round - 1) & 1, failed, status, kStatusEmptyWaitTimedOut);
                const uint32_t held = __popc(__ballot_sync(0xffffffffu, e >= 0));
                if (__ballot_sync(0xffffffffu, !ok)) ok = false;
                if (!ok) continue;
                if (lane == 0) mbar_arrive_expect_tx(full + st, held * 2 * bytes);
                __syncwarp();
                if (e >= 0) {
                    const size_t at = ((size_t)e * c.kv_heads + g.head) * bytes;
                    uint8_t* dst = smem + st * T::kStageBytes + lane * bytes;
                    bulk_load(dst, c.k + at, bytes, full + st);
                    bulk_load(dst + T::kTileBytes, c.v + at, bytes, full + st);
                }
                if (++st == T::kStages) st = 0, ++round;
            }
        }
        if (!ok) {  // gave up: wait (with a limit) for the copies in flight before the CTA may end
            const long long begun = clock64();
            for (uint32_t i = 0; i < T::kStages; ++i) {
                const uint32_t fills = round + (i < st);
                while (fills && !mbar_try_wait(full + i, (fills - 1) & 1) && clock64() - begun < 2000000000ll) {
                }
            }
        }
    } else if (warp == 4) {
        if (lane == 0) {
            constexpr uint32_t s_desc = umma_idesc(2, 1, 1, kKeys, T::kN);  // s32 sums, s8 codes x s8 digits of q
            constexpr uint32_t d_desc = umma_idesc(2, 1, 0, T::kM, T::kN);  // s32 sums, s8 codes x u8 digits of P
            const uint32_t q_addr = smem_u32(smem + T::kQAt), p_addr = smem_u32(smem + T::kPAt);
            uint32_t st = 0, round = 0, tile = 0, seg = 0;
            while (walk.next(c, s, group, RP, g)) {
                if (g.t0 == g.t1) continue;
                ok = ok && mbar_wait(q_full, seg++ & 1, failed, status, kStatusMmaWaitTimedOut);
                for (uint32_t t = g.t0; t < g.t1; ++t, ++tile) {
                    ok = ok && mbar_wait(full + st, round & 1, failed, status, kStatusFullWaitTimedOut);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t k_addr = smem_u32(smem + st * T::kStageBytes), v_addr = k_addr + T::kTileBytes;
#pragma unroll
                    for (uint32_t d = 0; d < DIM / 32; ++d)
                        umma_i8_ss(tmem, umma_desc_plain(k_addr + 256 * d, 128, 8 * DIM), umma_desc_plain(q_addr + 256 * d, 128, 8 * DIM), s_desc, d != 0);
                    umma_commit(s_full);
                    ok = mbar_wait(p_full, tile & 1, failed, status, kStatusMmaWaitTimedOut);
                    if (!ok) break;
                    tc_fence_after_sync();
#pragma unroll
                    for (uint32_t i = 0; i < kKeys / 32; ++i) {
                        // keys 32 i ..: two core matrices of one block, or (blocks of 16) of two
                        const uint32_t k0 = 32 * i, at = (k0 >> c.shift) * c.block * DIM + (k0 & (c.block - 1)) * 8;
                        const uint32_t step = c.shift == 4 ? 16 * DIM : 128;
                        umma_i8_ss(tmem + T::kCols, umma_desc_plain(v_addr + at, step, 8 * c.block), umma_desc_plain(p_addr + 256 * i, 128, 8 * kKeys),
                                   d_desc, i != 0);
                    }
                    umma_commit(d_full);
                    umma_commit(empty + st);
                    if (++st == T::kStages) st = 0, ++round;
                }
            }
        }
    } else {
        constexpr int kChunk = RP == 8 ? 8 : 16;
        const uint32_t comp = T::kM == 128 ? tid : 16 * warp + lane;  // the component of D on this thread's lane
        const bool owner = T::kM == 128 || (lane < 16 && comp < (uint32_t)DIM);
        uint32_t tile = 0;
        float O[RP], l[RP];
        auto drain = [&](uint32_t of_tile) {
            ok = ok && mbar_wait(d_full, of_tile & 1, failed, status, kStatusMmaWaitTimedOut);
            tc_fence_after_sync();
#pragma unroll
            for (int r0 = 0; r0 < RP; r0 += kChunk) {
                uint32_t d0[kChunk], d1[kChunk], d2[kChunk];
                const uint32_t at = tmem_addr(tmem, 32 * warp, T::kCols + r0);
                tmem_ld_cols(at, d0), tmem_ld_cols(at + RP, d1), tmem_ld_cols(at + 2 * RP, d2);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < kChunk; ++i) O[r0 + i] = __fmaf_rn(join(d0[i], d1[i], d2[i]), rowbuf[warp * RP + r0 + i].w, O[r0 + i]);
            }
        };
        while (walk.next(c, s, group, RP, g)) {
            // q's rows as three signed digits: lanes of four components
            {
                constexpr uint32_t kLanes = DIM / 4, kAtOnce = 128 / kLanes;
                const uint32_t sub = tid % kLanes, d = 4 * sub;
#pragma unroll 1
                for (uint32_t r = tid / kLanes; r < RP; r += kAtOnce) {
                    const uint32_t row = g.row0 + r, token = row / group;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < g.rows)
                        v = *reinterpret_cast<const float4*>(q + ((size_t)(walk.r.start + token) * heads + g.head * group + row % group) * DIM + d);
                    uint32_t m = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                                     max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
#pragma unroll
                    for (uint32_t o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                    const uint32_t e = max(m >> 23, 32u);  // 2^(e - 126) > max |q|
                    const float mult = e < 255 ? __uint_as_float((275u - e) << 23) : 0.0f;  // Q = rint(q 2^(22 - e)), |Q| <= 2^22
                    if (sub == 0) {
                        const float inv = e < 255 ? __uint_as_float((e - 21u) << 23) : __uint_as_float(0x7fc00000u);
                        const int seen = r < g.rows ? (int)min(walk.r.len + token, walk.r.keys - 1) : -1;
                        row_in[r] = make_float2(inv * scale, __int_as_float(seen));
                    }
                    const float x[4] = {v.x, v.y, v.z, v.w};
                    uint32_t w0 = 0, w1 = 0, w2 = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        int Q = __float2int_rn(x[i] * mult);
                        const int d0 = (int)(int8_t)Q;
                        Q = (Q - d0) >> 8;
                        const int d1 = (int)(int8_t)Q, d2 = (Q - d1) >> 8;
                        w0 |= ((uint32_t)d0 & 0xffu) << (8 * i), w1 |= ((uint32_t)d1 & 0xffu) << (8 * i), w2 |= ((uint32_t)d2 & 0xffu) << (8 * i);
                    }
                    uint8_t* qd = smem + T::kQAt;
                    *reinterpret_cast<uint32_t*>(qd + key_at(DIM, r, d)) = w0;
                    *reinterpret_cast<uint32_t*>(qd + key_at(DIM, RP + r, d)) = w1;
                    *reinterpret_cast<uint32_t*>(qd + key_at(DIM, 2 * RP + r, d)) = w2;
                }
            }
            named_barrier_sync(1, kKeys);  // row_in
            if (g.t0 < g.t1) {
                fence_proxy_async_smem();
                mbar_arrive(q_full);
            }
#pragma unroll
            for (int r = 0; r < RP; ++r) O[r] = l[r] = 0.0f;
            float M = kNone;  // of row `lane`
            const int32_t* table = c.table + (size_t)g.b * c.max_blocks;
            auto entry = [&](uint32_t t) {
                const uint32_t pos = t * kKeys + tid;
                return t < g.t1 && pos < walk.r.keys ? table[pos >> c.shift] : -1;
            };
            auto scales = [&](int32_t e) {
                if (e < 0 || (uint32_t)e >= c.blocks) return make_float2(0.0f, -1.0f);  // no such block
                const size_t at = (size_t)e * c.kv_heads + g.head;
                const float ks = c.kscale[at], vs = c.vscale[at];
                return make_float2(ks + 0.0f * (ks + vs), fabsf(vs));  // a scale that is no number makes the key's score none
            };
            float2 sc = scales(entry(g.t0));
            int32_t e_next = entry(g.t0 + 1);
            for (uint32_t t = g.t0; t < g.t1; ++t, ++tile) {
                const float2 sc_next = scales(e_next);
                e_next = entry(t + 2);
                if (t > g.t0) drain(tile - 1);
                const int pos = (int)(t * kKeys + tid);
                const bool there = !(sc.y < 0.0f) && (uint32_t)pos < walk.r.keys;
                const float lv = __log2f(sc.y);  // -inf for a block of zeros
                ok = ok && mbar_wait(s_full, tile & 1, failed, status, kStatusMmaWaitTimedOut);
                tc_fence_after_sync();
                float a[RP], mm = kNone, aa = kNone;
#pragma unroll
                for (int r0 = 0; r0 < RP; r0 += kChunk) {
                    uint32_t d0[kChunk], d1[kChunk], d2[kChunk];
                    const uint32_t at = tmem_addr(tmem, 32 * warp, r0);
                    tmem_ld_cols(at, d0), tmem_ld_cols(at + RP, d1), tmem_ld_cols(at + 2 * RP, d2);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) {
                        const float2 in = row_in[r0 + i];
                        const float v = join(d0[i], d1[i], d2[i]) * (in.x * sc.x);
                        a[r0 + i] = there && pos <= __float_as_int(in.y) ? v : kNone;
                        const float m = warp_max(a[r0 + i]), n = warp_max(a[r0 + i] + lv);
                        if (lane == (uint32_t)(r0 + i)) mm = m, aa = n;
                    }
                }
                float2* ex = exchange + (tile & 1) * 4 * RP;
                if (lane < (uint32_t)RP) ex[warp * RP + lane] = make_float2(mm, aa);
                named_barrier_sync(1, kKeys);
                bool moved = false;
                if (lane < (uint32_t)RP) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float2 o = ex[w * RP + lane];
                        mm = fmaxf(mm, o.x), aa = fmaxf(aa, o.y);
                    }
                    const float top = fmaxf(M, mm), at = top == kNone ? 0.0f : top, corr = exp2_fast(M - at);
                    const int n = (int)fminf(fmaxf(ceilf(aa - at + 0.001f), -100.0f), 128.0f);
                    rowbuf[warp * RP + lane] = make_float4(at, corr, pow2(24 - n), pow2(n - 24));
                    moved = corr != 1.0f;
                    M = top;
                }
                const bool rescale = __ballot_sync(0xffffffffu, moved) != 0;
                uint8_t* pd = smem + T::kPAt + (tid >> 4) * 128 + (tid & 15);
#pragma unroll
                for (int r = 0; r < RP; ++r) {
                    const float4 rb = rowbuf[warp * RP + r];
                    const float p = exp2_fast(a[r] - rb.x);
                    if (rescale) l[r] *= rb.y, O[r] *= rb.y;
                    l[r] += p;
                    const uint32_t P = min(__float2uint_rn(p * sc.y * rb.z), 0xffffffu);
                    auto at = [](uint32_t n) { return (n >> 3) * 8 * kKeys + (n & 7) * 16; };
                    pd[at(r)] = (uint8_t)P, pd[at(RP + r)] = (uint8_t)(P >> 8), pd[at(2 * RP + r)] = (uint8_t)(P >> 16);
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                mbar_arrive(p_full);
                sc = sc_next;
            }
            if (g.t0 < g.t1) drain(tile - 1);
            // the rows' sums over the keys, in a fixed order
#pragma unroll
            for (int r = 0; r < RP; ++r) {
                float v = l[r];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane == (uint32_t)r) lsum[warp * RP + r] = v;
            }
            named_barrier_sync(1, kKeys);
            auto sum_of = [&](uint32_t r) { return (lsum[r] + lsum[RP + r]) + (lsum[2 * RP + r] + lsum[3 * RP + r]); };
            auto out_at = [&](uint32_t r) {
                const uint32_t row = g.row0 + r;
                return out + ((size_t)(walk.r.start + row / group) * heads + g.head * group + row % group) * DIM;
            };
            if (g.whole) {
                if (owner)
#pragma unroll
                    for (int r = 0; r < RP; ++r)
                        if ((uint32_t)r < g.rows) {
                            const float sum = sum_of(r);
                            out_at(r)[comp] = sum == 0.0f ? 0.0f : __fdiv_rn(O[r], sum);
                        }
                named_barrier_sync(1, kKeys);  // lsum and row_in are free
                continue;
            }
            // a part of an item: what this CTA has, and the last CTA to arrive adds the parts up
            constexpr uint32_t kPart = RP * (DIM + 2);
            const uint64_t c0 = ((g.first + 1) * ctas - 1) / total, c1 = (g.last * ctas - 1) / total;
            auto part_of = [&](uint64_t cta) { return partials + (cta * 2 + (cta == c0 && range_at(c0) != g.first ? 1 : 0)) * kPart; };
            float* part = part_of(blockIdx.x);
            if (owner)
#pragma unroll
                for (int r = 0; r < RP; ++r) part[r * DIM + comp] = O[r];
            if (warp == 0 && lane < (uint32_t)RP) part[RP * DIM + lane] = M, part[RP * DIM + RP + lane] = sum_of(lane);
            __threadfence();
            named_barrier_sync(1, kKeys);
            if (tid == 0) *arrived = atomicAdd(counters + c0, 1u);
            named_barrier_sync(1, kKeys);
            const uint32_t parts = (uint32_t)(c1 - c0) + 1;
            if (*arrived != parts - 1) continue;
            __threadfence();
            if (tid == 0) counters[c0] = 0;  // ready for the next call
            constexpr uint32_t kVec = DIM / 32;  // components of a lane
            for (uint32_t r = warp; r < g.rows; r += 4) {
                float top = kNone;
                for (uint32_t i = lane; i < parts; i += 32) top = fmaxf(top, __ldcg(part_of(c0 + i) + RP * DIM + r));
                top = warp_max(top);
                const float at = top == kNone ? 0.0f : top;
                float sum = 0.0f, acc[kVec] = {};
                for (uint32_t i0 = 0; i0 < parts; i0 += 32) {
                    const uint32_t i = i0 + lane, here = min(32u, parts - i0);
                    float wgt = 0.0f;
                    if (i < parts) {
                        const float* pp = part_of(c0 + i) + RP * DIM + r;
                        wgt = exp2_fast(__ldcg(pp) - at);
                        sum = __fmaf_rn(wgt, __ldcg(pp + RP), sum);
                    }
#pragma unroll 8
                    for (uint32_t k = 0; k < here; ++k) {
                        const float w = __shfl_sync(0xffffffffu, wgt, k);
                        const float* pp = part_of(c0 + i0 + k) + r * DIM + lane;
#pragma unroll
                        for (uint32_t d = 0; d < kVec; ++d) acc[d] = __fmaf_rn(w, __ldcg(pp + 32 * d), acc[d]);
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
                for (uint32_t d = 0; d < kVec; ++d) out_at(r)[lane + 32 * d] = sum == 0.0f ? 0.0f : __fdiv_rn(acc[d], sum);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 4) tmem_dealloc(tmem, 2 * T::kCols);
}

template <int RP, int DIM>
void launch_split(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                  float* out, void* state, void* scratch) {
    using T = Split<RP, DIM>;
    const uint32_t per_sm = (227 * 1024) / (T::kSmem + 1024), ctas = sm_count * (per_sm < kMostPerSm ? per_sm : kMostPerSm);
    GQ_CUDA(cudaFuncSetAttribute(paged_attn_kernel<RP, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::kSmem));
    launch_after(paged_attn_kernel<RP, DIM>, dim3(ctas), dim3(kThreads), T::kSmem, s, c, st, q, heads, scale * 1.4426950408889634f, out,
                 reinterpret_cast<float*>(scratch), reinterpret_cast<uint32_t*>(state), status);
}

template <int RP>
void launch_rows(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                 float* out, void* state, void* scratch) {
    if (c.dim == 128) launch_split<RP, 128>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else if (c.dim == 64) launch_split<RP, 64>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else launch_split<RP, 32>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
}

}  // namespace

// A counter per CTA; two parts per CTA of at most 32 rows.
uint64_t paged_attn_state_bytes() { return 1024 * kMostPerSm * 4; }
uint64_t paged_attn_scratch_bytes(uint32_t dim, int sm_count) { return (uint64_t)sm_count * kMostPerSm * 2 * 32 * (dim + 2) * 4; }

void launch_paged_attn(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                       uint64_t max_count, float* out, void* state, void* scratch) {
    const uint64_t rows = max_count * (heads / c.kv_heads);
    if (rows <= 8) launch_rows<8>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else if (rows <= 16) launch_rows<16>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else launch_rows<32>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
}

}  // namespace gq
