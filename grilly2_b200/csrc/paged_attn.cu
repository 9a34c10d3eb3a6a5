// Causal grouped-query attention of a step's rows over the paged int8 KV cache, in exact integer products on the fifth-
// generation tensor cores (tcgen05.mma kind::i8), softmax in float32. No counterpart in the reference.
//
//   s[r][j] = scale (q_r . k_j),  w[r][j] = exp(s[r][j] - max),  out[r] = sum_j w[r][j] v_j / sum_j w[r][j]
//
// The cached codes are the A operand exactly as they lie in the pool (its blocks are core matrices of 8 x 16 bytes):
// k_j = kscale_j K_j with 128 keys on the lanes of tensor memory, v_j = vscale_j V_j with the components on the lanes. What
// meets them is held as an exact fixed-point integer in base-256 digits, so that three or four products in int32 and one join
// give a float32 result:
//   q_r = max|q_r| / (127 * 2^16) Q, Q in three signed digits (which hold 127 * 2^16); kscale_j is a factor of a lane;
//   w vscale = 2^-31 P, P in four unsigned digits. The value scales are folded into P because the sum over j runs across blocks:
//     so that P fits, the reference of a row's P is one of its contributions' s + log2 vscale (not of the scores). It follows the
//     tiles of 128 keys: up where a tile's largest contribution passes it, down where that lies 2^15 below it, so that what
//     an attention sink outweighs keeps its digits: a weight is off by 2^-32 of a reference that lies 2^15 above its own tile's
//     largest at most. (Three digits and one reference per row lost what lay 2^-24 below the row's largest: 1e-4 of
//     the row where a key of no value stood 10 nats above 4095 others, 2e-2 at 17 nats; now 4e-7 and 2e-5. They took 633 us
//     for the chunks below and 79.5 for the prompts.) The denominator sums the w themselves in float32, in P's reference.
// As long as no row of a warpgroup moves its reference D goes on adding up in int32, and is read, joined and added to the float32
// sums only when one does (or after 256 tiles, before a sum could leave 32 bits). References are whole numbers, so sums follow them exactly.
// A warp's 32 keys share one block and so one scale (blocks of 32 and more): the maximum is taken over the joined integers
// and scaled afterwards, and the exponent is one multiplication and addition of the integer.
// Scales of values from 2^-100 to 2^90 (and 0) lose nothing; larger, negative or non-finite ones read as NaN. (Below 2^-34 P's
// reference follows the tiles less far down, so that the weights' sum stays a number.)
//
// A CTA takes a contiguous range of all (request, row tile, KV head, 128-key tile) units, with two more units for what an (item
// = request, row tile, KV head) costs beside its tiles, equal ranges for all CTAs: with ragged lengths no CTA waits for a
// long request, and a single request fills the GPU. A row tile is RP rows of (token, head of the group), N = 3 RP digit
// rows. An item that ends inside one range is written out; the others leave (max, sum, weighted V) per CTA and the last CTA of an item to arrive adds them in order (deterministic).
//   last warp      copies the tile's K and V blocks into a ring of stages (bulk copies; the table gives the addresses)
//   the one before issues the products: S = K Q (128 x N) of the next tile as soon as S is read, D = V P (dim x N) when P is written
//   4 WG warps     a thread owns a key of S and RP / WG rows: joins the digits, one maximum over the 128 keys per row (warp
//                  reductions and one exchange), P's digits to shared memory (four keys to a word: a 4 x 4 transposition
//                  between neighbouring lanes; byte stores were 3/5 of the kernel); then it owns a component of D and adds it to
//                  its float32 sums
//
// Bound, and what was measured (B200):
//   long contexts (32 requests of 2000 to 15000 tokens, 32 heads over 8 of 128): the codes' bytes, 442 MB in 80 us = 5.5 TB/s
//   one request, a small batch (700 tokens, 11.7 us; 64 requests of up to 4095 tokens, 24 MB, 17.8 us): latency. The units' scan,
//     the first blocks, three dependent steps a tile and the joining of the parts through L2 are some 10 us
//   chunks of prompts (2 requests, 2795 rows over 3000 cached tokens each, 32 heads of 128): 174 GFLOP in 644 us. Three int8
//     products for S and four for D would take 184; the float32 work beside them is 42 warp instructions per 32 scores, issued at 0.61 of
//     the schedulers' rate
//   short prompts (300 to 1100 tokens, 14 heads over 2 of 64): 82 us, a good third of it items' beginnings and ends (2500 cycles for
//     q's digits, 3000 for the last sums and the output, beside 3300 a tile)
#include "gq_internal.h"
#include "paged.cuh"
#include "tc_common.cuh"

namespace gq {

namespace {

constexpr uint32_t kKeys = 128;    // keys of a tile
constexpr float kNone = -INFINITY;
constexpr uint32_t kMostPerSm = 4;  // CTAs of an SM
constexpr float kUnit = 2147483648.0f;  // 2^31: P's steps of the reference; P passes it by a factor of 2 at most and so has 32 bits
// (all log2) how far above a tile's largest contribution its reference is laid where the quarters' largest lie within kEven of each
// other, and how far that of a later tile may fall below the reference before this follows. Each move reads D out, a quarter of a
// tile's time (4, 8, 6: chunks 652 us, prompts 82.3; 5, 10, 6: 649, 81.6; 5, 10, 10: 643.6, 80.3; if nothing ever moved: 627, 77); 16
// of P's 32 bits and a sum over a tile's keys remain where the two lie farthest apart.
constexpr float kRoom = 5.0f, kEven = 10.0f, kDrop = 9.0f;
constexpr float kQMost = 127.0f * 65536.0f;

template <int RP, int WG, int DIM>
struct Split {
    static constexpr int kRows = RP / WG;                                        // rows of a thread
    static constexpr int kSoft = 128 * WG, kThreads = kSoft + 64;                // softmax threads; all
    static constexpr uint32_t kNw = (3 * kRows + 15) / 16 * 16, kN = WG * kNw;   // columns of S: digit d of a warpgroup's row r in its column d kRows + r
    static constexpr uint32_t kDw = 4 * kRows, kD = WG * kDw;                    // of D
    // bytes from a core matrix of P to that of the next 16 keys: 128 would have the two halves of a warp write the same banks
    static constexpr uint32_t kPStep = RP == 32 ? 192 : 128;
    static constexpr uint32_t kCols = kD <= 32 ? 32 : kD <= 64 ? 64 : 128;       // S at column 0, D at kCols (three digits' columns are fewer than four's)
    static constexpr uint32_t kM = DIM == 128 ? 128 : 64;                        // lanes of D: dim, at least 64
    static constexpr uint32_t kTileBytes = kKeys * DIM, kStageBytes = 2 * kTileBytes;
    static constexpr uint32_t kStages = DIM == 128 ? 2 : DIM == 64 ? 3 : 4;
    // (dim 32: the 64 lanes of D read 32 rows that are not there, up to 4 KB behind the last stage; nobody reads the sums)
    static constexpr uint32_t kQAt = kStages * kStageBytes + (DIM == 32 ? 4096 : 0);
    static constexpr uint32_t kPAt = kQAt + kN * DIM, kMiscAt = kPAt + kD * (kKeys / 16) * (kPStep / 8);
    // blocks' scales of each stage; rows' arrays: scale, last position seen, [4] sums, [2][4] maxima, [4] raw maximum or factor,
    // reference of O and (negative) of P, corrections of O and l, lift and the lift of what D holds, of each warp
    static constexpr uint32_t kSmem = kMiscAt + 1024 + kStages * 128 + RP * 4 * (1 + 1 + 4 + 8 + 28);
    // CTAs of an SM: what shared memory and tensor memory hold
    static constexpr uint32_t kBySmem = (227 * 1024) / (kSmem + 1024), kByTmem = 512 / (2 * kCols), kHeld = kBySmem < kByTmem ? kBySmem : kByTmem;
    static constexpr uint32_t kMost = RP == 16 ? 3 : kMostPerSm;  // (registers)
    static constexpr uint32_t kPerSm = kHeld < kMost ? kHeld : kMost;
    static_assert(kPerSm >= 1 && kPerSm * RP <= kMostPerSm * 32, "the scratch holds the parts");
    static_assert(kN <= kCols, "S and D lie side by side");
};

__device__ __forceinline__ float warp_max(float v) {  // the largest that is a number
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
template <int N>
struct Rows {
    static constexpr int value = N;
};
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[8]) { tmem_ld8(addr, r); }
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// a barrier of the softmax threads that tells every one of them whether all say yes
__device__ __forceinline__ bool all_of(bool mine, uint32_t threads) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, r;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.red.and.pred r, 9, %2, p;\n\t"
        "selp.u32 %0, 1, 0, r;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)mine), "r"(threads)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// A row's scale times a key's: what the joined integer is multiplied by. Never 0, so that the -inf of a key out of sight stays -inf.
__device__ __forceinline__ float factor_of(float row, float key) {
    const float f = row * key;
    return f < 1e-37f ? 1e-37f : f;
}
// 2^n for a whole n of at most 127, 0 below the normal numbers (and for what is no number)
__device__ __forceinline__ float power_of_two(float n) { return n > -127.0f ? __int_as_float(((int)n + 127) << 23) : 0.0f; }
// three digit sums of up to 22 bits, joined with two roundings
__device__ __forceinline__ float join(uint32_t d0, uint32_t d1, uint32_t d2) {
    return __fmaf_rn((float)(int)d2, 65536.0f, (float)((int)d0 + ((int)d1 << 8)));
}

// What the softmax needs to know of a block: x = its key scale; y = log2 of its value scale (of at least 2^-100; of a scale of 0, which
// contributes to the weights' sum alone, as if it were 2^-60) and a margin for the
// rounding, so that P stays below 2^32; z = the value scale times 2^31; w = 0, 1 where a scale is none (negative, beyond 2^90 or
// no number; x is 1 then), 2 where there is no block.
__device__ __forceinline__ float4 block_scale(float ks, float vs) {
    const bool good = vs >= 0.0f && vs <= 1.2379401e27f && ks >= 0.0f && ks <= 3.0e38f;
    return make_float4(good ? ks : 1.0f, fmaxf(__log2f(vs), vs == 0.0f ? -60.0f : -100.0f) + 0.001f, vs * kUnit, good ? 0.0f : 1.0f);
}

// sum of floor((a i + b) / m) for i < n, by Euclid's steps on (a, m): whole multiples of m are taken out of a and b, and what is left
// counts the lattice points under a line, which the transposed line counts with a and m exchanged (Graham, Knuth and Patashnik,
// Concrete Mathematics, section 3.5). The divisions in 32 bits where the numbers allow (a
// 64-bit one is a hundred instructions, and a range's start takes some twenty)
template <class U>
__device__ uint64_t floor_sum_in(U n, U m, U a, U b) {
    uint64_t sum = 0;
    while (n) {
        if (a >= m) sum += (uint64_t)n * (n - 1) / 2 * (a / m), a %= m;
        if (b >= m) sum += (uint64_t)n * (b / m), b %= m;
        const U y = a * n + b;
        if (y < m) break;
        n = y / m, b = y % m;
        const U t = m;
        m = a, a = t;
    }
    return sum;
}
__device__ uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
    return a * n + b < (1ull << 32) && m < (1ull << 32) ? floor_sum_in<uint32_t>((uint32_t)n, (uint32_t)m, (uint32_t)a, (uint32_t)b)
                                                        : floor_sum_in<uint64_t>(n, m, a, b);
}

// What an item's beginning and end cost, in tiles: q's digits, the last sums, the output. Where items have few tiles
// ranges of equal tiles would leave some CTAs with many items (with 0 / 1 / 2 / 3 / 4: prompts of 300 to 1100 tokens
// 115 / 84 / 79 / 82 / 84 us, 64 single tokens 20.2 / 18.8 / 18.1 / 18.6 / 18.8, chunks 646 / 643 / 640 / 640 / 638).
constexpr uint32_t kItem = 2;

// One request's share of the units. A row tile's units are kItem and the 128-key tiles that its last row sees: all of the
// request's for the last row tile, floor((len + last token) / 128) + 1 for the others.
struct Request {
    uint32_t start, rows, len, keys, tiles, row_tiles, group, kv_heads;  // keys = cached and new ones, inside the table
    uint32_t rp;
    __device__ uint32_t tiles_of(uint32_t qt) const { return qt + 1 == row_tiles ? tiles : (len + ((qt + 1) * rp - 1) / group) / kKeys + 1; }
    __device__ uint64_t units_before(uint32_t qt) const {  // qt < row_tiles
        return qt ? kv_heads * ((uint64_t)qt * (1 + kItem) + floor_sum(qt, (uint64_t)kKeys * group, rp, (uint64_t)len * group + rp - 1)) : 0;
    }
    __device__ uint64_t units() const { return row_tiles ? units_before(row_tiles - 1) + (uint64_t)kv_heads * (tiles + kItem) : 0; }
};
__device__ __forceinline__ Request request_of(const PagedView& c, const StepView& s, uint32_t b, uint32_t group, uint32_t rp) {
    Request r;
    r.start = paged_start(s, b);
    const uint32_t end = paged_start(s, b + 1), count = end > r.start ? end - r.start : 0;
    r.rows = count * group, r.len = paged_len(c, b), r.group = group, r.kv_heads = c.kv_heads, r.rp = rp;
    r.keys = min(r.len + count, c.max_blocks << c.shift);
    r.tiles = (r.keys + kKeys - 1) / kKeys, r.row_tiles = (r.rows + rp - 1) / rp;
    return r;
}

// What a stretch of one item's tiles is. The warp that copies walks the CTA's units and hands the segments to the other roles
// through a ring in shared memory.
struct Segment {
    uint32_t b, t0, t1;          // tiles [t0, t1): those with a key that some row of the item sees
    uint32_t row0, rows, head;   // rows of the request's count * group, KV head
    uint32_t clear;              // keys that every row of the item sees
    uint32_t start, len, keys;   // of the request
    uint32_t whole, more;        // the item is this segment; 0: no segment, the end
    uint32_t c0, parts, second;  // the item's first CTA, how many have a part of it, whether the first one's is its second part
    uint64_t first, last;        // the item's units [first, last), of which the first kItem are no tiles
};
constexpr uint32_t kSegments = 4;  // of the ring

// Walks the units [u, hi) of this CTA, segment by segment.
struct Walk {
    uint64_t u, hi, base;  // base = the units before row tile qt of request b
    uint32_t b, qt;
    Request r;
    __device__ bool next(const PagedView& c, const StepView& s, Segment& g) {
        for (;;) {
            g.more = u < hi;
            if (!g.more) return false;
            const uint32_t cost = qt < r.row_tiles ? r.tiles_of(qt) + kItem : 0;  // of an item
            if (cost == 0) {
                r = request_of(c, s, ++b, r.group, r.rp), qt = 0;
                continue;
            }
            if (u >= base + (uint64_t)r.kv_heads * cost) {
                base += (uint64_t)r.kv_heads * cost, ++qt;
                continue;
            }
            const uint32_t v = (uint32_t)(u - base);
            g.head = v / cost;
            const uint32_t at = v - g.head * cost;  // of the item's units; the first kItem are no tiles
            g.first = base + (uint64_t)g.head * cost, g.last = g.first + cost;
            const uint64_t end = min(hi, g.last);
            u = end;
            if (end <= g.first + kItem) continue;  // none of the item's tiles
            g.b = b, g.start = r.start, g.len = r.len, g.keys = r.keys;
            g.whole = at <= kItem && end == g.last;
            g.row0 = qt * r.rp, g.rows = min(r.rp, r.rows - g.row0);
            const uint32_t seen = min(r.len + (g.row0 + g.rows - 1) / r.group + 1, r.keys);  // keys of the tile's last token
            g.clear = min(r.len + g.row0 / r.group + 1, r.keys);
            g.t0 = max(at, kItem) - kItem;
            g.t1 = max(g.t0, min((uint32_t)(end - g.first) - kItem, (seen + kKeys - 1) / kKeys));
            return true;
        }
    }
};

// ONE: the keys of a warp share a block (blocks of 32 tokens and more).
template <int RP, int WG, int DIM, bool ONE>
__global__ void __launch_bounds__((Split<RP, WG, DIM>::kThreads), (Split<RP, WG, DIM>::kPerSm))
    paged_attn_kernel(PagedView c, StepView s, const float* __restrict__ q, uint32_t heads, float scale, float* __restrict__ out,
                      float* __restrict__ partials, uint32_t* counters, uint32_t* status) {
    using T = Split<RP, WG, DIM>;
    constexpr int R = T::kRows;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* misc = smem + T::kMiscAt;
    uint64_t* full = reinterpret_cast<uint64_t*>(misc);  // [kStages] a stage's blocks have landed
    uint64_t* empty = full + 4;                          // [kStages] its products are complete
    uint64_t* s_full = empty + 4;                        // S is complete
    uint64_t* s_read = s_full + 1;                       // S is read
    uint64_t* p_full = s_read + 1;                       // [2] a warpgroup's P is written
    uint64_t* d_full = p_full + 2;                       // [2] its D is complete
    uint64_t* q_full = d_full + 2;                       // Q is written
    uint64_t* seg_full = q_full + 1;                     // [kSegments] a segment is written
    uint64_t* seg_free = seg_full + kSegments;           // [kSegments] ... and done with
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(seg_free + kSegments);
    uint32_t* arrived = tmem_slot + 1;
    volatile uint32_t* failed = arrived + 1;
    volatile uint32_t* go_on = arrived + 2;              // [2] whether a warpgroup's D goes on adding up
    float* low_scale = reinterpret_cast<float*>(misc + 256);      // [kStages] the smallest log2 of a value scale up to the tile
    Segment* segments = reinterpret_cast<Segment*>(misc + 512);   // [kSegments]
    float4* block_scales = reinterpret_cast<float4*>(misc + 1024);  // [kStages][8] what block_scale() gives
    float* row_scale = reinterpret_cast<float*>(misc + 1024 + T::kStages * 128);  // [RP] scale of a row's Q, times log2 e
    int* row_seen = reinterpret_cast<int*>(row_scale + RP);     // [RP] the last position it sees
    float* lsum = reinterpret_cast<float*>(row_seen + RP);      // [4][RP]
    float* exchange = lsum + 4 * RP;                            // [2][RP][4] warps' maxima
    float* refs = exchange + 8 * RP;                            // [4][RP] the rows' references (negative), a copy per warp
    float* corrs = refs + 4 * RP;                               // [4][RP] what older sums are multiplied by
    float* l_corrs = corrs + 4 * RP;                            // [4][RP] ... the older weights' sum
    float* lifts = l_corrs + 4 * RP;                            // [4][RP] 2^(reference of P - reference of O)
    float* held_lifts = lifts + 4 * RP;                         // [4][RP] ... of what is in D
    float* sum_refs = held_lifts + 4 * RP;                      // [4][RP] the references of O
    float* factors = sum_refs + 4 * RP;                        // [4][RP] a warp's raw maxima, then the row's scale times the warp's key scale

    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = heads / c.kv_heads;
    if (tid == 0) {
        for (uint32_t i = 0; i < T::kStages; ++i) mbar_init(full + i, 2), mbar_init(empty + i, 1);
        for (uint32_t i = 0; i < kSegments; ++i) mbar_init(seg_full + i, 1), mbar_init(seg_free + i, T::kSoft + 1);
        for (uint32_t i = 0; i < WG; ++i) mbar_init(p_full + i, 128), mbar_init(d_full + i, 1);
        mbar_init(s_full, 1), mbar_init(s_read, T::kSoft), mbar_init(q_full, T::kSoft);
        *failed = 0;
        mbar_fence_init();
    }
    __syncthreads();
    // Before any tensor memory is taken: a kernel ahead that lets this one start before it has its own columns would wait for those
    // held here, and this one for its end. (Behind the barriers' set-up it costs 0.4 us less than as the first statement.)
    GQ_GRID_DEP_SYNC();
    if (warp == 4 * WG) {
        tmem_alloc(tmem_slot, 2 * T::kCols);
        tc_fence_before_sync();
    }
    uint32_t tmem = 0;
    if (warp != 4 * WG + 1) {  // (the copying warp needs none and goes ahead)
        named_barrier_sync(10, T::kSoft + 32);
        tc_fence_after_sync();
        tmem = *tmem_slot;
    }

    bool ok = true;

    if (warp == 4 * WG + 1) {
        // the units of all requests: lane = a stretch of requests
        const uint32_t per = (c.seqs + 31) / 32, b0 = min(lane * per, c.seqs), b1 = min(b0 + per, c.seqs);
        uint64_t mine = 0;
#pragma unroll 4
        for (uint32_t b = b0; b < b1; ++b) mine += request_of(c, s, b, group, RP).units();
        auto scanned = [&](uint64_t v) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= (uint32_t)o) v += y;
            }
            return v;
        };
        const uint64_t upto = scanned(mine), total = __shfl_sync(0xffffffffu, upto, 31);
        // ranges of `share` units, the first `extra` ones of one more
        const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, total);
        const uint64_t share = ctas ? (total >> 32 ? total / ctas : (uint32_t)total / ctas) : 0, extra = total - share * ctas;
        auto range_at = [&](uint32_t i) { return i * share + min((uint64_t)i, extra); };
        auto cta_of = [&](uint64_t u) {  // whose range holds unit u
            const uint64_t longer = extra * (share + 1);
            const uint64_t v = u < longer ? u : u - longer, by = u < longer ? share + 1 : share;
            return (uint32_t)((u < longer ? 0 : extra) + (v >> 32 || by >> 32 ? v / by : (uint32_t)v / (uint32_t)by));
        };
        Walk walk;
        walk.u = walk.hi = 0;
        if (blockIdx.x < ctas) {
            walk.u = range_at(blockIdx.x), walk.hi = range_at(blockIdx.x + 1);
            // the request that the range starts in: its stretch, then the stretch request by request
            const int in = __ffs(__ballot_sync(0xffffffffu, walk.u >= upto - mine && walk.u < upto)) - 1;
            const uint32_t end = __shfl_sync(0xffffffffu, b1, in);
            walk.b = __shfl_sync(0xffffffffu, b0, in), walk.base = __shfl_sync(0xffffffffu, upto - mine, in), walk.qt = 0;
            while (per > 1) {
                const uint64_t units = walk.b + lane < end ? request_of(c, s, walk.b + lane, group, RP).units() : 0, through = scanned(units);
                const uint32_t hit = __ballot_sync(0xffffffffu, walk.u < walk.base + through);
                const int at = hit ? __ffs(hit) - 1 : 31;
                walk.base += __shfl_sync(0xffffffffu, hit ? through - units : through, at), walk.b += hit ? at : 32;
                if (hit || walk.b >= end) break;
            }
            walk.r = request_of(c, s, walk.b, group, RP);
            if (walk.r.row_tiles > 1) {  // the last row tile that begins at or before u, 32 candidates a round
                const uint64_t v = walk.u - walk.base;
                uint64_t before = 0;
                uint32_t lo = 0, hi = walk.r.row_tiles;
                while (hi - lo > 1) {
                    const uint32_t step = (hi - lo + 31) / 32, k = lo + lane * step;
                    const uint64_t units = k < hi ? walk.r.units_before(k) : ~0ull;
                    const uint32_t at = 31 - __clz(__ballot_sync(0xffffffffu, units <= v));
                    before = __shfl_sync(0xffffffffu, units, at);
                    lo += at * step, hi = min(hi, lo + step);
                }
                walk.base += before, walk.qt = lo;
            }
        }
        uint32_t st = 0, round = 0;
        const uint32_t per_tile = kKeys >> c.shift, bytes = c.block * DIM;  // (at most max_blocks blocks hold the keys)
        for (uint32_t seg = 0; ok; ++seg) {
            Segment g;
            const bool more = walk.next(c, s, g);
            if (seg >= kSegments) ok = mbar_wait(seg_free + seg % kSegments, (seg / kSegments - 1) & 1, failed, status, kStatusEmptyWaitTimedOut);
            if (__ballot_sync(0xffffffffu, !ok)) ok = false;
            if (!ok) break;
            const int32_t* table = c.table + (more ? (size_t)g.b * c.max_blocks : 0);
            auto entry = [&](uint32_t t) {  // one lane per block
                const uint32_t j = t * per_tile + lane;
                return t < g.t1 && lane < per_tile && (j << c.shift) < g.keys ? table[j] : -1;
            };
            int32_t e = more ? entry(g.t0) : -1;  // (requested before the divisions below)
            if (more && !g.whole) g.c0 = cta_of(g.first + kItem), g.parts = cta_of(g.last - 1) - g.c0 + 1, g.second = range_at(g.c0) < g.first;
            if (lane == 0) {
                segments[seg % kSegments] = g;
                mbar_arrive(seg_full + seg % kSegments);
            }
            if (!more) break;
            float low = 0.0f;
            for (uint32_t t = g.t0; t < g.t1; ++t) {
                const int32_t e_next = entry(t + 1);
                e = e >= 0 && (uint32_t)e < c.blocks ? e : -1;
                const size_t at = ((size_t)max(e, 0) * c.kv_heads + g.head);
                const float ks = e >= 0 ? c.kscale[at] : 0.0f, vs = e >= 0 ? c.vscale[at] : 0.0f;
                if (round) ok = ok && mbar_wait(empty + st, (round - 1) & 1, failed, status, kStatusEmptyWaitTimedOut);
                const uint32_t held = __popc(__ballot_sync(0xffffffffu, e >= 0));
                if (__ballot_sync(0xffffffffu, !ok)) ok = false;
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(full + st, held * 2 * bytes);
                __syncwarp();
                if (e >= 0) {
                    uint8_t* dst = smem + st * T::kStageBytes + lane * bytes;
                    bulk_load(dst, c.k + at * bytes, bytes, full + st);
                    bulk_load(dst + T::kTileBytes, c.v + at * bytes, bytes, full + st);
                }
                const float4 sc = e >= 0 ? block_scale(ks, vs) : make_float4(1.0f, 0.0f, 0.0f, 2.0f);
                if (lane < per_tile) block_scales[st * 8 + lane] = sc;
                low = fminf(low, -warp_max(-sc.y));
                if (lane == 0) low_scale[st] = low;
                __syncwarp();
                if (lane == 0) mbar_arrive(full + st);
                e = e_next;
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
    } else if (warp == 4 * WG) {
        if (lane == 0) {
            constexpr uint32_t s_desc = umma_idesc(2, 1, 1, kKeys, T::kN);  // s32 sums, s8 codes x s8 digits of q
            constexpr uint32_t d_desc = umma_idesc(2, 1, 0, T::kM, T::kDw);  // s32 sums, s8 codes x u8 digits of P
            const uint32_t q_addr = smem_u32(smem + T::kQAt), p_addr = smem_u32(smem + T::kPAt);
            uint32_t st = 0, round = 0, tile = 0;
            auto score = [&](uint32_t stage, uint32_t parity) {  // S of the tile in `stage`
                ok = ok && mbar_wait(full + stage, parity, failed, status, kStatusFullWaitTimedOut);
                if (!ok) return;
                tc_fence_after_sync();
                const uint32_t k_addr = smem_u32(smem + stage * T::kStageBytes);
#pragma unroll
                for (uint32_t d = 0; d < DIM / 32; ++d)
                    umma_i8_ss(tmem, umma_desc_plain(k_addr + 256 * d, 128, 8 * DIM), umma_desc_plain(q_addr + 256 * d, 128, 8 * DIM), s_desc, d != 0);
                umma_commit(s_full);
            };
            for (uint32_t i = 0, turn = 0; ok; ++i) {
                ok = mbar_wait(seg_full + i % kSegments, (i / kSegments) & 1, failed, status, kStatusMmaWaitTimedOut);
                if (!ok) break;
                const uint32_t more = segments[i % kSegments].more, tiles = segments[i % kSegments].t1 - segments[i % kSegments].t0;
                mbar_arrive(seg_free + i % kSegments);
                if (!more) break;
                if (tiles == 0) continue;
                ok = mbar_wait(q_full, turn++ & 1, failed, status, kStatusMmaWaitTimedOut);
                score(st, round & 1);
                for (uint32_t t = 0; t < tiles && ok; ++t, ++tile) {
                    const uint32_t here = st;
                    if (++st == T::kStages) st = 0, ++round;
                    ok = mbar_wait(s_read, tile & 1, failed, status, kStatusMmaWaitTimedOut);
                    if (t + 1 < tiles) score(st, round & 1);  // while the tile's weights are computed
                    const uint32_t v_addr = smem_u32(smem + here * T::kStageBytes) + T::kTileBytes;
#pragma unroll
                    for (uint32_t w = 0; w < WG; ++w) {
                        ok = ok && mbar_wait(p_full + w, tile & 1, failed, status, kStatusMmaWaitTimedOut);
                        if (!ok) break;
                        tc_fence_after_sync();
                        const bool more = go_on[w] != 0;
#pragma unroll
                        for (uint32_t i = 0; i < kKeys / 32; ++i) {
                            // keys 32 i ..: two core matrices of one block, or (blocks of 16) of two
                            const uint32_t k0 = 32 * i, at = (k0 >> c.shift) * c.block * DIM + (k0 & (c.block - 1)) * 8;
                            const uint32_t step = c.shift == 4 ? 16 * DIM : 128;
                            umma_i8_ss(tmem + T::kCols + w * T::kDw, umma_desc_plain(v_addr + at, step, 8 * c.block),
                                       umma_desc_plain(p_addr + w * T::kDw * T::kPStep + 2 * T::kPStep * i, T::kPStep, 8 * T::kPStep), d_desc, i != 0 || more);
                        }
                        umma_commit(d_full + w);
                    }
                    if (!ok) break;
                    umma_commit(empty + here);
                }
            }
        }
    } else {
        const uint32_t quarter = warp & 3, wg = warp >> 2, key = tid & 127, wrow = wg * R;  // this thread's key, its first row
        const uint32_t comp = T::kM == 128 ? key : 16 * quarter + lane;                    // the component of D on its lane
        const bool owner = T::kM == 128 || (lane < 16 && comp < (uint32_t)DIM);
        // Four neighbouring lanes give each other their keys' words, a row to a lane: whose words come first, and how a row's four words
        // (of this lane's key, its neighbour's, and the two of the other pair) become its four digits, one key to a byte
        const bool odd = lane & 1, upper = lane & 2;
        const uint32_t sel1 = odd ? 0x1504u : 0x5140u, sel2 = upper ? 0x1054u : 0x5410u;
        uint8_t* const p_at = smem + T::kPAt + wg * T::kDw * T::kPStep + (2 * quarter + (lane >> 4)) * T::kPStep + (lane & 3) * 16 + ((lane >> 2) & 3) * 4;
        float* const my_refs = refs + quarter * RP + wrow;
        float* const my_corrs = corrs + quarter * RP + wrow;
        float* const my_factors = factors + quarter * RP + wrow;
        float* const my_sum_refs = sum_refs + quarter * RP + wrow;
        float* const my_l_corrs = l_corrs + quarter * RP + wrow;
        float* const my_lifts = lifts + quarter * RP + wrow;
        float* const my_held = held_lifts + quarter * RP + wrow;
        uint32_t tile = 0, st = 0, round = 0;
        float O[R], l[R];
        auto products = [&](uint32_t of_tile) {  // D of the tile is complete, P may be written
            ok = ok && mbar_wait(d_full + wg, of_tile & 1, failed, status, kStatusMmaWaitTimedOut);
        };
        auto drain = [&](const float* held, auto at_once) {  // adds D, times its rows' lifts, to the float32 sums, some rows at a time
            tc_fence_after_sync();
            constexpr int kAtOnce = decltype(at_once)::value;
#pragma unroll
            for (int r0 = 0; r0 < R; r0 += kAtOnce) {
                uint32_t d[4][kAtOnce];
                const uint32_t at = tmem_addr(tmem, 32 * quarter, T::kCols + wg * T::kDw + r0);
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld(at + i * R, d[i]);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const float low = __fmaf_rn((float)(int)d[1][i], 256.0f, (float)(int)d[0][i]);
                    const float sum = __fmaf_rn((float)(int)d[3][i], 16777216.0f, __fmaf_rn((float)(int)d[2][i], 65536.0f, low));
                    O[r0 + i] = __fmaf_rn(sum, held[r0 + i], O[r0 + i]);
                }
            }
            tc_fence_before_sync();
        };
        for (uint32_t seg = 0;; ++seg) {
            ok = ok && mbar_wait(seg_full + seg % kSegments, (seg / kSegments) & 1, failed, status, kStatusMmaWaitTimedOut);
            if (!all_of(ok, T::kSoft)) break;  // one verdict for all: they meet at barriers below
            const Segment& g = segments[seg % kSegments];
            if (!g.more) break;
            const uint32_t t0 = g.t0, t1 = g.t1, clear_keys = g.clear;
            // q's rows as three signed digits: lanes of four components
            {
                constexpr uint32_t kLanes = DIM / 4, kAtOnce = T::kSoft / kLanes, kTurns = (RP + kAtOnce - 1) / kAtOnce;
                const uint32_t sub = tid % kLanes, d = 4 * sub;
                float4 row_q[kTurns];  // all loads in flight together
#pragma unroll
                for (uint32_t i = 0; i < kTurns; ++i) {
                    const uint32_t r = tid / kLanes + i * kAtOnce, row = g.row0 + r;
                    row_q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < g.rows)
                        row_q[i] = *reinterpret_cast<const float4*>(q + ((size_t)(g.start + row / group) * heads + g.head * group + row % group) * DIM + d);
                }
#pragma unroll
                for (uint32_t i = 0; i < kTurns; ++i) {
                    const uint32_t r = tid / kLanes + i * kAtOnce, token = (g.row0 + r) / group;
                    if (kTurns * kAtOnce > RP && r >= RP) break;
                    const float4 v = row_q[i];
                    uint32_t m = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                                     max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
#pragma unroll
                    for (uint32_t o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                    const bool finite = m < 0x7f800000u;
                    const float most = fmaxf(__uint_as_float(m), 1e-30f), mult = finite ? copysignf(__fdiv_rn(kQMost, most), scale) : 0.0f;
                    if (sub == 0) {
                        row_scale[r] = finite ? __fdiv_rn(most, kQMost) * fabsf(scale) : __uint_as_float(0x7fc00000u);
                        row_seen[r] = r < g.rows ? (int)min(g.len + token, g.keys - 1) : -1;
                    }
                    const float x[4] = {v.x, v.y, v.z, v.w};
                    uint32_t w0 = 0, w1 = 0, w2 = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        int Q = __float2int_rn(x[j] * mult);  // +-q in steps of its row; |Q| <= 127 * 2^16
                        const int d0 = (int)(int8_t)Q;
                        Q = (Q - d0) >> 8;
                        const int d1 = (int)(int8_t)Q, d2 = (Q - d1) >> 8;
                        w0 |= ((uint32_t)d0 & 0xffu) << (8 * j), w1 |= ((uint32_t)d1 & 0xffu) << (8 * j), w2 |= ((uint32_t)d2 & 0xffu) << (8 * j);
                    }
                    uint8_t* qd = smem + T::kQAt;
                    const uint32_t n = r / R * T::kNw + r % R;
                    *reinterpret_cast<uint32_t*>(qd + key_at(DIM, n, d)) = w0;
                    *reinterpret_cast<uint32_t*>(qd + key_at(DIM, n + R, d)) = w1;
                    *reinterpret_cast<uint32_t*>(qd + key_at(DIM, n + 2 * R, d)) = w2;
                }
            }
            named_barrier_sync(8, T::kSoft);  // row_scale, row_seen
            if (t0 < t1) {
                fence_proxy_async_smem();
                mbar_arrive(q_full);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) O[r] = l[r] = 0.0f;
            uint32_t since = 0;  // tiles in D
            if (lane < (uint32_t)R) my_sum_refs[lane] = kNone, my_refs[lane] = 0.0f, my_lifts[lane] = 0.0f;  // (a row that sees no key keeps these)
            __syncwarp();
            for (uint32_t t = t0; t < t1; ++t, ++tile) {
                ok = ok && mbar_wait(full + st, round & 1, failed, status, kStatusFullWaitTimedOut);
                const float4 sc = block_scales[st * 8 + (key >> c.shift)];
                const float* const low = low_scale + st;
                if (++st == T::kStages) st = 0, ++round;
                ok = ok && mbar_wait(s_full, tile & 1, failed, status, kStatusMmaWaitTimedOut);
                tc_fence_after_sync();
                float a[R];  // q . k in units of the row's and the key's scales
#pragma unroll
                for (int r0 = 0; r0 < R; r0 += 8) {
                    uint32_t d0[8], d1[8], d2[8];
                    const uint32_t at = tmem_addr(tmem, 32 * quarter, wg * T::kNw + r0);
                    tmem_ld8(at, d0), tmem_ld8(at + R, d1), tmem_ld8(at + 2 * R, d2);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) a[r0 + i] = join(d0[i], d1[i], d2[i]);
                }
                tc_fence_before_sync();
                mbar_arrive(s_read);
                // Where some row does not see some key, or a scale is none: a key out of sight scores -inf, and a row that sees a
                // key without a scale has no sum. (The factors are finite and not 0, so that -inf stays -inf.)
                if ((t + 1) * kKeys > clear_keys || __any_sync(0xffffffffu, sc.w != 0.0f)) {
                    const int pos = sc.w == 2.0f ? 0x7fffffff : (int)(t * kKeys + key);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const bool seen = pos <= row_seen[wrow + r];
                        if (!seen) a[r] = kNone;
                        else if (sc.w != 0.0f) l[r] = __uint_as_float(0x7fc00000u);
                    }
                }
                float* ex = exchange + ((tile & 1) * RP + wrow) * 4;
#pragma unroll
                for (int r = 0; r < R; r += 4) {
                    float m[4];
                    float4 rs;
                    if (!ONE) rs = *reinterpret_cast<const float4*>(row_scale + wrow + r);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        m[i] = warp_max(ONE ? a[r + i] : __fmaf_rn(a[r + i], factor_of(i == 0 ? rs.x : i == 1 ? rs.y : i == 2 ? rs.z : rs.w, sc.x), sc.y));
                    if (lane == 0) *reinterpret_cast<float4*>(my_factors + r) = make_float4(m[0], m[1], m[2], m[3]);
                }
                __syncwarp();
                if (lane < (uint32_t)R) {
                    const float raw = my_factors[lane], f = factor_of(row_scale[wrow + lane], sc.x);
                    ex[lane * 4 + quarter] = ONE ? __fmaf_rn(raw, f, sc.y) : raw;
                    if (ONE) my_factors[lane] = f;
                }
                named_barrier_sync(1 + wg, 128);
                // References are whole numbers: what older sums are multiplied by, and D on its way into O, are exact powers of two.
                // P's lies up to 2^60 below O's, and by less where a weight is many times its contribution: l stays below 2^127.
                bool moved = false, raised = false;
                if (lane < (uint32_t)R) {
                    const float4 m = *reinterpret_cast<const float4*>(ex + lane * 4);
                    const float top = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w)), M = my_sum_refs[lane], mu = -my_refs[lane];
                    raised = top > M + 1.0f;  // (-inf passes nothing, anything passes -inf)
                    // room above for the tiles to come, except for a tile in which some keys tower over the others
                    const float room = ceilf(top) + (top - fminf(fminf(m.x, m.y), fminf(m.z, m.w)) < kEven ? kRoom : 0.0f);
                    const float next = raised ? room : fmaxf(room, M - fmaxf(fminf(94.0f + *low, 60.0f), 0.0f));
                    moved = raised || top > mu + 1.0f || (next < mu - kDrop && top > kNone);
                    my_held[lane] = my_lifts[lane];
                    my_corrs[lane] = raised ? power_of_two(M - next) : 1.0f;
                    my_l_corrs[lane] = !moved ? 1.0f : M == kNone ? 0.0f : power_of_two(mu - next);
                    if (raised) my_sum_refs[lane] = next;
                    if (moved) my_refs[lane] = -next, my_lifts[lane] = raised ? 1.0f : power_of_two(next - M);
                }
                __syncwarp();
                // the same in all four warps of the warpgroup
                const uint32_t rows_moved = __ballot_sync(0xffffffffu, moved);
                const bool more = t > t0 && !rows_moved && since < 255;
                if (t > t0) products(tile - 1);
                if (t > t0 && !more) drain(my_held, Rows<R == 16 ? 4 : 8>());  // (fewer registers beside the scores)
                since = more ? since + 1 : 0;
                if (key == 0) go_on[wg] = more;
                if (rows_moved) {
#pragma unroll
                    for (int r = 0; r < R; r += 4)
                        if (rows_moved >> r & 15u) {
                            const float4 cr = *reinterpret_cast<const float4*>(my_corrs + r), lr = *reinterpret_cast<const float4*>(my_l_corrs + r);
                            O[r] *= cr.x, O[r + 1] *= cr.y, O[r + 2] *= cr.z, O[r + 3] *= cr.w;
                            l[r] *= lr.x, l[r + 1] *= lr.y, l[r + 2] *= lr.z, l[r + 3] *= lr.w;
                        }
                }
#pragma unroll
                for (int r = 0; r < R; r += 4) {
                    const float4 rf = *reinterpret_cast<const float4*>(my_refs + r);
                    const float4 fc = *reinterpret_cast<const float4*>((ONE ? my_factors : row_scale + wrow) + r);
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = i == 0 ? fc.x : i == 1 ? fc.y : i == 2 ? fc.z : fc.w, ref = i == 0 ? rf.x : i == 1 ? rf.y : i == 2 ? rf.z : rf.w;
                        const float p = exp2_fast(__fmaf_rn(a[r + i], ONE ? f : factor_of(f, sc.x), ref));
                        l[r + i] += p;
                        x[i] = __float2uint_rn(p * sc.z);  // P
                    }
                    const uint32_t k0 = odd ? x[1] : x[0], k1 = odd ? x[3] : x[2];
                    const uint32_t g0 = __shfl_xor_sync(0xffffffffu, odd ? x[0] : x[1], 1), g1 = __shfl_xor_sync(0xffffffffu, odd ? x[2] : x[3], 1);
                    const uint32_t own = upper ? k1 : k0, next = upper ? g1 : g0;  // row r + lane % 4 of this lane's key and its neighbour's
                    const uint32_t far = __shfl_xor_sync(0xffffffffu, upper ? k0 : k1, 2), last = __shfl_xor_sync(0xffffffffu, upper ? g0 : g1, 2);
                    const uint32_t a01 = __byte_perm(own, next, sel1), a23 = __byte_perm(own, next, sel1 + 0x2222u);
                    const uint32_t b01 = __byte_perm(far, last, sel1), b23 = __byte_perm(far, last, sel1 + 0x2222u);
                    const uint32_t w[4] = {__byte_perm(a01, b01, sel2), __byte_perm(a01, b01, sel2 + 0x2222u), __byte_perm(a23, b23, sel2),
                                           __byte_perm(a23, b23, sel2 + 0x2222u)};
#pragma unroll
                    for (uint32_t d = 0; d < 4; ++d) {
                        const uint32_t n = d * R + r;
                        *reinterpret_cast<uint32_t*>(p_at + (n >> 3) * 8 * T::kPStep + (n & 7) * 16) = w[d];
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                mbar_arrive(p_full + wg);
            }
            if (t0 < t1) products(tile - 1), drain(my_lifts, Rows<8>());
            // the rows' sums over the keys, in a fixed order: a lane gives away half of its rows with each step, until it has row
            // lane / kShare
            constexpr uint32_t kShare = 32 / R;
#pragma unroll
            for (uint32_t w = R / 2, o = 16; o > 0; w >>= 1, o >>= 1) {
                if (w == 0) l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
#pragma unroll
                for (uint32_t i = 0; i < w; ++i) {
                    const float keep = lane & o ? l[i + w] : l[i], give = lane & o ? l[i] : l[i + w];
                    l[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            }
            if (lane % kShare == 0) lsum[quarter * RP + wrow + lane / kShare] = l[0];
            named_barrier_sync(8, T::kSoft);  // (the next segment's first barrier keeps lsum until all have read it)
            // of row r, in O's reference
            auto sum_of = [&](uint32_t r) { return ((lsum[r] + lsum[RP + r]) + (lsum[2 * RP + r] + lsum[3 * RP + r])) * lifts[r]; };
            // a row that saw no key has neither sum and gives zeros. (P's unit is taken out of the other sum: where value scales are near
            // 2^-100, so that the weights' sum is beyond 2^100, the quotient would leave the normal numbers with it.)
            auto share_of = [](float sum) { return sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum); };
            if (g.whole) {
                float share = 0.0f;  // of row `lane`, and its place
                int place = -1;
                if (lane < (uint32_t)R) {
                    const uint32_t row = g.row0 + wrow + lane;
                    share = share_of(sum_of(wrow + lane));
                    if (wrow + lane < g.rows) place = (int)(row / group * heads + row % group);
                }
                float* at = out + ((size_t)g.start * heads + g.head * group) * DIM + comp;
                mbar_arrive(seg_free + seg % kSegments);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int row = __shfl_sync(0xffffffffu, place, r);
                    const float v = O[r] * (1.0f / kUnit) * __shfl_sync(0xffffffffu, share, r);
                    if (owner && row >= 0) at[(size_t)row * DIM] = v;
                }
                continue;
            }
            // a part of an item: what this CTA has, and the last CTA to arrive adds the parts up
            constexpr uint32_t kPart = RP * (DIM + 2);
            const uint32_t c0 = g.c0, parts = g.parts, second = g.second;
            auto part_of = [&](uint32_t cta) { return partials + (size_t)(cta * 2 + (cta == c0 ? second : 0)) * kPart; };
            float* part = part_of(blockIdx.x);
            if (owner)
#pragma unroll
                for (int r = 0; r < R; ++r) part[(wrow + r) * DIM + comp] = O[r];
            if (quarter == 0 && lane < (uint32_t)R) part[RP * DIM + wrow + lane] = my_sum_refs[lane], part[RP * DIM + RP + wrow + lane] = sum_of(wrow + lane);
            __threadfence();
            named_barrier_sync(8, T::kSoft);
            if (tid == 0) *arrived = atomicAdd(counters + c0, 1u);
            named_barrier_sync(8, T::kSoft);
            if (*arrived != parts - 1) {
                mbar_arrive(seg_free + seg % kSegments);
                continue;
            }
            __threadfence();
            if (tid == 0) counters[c0] = 0;  // ready for the next call
            auto out_at = [&](uint32_t r) {
                const uint32_t row = g.row0 + r;
                return out + ((size_t)(g.start + row / group) * heads + g.head * group + row % group) * DIM;
            };
            constexpr uint32_t kVec = DIM / 32;  // components of a lane
            for (uint32_t r = warp; r < g.rows; r += 4 * WG) {
                float top = kNone;
                for (uint32_t i = lane; i < parts; i += 32) top = fmaxf(top, __ldcg(part_of(c0 + i) + RP * DIM + r));
                top = warp_max(top);
                const float ref = top == kNone ? 0.0f : top;
                float sum = 0.0f, acc[kVec] = {};
                for (uint32_t i0 = 0; i0 < parts; i0 += 32) {
                    const uint32_t i = i0 + lane, here = min(32u, parts - i0);
                    float wgt = 0.0f;
                    if (i < parts) {
                        const float* pp = part_of(c0 + i) + RP * DIM + r;
                        wgt = exp2_fast(__ldcg(pp) - ref);
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
                const float factor = share_of(sum);
#pragma unroll
                for (uint32_t d = 0; d < kVec; ++d) out_at(r)[lane + 32 * d] = acc[d] * (1.0f / kUnit) * factor;
            }
            mbar_arrive(seg_free + seg % kSegments);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 4 * WG) tmem_dealloc(tmem, 2 * T::kCols);
}

template <int RP, int WG, int DIM, bool ONE>
void launch_split(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                  float* out, void* state, void* scratch) {
    using T = Split<RP, WG, DIM>;
    GQ_CUDA(cudaFuncSetAttribute(paged_attn_kernel<RP, WG, DIM, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::kSmem));
    launch_after(paged_attn_kernel<RP, WG, DIM, ONE>, dim3(sm_count * T::kPerSm), dim3(T::kThreads), T::kSmem, s, c, st, q, heads, scale * 1.4426950408889634f, out,
                 reinterpret_cast<float*>(scratch), reinterpret_cast<uint32_t*>(state), status);
}

template <int RP, int WG, bool ONE>
void launch_rows(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                 float* out, void* state, void* scratch) {
    if (c.dim == 128) launch_split<RP, WG, 128, ONE>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else if (c.dim == 64) launch_split<RP, WG, 64, ONE>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else launch_split<RP, WG, 32, ONE>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
}
template <bool ONE>
void launch_blocks(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                   uint64_t rows, float* out, void* state, void* scratch) {
    // Rows of a tile: as few as hold a request's rows while these are few, since a score costs the same whether its row is real
    // or not. Tiles of 8 / 16 / 32 rows (before items had units of their own): 64 requests with one token of 7 heads a group 20.1 / 24.3 / 30.3 us, 32 long
    // contexts of 4 heads a group 81 / 101 / 125; prompts of 300 to 1100 tokens 165 / 140 / 116, chunks of 1400 tokens
    // 1118 / 923 / 647. Many rows: 32 over two warpgroups, two CTAs an SM, took 638 us for the chunks and 112 for the
    // prompts, tiles of 40 rows 696 and 122, of 64 rows
    // over four warpgroups 726 and 127, over two 794, of 32 over one 788 (all before the weights had 24 bits, which cost 2 %).
    if (rows <= 8) launch_rows<8, 1, ONE>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else if (rows <= 16) launch_rows<16, 1, ONE>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
    else launch_rows<32, 2, ONE>(s, sm_count, status, c, st, q, heads, scale, out, state, scratch);
}

}  // namespace

// A counter per CTA; two parts per CTA, of at most 32 rows with kMostPerSm CTAs an SM.
uint64_t paged_attn_state_bytes() { return 1024 * kMostPerSm * 4; }
uint64_t paged_attn_scratch_bytes(uint32_t dim, int sm_count) { return (uint64_t)sm_count * kMostPerSm * 2 * 32 * (dim + 2) * 4; }

void launch_paged_attn(cudaStream_t s, int sm_count, uint32_t* status, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale,
                       uint64_t max_count, float* out, void* state, void* scratch) {
    const uint64_t rows = max_count * (heads / c.kv_heads);
    if (c.block >= 32) launch_blocks<true>(s, sm_count, status, c, st, q, heads, scale, rows, out, state, scratch);
    else launch_blocks<false>(s, sm_count, status, c, st, q, heads, scale, rows, out, state, scratch);
}

}  // namespace gq
