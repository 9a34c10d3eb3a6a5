// Causal grouped-query attention of a step's rows over the paged int8 KV cache. One warp per (row, head): lanes take
// keys for q k^T, components for the weighted sum; online softmax in float32.
#include "gq_internal.h"
#include "paged.cuh"

namespace gq {

namespace {

constexpr int kWarps = 4;

__global__ void __launch_bounds__(kWarps * 32) paged_attn_kernel(PagedView c, StepView s, const float* __restrict__ q, uint32_t heads, float scale,
                                                                float* __restrict__ out) {
    GQ_GRID_DEP_SYNC();
    __shared__ float s_q[kWarps][128];
    const uint32_t w = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = c.dim, per = dim / 32;
    const uint64_t item = (uint64_t)blockIdx.x * kWarps + w;
    const uint32_t t = (uint32_t)(item / heads), h = (uint32_t)(item - (uint64_t)t * heads), g = h / (heads / c.kv_heads);
    if (t >= paged_start(s, c.seqs)) return;
    uint32_t lo = 0, hi = c.seqs;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (paged_start(s, mid) <= t) lo = mid;
        else hi = mid;
    }
    const uint32_t keys = min(paged_len(c, lo) + (t - paged_start(s, lo)) + 1, c.max_blocks << c.shift);
    const int32_t* table = c.table + (size_t)lo * c.max_blocks;
    for (uint32_t d = lane; d < dim; d += 32) s_q[w][d] = q[((size_t)t * heads + h) * dim + d] * scale;
    __syncwarp();
    const float none = __uint_as_float(0xff800000u);
    float m = none, l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t j0 = 0; j0 < keys; j0 += 32) {
        const uint32_t j = j0 + lane;
        const int32_t e = j < keys ? table[j >> c.shift] : -1;
        const bool seen = e >= 0 && (uint32_t)e < c.blocks;
        float a = none, vs = 0.0f;
        if (seen) {
            const int8_t* kp = c.k + ((size_t)e * c.kv_heads + g) * c.block * dim;
            const uint32_t tok = j & (c.block - 1);
            a = 0.0f;
            for (uint32_t d = 0; d < dim; ++d) a = __fmaf_rn(s_q[w][d], (float)kp[key_at(dim, tok, d)], a);
            vs = c.vscale[(size_t)e * c.kv_heads + g];
            a *= c.kscale[(size_t)e * c.kv_heads + g];
        }
        float cm = a;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
        const float mn = fmaxf(m, cm);
        if (mn == none && !__any_sync(0xffffffffu, a != a)) continue;  // nothing seen yet
        const float corr = m == mn ? 1.0f : expf(m - mn);
        const float p = seen ? expf(a - mn) : 0.0f;
        float ps = p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
        l = __fmaf_rn(l, corr, ps);
        for (uint32_t i = 0; i < 4; ++i) acc[i] *= corr;
        for (uint32_t jj = 0; jj < min(32u, keys - j0); ++jj) {
            const int32_t be = __shfl_sync(0xffffffffu, e, jj);
            const float pv = __shfl_sync(0xffffffffu, p * vs, jj);
            if (be < 0 || (uint32_t)be >= c.blocks) continue;
            const int8_t* vp = c.v + ((size_t)be * c.kv_heads + g) * c.block * dim;
            for (uint32_t i = 0; i < per; ++i) acc[i] = __fmaf_rn(pv, (float)vp[value_at(c.block, (j0 + jj) & (c.block - 1), lane + 32 * i)], acc[i]);
        }
        m = mn;
    }
    for (uint32_t i = 0; i < per; ++i) out[((size_t)t * heads + h) * dim + lane + 32 * i] = l == 0.0f ? 0.0f : __fdiv_rn(acc[i], l);
}

}  // namespace

void launch_paged_attn(cudaStream_t s, const PagedView& c, const StepView& st, const float* q, uint32_t heads, float scale, float* out) {
    const uint64_t items = (uint64_t)st.tokens * heads;
    launch_after(paged_attn_kernel, dim3((uint32_t)((items + kWarps - 1) / kWarps)), dim3(kWarps * 32), 0, s, c, st, q, heads, scale, out);
}

}  // namespace gq
