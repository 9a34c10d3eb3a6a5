// The next token of every row with settings of its own: temperature, top-k, top-p, min-p, and the draw by the inverse CDF in
// token order. One CTA per row; thresholds by bisection over the order-preserving bits of the logits, every sum in
// float64 in a fixed order.
#include "gq_internal.h"

namespace gq {

namespace {

constexpr int kThreads = 1024;

__device__ __forceinline__ uint32_t key_of(float f) {  // a < b as floats <=> key_of(a) < key_of(b); NaN as -inf
    const uint32_t b = f == f ? __float_as_uint(f) : 0xff800000u;
    return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }

template <typename T>
__device__ T sum_all(T v, T* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    T t = 0;
    for (int w = 0; w < kThreads / 32; ++w) t += red[w];
    return t;
}

__global__ void __launch_bounds__(kThreads) sample_rows_kernel(const float* __restrict__ logits, uint32_t vocab, const float* __restrict__ temperature,
                                                              const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                                                              const float* __restrict__ min_p, const float* __restrict__ uniforms, uint32_t uniform_rows,
                                                              uint32_t* draws, int32_t* tokens, float* probs, uint32_t* ticket) {
    GQ_GRID_DEP_SYNC();
    __shared__ double red_d[32];
    __shared__ uint32_t red_u[32];
    __shared__ double part[kThreads];
    
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float* x = logits + (size_t)row * vocab;
    const float u = uniforms[(size_t)(draws ? *draws % uniform_rows : 0u) * gridDim.x + row];
    if (draws) {  // the last row to have read the counter advances it
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            if (atomicAdd(ticket, 1u) == gridDim.x - 1) *ticket = 0, *draws += 1;
        }
    }
    uint32_t mk = 0;
    for (uint32_t i = tid; i < vocab; i += kThreads) mk = max(mk, key_of(x[i]));
    mk = __reduce_max_sync(0xffffffffu, mk);
    if ((tid & 31) == 0) red_u[tid >> 5] = mk;
    __syncthreads();
    for (int w = 0; w < 32; ++w) mk = max(mk, red_u[w]);
    __syncthreads();
    const uint32_t floor_key = key_of(__uint_as_float(0xff800000u));
    const double top = (double)value_of(mk), temp = (double)temperature[row];
    auto weight = [&](uint32_t key) { return key == mk ? 1.0 : exp(((double)value_of(key) - top) / temp); };
    uint32_t low = floor_key + 1;  // keep keys >= low
    const bool greedy = !(temp > 0.0);
    if (mk == floor_key) {
        if (tid == 0) {
            tokens[row] = -1;
            if (probs) probs[row] = 0.0f;
        }
        return;
    }
    if (greedy) {
        low = mk;
    } else {
        const int32_t k = top_k[row];
        if (k > 0 && (uint32_t)k < vocab) {
            uint32_t lo = low, hi = mk;  // the largest key that at least k tokens reach
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                uint32_t n = 0;
                for (uint32_t i = tid; i < vocab; i += kThreads) n += key_of(x[i]) >= mid;
                if (sum_all(n, red_u) >= (uint32_t)k) lo = mid;
                else hi = mid - 1;
            }
            low = lo;
        }
        const double p = (double)top_p[row];
        if (p < 1.0) {
            double z = 0.0;
            for (uint32_t i = tid; i < vocab; i += kThreads) z += key_of(x[i]) >= low ? weight(key_of(x[i])) : 0.0;
            const double target = p * sum_all(z, red_d);
            uint32_t lo = low, hi = mk;  // the smallest key above which there is less than the target
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                double above = 0.0;
                for (uint32_t i = tid; i < vocab; i += kThreads) above += key_of(x[i]) > mid ? weight(key_of(x[i])) : 0.0;
                if (sum_all(above, red_d) < target) hi = mid;
                else lo = mid + 1;
            }
            low = lo;
        }
    }
    const double least = greedy ? 0.0 : (double)min_p[row];
    auto kept = [&](uint32_t key) -> double {
        if (key < low) return 0.0;
        const double w = weight(key);
        return w >= least || key == mk ? w : 0.0;
    };
    const uint32_t per = (vocab + kThreads - 1) / kThreads, i0 = min(tid * per, vocab), i1 = min(i0 + per, vocab);
    double mine = 0.0;
    for (uint32_t i = i0; i < i1; ++i) mine += kept(key_of(x[i]));
    part[tid] = mine;
    __syncthreads();
    if (tid == 0) {
        double total = 0.0;
        for (int t = 0; t < kThreads; ++t) total += part[t];
        const double target = greedy ? 0.0 : (double)u * total;
        double before = 0.0, behind = 0.0;
        uint32_t owner = 0, chosen = 0;
        for (uint32_t t = 0; t < kThreads; ++t) {
            if (part[t] == 0.0) continue;
            before = behind, owner = t, behind += part[t];
            if (behind > target) break;  // else the last thread with anything kept
        }
        double run = before;
        for (uint32_t i = owner * per; i < min(owner * per + per, vocab); ++i) {
            const double w = kept(key_of(x[i]));
            if (w == 0.0) continue;
            chosen = i, run += w;
            if (run > target) break;
        }
        tokens[row] = (int32_t)chosen;
        if (probs) probs[row] = (float)(kept(key_of(x[chosen])) / total);
    }
}

}  // namespace

void launch_sample_rows(cudaStream_t s, const float* logits, uint32_t rows, uint32_t vocab, const float* temperature, const int32_t* top_k,
                        const float* top_p, const float* min_p, const float* uniforms, uint32_t uniform_rows, uint32_t* draws, int32_t* tokens, float* probs,
                        uint32_t* ticket) {
    launch_after(sample_rows_kernel, dim3(rows), dim3(kThreads), 0, s, logits, vocab, temperature, top_k, top_p, min_p, uniforms, uniform_rows, draws, tokens, probs, ticket);
}

}  // namespace gq
