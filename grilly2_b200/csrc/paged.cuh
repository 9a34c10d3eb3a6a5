// What the kernels of the paged int8 KV cache share (paged.cu, paged_attn.cu): the cache as device pointers, and the
// checks that keep every index a device buffer supplies inside the pool.
#pragma once

#include <cstdint>

namespace gq {

struct PagedView {
    int8_t* k = nullptr;  // this layer's pool: [blocks][kv_heads][block * dim]
    int8_t* v = nullptr;
    float* kscale = nullptr;  // [blocks][kv_heads]
    float* vscale = nullptr;
    int32_t* table = nullptr;  // [seqs][max_blocks]
    int32_t* lens = nullptr;   // [seqs]
    uint32_t blocks = 0, block = 0, shift = 0, kv_heads = 0, dim = 0, seqs = 0, max_blocks = 0;  // block = 1 << shift
};
struct StepView {
    int32_t *starts = nullptr, *slots = nullptr, *positions = nullptr, *runs = nullptr, *last = nullptr, *info = nullptr;
    uint32_t tokens = 0, runs_cap = 0;
};

constexpr uint32_t kPagedMaxSeqs = 4096;

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t paged_len(const PagedView& c, uint32_t b) {
    return (uint32_t)min(max(c.lens[b], 0), (int32_t)(c.max_blocks << c.shift));
}
// rows before request b, inside the step whatever the buffer holds
__device__ __forceinline__ uint32_t paged_start(const StepView& s, uint32_t b) { return (uint32_t)min(max(s.starts[b], 0), (int32_t)s.tokens); }
// byte of (token, component) in a key block and of (component, token) in a value block
__device__ __forceinline__ uint32_t key_at(uint32_t dim, uint32_t t, uint32_t d) { return (t >> 3) * 8 * dim + (d >> 4) * 128 + (t & 7) * 16 + (d & 15); }
__device__ __forceinline__ uint32_t value_at(uint32_t block, uint32_t t, uint32_t d) {
    return (d >> 3) * 8 * block + (t >> 4) * 128 + (d & 7) * 16 + (t & 15);
}
#endif

}  // namespace gq
