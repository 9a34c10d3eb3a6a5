// C ABI of the paged int8 KV cache and of sampling by rows (include/gq.h): argument checks against buffer sizes, then the
// launchers of paged.cu, paged_attn.cu and sample_rows.cu.
#include "gq_internal.h"
#include "paged.cuh"

using namespace gq;

namespace {

using ull = unsigned long long;

// The geometry of a cache, refused where a kernel's index could leave its buffer or 32 bits.
PagedView cache_view(gq_ctx* ctx, const char* op, const gq_paged_cache* c, uint64_t layer, bool pool) {
    if (!c) fail("%s: null cache", op);
    if (c->block_size != 16 && c->block_size != 32 && c->block_size != 64 && c->block_size != 128)
        fail("%s: block_size must be 16, 32, 64 or 128, got %llu", op, (ull)c->block_size);
    if (c->seqs == 0 || c->seqs > kPagedMaxSeqs) fail("%s: 1 to %u requests, got %llu", op, kPagedMaxSeqs, (ull)c->seqs);
    if (c->blocks == 0 || c->max_blocks == 0) fail("%s: a cache of no blocks", op);
    check_dims(op, c->blocks, c->max_blocks, c->layers);
    if (c->blocks * c->block_size > 0x7fffffffull || c->seqs * c->max_blocks > 0x7fffffffull || c->max_blocks * c->block_size > 0x7fffffffull)
        fail("%s: the pool and the tables must stay below 2^31 tokens and entries", op);
    PagedView v;
    v.blocks = (uint32_t)c->blocks, v.block = (uint32_t)c->block_size, v.seqs = (uint32_t)c->seqs, v.max_blocks = (uint32_t)c->max_blocks;
    while ((1u << v.shift) < v.block) ++v.shift;
    v.table = (int32_t*)view(ctx, c->table, 0, c->seqs * c->max_blocks, 4, "the block table");
    v.lens = (int32_t*)view(ctx, c->lens, 0, c->seqs, 4, "the cached lengths");
    if (!pool) return v;
    if (c->kv_heads == 0 || c->kv_heads > 4096) fail("%s: 1 to 4096 KV heads, got %llu", op, (ull)c->kv_heads);
    if (c->dim != 32 && c->dim != 64 && c->dim != 128) fail("%s: head_dim must be 32, 64 or 128, got %llu", op, (ull)c->dim);
    if (layer >= c->layers) fail("%s: layer %llu of %llu", op, (ull)layer, (ull)c->layers);
    v.kv_heads = (uint32_t)c->kv_heads, v.dim = (uint32_t)c->dim;
    const uint64_t scales = c->blocks * c->kv_heads, codes = scales * c->block_size * c->dim;  // < 2^31 * 2^12 * 2^7
    v.k = (int8_t*)view(ctx, c->k, layer * codes, codes, 1, "the key pool");
    v.v = (int8_t*)view(ctx, c->v, layer * codes, codes, 1, "the value pool");
    v.kscale = (float*)view(ctx, c->kscale, layer * scales, scales, 4, "the key scales");
    v.vscale = (float*)view(ctx, c->vscale, layer * scales, scales, 4, "the value scales");
    if (((uintptr_t)v.k | (uintptr_t)v.v) & 15) fail("%s: the pool must lie on 16-byte boundaries", op);
    return v;
}

StepView step_view(gq_ctx* ctx, const char* op, const gq_paged_cache* c, const gq_paged_step* st) {
    if (!st) fail("%s: null step", op);
    check_dims(op, st->max_tokens, 1);
    if (st->max_tokens == 0) fail("%s: a step of no rows", op);
    StepView v;
    v.tokens = (uint32_t)st->max_tokens, v.runs_cap = (uint32_t)GQ_PAGED_RUNS(st->max_tokens, c->block_size, c->seqs);
    v.starts = (int32_t*)view(ctx, st->starts, 0, c->seqs + 1, 4, "the step's starts");
    v.slots = (int32_t*)view(ctx, st->slots, 0, st->max_tokens, 4, "the step's slots");
    v.positions = (int32_t*)view(ctx, st->positions, 0, st->max_tokens, 4, "the step's positions");
    v.runs = (int32_t*)view(ctx, st->runs, 0, (uint64_t)v.runs_cap + 1, 4, "the step's runs");
    v.last = (int32_t*)view(ctx, st->last, 0, c->seqs, 4, "the step's last rows");
    v.info = (int32_t*)view(ctx, st->info, 0, 2, 4, "the step's info");
    return v;
}

void check_aligned(const char* op, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if ((uintptr_t)p & 15) fail("%s: buffers must lie on 16-byte boundaries", op);
}

// A kernel's CTAs write some buffers while others read theirs: what is written must lie apart from all else the call names.
struct Range {
    const char* what;
    const void* p;
    uint64_t bytes;
};
void check_apart(const char* op, std::initializer_list<Range> written, std::initializer_list<Range> read) {
    for (const Range* w = written.begin(); w != written.end(); ++w) {
        for (const Range* o = w + 1; o != written.end(); ++o)
            if (ranges_overlap(w->p, w->bytes, o->p, o->bytes)) fail("%s: %s must not overlap %s", op, w->what, o->what);
        for (const Range& r : read)
            if (ranges_overlap(w->p, w->bytes, r.p, r.bytes)) fail("%s: %s must not overlap %s", op, w->what, r.what);
    }
}
uint64_t table_bytes(const PagedView& c) { return (uint64_t)c.seqs * c.max_blocks * 4; }
uint64_t code_bytes(const PagedView& c) { return (uint64_t)c.blocks * c.kv_heads * c.dim << c.shift; }
uint64_t scale_bytes(const PagedView& c) { return (uint64_t)c.blocks * c.kv_heads * 4; }

uint64_t check_heads(const char* op, const PagedView& c, uint64_t heads) {
    if (heads == 0 || heads > 65536 || heads % c.kv_heads)
        fail("%s: %llu heads do not group over %u kv heads", op, (ull)heads, c.kv_heads);
    return heads * c.dim;
}

}  // namespace

extern "C" {

int32_t gq_paged_plan(gq_ctx* ctx, const gq_paged_cache* cache, gq_buf counts, gq_buf free_list, gq_buf free_count, const gq_paged_step* step) {
    return guarded([&] {
        Locked l(ctx);
        const PagedView c = cache_view(ctx, "gq_paged_plan", cache, 0, false);
        const StepView st = step_view(ctx, "gq_paged_plan", cache, step);
        auto np = (const int32_t*)view(ctx, counts, 0, c.seqs, 4, "gq_paged_plan counts");
        auto fp = (const int32_t*)view(ctx, free_list, 0, c.blocks, 4, "gq_paged_plan free list");
        auto fc = (int32_t*)view(ctx, free_count, 0, 1, 4, "gq_paged_plan free count");
        const uint64_t per_seq = (uint64_t)c.seqs * 4, per_row = (uint64_t)st.tokens * 4;
        check_apart("gq_paged_plan",
                    {{"the step's starts", st.starts, per_seq + 4}, {"the step's slots", st.slots, per_row}, {"the step's positions", st.positions, per_row},
                     {"the step's runs", st.runs, (uint64_t)st.runs_cap * 4 + 4}, {"the step's last rows", st.last, per_seq}, {"the step's info", st.info, 8},
                     {"the block table", c.table, table_bytes(c)}, {"the free count", fc, 4}},
                    {{"the counts", np, per_seq}, {"the cached lengths", c.lens, per_seq}, {"the free list", fp, (uint64_t)c.blocks * 4}});
        launch_paged_plan(ctx->stream, c, st, np, fp, fc);
        after_launch(ctx, "paged_plan", {cache->table, cache->lens, counts, free_list, free_count, step->starts, step->slots, step->positions, step->runs,
                                         step->last, step->info});
    });
}

int32_t gq_paged_advance(gq_ctx* ctx, const gq_paged_cache* cache, const gq_paged_step* step) {
    return guarded([&] {
        Locked l(ctx);
        const PagedView c = cache_view(ctx, "gq_paged_advance", cache, 0, false);
        const StepView st = step_view(ctx, "gq_paged_advance", cache, step);
        check_apart("gq_paged_advance", {{"the cached lengths", c.lens, (uint64_t)c.seqs * 4}}, {{"the step's starts", st.starts, (uint64_t)c.seqs * 4 + 4}});
        launch_paged_advance(ctx->stream, c, st);
        after_launch(ctx, "paged_advance", {cache->table, cache->lens, step->starts});
    });
}

int32_t gq_paged_release(gq_ctx* ctx, const gq_paged_cache* cache, gq_buf which, gq_buf free_list, gq_buf free_count) {
    return guarded([&] {
        Locked l(ctx);
        const PagedView c = cache_view(ctx, "gq_paged_release", cache, 0, false);
        auto wp = (const int32_t*)view(ctx, which, 0, c.seqs, 4, "gq_paged_release requests");
        auto fp = (int32_t*)view(ctx, free_list, 0, c.blocks, 4, "gq_paged_release free list");
        auto fc = (int32_t*)view(ctx, free_count, 0, 1, 4, "gq_paged_release free count");
        check_apart("gq_paged_release",
                    {{"the block table", c.table, table_bytes(c)}, {"the cached lengths", c.lens, (uint64_t)c.seqs * 4},
                     {"the free list", fp, (uint64_t)c.blocks * 4}, {"the free count", fc, 4}},
                    {{"the requests", wp, (uint64_t)c.seqs * 4}});
        launch_paged_release(ctx->stream, c, wp, fp, fc);
        after_launch(ctx, "paged_release", {cache->table, cache->lens, which, free_list, free_count});
    });
}

int32_t gq_paged_append(gq_ctx* ctx, const gq_paged_cache* cache, uint64_t layer, gq_buf qkv, uint64_t heads, gq_buf cos, gq_buf sin,
                        uint64_t max_pos, const gq_paged_step* step, gq_buf q_out) {
    return guarded([&] {
        Locked l(ctx);
        const char* op = "gq_paged_append";
        const PagedView c = cache_view(ctx, op, cache, layer, true);
        const StepView st = step_view(ctx, op, cache, step);
        const uint64_t width = check_heads(op, c, heads), row = width + 2 * (uint64_t)c.kv_heads * c.dim;
        check_dims(op, max_pos, row);
        if (max_pos == 0) fail("%s: rotary tables of no positions", op);
        auto qp = (const float*)view(ctx, qkv, 0, st.tokens * row, 4, "gq_paged_append qkv");
        auto cp = (const float*)view(ctx, cos, 0, max_pos * c.dim, 4, "gq_paged_append cos");
        auto sp = (const float*)view(ctx, sin, 0, max_pos * c.dim, 4, "gq_paged_append sin");
        auto op_ = (float*)view(ctx, q_out, 0, st.tokens * width, 4, "gq_paged_append q output");
        check_aligned(op, {qp, cp, sp, op_});
        check_apart(op,
                    {{"the output", op_, st.tokens * width * 4}, {"the key pool", c.k, code_bytes(c)}, {"the value pool", c.v, code_bytes(c)},
                     {"the key scales", c.kscale, scale_bytes(c)}, {"the value scales", c.vscale, scale_bytes(c)}},
                    {{"qkv", qp, st.tokens * row * 4}, {"cos", cp, max_pos * c.dim * 4}, {"sin", sp, max_pos * c.dim * 4},
                     {"the step's starts", st.starts, (uint64_t)c.seqs * 4 + 4}, {"the step's slots", st.slots, (uint64_t)st.tokens * 4},
                     {"the step's positions", st.positions, (uint64_t)st.tokens * 4}, {"the step's runs", st.runs, (uint64_t)st.runs_cap * 4 + 4}});
        launch_paged_append(ctx->stream, c, st, qp, (uint32_t)heads, cp, sp, (uint32_t)max_pos, op_);
        after_launch(ctx, "paged_append", {cache->k, cache->v, cache->kscale, cache->vscale, cache->table, cache->lens, qkv, cos, sin, step->starts,
                                           step->slots, step->positions, step->runs, q_out});
    });
}

int32_t gq_paged_attn(gq_ctx* ctx, const gq_paged_cache* cache, uint64_t layer, gq_buf q, uint64_t heads, float scale, const gq_paged_step* step,
                      uint64_t max_count, gq_buf out) {
    return guarded([&] {
        Locked l(ctx);
        const char* op = "gq_paged_attn";
        const PagedView c = cache_view(ctx, op, cache, layer, true);
        const StepView st = step_view(ctx, op, cache, step);
        const uint64_t width = check_heads(op, c, heads);
        check_dims(op, max_count, 1);
        if (max_count == 0) fail("%s: max_count must be at least 1", op);
        check_dims(op, st.tokens * heads, 1);
        // a row tile's units (key tiles and two more, over all KV heads) are numbered in 32 bits
        if (c.kv_heads * (((uint64_t)c.max_blocks << c.shift) / 128 + 3) > 0xffffffffull)
            fail("%s: %u KV heads over requests of up to %llu tokens: more than 2^32 tiles of 128 keys", op, c.kv_heads, (ull)c.max_blocks << c.shift);
        auto qp = (const float*)view(ctx, q, 0, st.tokens * width, 4, "gq_paged_attn q");
        auto yp = (float*)view(ctx, out, 0, st.tokens * width, 4, "gq_paged_attn output");
        check_aligned(op, {qp, yp});
        check_apart(op, {{"the output", yp, st.tokens * width * 4}},
                    {{"q", qp, st.tokens * width * 4}, {"the key pool", c.k, code_bytes(c)}, {"the value pool", c.v, code_bytes(c)},
                     {"the key scales", c.kscale, scale_bytes(c)}, {"the value scales", c.vscale, scale_bytes(c)}, {"the block table", c.table, table_bytes(c)},
                     {"the cached lengths", c.lens, (uint64_t)c.seqs * 4}, {"the step's starts", st.starts, (uint64_t)c.seqs * 4 + 4}});
        const int sms = ctx->prop.multiProcessorCount;
        void* scratch = context_scratch(ctx, paged_attn_scratch_bytes(c.dim, sms));
        launch_paged_attn(ctx->stream, sms, ctx->status_dev, c, st, qp, (uint32_t)heads, scale, max_count, yp, ctx->paged_state, scratch);
        after_launch(ctx, "paged_attn", {cache->k, cache->v, cache->kscale, cache->vscale, cache->table, cache->lens, q, step->starts, out});
    });
}

int32_t gq_sample_rows(gq_ctx* ctx, gq_buf logits, uint64_t l_off, uint64_t rows, uint64_t vocab, gq_buf temperature, gq_buf top_k, gq_buf top_p,
                       gq_buf min_p, gq_buf uniforms, uint64_t uniform_rows, gq_buf draws, gq_buf tokens, gq_buf probs) {
    return guarded([&] {
        Locked l(ctx);
        check_dims("gq_sample_rows", rows, vocab, uniform_rows);
        if (vocab > (1u << 23) || rows > (1u << 24)) fail("gq_sample_rows: at most 2^23 tokens and 2^24 rows");
        if (uniform_rows == 0) fail("gq_sample_rows: sampling needs at least one row of uniform numbers");
        if (vocab == 0) fail("gq_sample_rows: expected (batch, vocab) with vocab > 0");
        auto lp = (const float*)view(ctx, logits, l_off, rows * vocab, 4, "gq_sample_rows logits");
        auto tp = (const float*)view(ctx, temperature, 0, rows, 4, "gq_sample_rows temperature");
        auto kp = (const int32_t*)view(ctx, top_k, 0, rows, 4, "gq_sample_rows top_k");
        auto pp = (const float*)view(ctx, top_p, 0, rows, 4, "gq_sample_rows top_p");
        auto mp = (const float*)view(ctx, min_p, 0, rows, 4, "gq_sample_rows min_p");
        auto up = (const float*)view(ctx, uniforms, 0, uniform_rows * rows, 4, "gq_sample_rows uniforms");
        auto dp = draws ? (uint32_t*)view(ctx, draws, 0, 1, 4, "gq_sample_rows draw counter") : nullptr;
        auto op = (int32_t*)view(ctx, tokens, 0, rows, 4, "gq_sample_rows tokens");
        auto rp = probs ? (float*)view(ctx, probs, 0, rows, 4, "gq_sample_rows probabilities") : nullptr;
        // a row's CTAs read its settings, logits and numbers while other rows' results are written
        const std::pair<const void*, uint64_t> read[] = {{lp, rows * vocab}, {tp, rows}, {kp, rows}, {pp, rows}, {mp, rows}, {up, uniform_rows * rows}, {dp, dp ? 1 : 0}};
        for (const auto& in : read)
            if (ranges_overlap(op, rows * 4, in.first, in.second * 4) || (rp && ranges_overlap(rp, rows * 4, in.first, in.second * 4)))
                fail("gq_sample_rows: the outputs must not overlap the inputs");
        if (rp && ranges_overlap(op, rows * 4, rp, rows * 4)) fail("gq_sample_rows: tokens and probabilities must not overlap");
        if (rows == 0) return;
        launch_sample_rows(ctx->stream, ctx->prop.multiProcessorCount, lp, (uint32_t)rows, (uint32_t)vocab, tp, kp, pp, mp, up, (uint32_t)uniform_rows, dp, op, rp,
                           (uint32_t*)ctx->sample_state);
        after_launch(ctx, "sample_rows", {logits, temperature, top_k, top_p, min_p, uniforms, draws, tokens, probs});
    });
}

}  // extern "C"
