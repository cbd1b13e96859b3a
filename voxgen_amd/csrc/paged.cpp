// C ABI of the paged KV cache: argument checks and launches (kernels_paged.hip,
// kernels_paged_attn.hip). Every call checks its push and the bound buffers before it
// enqueues anything; what device buffers hold (lengths, tables, a plan, a selection) is
// bounded by the kernels themselves.
#include "cache_checks.h"
#include "paged.h"

using namespace vx;

namespace vx {

PagedShape paged_shape(const vx_paged_batch &b) {
    PagedShape s{};
    const uint32_t group = b.q_heads / b.geom.kv_heads, rows = b.max_count * group;
    // Of eight rows both f16 terms go through the products side by side, not one behind the other, and scratch
    // has eight rows, not sixteen (one token over 32700: 8.6 us and 4.7 to join, else 9.0 and 4.5; 64 requests over
    // up to 24000, which wait for memory: 184 and 5.2, else 181 and 8.0). Tiles of 32 rows ask for K and V half
    // as often as those of 16 (919 tokens: 58 us, with 16 rows 77 and 34 to join; 5 tokens of 64 requests over
    // 8000: 111, 129 and 21; but 60 tokens at 1000 13.6, 11.7). They have eight waves, and of heads of 256 four,
    // for which there are registers (400 tokens at 2000 of those: 54).
    s.packed = rows <= 8u;
    s.tile_rows = s.packed ? 8u : rows <= 16u ? 16u : 32u;
    s.waves = s.tile_rows > 16u && b.geom.head_dim < 256u ? 8u : 4u;
    // A CU holds four of the workgroups of 16 rows at most, or one of heads of 256, whose are half as many (16
    // requests over up to 8000, of one KV head: 19.6 us, with 1024 25.4), and one of 32 rows.
    s.workgroups = s.tile_rows > 16u ? 8u : b.geom.head_dim < 256u ? 10u : 9u;
    // A part has two chunks a wave at least, so that one is fetched while it works; of tables of `whole` chunks
    // or fewer no request is divided.
    const uint32_t whole = s.tile_rows > 16u && s.waves == 4u ? kPagedWholeWide : kPagedWhole;
    s.least = (uint64_t)b.table_width * b.geom.page_size <= 32u * whole ? whole : 2u * s.waves;
    // Tiles: at most one for each request of so few rows, else a request's last may be part of one. Parts
    // of a tile: what its keys divide into, of which in all a KV head's share of the workgroups comes on top.
    const uint32_t requests = std::min(b.requests, b.max_rows);
    const uint64_t tiles = rows <= s.tile_rows ? requests : (uint64_t)b.max_rows * group / s.tile_rows + requests;
    const uint32_t share = ((1u << s.workgroups) + b.geom.kv_heads - 1u) / b.geom.kv_heads;
    const uint64_t chunks = ((uint64_t)b.table_width * b.geom.page_size + 31u) / 32u, most = (chunks + s.least - 1u) / s.least;
    s.items = (uint32_t)std::min(tiles + share, tiles * most);
    s.joins = most > 1u ? (uint32_t)std::min<uint64_t>(share, tiles) : 0u;
    s.parts = most > 1u ? (uint32_t)std::min<uint64_t>(2u * share, tiles * most) : 0u;
    s.runs = (uint32_t)std::min<uint64_t>(b.max_rows, (uint64_t)b.max_rows / b.geom.page_size + 2ull * b.requests);
    s.slots = VX_PAGED_PLAN_ROWS;
    s.requests = s.slots + b.max_rows;
    s.positions = s.requests + b.max_rows;
    s.granted = s.positions + b.max_rows;
    s.run_at = (s.granted + b.requests + 3u) / 4u * 4u;
    s.item_at = s.run_at + (uint64_t)s.runs * (sizeof(PagedRun) / 4u);
    s.join_at = s.item_at + (uint64_t)s.items * (sizeof(PagedItem) / 4u);
    s.page_at = s.join_at + (uint64_t)s.joins * (sizeof(PagedJoin) / 4u);
    s.words = s.page_at + (s.tile_rows <= 16u ? (uint64_t)s.items * kPagedListed : 0u);
    return s;
}

}  // namespace vx

namespace {

int check_geom(const vx_paged_geom &g, const char *what) {
    if (!g.layers || !g.pages || !g.kv_heads)
        return fail(VX_ERR_INVALID_ARG, "%s: a size of the geometry is zero", what);
    if (g.head_dim != 64u && g.head_dim != 128u && g.head_dim != 256u)
        return fail(VX_ERR_UNSUPPORTED, "%s: head_dim %u (64, 128 or 256)", what, g.head_dim);
    if (g.page_size < 16u || g.page_size > 256u || (g.page_size & (g.page_size - 1u)))
        return fail(VX_ERR_UNSUPPORTED, "%s: page_size %u (16, 32, 64, 128 or 256)", what, g.page_size);
    if (g.layers > 65535u || g.kv_heads > 65535u || (uint64_t)g.pages * g.page_size >= 0xFFFFFFFFull)
        return fail(VX_ERR_UNSUPPORTED, "%s: at most 65535 layers, 65535 KV heads and 2^32 - 2 slots", what);
    // a layer's units of 16 slots are counted in 32 bits
    if ((unsigned __int128)g.pages * g.page_size * g.kv_heads >> 36 ||
        (unsigned __int128)g.layers * g.pages * g.page_size * g.kv_heads * g.head_dim * 2u >> 47)
        return fail(VX_ERR_UNSUPPORTED, "%s: a layer of 2^36 slots or a cache of 2^47 bytes, or more", what);
    return VX_OK;
}

uint64_t cache_bytes(const vx_paged_geom &g) {
    return (uint64_t)g.layers * g.pages * g.page_size * g.kv_heads * g.head_dim * 2u;
}
uint64_t bounds_bytes(const vx_paged_geom &g) { return (uint64_t)g.layers * g.pages * g.kv_heads * g.head_dim * 4u; }

int check_batch(const vx_paged_batch &b, const char *what) {
    VX_CHECK(check_geom(b.geom, what));
    if (!b.requests || !b.table_width || !b.max_rows || !b.max_count)
        return fail(VX_ERR_INVALID_ARG, "%s: a size of the batch is zero", what);
    if (b.requests > kPagedRequests || (uint64_t)b.table_width * b.geom.page_size > kPagedMaxTokens)
        return fail(VX_ERR_UNSUPPORTED, "%s: at most %u requests of 2^28 positions", what, kPagedRequests);
    if (b.max_count > b.max_rows)
        return fail(VX_ERR_SHAPE, "%s: %u rows of a request, %u of the step", what, b.max_count, b.max_rows);
    if (!b.q_heads || b.q_heads % b.geom.kv_heads)
        return fail(VX_ERR_SHAPE, "%s: q_heads %u is not a multiple of kv_heads %u", what, b.q_heads, b.geom.kv_heads);
    if (b.q_heads / b.geom.kv_heads > 1024u || (uint64_t)b.max_rows * b.q_heads > kPagedMaxRowHeads ||
        (uint64_t)b.max_count * (b.q_heads / b.geom.kv_heads) > 1u << 22)
        return fail(VX_ERR_UNSUPPORTED, "%s: %u query heads for %u KV heads with %u rows", what, b.q_heads, b.geom.kv_heads,
                    b.max_rows);
    return VX_OK;
}

int check_layer(const vx_paged_batch &b, uint32_t layer, const char *what) {
    VX_CHECK(check_batch(b, what));
    if (layer >= b.geom.layers) return fail(VX_ERR_SHAPE, "%s: layer %u of %u", what, layer, b.geom.layers);
    return VX_OK;
}

uint64_t table_bytes(const vx_paged_batch &b) { return (uint64_t)b.requests * b.table_width * 4u; }
uint64_t pool_bytes(const vx_paged_geom &g) { return ((uint64_t)g.pages + 1u) * 4u; }

template <class T>
T *at(const vx_buf *b) {
    return static_cast<T *>(b->ptr);
}

int row_width(uint32_t heads, uint32_t head_dim, uint32_t *width, const char *what) {
    const uint64_t wide = (uint64_t)heads * head_dim;
    if (wide > 0xFFFFFFFFu) return fail(VX_ERR_UNSUPPORTED, "%s: a row of %llu values", what, (unsigned long long)wide);
    *width = (uint32_t)wide;
    return VX_OK;
}

int check_budget(const vx_paged_batch &b, uint32_t budget, const char *what) {
    if ((uint64_t)budget * b.geom.page_size > kPagedMaxTokens)
        return fail(VX_ERR_UNSUPPORTED, "%s: %u pages of %u slots selected", what, budget, b.geom.page_size);
    return VX_OK;
}

int check_attention(const vx_paged_attention_push *pc, const char *what) {
    VX_CHECK(check_layer(pc->batch, pc->layer, what));
    VX_CHECK(check_budget(pc->batch, pc->budget, what));
    return VX_OK;
}

int check_select(const vx_paged_select_push *pc, const char *what) {
    VX_CHECK(check_layer(pc->batch, pc->layer, what));
    if (!pc->budget || !pc->recent) return fail(VX_ERR_INVALID_ARG, "%s: no budget, or no recent page", what);
    VX_CHECK(check_budget(pc->batch, pc->budget, what));
    if ((uint64_t)pc->sinks + pc->recent > pc->budget)
        return fail(VX_ERR_SHAPE, "%s: %u first and %u last pages do not fit %u", what, pc->sinks, pc->recent, pc->budget);
    return VX_OK;
}

uint64_t selected_bytes(const vx_paged_batch &b, uint32_t budget) {
    return (uint64_t)b.max_rows * b.geom.kv_heads * budget * 4u;
}

}  // namespace

extern "C" {

uint64_t vx_paged_cache_bytes(const vx_paged_geom *geom) {
    if (!geom || check_geom(*geom, "vx_paged_cache_bytes") != VX_OK) return 0;
    return cache_bytes(*geom);
}

uint64_t vx_paged_bounds_bytes(const vx_paged_geom *geom) {
    if (!geom || check_geom(*geom, "vx_paged_bounds_bytes") != VX_OK) return 0;
    return bounds_bytes(*geom);
}

uint64_t vx_paged_plan_bytes(const vx_paged_batch *batch) {
    if (!batch || check_batch(*batch, "vx_paged_plan_bytes") != VX_OK) return 0;
    return paged_shape(*batch).words * 4u;
}

int vx_paged_reset(vx_ctx *ctx, vx_buf *lengths, vx_buf *tables, vx_buf *pool, const vx_paged_batch *batch) {
    if (!ctx || !batch) return fail(VX_ERR_INVALID_ARG, "vx_paged_reset: null context or batch");
    VX_CHECK(check_batch(*batch, "vx_paged_reset"));
    VX_CHECK(need_buf(lengths, (uint64_t)batch->requests * 4u, "vx_paged_reset lengths"));
    VX_CHECK(need_buf(tables, table_bytes(*batch), "vx_paged_reset tables"));
    VX_CHECK(need_buf(pool, pool_bytes(batch->geom), "vx_paged_reset pool"));
    VX_CHECK(check_apart("vx_paged_reset", {lengths, tables, pool}, {}));
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.reset");
    return launch_paged_reset(ctx->stream, *batch, at<uint32_t>(lengths), at<uint32_t>(tables), at<uint32_t>(pool));
}

int vx_paged_plan(vx_ctx *ctx, const vx_buf *lengths, const vx_buf *counts, vx_buf *tables, const vx_buf *pool,
                  vx_buf *plan, const vx_paged_batch *batch) {
    if (!ctx || !batch) return fail(VX_ERR_INVALID_ARG, "vx_paged_plan: null context or batch");
    VX_CHECK(check_batch(*batch, "vx_paged_plan"));
    PagedPlan l;
    l.b = *batch;
    l.s = paged_shape(*batch);
    VX_CHECK(need_buf(lengths, (uint64_t)batch->requests * 4u, "vx_paged_plan lengths"));
    VX_CHECK(need_buf(counts, (uint64_t)batch->requests * 4u, "vx_paged_plan counts"));
    VX_CHECK(need_buf(tables, table_bytes(*batch), "vx_paged_plan tables"));
    VX_CHECK(need_buf(pool, pool_bytes(batch->geom), "vx_paged_plan pool"));
    VX_CHECK(need_buf(plan, l.s.words * 4u, "vx_paged_plan plan"));
    VX_CHECK(check_apart("vx_paged_plan", {tables, plan}, {lengths, counts, pool}));
    l.lengths = at<uint32_t>(lengths);
    l.counts = at<uint32_t>(counts);
    l.pool = at<uint32_t>(pool);
    l.tables = at<uint32_t>(tables);
    l.plan = at<uint32_t>(plan);
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.plan");
    return launch_paged_plan(ctx->stream, l);
}

int vx_paged_advance(vx_ctx *ctx, const vx_buf *plan, vx_buf *lengths, vx_buf *pool, const vx_paged_batch *batch) {
    if (!ctx || !batch) return fail(VX_ERR_INVALID_ARG, "vx_paged_advance: null context or batch");
    VX_CHECK(check_batch(*batch, "vx_paged_advance"));
    VX_CHECK(need_buf(plan, paged_shape(*batch).words * 4u, "vx_paged_advance plan"));
    VX_CHECK(need_buf(lengths, (uint64_t)batch->requests * 4u, "vx_paged_advance lengths"));
    VX_CHECK(need_buf(pool, pool_bytes(batch->geom), "vx_paged_advance pool"));
    VX_CHECK(check_apart("vx_paged_advance", {lengths, pool}, {plan}));
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.advance");
    return launch_paged_advance(ctx->stream, *batch, at<uint32_t>(plan), at<uint32_t>(lengths), at<uint32_t>(pool));
}

int vx_paged_cut(vx_ctx *ctx, const vx_buf *keep, vx_buf *lengths, vx_buf *tables, vx_buf *pool,
                 const vx_paged_batch *batch) {
    if (!ctx || !batch) return fail(VX_ERR_INVALID_ARG, "vx_paged_cut: null context or batch");
    VX_CHECK(check_batch(*batch, "vx_paged_cut"));
    VX_CHECK(need_buf(keep, (uint64_t)batch->requests * 4u, "vx_paged_cut keep"));
    VX_CHECK(need_buf(lengths, (uint64_t)batch->requests * 4u, "vx_paged_cut lengths"));
    VX_CHECK(need_buf(tables, table_bytes(*batch), "vx_paged_cut tables"));
    VX_CHECK(need_buf(pool, pool_bytes(batch->geom), "vx_paged_cut pool"));
    VX_CHECK(check_apart("vx_paged_cut", {lengths, tables, pool}, {keep}));
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.cut");
    return launch_paged_cut(ctx->stream, *batch, at<uint32_t>(keep), at<uint32_t>(lengths), at<uint32_t>(tables),
                            at<uint32_t>(pool));
}

int vx_paged_store(vx_ctx *ctx, const vx_buf *k, const vx_buf *v, vx_buf *k_cache, vx_buf *v_cache, vx_buf *bounds,
                   const vx_buf *plan, const vx_paged_store_push *pc) {
    if (!ctx || !pc) return fail(VX_ERR_INVALID_ARG, "vx_paged_store: null context or push struct");
    const vx_paged_batch &b = pc->batch;
    VX_CHECK(check_layer(b, pc->layer, "vx_paged_store"));
    PagedStore l;
    l.b = b;
    l.s = paged_shape(b);
    uint32_t width = 0;
    VX_CHECK(row_width(b.geom.kv_heads, b.geom.head_dim, &width, "vx_paged_store"));
    VX_CHECK(check_rows(k, b.max_rows, pc->k_stride, pc->k_base, width, "vx_paged_store k"));
    VX_CHECK(check_rows(v, b.max_rows, pc->v_stride, pc->v_base, width, "vx_paged_store v"));
    VX_CHECK(need_buf(k_cache, cache_bytes(b.geom), "vx_paged_store k_cache"));
    VX_CHECK(need_buf(v_cache, cache_bytes(b.geom), "vx_paged_store v_cache"));
    if (bounds) VX_CHECK(need_buf(bounds, bounds_bytes(b.geom), "vx_paged_store bounds"));
    VX_CHECK(need_buf(plan, l.s.words * 4u, "vx_paged_store plan"));
    VX_CHECK(check_apart("vx_paged_store", {k_cache, v_cache, bounds}, {k, v, plan}));
    l.layer = pc->layer;
    l.k_stride = pc->k_stride;
    l.v_stride = pc->v_stride;
    l.k = at<float>(k) + pc->k_base;
    l.v = at<float>(v) + pc->v_base;
    l.kc = at<uint8_t>(k_cache);
    l.vc = at<uint8_t>(v_cache);
    l.bounds = bounds ? at<uint8_t>(bounds) : nullptr;
    l.plan = at<uint32_t>(plan);
    l.vec = aligned(pc->k_stride, pc->k_base) && aligned(pc->v_stride, pc->v_base);
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.store");
    return launch_paged_store(ctx->stream, l);
}

uint64_t vx_paged_attention_scratch_bytes(const vx_paged_attention_push *pc) {
    if (!pc || check_attention(pc, "vx_paged_attention_scratch_bytes") != VX_OK) return 0;
    return paged_attn_scratch_bytes(pc->batch, pc->budget);
}

int vx_paged_attention(vx_ctx *ctx, const vx_buf *q, const vx_buf *k_cache, const vx_buf *v_cache, vx_buf *out,
                       const vx_buf *tables, const vx_buf *plan, const vx_buf *selected, vx_buf *scratch,
                       const vx_paged_attention_push *pc) {
    if (!ctx || !pc) return fail(VX_ERR_INVALID_ARG, "vx_paged_attention: null context or push struct");
    const vx_paged_batch &b = pc->batch;
    VX_CHECK(check_attention(pc, "vx_paged_attention"));
    if ((selected != nullptr) != (pc->budget != 0))
        return fail(VX_ERR_INVALID_ARG, "vx_paged_attention: a budget without selected pages, or the other way round");
    PagedAttn l;
    l.b = b;
    l.s = paged_shape(b);
    uint32_t width = 0;
    VX_CHECK(row_width(b.q_heads, b.geom.head_dim, &width, "vx_paged_attention"));
    VX_CHECK(check_rows(q, b.max_rows, pc->q_stride, pc->q_base, width, "vx_paged_attention q"));
    VX_CHECK(check_rows(out, b.max_rows, pc->out_stride, pc->out_base, width, "vx_paged_attention out"));
    VX_CHECK(need_buf(k_cache, cache_bytes(b.geom), "vx_paged_attention k_cache"));
    VX_CHECK(need_buf(v_cache, cache_bytes(b.geom), "vx_paged_attention v_cache"));
    VX_CHECK(need_buf(tables, table_bytes(b), "vx_paged_attention tables"));
    VX_CHECK(need_buf(plan, l.s.words * 4u, "vx_paged_attention plan"));
    if (selected) VX_CHECK(need_buf(selected, selected_bytes(b, pc->budget), "vx_paged_attention selected"));
    VX_CHECK(need_buf(scratch, paged_attn_scratch_bytes(b, pc->budget), "vx_paged_attention scratch"));
    VX_CHECK(check_apart("vx_paged_attention", {out, scratch}, {k_cache, v_cache, tables, plan, selected}));
    VX_CHECK(check_apart("vx_paged_attention", {scratch}, {q}));
    VX_CHECK(check_rows_apart("vx_paged_attention: q and out", q, pc->q_stride, pc->q_base, out, pc->out_stride,
                              pc->out_base, b.max_rows, width));
    l.layer = pc->layer;
    l.q_stride = pc->q_stride;
    l.out_stride = pc->out_stride;
    l.budget = pc->budget;
    l.q = at<float>(q) + pc->q_base;
    l.kc = at<uint8_t>(k_cache);
    l.vc = at<uint8_t>(v_cache);
    l.out = at<float>(out) + pc->out_base;
    l.scratch = at<float>(scratch);
    l.tables = at<uint32_t>(tables);
    l.plan = at<uint32_t>(plan);
    l.selected = selected ? at<uint32_t>(selected) : nullptr;
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.attention");
    return launch_paged_attention(ctx->stream, l);
}

uint64_t vx_paged_select_scratch_bytes(const vx_paged_select_push *pc) {
    if (!pc || check_select(pc, "vx_paged_select_scratch_bytes") != VX_OK) return 0;
    return paged_select_scratch_bytes(pc->batch);
}

int vx_paged_select(vx_ctx *ctx, const vx_buf *q, const vx_buf *bounds, const vx_buf *tables, const vx_buf *plan,
                    vx_buf *selected, vx_buf *scratch, const vx_paged_select_push *pc) {
    if (!ctx || !pc) return fail(VX_ERR_INVALID_ARG, "vx_paged_select: null context or push struct");
    const vx_paged_batch &b = pc->batch;
    VX_CHECK(check_select(pc, "vx_paged_select"));
    PagedSelect l;
    l.b = b;
    l.s = paged_shape(b);
    uint32_t width = 0;
    VX_CHECK(row_width(b.q_heads, b.geom.head_dim, &width, "vx_paged_select"));
    VX_CHECK(check_rows(q, b.max_rows, pc->q_stride, pc->q_base, width, "vx_paged_select q"));
    VX_CHECK(need_buf(bounds, bounds_bytes(b.geom), "vx_paged_select bounds"));
    VX_CHECK(need_buf(tables, table_bytes(b), "vx_paged_select tables"));
    VX_CHECK(need_buf(plan, l.s.words * 4u, "vx_paged_select plan"));
    VX_CHECK(need_buf(selected, selected_bytes(b, pc->budget), "vx_paged_select selected"));
    VX_CHECK(need_buf(scratch, paged_select_scratch_bytes(b), "vx_paged_select scratch"));
    VX_CHECK(check_apart("vx_paged_select", {selected, scratch}, {q, bounds, tables, plan}));
    l.layer = pc->layer;
    l.q_stride = pc->q_stride;
    l.budget = pc->budget;
    l.sinks = pc->sinks;
    l.recent = pc->recent;
    l.q = at<float>(q) + pc->q_base;
    l.bounds = at<uint8_t>(bounds);
    l.tables = at<uint32_t>(tables);
    l.plan = at<uint32_t>(plan);
    l.selected = at<uint32_t>(selected);
    l.scratch = at<uint64_t>(scratch);
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "paged.select");
    return launch_paged_select(ctx->stream, l);
}

}  // extern "C"
