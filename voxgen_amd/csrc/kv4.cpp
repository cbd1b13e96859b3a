// C ABI of the 4-bit KV cache: argument checks and launches (kernels_kv4.hip). Every
// call checks its push and the bound buffers before it enqueues anything; what device
// buffers hold (slot counts, positions, a plan) is bounded by the kernels themselves.
#include "cache_checks.h"
#include "kv4.h"

using namespace vx;

namespace {

int check_geom(const vx_kv4_geom &g, const char *what) {
    if (!g.layers || !g.sequences || !g.kv_heads || !g.context)
        return fail(VX_ERR_INVALID_ARG, "%s: a size of the geometry is zero", what);
    if (g.head_dim != 64u && g.head_dim != 128u && g.head_dim != 256u)
        return fail(VX_ERR_UNSUPPORTED, "%s: head_dim %u (64, 128 or 256)", what, g.head_dim);
    if (g.layers > 65535u || (uint64_t)g.sequences * g.kv_heads > 65535u || g.context > kKv4MaxContext)
        return fail(VX_ERR_UNSUPPORTED, "%s: at most 65535 layers, 65535 sequences x KV heads and 2^28 slots", what);
    if ((unsigned __int128)g.layers * g.sequences * g.kv_heads * kv4_plane_bytes(g) >> 47)
        return fail(VX_ERR_UNSUPPORTED, "%s: a cache of 2^47 bytes or more", what);
    return VX_OK;
}

uint64_t planes(const vx_kv4_geom &g) { return (uint64_t)g.layers * g.sequences * g.kv_heads; }

int check_sequences(const vx_kv4_geom &g, uint32_t first, uint32_t n, const char *what) {
    if (!n) return fail(VX_ERR_INVALID_ARG, "%s: no sequences", what);
    if (first >= g.sequences || n > g.sequences - first)
        return fail(VX_ERR_SHAPE, "%s: sequences %u..+%u of %u", what, first, n, g.sequences);
    return VX_OK;
}

int check_call(const vx_kv4_geom &g, uint32_t layer, uint32_t first, uint32_t n, uint32_t tokens, const char *what) {
    VX_CHECK(check_geom(g, what));
    VX_CHECK(check_sequences(g, first, n, what));
    if (layer >= g.layers) return fail(VX_ERR_SHAPE, "%s: layer %u of %u", what, layer, g.layers);
    if (!tokens) return fail(VX_ERR_INVALID_ARG, "%s: no tokens", what);
    if (tokens > g.context) return fail(VX_ERR_SHAPE, "%s: %u tokens, context %u", what, tokens, g.context);
    if (tokens > kKv4MaxRows) return fail(VX_ERR_UNSUPPORTED, "%s: %u tokens in one call", what, tokens);
    return VX_OK;
}

int check_caches(const vx_kv4_geom &g, const vx_buf *k_cache, const vx_buf *v_cache, const char *what) {
    const uint64_t bytes = planes(g) * kv4_plane_bytes(g);
    VX_CHECK(need_buf(k_cache, bytes, what));
    VX_CHECK(need_buf(v_cache, bytes, what));
    if (k_cache == v_cache) return fail(VX_ERR_INVALID_ARG, "%s: K and V cache are one buffer", what);
    return VX_OK;
}

int rows_call(vx_ctx *ctx, const vx_kv4_rows_push *pc, const vx_buf *slots, const char *what, Kv4Rows *l) {
    if (!ctx || !pc) return fail(VX_ERR_INVALID_ARG, "%s: null context or push struct", what);
    VX_CHECK(check_call(pc->geom, pc->layer, pc->first_sequence, pc->n_sequences, pc->tokens, what));
    VX_CHECK(need_buf(slots, (uint64_t)pc->geom.sequences * 4u, what));
    l->g = pc->geom;
    l->layer = pc->layer;
    l->first = pc->first_sequence;
    l->n = pc->n_sequences;
    l->tokens = pc->tokens;
    l->k_stride = pc->k_stride;
    l->v_stride = pc->v_stride;
    l->slots = static_cast<const uint32_t *>(slots->ptr);
    l->vec = aligned(pc->k_stride, pc->k_base) && aligned(pc->v_stride, pc->v_base);
    return VX_OK;
}

int attn_shape(const vx_kv4_attention_push *pc, const char *what) {
    const vx_kv4_geom &g = pc->geom;
    VX_CHECK(check_call(g, pc->layer, pc->first_sequence, pc->n_sequences, pc->tokens, what));
    if (!pc->q_heads || pc->q_heads % g.kv_heads)
        return fail(VX_ERR_SHAPE, "%s: q_heads %u is not a multiple of kv_heads %u", what, pc->q_heads, g.kv_heads);
    if (pc->q_heads / g.kv_heads > 1024u || (uint64_t)pc->tokens * (pc->q_heads / g.kv_heads) > kKv4MaxRows)
        return fail(VX_ERR_UNSUPPORTED, "%s: %u query heads per KV head with %u tokens", what,
                    pc->q_heads / g.kv_heads, pc->tokens);
    return VX_OK;
}

Kv4Attn attn_launch(const vx_kv4_attention_push *pc) {
    Kv4Attn l;
    l.g = pc->geom;
    l.layer = pc->layer;
    l.first = pc->first_sequence;
    l.n = pc->n_sequences;
    l.tokens = pc->tokens;
    l.q_heads = pc->q_heads;
    l.q_stride = pc->q_stride;
    l.out_stride = pc->out_stride;
    l.decay = pc->decay;
    return l;
}

int evict_call(const vx_kv4_evict_push *pc, const char *what, Kv4Evict *l) {
    if (!pc) return fail(VX_ERR_INVALID_ARG, "%s: null push struct", what);
    VX_CHECK(check_geom(pc->geom, what));
    VX_CHECK(check_sequences(pc->geom, pc->first_sequence, pc->n_sequences, what));
    if (!pc->keep || pc->keep >= pc->geom.context)
        return fail(VX_ERR_SHAPE, "%s: keep %u of %u slots", what, pc->keep, pc->geom.context);
    if ((uint64_t)pc->sinks + pc->recent > pc->keep)
        return fail(VX_ERR_SHAPE, "%s: %u first and %u last positions do not fit %u slots", what, pc->sinks,
                    pc->recent, pc->keep);
    l->g = pc->geom;
    l->first = pc->first_sequence;
    l->n = pc->n_sequences;
    l->keep = pc->keep;
    l->sinks = pc->sinks;
    l->recent = pc->recent;
    l->moves = pc->keep < pc->geom.context - pc->keep ? pc->keep : pc->geom.context - pc->keep;
    return VX_OK;
}

uint64_t plan_bytes(const Kv4Evict &l) {
    return (uint64_t)l.g.layers * l.n * l.g.kv_heads * l.moves * 8u;
}

}  // namespace

extern "C" {

uint64_t vx_kv4_cache_bytes(const vx_kv4_geom *geom) {
    if (!geom || check_geom(*geom, "vx_kv4_cache_bytes") != VX_OK) return 0;
    return planes(*geom) * kv4_plane_bytes(*geom);
}

int vx_kv4_store(vx_ctx *ctx, const vx_buf *k, const vx_buf *v, vx_buf *k_cache, vx_buf *v_cache,
                 const vx_buf *slots, const vx_buf *positions, vx_buf *slot_positions,
                 const vx_kv4_rows_push *pc) {
    Kv4Rows l;
    VX_CHECK(rows_call(ctx, pc, slots, "vx_kv4_store", &l));
    const vx_kv4_geom &g = pc->geom;
    const uint64_t rows = (uint64_t)pc->n_sequences * pc->tokens;
    const uint32_t width = g.kv_heads * g.head_dim;
    VX_CHECK(check_rows(k, rows, pc->k_stride, pc->k_base, width, "vx_kv4_store k"));
    VX_CHECK(check_rows(v, rows, pc->v_stride, pc->v_base, width, "vx_kv4_store v"));
    VX_CHECK(check_caches(g, k_cache, v_cache, "vx_kv4_store cache"));
    if (positions) VX_CHECK(need_buf(positions, (uint64_t)g.sequences * 4u, "vx_kv4_store positions"));
    if (slot_positions)
        VX_CHECK(need_buf(slot_positions, planes(g) * g.context * 4u, "vx_kv4_store slot_positions"));
    VX_CHECK(check_apart("vx_kv4_store", {k_cache, v_cache, slot_positions}, {k, v, slots, positions}));
    l.k = static_cast<float *>(k->ptr) + pc->k_base;
    l.v = static_cast<float *>(v->ptr) + pc->v_base;
    l.kc = static_cast<uint8_t *>(k_cache->ptr);
    l.vc = static_cast<uint8_t *>(v_cache->ptr);
    l.positions = positions ? static_cast<const uint32_t *>(positions->ptr) : nullptr;
    l.slot_positions = slot_positions ? static_cast<uint32_t *>(slot_positions->ptr) : nullptr;
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "kv4.store");
    return launch_kv4_store(ctx->stream, l);
}

int vx_kv4_load(vx_ctx *ctx, const vx_buf *k_cache, const vx_buf *v_cache, vx_buf *k, vx_buf *v,
                const vx_buf *slots, const vx_kv4_rows_push *pc) {
    Kv4Rows l;
    VX_CHECK(rows_call(ctx, pc, slots, "vx_kv4_load", &l));
    const vx_kv4_geom &g = pc->geom;
    const uint64_t rows = (uint64_t)pc->n_sequences * pc->tokens;
    const uint32_t width = g.kv_heads * g.head_dim;
    if (!k && !v) return fail(VX_ERR_INVALID_ARG, "vx_kv4_load: neither k nor v");
    if (k) VX_CHECK(check_rows(k, rows, pc->k_stride, pc->k_base, width, "vx_kv4_load k"));
    if (v) VX_CHECK(check_rows(v, rows, pc->v_stride, pc->v_base, width, "vx_kv4_load v"));
    VX_CHECK(check_caches(g, k_cache, v_cache, "vx_kv4_load cache"));
    VX_CHECK(check_apart("vx_kv4_load", {k}, {k_cache, v_cache, slots}));
    VX_CHECK(check_apart("vx_kv4_load", {v}, {k_cache, v_cache, slots}));
    if (k && v)
        VX_CHECK(check_rows_apart("vx_kv4_load: k and v", k, pc->k_stride, pc->k_base, v, pc->v_stride, pc->v_base, rows, width));
    if (k) l.k = static_cast<float *>(k->ptr) + pc->k_base;
    if (v) l.v = static_cast<float *>(v->ptr) + pc->v_base;
    l.kc = static_cast<uint8_t *>(k_cache->ptr);
    l.vc = static_cast<uint8_t *>(v_cache->ptr);
    l.vec = (!k || aligned(pc->k_stride, pc->k_base)) && (!v || aligned(pc->v_stride, pc->v_base));
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "kv4.load");
    return launch_kv4_load(ctx->stream, l);
}

int vx_kv4_advance(vx_ctx *ctx, vx_buf *slots, vx_buf *positions, uint32_t first_sequence, uint32_t n_sequences,
                   uint32_t tokens, uint32_t context) {
    if (!ctx) return fail(VX_ERR_INVALID_ARG, "vx_kv4_advance: null context");
    if (!n_sequences || !tokens || !context)
        return fail(VX_ERR_INVALID_ARG, "vx_kv4_advance: no sequences, tokens or context");
    if (context > kKv4MaxContext || tokens > context)
        return fail(VX_ERR_SHAPE, "vx_kv4_advance: %u tokens, context %u", tokens, context);
    const uint64_t bytes = ((uint64_t)first_sequence + n_sequences) * 4u;
    VX_CHECK(need_buf(slots, bytes, "vx_kv4_advance slots"));
    if (positions) VX_CHECK(need_buf(positions, bytes, "vx_kv4_advance positions"));
    VX_CHECK(check_apart("vx_kv4_advance", {slots, positions}, {}));
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "kv4.advance");
    return launch_kv4_advance(ctx->stream, static_cast<uint32_t *>(slots->ptr) + first_sequence,
                              positions ? static_cast<uint32_t *>(positions->ptr) + first_sequence : nullptr,
                              n_sequences, tokens, context);
}

uint64_t vx_kv4_attention_scratch_bytes(const vx_kv4_attention_push *pc, uint32_t with_weights) {
    if (!pc || attn_shape(pc, "vx_kv4_attention_scratch_bytes") != VX_OK) return 0;
    return kv4_attn_scratch_bytes(attn_launch(pc), with_weights != 0);
}

int vx_kv4_attention(vx_ctx *ctx, const vx_buf *q, const vx_buf *k_cache, const vx_buf *v_cache, vx_buf *out,
                     vx_buf *weights, const vx_buf *slots, vx_buf *scratch, const vx_kv4_attention_push *pc) {
    if (!ctx || !pc) return fail(VX_ERR_INVALID_ARG, "vx_kv4_attention: null context or push struct");
    VX_CHECK(attn_shape(pc, "vx_kv4_attention"));
    const vx_kv4_geom &g = pc->geom;
    if (!(pc->decay >= 0.0f && pc->decay <= 1.0f))
        return fail(VX_ERR_INVALID_ARG, "vx_kv4_attention: decay %g is outside 0..1", (double)pc->decay);
    const uint64_t rows = (uint64_t)pc->n_sequences * pc->tokens;
    const uint64_t wide = (uint64_t)pc->q_heads * g.head_dim;
    if (wide > 0xFFFFFFFFu) return fail(VX_ERR_UNSUPPORTED, "vx_kv4_attention: a row of %llu values",
                                        (unsigned long long)wide);
    const uint32_t width = (uint32_t)wide;
    VX_CHECK(check_rows(q, rows, pc->q_stride, pc->q_base, width, "vx_kv4_attention q"));
    VX_CHECK(check_rows(out, rows, pc->out_stride, pc->out_base, width, "vx_kv4_attention out"));
    VX_CHECK(check_caches(g, k_cache, v_cache, "vx_kv4_attention cache"));
    VX_CHECK(need_buf(slots, (uint64_t)g.sequences * 4u, "vx_kv4_attention slots"));
    if (weights) VX_CHECK(need_buf(weights, planes(g) * g.context * 4u, "vx_kv4_attention weights"));
    Kv4Attn l = attn_launch(pc);
    VX_CHECK(need_buf(scratch, kv4_attn_scratch_bytes(l, weights != nullptr), "vx_kv4_attention scratch"));
    VX_CHECK(check_apart("vx_kv4_attention", {out, weights, scratch}, {k_cache, v_cache, slots}));
    VX_CHECK(check_apart("vx_kv4_attention", {weights, scratch}, {q}));
    VX_CHECK(check_rows_apart("vx_kv4_attention: q and out", q, pc->q_stride, pc->q_base, out, pc->out_stride, pc->out_base,
                              rows, width));
    l.q = static_cast<const float *>(q->ptr) + pc->q_base;
    l.kc = static_cast<const uint8_t *>(k_cache->ptr);
    l.vc = static_cast<const uint8_t *>(v_cache->ptr);
    l.out = static_cast<float *>(out->ptr) + pc->out_base;
    l.weights = weights ? static_cast<float *>(weights->ptr) : nullptr;
    l.slots = static_cast<const uint32_t *>(slots->ptr);
    l.scratch = static_cast<float *>(scratch->ptr);
    l.qvec = aligned(pc->q_stride, pc->q_base);
    l.ovec = aligned(pc->out_stride, pc->out_base);
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "kv4.attention");
    return launch_kv4_attention(ctx->stream, l);
}

uint64_t vx_kv4_plan_bytes(const vx_kv4_evict_push *pc) {
    Kv4Evict l;
    return evict_call(pc, "vx_kv4_plan_bytes", &l) == VX_OK ? plan_bytes(l) : 0;
}

int vx_kv4_select(vx_ctx *ctx, const vx_buf *weights, const vx_buf *slot_positions, const vx_buf *slots,
                  vx_buf *plan, const vx_kv4_evict_push *pc) {
    if (!ctx) return fail(VX_ERR_INVALID_ARG, "vx_kv4_select: null context");
    Kv4Evict l;
    VX_CHECK(evict_call(pc, "vx_kv4_select", &l));
    const uint64_t table = planes(l.g) * l.g.context * 4u;
    VX_CHECK(need_buf(weights, table, "vx_kv4_select weights"));
    VX_CHECK(need_buf(slot_positions, table, "vx_kv4_select slot_positions"));
    VX_CHECK(need_buf(slots, (uint64_t)l.g.sequences * 4u, "vx_kv4_select slots"));
    VX_CHECK(need_buf(plan, plan_bytes(l), "vx_kv4_select plan"));
    VX_CHECK(check_apart("vx_kv4_select", {plan}, {weights, slot_positions, slots}));
    l.weights = static_cast<float *>(weights->ptr);
    l.slot_positions = static_cast<uint32_t *>(slot_positions->ptr);
    l.slots = static_cast<uint32_t *>(slots->ptr);
    l.plan = static_cast<uint32_t *>(plan->ptr);
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "kv4.select");
    return launch_kv4_select(ctx->stream, l);
}

int vx_kv4_compact(vx_ctx *ctx, const vx_buf *plan, vx_buf *k_cache, vx_buf *v_cache, vx_buf *weights,
                   vx_buf *slot_positions, vx_buf *slots, const vx_kv4_evict_push *pc) {
    if (!ctx) return fail(VX_ERR_INVALID_ARG, "vx_kv4_compact: null context");
    Kv4Evict l;
    VX_CHECK(evict_call(pc, "vx_kv4_compact", &l));
    const uint64_t table = planes(l.g) * l.g.context * 4u;
    VX_CHECK(need_buf(plan, plan_bytes(l), "vx_kv4_compact plan"));
    if (k_cache || v_cache) VX_CHECK(check_caches(l.g, k_cache, v_cache, "vx_kv4_compact cache"));
    if (weights) VX_CHECK(need_buf(weights, table, "vx_kv4_compact weights"));
    if (slot_positions) VX_CHECK(need_buf(slot_positions, table, "vx_kv4_compact slot_positions"));
    VX_CHECK(need_buf(slots, (uint64_t)l.g.sequences * 4u, "vx_kv4_compact slots"));
    VX_CHECK(check_apart("vx_kv4_compact", {k_cache, v_cache, weights, slot_positions, slots}, {plan}));
    l.plan_in = static_cast<const uint32_t *>(plan->ptr);
    l.kc = k_cache ? static_cast<uint8_t *>(k_cache->ptr) : nullptr;
    l.vc = v_cache ? static_cast<uint8_t *>(v_cache->ptr) : nullptr;
    l.weights = weights ? static_cast<float *>(weights->ptr) : nullptr;
    l.slot_positions = slot_positions ? static_cast<uint32_t *>(slot_positions->ptr) : nullptr;
    l.slots = static_cast<uint32_t *>(slots->ptr);
    OnDevice on(ctx->device);
    ProfSpan span(ctx, "kv4.compact");
    return launch_kv4_compact(ctx->stream, l);
}

}  // extern "C"
