// The paged KV cache (include/voxhip.h, vx_paged_*): the plan's layout and the launch
// descriptions shared by the C ABI checks (paged.cpp) and the kernels (kernels_paged*.hip).
#pragma once

#include <cmath>

#include "vx_internal.h"

namespace vx {

constexpr uint32_t kPagedRequests = 4096;        // what one workgroup's scan of the requests holds in LDS
constexpr uint32_t kPagedMaxTokens = 1u << 28;   // positions of a request
constexpr uint32_t kPagedMaxRowHeads = 1u << 22; // rows of a step times query heads: bounds every grid
constexpr uint32_t kPagedUnit = 16;              // slots of a unit: 32 * head_dim bytes of K, and of V
constexpr uint32_t kPagedMaxSplits = 256;        // of a tile of query rows
constexpr uint32_t kPagedListed = 64;            // units of an item whose pages the plan lists, for tiles of 16 rows or fewer:
                                                 // the attention need not wait for the table, which has the last word

// Chunks of a table whose requests are not divided, so that no join is launched: a CU takes 0.117 us for one (16 KB of heads
// of 128, 64 bytes a clock), the launch that joins parts 4 (one token: 47 chunks whole 9.9 us, 63 divided 6.0 and 4.1). What
// a table can hold decides, for the host launches the join and knows no lengths: 511 tokens take 6.0 in a table of 17
// pages, 5.4 and 4.2 in one of 1024; 1000 tokens 7.8, and 5.7 and 4.2.
constexpr uint32_t kPagedWhole = 48;
// Of tiles of 32 rows with four waves, each of which takes 3 us for a chunk (heads of 256: 20 tokens of two requests at
// 1300 whole 32 us, divided 16.7 and 4.6; 100 at 1000 29, 17.9 and 7.5; but 600 at 600 50, 49.6 and 4.6).
constexpr uint32_t kPagedWholeWide = 32;

inline uint32_t paged_shift(uint32_t page_size) { return 31u - (uint32_t)__builtin_clz(page_size); }

// How the attention divides a step, from the sizes that a batch fixes: max_count decides the tile, the table's width
// whether requests are divided. A tile is tile_rows query rows (tokens times query heads of a KV head) of one
// request; its keys, in chunks of 32, are divided so that about `workgroups` workgroups come out, of least chunks or more.
// A batch that allows for more than a step has costs time: one token over 32700 with a max_count of 64 takes 12.2 us and
// 3.9 to join, with one of 1 6.9 and 5.1; 64 over up to 24000 216 and 8.4, 180 and 5.2.
struct PagedShape {
    uint32_t tile_rows, waves;
    bool packed;                     // both f16 terms of eight rows in one column tile
    uint32_t workgroups, least;      // 2^workgroups
    uint32_t runs, items, joins, parts;              // most of each; items, joins and parts of one KV head
    // words of the plan
    uint64_t slots, requests, positions, granted, run_at, item_at, join_at, page_at, words;
};
PagedShape paged_shape(const vx_paged_batch &b);

// Chunks of a part in a step whose tiles have so many in all (a sum in f32, rounded up enough for its order not to matter).
__host__ __device__ inline uint32_t paged_per(const PagedShape &s, uint32_t kv_heads, float chunks) {
    float share = chunks * 1.0001f * (float)kv_heads / (float)(1u << s.workgroups);
    // Of little work half the workgroups, all of which run at once, make fewer parts to join (16 requests over
    // up to 8000: 16.6 us, with twice as many 20.2); of much twice as many end together (64 over 24000: 200, 194).
    if (s.tile_rows <= 16u && share < 16.f) share *= 2.f;
    // a wave's chunks are alike in number
    const uint32_t shift = 31u - (uint32_t)__builtin_clz(s.waves), per = ((uint32_t)fminf(ceilf(share), 1e9f) + s.waves - 1u) >> shift << shift;
    return per > s.least ? per : s.least;
}
// Chunks of a part of a tile that has `chunks`, and the number of its parts; a request's tiles are all divided alike.
// Tiles of many rows are divided where twice the share would be exceeded: what they have to join
// takes longer then.
__host__ __device__ inline uint32_t paged_divide(const PagedShape &s, uint32_t per, uint32_t chunks, uint32_t &splits) {
    const uint32_t shift = 31u - (uint32_t)__builtin_clz(s.waves);
    splits = s.tile_rows > 16u ? chunks / per : (chunks + per - 1u) / per;
    if (s.tile_rows > 16u && splits == 0u) splits = 1u;
    if (splits > kPagedMaxSplits) splits = kPagedMaxSplits;
    if (splits <= 1u) return chunks ? chunks : 1u;
    const uint32_t by = ((chunks + splits - 1u) / splits + s.waves - 1u) >> shift << shift;
    splits = (chunks + by - 1u) / by;
    return by;
}

// Records of a plan. Rows of a request that lie in one page.
struct PagedRun {
    uint32_t row, n, slot, unused;   // first row, rows, slot of the first (VX_PAGED_NONE: no page)
};
// One workgroup's share: a tile of query rows over chunks [first, first + n) of its keys.
struct PagedItem {
    uint32_t request, row, base, count;   // the request, its first row, tokens cached before it, its rows
    uint32_t tile, first, n, part;        // the tile's first query row; where its partial sums go (VX_PAGED_NONE: none)
};
// Whether an item is one: its rows are rows of the step, their positions (below cap) within the table, its chunks such as
// they attend to, its part one of `parts`. What else a plan's buffer may hold is no work, however long, and reaches nothing.
__host__ __device__ inline bool paged_is_item(const PagedItem &it, uint32_t requests, uint32_t max_rows, uint32_t group, uint32_t cap,
                                              uint32_t parts) {
    if (it.request >= requests || it.row >= max_rows || it.count > max_rows - it.row || it.base > cap || it.count > cap - it.base ||
        it.tile >= it.count * group || (it.part >= parts && it.part != VX_PAGED_NONE))
        return false;
    const uint32_t chunks = (it.base + it.count + 31u) / 32u;
    return it.first <= chunks && it.n <= chunks - it.first;
}
// A tile whose keys are divided: partial sums first_part.. + parts.
struct PagedJoin {
    uint32_t row, base, count, tile, part, per, unused[2];   // per: chunks of a part
};

struct PagedPlan {
    vx_paged_batch b;
    PagedShape s;
    const uint32_t *lengths = nullptr, *counts = nullptr, *pool = nullptr;
    uint32_t *tables = nullptr, *plan = nullptr;
};
int launch_paged_reset(hipStream_t s, const vx_paged_batch &b, uint32_t *lengths, uint32_t *tables, uint32_t *pool);
int launch_paged_plan(hipStream_t s, const PagedPlan &a);
int launch_paged_advance(hipStream_t s, const vx_paged_batch &b, const uint32_t *plan, uint32_t *lengths, uint32_t *pool);
int launch_paged_cut(hipStream_t s, const vx_paged_batch &b, const uint32_t *keep, uint32_t *lengths, uint32_t *tables,
                     uint32_t *pool);

struct PagedStore {
    vx_paged_batch b;
    PagedShape s;
    uint32_t layer = 0, k_stride = 0, v_stride = 0;
    const float *k = nullptr, *v = nullptr;     // at the push's base
    uint8_t *kc = nullptr, *vc = nullptr, *bounds = nullptr;
    const uint32_t *plan = nullptr;
    bool vec = false;                           // every row's address is 16-byte aligned
};
int launch_paged_store(hipStream_t s, const PagedStore &a);

struct PagedAttn {
    vx_paged_batch b;
    PagedShape s;
    uint32_t layer = 0, q_stride = 0, out_stride = 0, budget = 0;
    const float *q = nullptr;
    const uint8_t *kc = nullptr, *vc = nullptr;
    float *out = nullptr, *scratch = nullptr;
    const uint32_t *tables = nullptr, *plan = nullptr, *selected = nullptr;
};
uint64_t paged_attn_scratch_bytes(const vx_paged_batch &b, uint32_t budget);
int launch_paged_attention(hipStream_t s, const PagedAttn &a);

struct PagedSelect {
    vx_paged_batch b;
    PagedShape s;
    uint32_t layer = 0, q_stride = 0, budget = 0, sinks = 0, recent = 0;
    const float *q = nullptr;
    const uint8_t *bounds = nullptr;
    const uint32_t *tables = nullptr, *plan = nullptr;
    uint32_t *selected = nullptr;
    uint64_t *scratch = nullptr;
};
uint64_t paged_select_scratch_bytes(const vx_paged_batch &b);
int launch_paged_select(hipStream_t s, const PagedSelect &a);

}  // namespace vx
