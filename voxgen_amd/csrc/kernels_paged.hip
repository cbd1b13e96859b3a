// The paged KV cache but for its attention: the plan of a step, what follows from it for
// lengths and pool, storing rows, and the choice of the pages that a row attends to
// (include/voxhip.h, vx_paged_*, has the layouts). Everything that a step depends on is
// read from device memory, so that a captured step replays.
#include "attn_dev.h"
#include "paged.h"

namespace vx {
namespace {

__device__ __forceinline__ uint32_t add_up_to(uint32_t a, uint32_t b, uint32_t most) { return min(a + b, most); }

// v of another lane of the wave by a DPP control, 0 where there is none or ROWS does not have the lane's row.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_of(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}

// Sums over a workgroup's T threads up to and with each, and in `before` without it, each clipped to
// `most` (clipped addition of numbers below 2^31 is associative); all of them in `all`. `between`
// holds a word for each wave.
template <int N, uint32_t T>
__device__ __forceinline__ void scan(uint32_t (&v)[N], uint32_t (&before)[N], uint32_t (&all)[N], uint32_t most,
                                     uint32_t (*between)[N]) {
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        v[n] = add_up_to(v[n], lane_of<0x111, 0xf>(v[n]), most);   // row_shr 1, 2, 4, 8
        v[n] = add_up_to(v[n], lane_of<0x112, 0xf>(v[n]), most);
        v[n] = add_up_to(v[n], lane_of<0x114, 0xf>(v[n]), most);
        v[n] = add_up_to(v[n], lane_of<0x118, 0xf>(v[n]), most);
        v[n] = add_up_to(v[n], lane_of<0x142, 0xa>(v[n]), most);   // row_bcast 15, 31
        v[n] = add_up_to(v[n], lane_of<0x143, 0xc>(v[n]), most);
        before[n] = lane_of<0x138, 0xf>(v[n]);                     // wave_shr 1
        if (lane == 63u) between[w][n] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        uint32_t ahead = 0;
        all[n] = 0;
#pragma unroll
        for (uint32_t u = 0; u < T / 64u; ++u) {
            ahead = u == w ? all[n] : ahead;
            all[n] = add_up_to(all[n], between[u][n], most);
        }
        v[n] = add_up_to(v[n], ahead, most);
        before[n] = add_up_to(before[n], ahead, most);
    }
    __syncthreads();
}

// The least i with end[i] > x; ends rise, and the last is above x.
__device__ __forceinline__ uint32_t owner_of(const uint32_t *end, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n - 1u;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (end[mid] > x)
            hi = mid;
        else
            lo = mid + 1u;
    }
    return lo;
}

// Every workgroup scans all requests, and writes its share of what follows from that: so one
// launch does, and none waits for another. A thread has E requests one behind the other. Bound by
// what needs each other: lengths and counts, three sums over the requests, for each row the
// request that it is of, and its page. 16 requests 5.8 us, 512 with up to 64 rows 8.0.
template <uint32_t T, uint32_t E>
__global__ __launch_bounds__(T) void k_paged_plan(PagedPlan a) {
    constexpr uint32_t N = T * E, kPagedLists = 7;
    __shared__ uint32_t length_of[N], count_of[N], row_end[N], page_end[N], run_end[N], item_end[N], join_end[N], part_end[N];
    __shared__ uint32_t between[T / 64][6];
    __shared__ float work[T / 64];
    const uint32_t tid = threadIdx.x, n = a.b.requests, r0 = tid * E;
    const uint32_t pages = a.b.geom.pages, shift = 31u - __clz(a.b.geom.page_size), ps = a.b.geom.page_size;
    const uint32_t width = a.b.table_width, cap = width << shift, rows = a.b.max_rows;
    const uint32_t group = a.b.q_heads / a.b.geom.kv_heads, tile_shift = 31u - __clz(a.s.tile_rows);
    const uint32_t free = min(a.pool[0], pages);
    uint32_t len[E], count[E], need[E], v[1] = {0}, before[1], all[1];
    bool takes[E];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        len[e] = r0 + e < n ? a.lengths[r0 + e] : 0u;
        count[e] = r0 + e < n ? a.counts[r0 + e] : 0u;
    }
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        length_of[r0 + e] = len[e];
        count_of[r0 + e] = count[e];
        v[0] = add_up_to(v[0], min(count[e], rows + 1u), rows + 1u);
    }
    scan<1, T>(v, before, all, rows + 1u, reinterpret_cast<uint32_t (*)[1]>(between));
    const uint32_t all_rows = min(all[0], rows);
    // What the attention has to do, chunks of 32 keys by tiles of query rows, of requests that may take part.
    uint32_t at = before[0], tiles[E], chunks[E];
    float todo = 0.f;
    v[0] = 0;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        at = add_up_to(at, min(count[e], rows + 1u), rows + 1u);
        row_end[r0 + e] = at;
        takes[e] = count[e] != 0u && count[e] <= a.b.max_count && at <= rows && len[e] <= cap && count[e] <= cap - len[e];
        need[e] = takes[e] ? ((len[e] + count[e] + ps - 1u) >> shift) - ((len[e] + ps - 1u) >> shift) : 0u;
        v[0] = add_up_to(v[0], need[e], pages + 1u);
        tiles[e] = takes[e] ? (count[e] * group + a.s.tile_rows - 1u) >> tile_shift : 0u;
        chunks[e] = takes[e] ? (len[e] + count[e] + 31u) / 32u : 0u;
        todo += (float)tiles[e] * (float)chunks[e];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) todo += __shfl_xor(todo, d, 64);
    if ((tid & 63u) == 0) work[tid >> 6] = todo;
    scan<1, T>(v, before, all, pages + 1u, reinterpret_cast<uint32_t (*)[1]>(between));
    todo = 0.f;
#pragma unroll
    for (uint32_t u = 0; u < T / 64u; ++u) todo += work[u];
    const uint32_t per = paged_per(a.s, a.b.geom.kv_heads, todo);
    auto divided = [&](uint32_t many, uint32_t &splits) { return paged_divide(a.s, per, many, splits); };
    // runs, items, joins and parts of each request, and pages, rows and requests that take part
    uint32_t splits[E], w[6] = {0, 0, 0, 0, 0, 0}, done[6], sum[6], taking = 0;
    at = before[0];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        at = add_up_to(at, need[e], pages + 1u);
        page_end[r0 + e] = at;
        takes[e] = takes[e] && (need[e] == 0u || at <= free);
        divided(chunks[e], splits[e]);
        if (!takes[e]) continue;
        w[0] += ((len[e] + count[e] - 1u) >> shift) - (len[e] >> shift) + 1u;
        w[1] += tiles[e] * splits[e];
        w[2] += splits[e] > 1u ? tiles[e] : 0u;
        w[3] += splits[e] > 1u ? tiles[e] * splits[e] : 0u;
        w[4] += need[e];
        w[5] += count[e];
        taking += 1u;
    }
    scan<6, T>(w, done, sum, 0x7fffffffu, between);
    {
        uint32_t run = done[0], item = done[1], join = done[2], part = done[3];
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            if (takes[e]) {
                run += ((len[e] + count[e] - 1u) >> shift) - (len[e] >> shift) + 1u;
                item += tiles[e] * splits[e];
                join += splits[e] > 1u ? tiles[e] : 0u;
                part += splits[e] > 1u ? tiles[e] * splits[e] : 0u;
            }
            run_end[r0 + e] = run;
            item_end[r0 + e] = item;
            join_end[r0 + e] = join;
            part_end[r0 + e] = part;
        }
    }
    const uint32_t most_taking = __syncthreads_count(taking != 0u);   // of E 1 the requests that take part

    const uint32_t all_runs = min(sum[0], a.s.runs), all_items = min(sum[1], a.s.items), all_joins = min(sum[2], a.s.joins);
    const uint32_t taken = min(sum[4], free);
    // What is left is lists whose entries stand for themselves; each begins at another workgroup, so that
    // short ones are made at the same time.
    const uint32_t step = gridDim.x * T;
    auto turn = [&](uint32_t list) { return (blockIdx.x >= list ? blockIdx.x - list : blockIdx.x + gridDim.x - list) * T + tid; };
    auto begin = [&](const uint32_t *end, uint32_t i) { return i ? end[i - 1u] : 0u; };
    auto part_of = [&](uint32_t i) { return run_end[i] != begin(run_end, i); };
    // the page of position p of request i that takes part: one in use, or one from the top of the pool
    auto page_of = [&](uint32_t i, uint32_t length, uint32_t p) {
        const uint32_t have = (length + ps - 1u) >> shift, k = p >> shift;
        const uint32_t nth = begin(page_end, i) + k - have;
        const uint32_t *const from = k < have ? a.tables + (size_t)i * width + k : a.pool + (nth < free ? free - nth : 0u);
        const uint32_t page = *from;
        return k < have || nth < free ? page : VX_PAGED_NONE;
    };
    for (uint32_t r = turn(0); r < rows; r += step) {
        uint32_t slot = VX_PAGED_NONE, request = VX_PAGED_NONE, position = VX_PAGED_NONE;
        if (r < all_rows) {
            const uint32_t i = owner_of(row_end, n, r);
            if (part_of(i)) {
                request = i;
                position = length_of[i] + r - begin(row_end, i);
                const uint32_t page = page_of(i, length_of[i], position);
                if (page < pages) slot = (page << shift) + (position & (ps - 1u));
            }
        }
        a.plan[a.s.slots + r] = slot;
        a.plan[a.s.requests + r] = request;
        a.plan[a.s.positions + r] = position;
    }
    for (uint32_t g = turn(1); g < all_runs; g += step) {
        const uint32_t i = owner_of(run_end, n, g), length = length_of[i], k = g - begin(run_end, i);
        const uint32_t first = k ? ((length >> shift) + k) << shift : length;       // position of the run's first row
        const uint32_t last = min(((first >> shift) + 1u) << shift, length + count_of[i]);
        const uint32_t page = page_of(i, length, first);
        const PagedRun run = {begin(row_end, i) + first - length, last - first,
                              page < pages ? (page << shift) + (first & (ps - 1u)) : VX_PAGED_NONE, 0u};
        reinterpret_cast<PagedRun *>(a.plan + a.s.run_at)[g] = run;
    }
    for (uint32_t g = turn(2); g < all_items; g += step) {
        const uint32_t i = owner_of(item_end, n, g), length = length_of[i], cnt = count_of[i], k = g - begin(item_end, i);
        uint32_t s;
        const uint32_t by = divided((length + cnt + 31u) / 32u, s);
        // the tiles with the most keys first
        const uint32_t tile = ((cnt * group + a.s.tile_rows - 1u) >> tile_shift) - 1u - k / s, split = k % s;
        const uint32_t last_row = min((tile + 1u) << tile_shift, cnt * group) - 1u;
        const uint32_t many = (length + last_row / group) / 32u + 1u, first = split * by;
        const PagedItem it = {i, begin(row_end, i), length, cnt, tile << tile_shift, first,
                              first < many ? min(by, many - first) : 0u,
                              many > by ? begin(part_end, i) + tile * s + split : VX_PAGED_NONE};
        reinterpret_cast<PagedItem *>(a.plan + a.s.item_at)[g] = it;
    }
    if (a.s.tile_rows <= 16u) {   // a tile is few rows: the pages of its part's first units
        for (uint32_t g = turn(3); g < all_items * kPagedListed; g += step) {
            const uint32_t item = g / kPagedListed, i = owner_of(item_end, n, item), length = length_of[i], cnt = count_of[i];
            uint32_t s;
            const uint32_t by = divided((length + cnt + 31u) / 32u, s);
            const uint32_t at = (item - begin(item_end, i)) % s * by * 32u + g % kPagedListed * kPagedUnit;
            a.plan[a.s.page_at + g] = at < length + cnt ? page_of(i, length, at) : VX_PAGED_NONE;
        }
    }
    for (uint32_t g = turn(4); g < all_joins; g += step) {
        const uint32_t i = owner_of(join_end, n, g), length = length_of[i], cnt = count_of[i], tile = g - begin(join_end, i);
        uint32_t s;
        const uint32_t by = divided((length + cnt + 31u) / 32u, s);
        const PagedJoin j = {begin(row_end, i), length, cnt, tile << tile_shift, begin(part_end, i) + tile * s, by, {0, 0}};
        reinterpret_cast<PagedJoin *>(a.plan + a.s.join_at)[g] = j;
    }
    for (uint32_t i = turn(5); i < n; i += step) a.plan[a.s.granted + i] = part_of(i) ? count_of[i] : 0u;
    for (uint32_t g = turn(6); g < taken; g += step) {   // pages that requests that take part want: they are the first of all wanted
        const uint32_t i = owner_of(page_end, n, g), have = (length_of[i] + ps - 1u) >> shift;
        a.tables[(size_t)i * width + have + g - begin(page_end, i)] = a.pool[free - g];
    }
    if (blockIdx.x == kPagedLists) {
        uint32_t some = most_taking;
        if constexpr (E > 1) {
            some = taking;
#pragma unroll
            for (int d = 32; d; d >>= 1) some += __shfl_xor(some, d, 64);
            if ((tid & 63u) == 0) between[tid >> 6][0] = some;
            __syncthreads();
            some = 0;
            for (uint32_t u = 0; u < T / 64u; ++u) some += between[u][0];
        }
        const uint32_t head[8] = {all_rows, taken, some, sum[5], all_runs, all_items, all_joins, 0u};
        if (tid == 0) {
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) a.plan[u] = head[u];
        }
    }
}

__global__ __launch_bounds__(256) void k_paged_reset(vx_paged_batch b, uint32_t *lengths, uint32_t *tables, uint32_t *pool) {
    const size_t at = (size_t)blockIdx.x * 256u + threadIdx.x, step = (size_t)gridDim.x * 256u;
    if (at == 0) pool[0] = b.geom.pages;
    for (size_t i = at; i < b.requests; i += step) lengths[i] = 0u;
    for (size_t i = at; i < (size_t)b.requests * b.table_width; i += step) tables[i] = VX_PAGED_NONE;
    for (size_t i = at; i < b.geom.pages; i += step) pool[1u + i] = b.geom.pages - 1u - (uint32_t)i;
}

__global__ __launch_bounds__(256) void k_paged_advance(vx_paged_batch b, const uint32_t *plan, uint64_t granted, uint32_t *lengths,
                                                       uint32_t *pool) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i == 0) {
        const uint32_t free = min(pool[0], b.geom.pages);
        pool[0] = free - min(plan[1], free);
    }
    if (i >= b.requests) return;
    const uint32_t length = lengths[i], cap = b.table_width * b.geom.page_size, more = plan[granted + i];
    if (more && length <= cap) lengths[i] = length + min(more, cap - length);
}

constexpr uint32_t kCutThreads = 1024, kCutEach = kPagedRequests / kCutThreads;
// One workgroup: the pages that requests give back, in order, go on top of the pool.
__global__ __launch_bounds__(1024) void k_paged_cut(vx_paged_batch b, const uint32_t *keep, uint32_t *lengths, uint32_t *tables,
                                                    uint32_t *pool) {
    __shared__ uint32_t end[kPagedRequests], from[kPagedRequests];
    __shared__ uint32_t between[kCutThreads / 64][1];
    const uint32_t tid = threadIdx.x, n = b.requests, each = (n + kCutThreads - 1u) / kCutThreads, r0 = tid * each;
    const uint32_t shift = 31u - __clz(b.geom.page_size), ps = b.geom.page_size, pages = b.geom.pages;
    const uint32_t cap = b.table_width << shift, free = min(pool[0], pages);
    uint32_t back[kCutEach], v[1] = {0}, before[1], all[1];
#pragma unroll
    for (uint32_t e = 0; e < kCutEach; ++e) {
        back[e] = 0;
        if (e >= each || r0 + e >= n) continue;
        const uint32_t i = r0 + e, length = min(lengths[i], cap), stay = min(length, keep[i]);
        from[i] = (stay + ps - 1u) >> shift;
        back[e] = ((length + ps - 1u) >> shift) - from[i];
        if (stay != length) lengths[i] = stay;
        v[0] += back[e];
    }
    scan<1, kCutThreads>(v, before, all, 0x7fffffffu, between);
    uint32_t at = before[0];
#pragma unroll
    for (uint32_t e = 0; e < kCutEach; ++e) {
        at += back[e];
        if (e < each && r0 + e < n) end[r0 + e] = at;
    }
    __syncthreads();
    for (uint32_t g = tid; g < all[0]; g += kCutThreads) {
        const uint32_t i = owner_of(end, n, g), k = g - (i ? end[i - 1u] : 0u);
        uint32_t *const entry = tables + (size_t)i * b.table_width + from[i] + k;
        if (g < pages - free) pool[1u + free + g] = *entry;
        *entry = VX_PAGED_NONE;
    }
    if (tid == 0) pool[0] = free + min(all[0], pages - free);
}

// ------------------------------------------------------------------- rows
// A workgroup per run (rows of one request in one page) and KV head: lanes of eight dimensions,
// 256 / (HD / 8) slots at once. K's eighths go out as they are; V's are transposed through LDS, and
// a lane then owns an octet of slots of one dimension. Bound by three loads that need each other and, for
// pages of many rows, a workgroup's way through one: 16 rows 3.1 us; four prompts of up to 700 rows with
// bounds, 6.2 MB, 6.1.
template <int HD, bool BOUNDS>
__global__ __launch_bounds__(256) void k_paged_store(PagedStore a) {
    constexpr int W = HD / 8, R = 256 / W;
    __shared__ __attribute__((aligned(16))) _Float16 rows[R][HD + 8];
    const uint32_t tid = threadIdx.x, r = tid / W, c = tid % W, heads = a.b.geom.kv_heads;
    const uint32_t run = blockIdx.x / heads, head = blockIdx.x % heads, ps = a.b.geom.page_size, shift = 31u - __clz(ps);
    if (run >= min(a.plan[4], a.s.runs)) return;
    const PagedRun at = reinterpret_cast<const PagedRun *>(a.plan + a.s.run_at)[run];
    const uint32_t page = at.slot >> shift, first = at.slot & (ps - 1u);
    if (at.slot == VX_PAGED_NONE || page >= a.b.geom.pages || at.n > ps - first || at.row >= a.b.max_rows ||
        at.n > a.b.max_rows - at.row)
        return;
    const uint32_t end = first + at.n;
    const size_t in_cache = (((size_t)a.layer * a.b.geom.pages + page) * heads + head) * ps * HD;   // values
    _Float16 *const kc = reinterpret_cast<_Float16 *>(a.kc) + in_cache, *const vc = reinterpret_cast<_Float16 *>(a.vc) + in_cache;
    h8 lo = (h8)((_Float16)INFINITY), hi = -lo;
    uint32_t bad = 0;
    auto bound = [&](h8 x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) bad |= x[i] != x[i] ? 1u << i : 0u;
        lo = __builtin_elementwise_min(lo, x);
        hi = __builtin_elementwise_max(hi, x);
    };
    for (uint32_t s0 = BOUNDS ? 0u : first / 8u * 8u; s0 < end; s0 += R) {
        const uint32_t s = s0 + r;
        const bool live = s >= first && s < end;
        _Float16 *const to = kc + ((s / 16u * W + c) * 16u + s % 16u) * 8u;
        if (BOUNDS && s < first) bound(*reinterpret_cast<const h8 *>(to));
        float x[8], y[8];
        if (live) {
            const size_t row = at.row + s - first;
            load8(a.k + row * a.k_stride + head * HD + c * 8u, a.vec, x);
            load8(a.v + row * a.v_stride + head * HD + c * 8u, a.vec, y);
            h8 kx, vx;
#pragma unroll
            for (int i = 0; i < 8; ++i) kx[i] = (_Float16)x[i], vx[i] = (_Float16)y[i];
            *reinterpret_cast<h8 *>(to) = kx;
            if (BOUNDS) bound(kx);
            *reinterpret_cast<h8 *>(&rows[r][c * 8u]) = vx;
        }
        __syncthreads();
        const uint32_t o = tid / HD * 8u, dim = tid % HD, so = s0 + o;   // R / 8 octets of HD dimensions
        _Float16 *const vt = vc + ((size_t)(so / 8u) * HD + dim) * 8u;
        if (so >= first && so + 8u <= end) {
            h8 x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = rows[o + e][dim];
            *reinterpret_cast<h8 *>(vt) = x;
        } else if (so + 8u > first && so < end) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (so + e >= first && so + e < end) vt[e] = rows[o + e][dim];
        }
        __syncthreads();
    }
    if constexpr (BOUNDS) {
        __shared__ __attribute__((aligned(16))) _Float16 most[2][R][HD + 8];
        const _Float16 nan = (_Float16)__builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (bad >> i & 1u) lo[i] = hi[i] = nan;
        *reinterpret_cast<h8 *>(&most[0][r][c * 8u]) = lo;
        *reinterpret_cast<h8 *>(&most[1][r][c * 8u]) = hi;
        __syncthreads();
        for (uint32_t t = tid; t < 2u * HD; t += 256u) {
            const uint32_t which = t / HD, dim = t % HD;
            float x = (float)most[which][0][dim];
#pragma unroll
            for (int u = 1; u < R; ++u) {
                const float y = (float)most[which][u][dim];
                x = x != x ? x : y != y ? y : which ? fmaxf(x, y) : fminf(x, y);
            }
            reinterpret_cast<_Float16 *>(a.bounds)[(((size_t)a.layer * a.b.geom.pages + page) * heads + head) * 2u * HD + t] = (_Float16)x;
        }
    }
}

// ------------------------------------------------------------------- selection
// The most that a key within a page's bounds can score: sum over the group's heads j and the
// dimensions of max(q_j lo, q_j hi) = up . hi + down . lo, with up and down the sums over j of
// max(q_j, 0) and min(q_j, 0). In 64 bits: the choice falls at a border between sums that 32 bits,
// added up in one order or another, would swap.
//
// A page's order: sums as unsigned numbers that rise with them, NaN above all of them.
__device__ __forceinline__ uint64_t order_of(double x) {
    if (x != x) return ~0ull;
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);   // -0 as 0
    return u >> 63 ? ~u : u | 1ull << 63;
}

constexpr uint32_t kScorePages = 64;   // pages of a workgroup

// Sums of 2^k values a lane over the L lanes of its group (L 16, 32 or 64, N a divisor of L): each
// step halves what a lane holds, so that in the end lane l has the whole sum of value l % N.
template <int N, int L>
__device__ __forceinline__ double fold(double (&s)[N]) {
    const uint32_t lane = threadIdx.x & 63u;
    int n = N;
#pragma unroll
    for (int d = 1; d < N; d <<= 1) {
        n /= 2;
        const bool odd = lane & (uint32_t)d;
#pragma unroll
        for (int k = 0; k < N / 2; ++k)
            if (k < n) {
                // values 2 k and 2 k + 1 of those left are the ones that differ in this step's bit
                const double keep = odd ? s[2 * k + 1] : s[2 * k], give = odd ? s[2 * k] : s[2 * k + 1];
                s[k] = keep + __shfl_xor(give, d, 64);
            }
    }
    double x = s[0];
#pragma unroll
    for (int d = N; d < L; d <<= 1) x += __shfl_xor(x, d, 64);
    return x;
}

// A workgroup takes 64 pages of a row and KV head, a wave 16, L lanes a page. What is fetched does
// not wait for what it is multiplied by. Bound by four loads that need each other (the row's
// request, the table, the bounds; the queries beside them), then by the bytes of the bounds. 1020 pages 3.9 us,
// 512 of 16 requests (8.4 MB) 5.0.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_score(PagedSelect a, uint32_t blocks) {
    constexpr int L = HD / 4;              // lanes of a page: eight values each of lo, then hi
    constexpr int AT = 64 / L;             // pages of a wave at once
    constexpr int P = kScorePages / 4;     // pages of a wave
    constexpr int N = P / AT;              // of a group of L lanes: page n AT + lane / L
    __shared__ double ends[2][HD];         // down, up
    const uint32_t tid = threadIdx.x, lane = tid & 63u, w = tid >> 6, heads = a.b.geom.kv_heads;
    const uint32_t pair = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const uint32_t row = pair / heads, head = pair % heads, shift = 31u - __clz(a.b.geom.page_size);
    const uint32_t request = a.plan[a.s.requests + row], position = a.plan[a.s.positions + row];
    if (request >= a.b.requests) return;
    const uint32_t last = min(position >> shift, a.b.table_width - 1u);
    if (block * kScorePages > last) return;
    const uint32_t group = a.b.q_heads / heads, l = lane % L;
    const uint32_t *const table = a.tables + (size_t)request * a.b.table_width;
    const h8 *const bounds = reinterpret_cast<const h8 *>(a.bounds) + ((size_t)a.layer * a.b.geom.pages * heads + head) * L + l;
    uint64_t *const to = a.scratch + ((size_t)row * heads + head) * a.b.table_width;
    h8 x[N];
    uint32_t page[N];
    auto fetch = [&](uint32_t k) {
#pragma unroll
        for (int n = 0; n < N; ++n) page[n] = table[min(k + n * AT + lane / L, last)];
#pragma unroll
        for (int n = 0; n < N; ++n) x[n] = bounds[(size_t)min(page[n], a.b.geom.pages - 1u) * heads * L];
    };
    uint32_t k = block * kScorePages + w * P;
    if (k <= last) fetch(k);
    const float *const q = a.q + (size_t)row * a.q_stride + (size_t)head * group * HD;
    for (uint32_t d = tid; d < (uint32_t)HD; d += 256u) {
        double up = 0, down = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < group; ++j) {
            const float v = q[(size_t)j * HD + d];
            up += v > 0.f || v != v ? (double)v : 0.0;
            down += v < 0.f || v != v ? (double)v : 0.0;
        }
        ends[0][d] = down;
        ends[1][d] = up;
    }
    __syncthreads();
    double coef[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) coef[i] = ends[l / (L / 2)][l % (L / 2) * 8 + i];
    for (; k <= last; k += blocks * kScorePages) {
        if (k != block * kScorePages + w * P) fetch(k);
        double s[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            s[n] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[n] += coef[i] * (double)(float)x[n][i];
            if (page[n] >= a.b.geom.pages) s[n] = __builtin_nan("");
        }
        const double sum = fold<N, L>(s);
        const uint32_t p = k + l % N * AT + lane / L;
        if (l < (uint32_t)N && p <= last) to[p] = order_of(sum);
    }
}

// A workgroup a row and KV head, E orders a thread one behind the other (E 0: as many as it takes,
// read again each time). The pages that stay in any case are known by index. Of the others the least
// order that stays is found by histograms of 2048 bins over the range that is left: orders from lo to hi are
// binned by their distance from lo, and the bin that the border falls in is the next range, until it
// is taken whole or holds equal orders only, of which the first pages stay. Two passes as a rule. Bound by
// the passes' barriers and one workgroup's way through its orders: 1020 pages 5.5 us, 8125 12.4.
constexpr uint32_t kChoose = 512, kBins = 2048;
template <int E>
__global__ __launch_bounds__(512) void k_paged_choose(PagedSelect a) {
    __shared__ uint32_t bins[kBins], between[kChoose / 64][2], chosen[3];
    __shared__ uint64_t ends[2][kChoose / 64];
    const uint32_t tid = threadIdx.x, heads = a.b.geom.kv_heads, row = blockIdx.x / heads, head = blockIdx.x % heads;
    const uint32_t lane = tid & 63u, w = tid >> 6, shift = 31u - __clz(a.b.geom.page_size);
    const uint64_t *const keys = a.scratch + ((size_t)row * heads + head) * a.b.table_width;
    const uint32_t request = a.plan[a.s.requests + row], position = a.plan[a.s.positions + row];
    uint32_t *const out = a.selected + ((size_t)row * heads + head) * a.budget;
    const uint32_t n = request < a.b.requests ? min(position >> shift, a.b.table_width - 1u) + 1u : 0u;
    if (n <= a.budget) {
        for (uint32_t k = tid; k < a.budget; k += kChoose) out[k] = k < n ? k : VX_PAGED_NONE;
        return;
    }
    const uint32_t each = E ? E : (n + kChoose - 1u) / kChoose, k0 = min(tid * each, n), k1 = min(k0 + each, n);
    const uint32_t held0 = a.sinks, held1 = n - a.recent;           // pages below and from there on stay
    uint64_t mine[E ? E : 1];
    if constexpr (E != 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) mine[e] = k0 + e < n ? keys[k0 + e] : 0;
    }
    // every page that has to be chosen, with its order
    auto each_free = [&](auto &&f) {
        if constexpr (E != 0) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (k0 + e >= held0 && k0 + e < held1) f(k0 + e, mine[e]);
        } else {
            for (uint32_t k = max(k0, held0); k < min(k1, held1); ++k) f(k, keys[k]);
        }
    };
    uint64_t lo = ~0ull, hi = 0;
    each_free([&](uint32_t, uint64_t x) { lo = min(lo, x), hi = max(hi, x); });
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        lo = min(lo, (uint64_t)__shfl_xor((unsigned long long)lo, d, 64));
        hi = max(hi, (uint64_t)__shfl_xor((unsigned long long)hi, d, 64));
    }
    if (lane == 0) ends[0][w] = lo, ends[1][w] = hi;
    for (uint32_t k = tid; k < kBins; k += kChoose) bins[k] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < kChoose / 64; ++u) lo = min(lo, ends[0][u]), hi = max(hi, ends[1][u]);
    uint32_t left = a.budget - a.sinks - a.recent;   // pages to take of those from lo to hi
    bool some = false;                               // not all that equal lo are taken
    while (left) {
        const uint64_t range = hi - lo;
        const int by = range >> 11 ? 53 - __clzll(range) : 0;        // (hi - lo) >> by is below 2048
        each_free([&](uint32_t, uint64_t x) {
            if (x >= lo && x <= hi) atomicAdd(&bins[(x - lo) >> by], 1u);
        });
        __syncthreads();
        // four bins a thread, the highest first
        constexpr uint32_t BE = kBins / kChoose;
        uint32_t count[BE], v[1] = {0}, before[1], all[1];
#pragma unroll
        for (uint32_t e = 0; e < BE; ++e) count[e] = bins[kBins - 1u - (tid * BE + e)], v[0] += count[e];
        scan<1, kChoose>(v, before, all, 0x7fffffffu, reinterpret_cast<uint32_t (*)[1]>(between));
        if (before[0] < left && v[0] >= left) {
            uint32_t above = before[0];
            bool done = false;
#pragma unroll
            for (uint32_t e = 0; e < BE; ++e) {
                if (!done && above + count[e] >= left) {
                    done = true;
                    chosen[0] = kBins - 1u - (tid * BE + e);
                    chosen[1] = left - above;
                    chosen[2] = count[e];
                }
                if (!done) above += count[e];
            }
        }
        for (uint32_t k = tid; k < kBins; k += kChoose) bins[k] = 0;
        __syncthreads();
        lo += (uint64_t)chosen[0] << by;
        const uint64_t span = (1ull << by) - 1ull;
        hi = hi - lo < span ? hi : lo + span;
        left = chosen[1];
        const bool whole = chosen[2] == left;
        __syncthreads();
        if (whole) break;
        if (by == 0) {
            some = true;
            break;
        }
    }
    if (a.budget == a.sinks + a.recent) lo = ~0ull, some = true, left = 0;   // none but those that stay
    // in rising order; of those equal to lo the first `left` where not all are taken
    uint32_t v[2] = {0, 0}, before[2], all[2];
    auto count = [&](uint32_t k, uint64_t x) {
        const bool held = k < held0 || k >= held1;
        v[0] += held || x > lo || (x == lo && !some);
        v[1] += !held && some && x == lo;
    };
    if constexpr (E != 0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (k0 + e < n) count(k0 + e, mine[e]);
    } else {
        for (uint32_t k = k0; k < k1; ++k) count(k, keys[k]);
    }
    scan<2, kChoose>(v, before, all, 0x7fffffffu, between);
    uint32_t sure = before[0], equal = before[1];
    auto put = [&](uint32_t k, uint64_t x) {
        const bool held = k < held0 || k >= held1, take = held || x > lo || (x == lo && !some), tie = !held && some && x == lo;
        if (take || (tie && equal < left)) out[sure + min(equal, left)] = k;
        sure += take;
        equal += tie;
    };
    if constexpr (E != 0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (k0 + e < n) put(k0 + e, mine[e]);
    } else {
        for (uint32_t k = k0; k < k1; ++k) put(k, keys[k]);
    }
}

}  // namespace

int launch_paged_reset(hipStream_t s, const vx_paged_batch &b, uint32_t *lengths, uint32_t *tables, uint32_t *pool) {
    const uint64_t n = std::max<uint64_t>(std::max<uint64_t>(b.requests, (uint64_t)b.requests * b.table_width), b.geom.pages);
    k_paged_reset<<<(uint32_t)std::min<uint64_t>((n + 255u) / 256u, 4096u), 256, 0, s>>>(b, lengths, tables, pool);
    VX_LAUNCHED("k_paged_reset");
    return VX_OK;
}

int launch_paged_plan(hipStream_t s, const PagedPlan &a) {
    // a workgroup for so many rows, entries of a list or requests as it has threads; 64 for more, and one for
    // each of the lists and the header (16 requests of a token: 5.8 us, by one workgroup 7.1). As few threads
    // and requests a thread as hold them all (16: 5.8 us, with 512 threads 6.6, 1024 11.0; 512: 8.1, 11.7).
    const uint32_t most = std::max(std::max(a.b.max_rows, a.b.requests), a.s.items * (a.s.tile_rows <= 16u ? kPagedListed : 1u));
    auto blocks = [&](uint32_t threads) { return std::min(std::max((most + threads - 1u) / threads, 8u), 64u); };
    if (a.b.requests <= 256u)
        k_paged_plan<256, 1><<<blocks(256), 256, 0, s>>>(a);
    else if (a.b.requests <= 1024u)
        k_paged_plan<512, 2><<<blocks(512), 512, 0, s>>>(a);
    else
        k_paged_plan<1024, 4><<<blocks(1024), 1024, 0, s>>>(a);
    VX_LAUNCHED("k_paged_plan");
    return VX_OK;
}

int launch_paged_advance(hipStream_t s, const vx_paged_batch &b, const uint32_t *plan, uint32_t *lengths, uint32_t *pool) {
    k_paged_advance<<<(b.requests + 255u) / 256u, 256, 0, s>>>(b, plan, paged_shape(b).granted, lengths, pool);
    VX_LAUNCHED("k_paged_advance");
    return VX_OK;
}

int launch_paged_cut(hipStream_t s, const vx_paged_batch &b, const uint32_t *keep, uint32_t *lengths, uint32_t *tables,
                     uint32_t *pool) {
    k_paged_cut<<<1, kCutThreads, 0, s>>>(b, keep, lengths, tables, pool);
    VX_LAUNCHED("k_paged_cut");
    return VX_OK;
}

#define PAGED_HD(hd, call)                \
    switch (hd) {                         \
        case 64: call(64); break;         \
        case 128: call(128); break;       \
        default: call(256); break;        \
    }

int launch_paged_store(hipStream_t s, const PagedStore &a) {
    const dim3 grid(a.s.runs * a.b.geom.kv_heads);
#define CALL(HD)                                        \
    if (a.bounds)                                       \
        k_paged_store<HD, true><<<grid, 256, 0, s>>>(a); \
    else                                                \
        k_paged_store<HD, false><<<grid, 256, 0, s>>>(a)
    PAGED_HD(a.b.geom.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_paged_store");
    return VX_OK;
}

uint64_t paged_select_scratch_bytes(const vx_paged_batch &b) {
    return (uint64_t)b.max_rows * b.geom.kv_heads * b.table_width * 8u;
}

int launch_paged_select(hipStream_t s, const PagedSelect &a) {
    const uint32_t pairs = a.b.max_rows * a.b.geom.kv_heads;
    // at most 2^14 workgroups, or one a pair: the pages beyond are taken in turns
    const uint32_t blocks = std::min((a.b.table_width + kScorePages - 1u) / kScorePages, std::max(16384u / pairs, 1u));
#define CALL(HD) k_paged_score<HD><<<blocks * pairs, 256, 0, s>>>(a, blocks)
    PAGED_HD(a.b.geom.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_paged_score");
    // orders in registers up to 16 a thread, as few as hold them (1020 pages: 2 a thread 5.5 us, 4 5.6, 16 9.0,
    // none 6.4; 2044: 4 5.9, 16 9.0, none 7.1; 8125: 16 12.4, none 23)
    const uint32_t each = (a.b.table_width + kChoose - 1u) / kChoose;
    if (each <= 1u)
        k_paged_choose<1><<<pairs, kChoose, 0, s>>>(a);
    else if (each <= 2u)
        k_paged_choose<2><<<pairs, kChoose, 0, s>>>(a);
    else if (each <= 4u)
        k_paged_choose<4><<<pairs, kChoose, 0, s>>>(a);
    else if (each <= 16u)
        k_paged_choose<16><<<pairs, kChoose, 0, s>>>(a);
    else
        k_paged_choose<0><<<pairs, kChoose, 0, s>>>(a);
    VX_LAUNCHED("k_paged_choose");
    return VX_OK;
}

}  // namespace vx
