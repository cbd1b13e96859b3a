// Attention over the paged KV cache (include/voxhip.h, vx_paged_attention): all pages that a row
// attends to, or those of a selection.
//
// With S^T = K . Q^T and O^T = V^T . P^T, a lane of v_mfma_f32_16x16x32_f16 holds as its A operand
// eight values along the summed axis of one row: of K eight dimensions of a slot, of V^T eight
// slots of a dimension, 16 bytes each as the pages have them. Which row of the first product is
// which slot is free, so K's slots are taken in the order that leaves each lane with eight
// consecutive slots of its query row in S^T: the P^T operand of the second product, already in the
// lane's registers. Keys go by chunks of 32 slots, of two units of 16; a unit lies in one page, and
// K's and V's 16 slots at the same 32 * head_dim bytes of their caches.
#include <algorithm>
#include <type_traits>

#include "attn_dev.h"
#include "paged.h"

namespace vx {
namespace {

constexpr uint32_t kFar = 1u << 30;   // the position of a unit that holds no slots: above every row's

// Flat and with what a workgroup asks for first in front: its arguments are memory too, line by line.
struct AttnArgs {
    const PagedItem *items;          // of the plan
    const uint32_t *lists;           // of the plan: pages of items; of a selection: [row][KV head][budget] pages
    const uint32_t *header;          // of the plan
    const uint32_t *tables;
    const float *q;
    uint32_t budget, shift;          // log2 of the page size
    uint32_t table_width, requests, max_rows, pages;
    uint32_t group, by_group;        // query heads a KV head; 2^32 / group, rounded up (0 where group is 1)
    uint32_t q_stride, out_stride;
    uint32_t tile_rows, tiles, by_tiles, splits, per;   // tiles of a row, splits of its list, chunks of one (of a selection)
    uint32_t parts;                  // of one KV head
    const uint8_t *kc, *vc;          // of the layer
    float *out;
    float *ml, *acc;                 // [KV head][part][tile rows][2], [..][tile rows][HD]
    const uint32_t *row_requests, *row_positions;       // of the plan
    const PagedJoin *joins;          // of the plan
};

// What a kernel attends to: all pages; all, each read once; those of a selection.
enum Mode { kDense, kOnce, kSelected };

// The token of a row. The product with 2^32 / group rounded up is exact for rows below 2^22
// and groups up to 2^10: it is over by less than 2^22 2^10 / 2^32 / group.
__device__ __forceinline__ uint32_t token_of(const AttnArgs &p, uint32_t row) {
    return p.by_group ? __umulhi(row, p.by_group) : row;
}

// A tile of query rows: those of one request from `tile` on, the request's row 0 being row `row`
// of the step at position `base`. In bounds whatever the plan's buffer holds.
struct Tile {
    uint32_t request, row, base, count, tile, first, n, part;
    bool ok;
};
template <Mode MODE>
__device__ __forceinline__ Tile tile_of(const AttnArgs &p) {
    Tile t;
    const uint32_t index = blockIdx.x, cap = p.table_width << p.shift;
    if constexpr (MODE == kSelected) {
        t.row = p.by_tiles ? __umulhi(index, p.by_tiles) : index;   // exact: an index is below 2^22, tiles at most 2^10
        t.tile = (index - t.row * p.tiles) * p.tile_rows;
        t.request = p.row_requests[t.row];
        t.base = p.row_positions[t.row];
        t.count = 1;
        t.ok = t.request < p.requests && t.base < cap;
        const uint32_t chunks = ((min(p.budget, (t.base >> p.shift) + 1u) << p.shift) + 31u) / 32u;
        t.first = blockIdx.z * p.per;
        t.n = t.first < chunks ? min(p.per, chunks - t.first) : 0u;
        t.part = chunks > p.per ? index * p.splits + blockIdx.z : VX_PAGED_NONE;
    } else {
        const PagedItem it = p.items[index];
        t = {it.request, it.row, it.base, it.count, it.tile, it.first, it.n, it.part, false};
        t.ok = index < p.header[5] && paged_is_item(it, p.requests, p.max_rows, p.group, cap, p.parts);
    }
    return t;
}

// Into scalar registers: the compiler does not see that loads by the workgroup's index are uniform.
__device__ __forceinline__ Tile uniform(Tile t) {
    uint32_t *const f[8] = {&t.request, &t.row, &t.base, &t.count, &t.tile, &t.first, &t.n, &t.part};
#pragma unroll
    for (int k = 0; k < 8; ++k) *f[k] = __builtin_amdgcn_readfirstlane(*f[k]);
    t.ok = __builtin_amdgcn_readfirstlane(t.ok) != 0;
    return t;
}

// log2(e) / sqrt(HD): weights are powers of two.
template <int HD>
constexpr float kScale = kLog2e / (HD == 64 ? 8.0f : HD == 128 ? 11.3137085f : 16.0f);

// Sixteen query rows as the B operand: lane (i, q) holds row i, dimensions 32 u + 8 q + 0..7 in
// step u; split() makes two f16 terms of the row, with log2(e) / sqrt(HD) in it and scaled, and
// returns the scale that is left to the scores. It is a power of two: products with it are exact,
// so that a score less the reference, an fma, is what it would be of rounded scores.
template <int HD>
struct QRow {
    static constexpr int U = HD / 32;
    float x[U][8];
    // Rows lie at any multiple of four bytes, which loads of sixteen take: a branch for those at sixteen would
    // make what is loaded wait at its end.
    __device__ __forceinline__ void load(const AttnArgs &p, const Tile &t, uint32_t head, uint32_t row, uint32_t q) {
        const uint32_t k = token_of(p, row), j = row - k * p.group;
        const float *src = p.q + (size_t)(t.row + k) * p.q_stride + (size_t)(head * p.group + j) * HD + q * 8u;
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(x[u], src + 32 * u, 32);
    }
    __device__ __forceinline__ float split(h8 *qh, h8 *ql) const {
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[u][i]));
        constexpr float c = kScale<HD>;
        const int e = scale_of(row_max(top) * c);
        const float up = ldexpf(c, 10 - e);
#pragma unroll
        for (int u = 0; u < U; ++u) split8(x[u], up, qh[u], ql[u]);
        return ldexpf(1.0f, e - 10);
    }
};

// Eight values; ONCE: not kept in the caches behind them.
template <bool ONCE>
__device__ __forceinline__ h8 load_once(const uint8_t *from) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const h8 *>(from));
    return *reinterpret_cast<const h8 *>(from);
}

// A lane's share of a chunk of K: for both of the product's row tiles tt, slot 8 (i / 4) + 4 tt +
// i % 4. Lane (i, q) of the product S^T then holds the scores of query row i and slots 8 q + 4 tt + r:
// eight consecutive ones.
template <int HD>
struct KFrag {
    static constexpr int U = HD / 32;
    h8 x[2][U];
    template <bool ONCE>
    __device__ __forceinline__ void load(const uint8_t *unit, uint32_t i, uint32_t q) {
        const uint8_t *const at = unit + (8u * (i / 4u % 2u) + i % 4u) * 16u + q * 256u;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int u = 0; u < U; ++u) x[tt][u] = load_once<ONCE>(at + tt * 64 + u * 1024);
    }
};
// Of V^T: octet q of the chunk's slots, dimensions 16 dt + i.
template <int HD>
struct VFrag {
    static constexpr int DT = HD / 16;
    h8 x[DT];
    template <bool ONCE>
    __device__ __forceinline__ void load(const uint8_t *unit, uint32_t i, uint32_t q) {
        const uint8_t *const at = unit + (q % 2u) * (HD * 16u) + i * 16u;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) x[dt] = load_once<ONCE>(at + dt * 256);
    }
};

typedef uint32_t U4 __attribute__((ext_vector_type(4)));
// All ones in the first n of eight halves.
__device__ __forceinline__ U4 halves_below(uint32_t n) {
    U4 m;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) m[k] = n > 2u * k + 1u ? ~0u : n > 2u * k ? 0xffffu : 0u;
    return m;
}
__device__ __forceinline__ bool finite(_Float16 x) {
    return (__builtin_bit_cast(uint16_t, x) & 0x7c00u) != 0x7c00u;
}
__device__ __forceinline__ bool infinite(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7fffu) == 0x7c00u; }

// Over the 16 lanes of a row of lanes, in each of them (row_ror 8, 4, 2, 1).
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, dpp<0x128>(v));
    v = fmaxf(v, dpp<0x124>(v));
    v = fmaxf(v, dpp<0x122>(v));
    return fmaxf(v, dpp<0x121>(v));
}
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0x128>(v);
    v += dpp<0x124>(v);
    v += dpp<0x122>(v);
    return v + dpp<0x121>(v);
}

// A kernel's arguments once more, from where they lie: the compiler need not keep them in registers for a rare path, nor
// from one turn of its loops to the next.
typedef decltype(__builtin_amdgcn_kernarg_segment_ptr()) Arguments;
__device__ __forceinline__ const AttnArgs &again(Arguments args) {
    asm("" : "+s"(args));
    return *(const AttnArgs *)args;
}

// The first position of unit h of chunk c of a tile's part, and where it lies in the caches (bytes); kFar where there is
// no such unit, or no slot that some row of the tile attends to. Uniform.
template <Mode MODE>
__device__ __forceinline__ uint32_t unit_at(Arguments args, const Tile &t, uint32_t head, uint32_t last_pos, uint32_t c,
                                            uint32_t h, size_t unit_bytes, size_t *at) {
    const AttnArgs &p = again(args);
    const uint32_t first = (t.first + c) * 32u + kPagedUnit * h, mask = (1u << p.shift) - 1u;
    uint32_t index = first >> p.shift;
    if constexpr (MODE == kSelected) {
        const uint32_t own = t.base >> p.shift;
        if (index >= min(p.budget, own + 1u)) return kFar;
        index = p.lists[((size_t)t.row * gridDim.y + head) * p.budget + index];
        if (index > own) return kFar;
    }
    if (index >= p.table_width) return kFar;
    const uint32_t pos = (index << p.shift) + (first & mask), page = p.tables[(size_t)t.request * p.table_width + index];
    if (page >= p.pages || pos > last_pos) return kFar;
    *at = (size_t)((page * gridDim.y + head) * ((mask + 1u) / kPagedUnit) + (first & mask) / kPagedUnit) * unit_bytes;
    return pos;
}

// The rare path of a part in whose keys there are infinities. Times the two terms of a query these are infinities of
// both signs, or NaN, where the key's product with the query is one infinity: -inf, say, whose slot has a weight of 0. So the
// tile's rows are made by the formula in f32, as IEEE arithmetic has it: a wave takes some rows through 16 slots at a time,
// without matrix products (2000 tokens at 6000, one infinite key: 6.3 ms in place of 0.25; one token over 1000: 0.14). And of a
// part whose pages are not those that the plan has listed (`must`). False, and nothing is done, where there is no need. Its
// arguments and a lane's numbers are made anew, so that what comes before has the registers and the time that it has without it.
template <int HD, int RT, int W, Mode MODE>
__device__ __forceinline__ bool by_formula(bool must, uint32_t *endless) {
    constexpr int U = HD / 32, D = HD / 64;   // D dimensions of a lane: lane + 64 d
    constexpr size_t UNIT = 32 * HD;
    uint32_t tid = threadIdx.x;
    asm("" : "+v"(tid));   // nor are a lane's numbers kept
    const uint32_t lane = tid & 63u, i = lane & 15u, q = lane >> 4, head = blockIdx.y, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Arguments args = __builtin_amdgcn_kernarg_segment_ptr();
    const Tile t = uniform(tile_of<MODE>(again(args)));
    const uint32_t rows = t.count * again(args).group, last_pos = t.base + token_of(again(args), min(t.tile + RT, rows) - 1u);
    size_t at = 0;
    for (uint32_t c = w; c < 2u * t.n && !must; c += W) {
        const uint32_t pos = unit_at<MODE>(args, t, head, last_pos, c / 2u, c & 1u, UNIT, &at);
        if (pos == kFar) continue;
        uint32_t some = 0;
        for (uint32_t e = lane; e < 2u * HD; e += 64u) {   // eighths [head_dim / 8][slot]
            const h8 x = *reinterpret_cast<const h8 *>(again(args).kc + at + e * 16u);
#pragma unroll
            for (int k = 0; k < 8; ++k) some |= infinite(x[k]) && pos + e % 16u <= last_pos;
        }
        if (some) *endless = 1u;
    }
    __syncthreads();
    if (!must && *endless == 0u) return false;
    constexpr int N = HD < 256 ? RT / W : 2;   // rows of a wave at once, as many as registers hold: r + W n
    for (uint32_t r = w; r < (uint32_t)RT && t.tile + r < rows; r += W * N) {
        float top[N], sum[N], o[N][D];
        bool any[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            top[n] = -INFINITY, sum[n] = 0.f, any[n] = false;
#pragma unroll
            for (int d = 0; d < D; ++d) o[n][d] = 0.f;
        }
        for (uint32_t c = 0; c < 2u * t.n; ++c) {
            const uint32_t pos = unit_at<MODE>(args, t, head, last_pos, c / 2u, c & 1u, UNIT, &at);
            if (pos == kFar) continue;
            const AttnArgs &p = again(args);
            h8 k[U], x[2][D];
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = *reinterpret_cast<const h8 *>(p.kc + at + (4u * u + q) * 256u + i * 16u);
            bool wild = false;                    // some value is not finite
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    x[h][d] = *reinterpret_cast<const h8 *>(p.vc + at + (h * HD + lane + 64u * d) * 16u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) wild = wild || !finite(x[h][d][e]);
                }
            wild = __any(wild);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const uint32_t row = t.tile + r + W * n, token = token_of(p, row), last = t.base + token;
                if (row >= rows || pos > last) continue;
                any[n] = true;
                const float *const src = p.q + (size_t)(t.row + token) * p.q_stride + (size_t)(head * p.group + row - token * p.group) * HD + 8u * q;
                float s = 0.f;                    // of slot i
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)k[u][e], src[32 * u + e], s);
                s = row_sum(s) * kScale<HD>;
                const bool sees = pos + i <= last;
                const float most = fmaxf(top[n], max16(sees ? s : -INFINITY)), ref = most == -INFINITY ? 0.f : most;
                const float alpha = most == top[n] ? 1.f : __builtin_amdgcn_exp2f(top[n] - most);
                const float weight = sees ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
                auto of = [&](uint32_t e) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, weight), e)); };
                top[n] = most;
                sum[n] = sum[n] * alpha + sum16(weight);
#pragma unroll
                for (int d = 0; d < D; ++d) o[n][d] = __builtin_isfinite(o[n][d]) ? o[n][d] * alpha : o[n][d];
                if (!wild) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
#pragma unroll
                        for (int d = 0; d < D; ++d) o[n][d] = __builtin_fmaf(of(e), (float)x[e / 8][d][e % 8], o[n][d]);
                    continue;
                }
                const uint32_t seen = (uint32_t)__ballot(sees), none = (uint32_t)__ballot(s == -INFINITY);
#pragma unroll 1
                for (uint32_t e = 0; e < 16u; ++e) {
                    if (!(seen >> e & 1u)) continue;
#pragma unroll
                    for (int d = 0; d < D; ++d) {   // an infinity is itself by any weight but that of -inf, the one that is 0
                        const _Float16 v = reinterpret_cast<const _Float16 *>(p.vc + at)[(e / 8u * HD + lane + 64u * d) * 8u + e % 8u];
                        o[n][d] += finite(v) || (none >> e & 1u) ? of(e) * (float)v : (float)v;
                    }
                }
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const AttnArgs &p = again(args);
            const uint32_t row = t.tile + r + W * n, token = token_of(p, row);
            if (row >= rows) continue;
            if (t.part == VX_PAGED_NONE) {
                float *const to = p.out + (size_t)(t.row + token) * p.out_stride + (size_t)(head * p.group + row - token * p.group) * HD + lane;
#pragma unroll
                for (int d = 0; d < D; ++d) to[64 * d] = any[n] ? o[n][d] * (1.0f / sum[n]) : 0.f;
            } else {
                const size_t record = ((size_t)head * p.parts + t.part) * RT + r + W * n;
#pragma unroll
                for (int d = 0; d < D; ++d) p.acc[record * HD + lane + 64u * d] = o[n][d];
                if (lane == 0) p.ml[record * 2u] = top[n], p.ml[record * 2u + 1u] = any[n] ? sum[n] : -1.f;
            }
        }
    }
    return true;
}

// One workgroup: a tile of 16 NT query rows (tokens x the KV head's query heads) of a request over
// a part of its chunks, which the waves take in turn, each with its own running maximum and sum;
// they join in LDS. A tile with one part is finished here, the others' partial sums go to scratch.
// PK, of at most eight rows: columns 0..7 of the products take the high terms of the rows,
// columns 8..15 the low ones, so that one product does for both; the scores of the two
// columns of a row are added, and so are its sums at the end.
//
// Bound, with heads of 128: one token over 511, 6.0 us, by what needs each other, the part, its pages, q and K,
// four chunks a wave and the join in LDS; 64 requests over up to 24000, 183, by reading 1.06 GB (5.8 TB/s; a kernel
// that only reads: 6.25); 919 tokens of two requests, 58, by the issue of products (0.46 of the CUs' busy time) and other
// vector instructions (0.33), and by 460 tiles on 256 CUs (busy 0.69 of it): 790 TFLOP/s of two-term products.
template <int HD, int NT, int W, bool PK, Mode MODE>
__global__ __launch_bounds__(64 * W, NT > 1 || HD > 128 ? 1 : 2) void k_paged_attn(AttnArgs p) {
    constexpr int U = HD / 32, DT = HD / 16, OROW = HD + 4, R = 16 * NT, RT = PK ? 8 : R;
    constexpr int QLDS = NT > 1 ? R * HD : 0;   // floats: two f16 planes
    constexpr int LDS = W * R * OROW > QLDS ? W * R * OROW : QLDS;
    constexpr size_t UNIT = 32 * HD;            // bytes
    __shared__ __attribute__((aligned(16))) float lds[LDS];
    static_assert((!PK || NT == 1) && (W == 4 || W == 8), "one column tile of both terms; a wave or two a SIMD");
    __shared__ float ms[W][R], ls[W][R], fs[R];
    // by dimension the first position of a +inf or NaN in V, and of a -inf or NaN
    __shared__ uint32_t odd[2][HD], odd_in[W], endless;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, i = lane & 15u, q = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t heads = gridDim.y, head = blockIdx.y;
    // What the first chunks' pages are is asked for together with what the tile is: the plan's list of the
    // item's pages, or the row's list of a selection.
    constexpr bool ONCE = MODE == kOnce, LISTED = NT == 1 && MODE != kSelected;
    uint32_t early = VX_PAGED_NONE;
    if constexpr (NT == 1) {
        const uint32_t k = 2u * (w + W * (lane / 2u)) + (lane & 1u);   // unit of the part
        if constexpr (MODE == kSelected) {
            const uint32_t entry = (blockIdx.z * p.per * 32u + kPagedUnit * k) >> p.shift;
            const uint32_t row = p.by_tiles ? __umulhi(blockIdx.x, p.by_tiles) : blockIdx.x;
            early = p.lists[((size_t)row * heads + head) * p.budget + min(entry, p.budget - 1u)];
        } else {
            early = p.lists[(size_t)blockIdx.x * kPagedListed + min(k, kPagedListed - 1u)];
        }
    }
    const Tile t = uniform(tile_of<MODE>(p));
    if (!t.ok || t.n == 0) return;
    const uint32_t rows = t.count * p.group, r0 = t.tile, ri = PK ? i & 7u : i;
    const uint32_t sees_all = t.base + token_of(p, r0);                               // last position that every row attends to
    const uint32_t last_pos = t.base + token_of(p, min(r0 + RT, rows) - 1u);          // and that some row does
    const uint8_t *const kc = p.kc, *const vc = p.vc;

    // The wave's chunks t.first + w + W j: lane 2 (j - start) + h holds unit h of the j-th, up to 32 chunks
    // at once, in the first place as many as `early` has.
    // The table has the last word on pages: what it says of those that the plan has listed is asked for with the first
    // chunk, and compared with the list at the end.
    uint32_t unit = 0, where = kFar, start = 0, tabled = 0;
    uint64_t pages_in = 0;   // lanes with a unit that some row attends to
    uint32_t stop = NT > 1 || MODE == kSelected ? 32u : kPagedListed / 2u / W;
    const uint32_t mask = (1u << p.shift) - 1u, units = (mask + 1u) / kPagedUnit;
    auto look_up = [&](uint32_t j0, auto is_early) {
        constexpr bool first = decltype(is_early)::value;
        const uint32_t c = w + W * (j0 + lane / 2u), at = (t.first + c) * 32u + kPagedUnit * (lane & 1u);
        uint32_t index = at >> p.shift;
        bool there = c < t.n;
        if constexpr (MODE == kSelected) {
            there = there && index < min(p.budget, (t.base >> p.shift) + 1u);
            if constexpr (first)
                index = early;
            else
                index = there ? p.lists[((size_t)t.row * heads + head) * p.budget + index] : 0u;
            there = there && index <= t.base >> p.shift;
        }
        there = there && index < p.table_width;
        const uint32_t off = at & mask, pos = (index << p.shift) + off;
        there = there && pos <= last_pos;
        uint32_t page = p.tables[(size_t)t.request * p.table_width + (there ? index : 0u)];
        if constexpr (first && MODE != kSelected) tabled = page, pages_in = __ballot(there), page = early;
        there = there && page < p.pages;
        unit = there ? (page * heads + head) * units + off / kPagedUnit : 0u;
        where = there ? pos : kFar;
    };
    auto unit_of = [&](uint32_t j, bool second) {   // bytes
        const uint32_t at = (j - start) * 2u, u0 = __builtin_amdgcn_readlane(unit, at), u1 = __builtin_amdgcn_readlane(unit, at + 1u);
        return (size_t)(second ? u1 : u0) * UNIT;
    };
    auto where_is = [&](uint32_t j, uint32_t h) { return (uint32_t)__builtin_amdgcn_readlane(where, (j - start) * 2u + h); };
    // Loads come back in order: the queries first, which are worked on while the first chunk is on its way.
    QRow<HD> qr;
    if constexpr (NT == 1) qr.load(p, t, head, min(r0 + ri, rows - 1u), q);   // rows behind the last are it once more
    look_up(0, std::bool_constant<NT == 1>{});
    const uint32_t mine = t.n > w ? (t.n - w + W - 1u) / W : 0u;   // the wave's chunks
    KFrag<HD> kf;
    VFrag<HD> vf;
    // K and V of a chunk are fetched when the one ahead is done with them; not of tiles of 32 rows: heads of 128 and 256
    // have no registers for it, and heads of 64 take 138, with which a CU has one workgroup and not two (2000 tokens at 6000
    // 158 us in place of 128, but 5 drafted tokens of 64 requests 60 in place of 73).
    constexpr bool AHEAD = NT == 1;
    if constexpr (AHEAD) {   // a wave without chunks fetches unit 0: a branch here would have the queries wait for what is in it
        kf.template load<ONCE>(kc + unit_of(0, i >= 8u), i, q);
        vf.template load<ONCE>(vc + unit_of(0, q >= 2u), i, q);
    }

    for (uint32_t d = tid; d < 2u * HD; d += 64u * W) odd[d / HD][d % HD] = ~0u;
    if (tid == 0) endless = 0u;
    uint32_t found = 0;
    // The two terms of the queries, in registers where these do; the tiles of 32 rows get them through LDS, which the other
    // heads' read again each chunk (heads of 128: 919 tokens 60.3 us, read each time 62.4; 2000 at 6000 267 and 288;
    // but heads of 64, of which a CU then holds one workgroup and not two, 160 and 137).
    constexpr bool HELD = NT == 1 || HD == 128;
    h8 qh[HELD ? NT : 1][U], ql[HELD ? NT : 1][U];
    float factor[NT];
    h8 *const qs = reinterpret_cast<h8 *>(lds);   // [NT][U][hi, lo][64]
    if constexpr (NT == 1) {
        factor[0] = qr.split(qh[0], ql[0]);
        if constexpr (PK) {
#pragma unroll
            for (int u = 0; u < U; ++u) qh[0][u] = i < 8u ? qh[0][u] : ql[0][u];
        }
    } else {
        for (uint32_t c = w; c < NT; c += W) {
            const uint32_t row = r0 + 16u * c + i;
            qr.load(p, t, head, min(row, rows - 1u), q);
            const float f = qr.split(qh[0], ql[0]);
            if (q == 0) fs[16u * c + i] = f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                qs[((c * U + u) * 2u) * 64u + lane] = qh[0][u];
                qs[((c * U + u) * 2u + 1u) * 64u + lane] = ql[0][u];
            }
        }
    }
    if constexpr (NT > 1) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NT; ++c) factor[c] = fs[16 * c + i];
        if constexpr (HELD) {
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    qh[c][u] = qs[((c * U + u) * 2u) * 64u + lane];
                    ql[c][u] = qs[((c * U + u) * 2u + 1u) * 64u + lane];
                }
        }
    }
    // last position that the lane's row of a column tile attends to
    auto limit = [&](int c) { return t.base + token_of(p, min(r0 + 16u * c + ri, rows - 1u)); };

    float m[NT], l[NT];
    bool saw[NT];   // the lane's row attends to some slot
    f4 o[NT][DT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        saw[c] = false;
        m[c] = -INFINITY;
        l[c] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[c][dt] = f4{0.f, 0.f, 0.f, 0.f};
    }
    float minus = PK && i < 8u ? 0.0f : -1.0f;
    asm("" : "+v"(minus));
    const bool partly = last_pos != sees_all;   // some row does not attend to all that another does

    // A chunk; at an edge, some row attends to a part of it only. (One body for both: with two, the
    // compiler moves the sums from registers to registers between them.)
    bool whole = false;   // some chunk was none at an edge
    auto step = [&](uint32_t j, uint32_t w0, uint32_t w1, bool edge) {
        const uint8_t *const vu = vc + unit_of(j, q >= 2u);
        if constexpr (!AHEAD) kf.template load<ONCE>(kc + unit_of(j, i >= 8u), i, q);
        // Behind the last chunk it is fetched once more, without a branch: with one between the products
        // and what reads them, this compiler lost count of the wait that that needs.
        const uint32_t next = min(j + 1u, mine - 1u);
        if (next == stop && next != j) {
            look_up(next, std::false_type{});
            start = next;
            stop = next + 32u;
        }
        const uint8_t *const ku = kc + unit_of(next, i >= 8u), *const vnext = vc + unit_of(next, q >= 2u);
        f4 x[NT][2];
#pragma unroll
        for (int c = 0; c < NT; ++c) x[c][0] = x[c][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const h8 hi = HELD ? qh[HELD ? c : 0][u] : qs[((c * U + u) * 2u) * 64u + lane];
                const h8 lo = HELD ? ql[HELD ? c : 0][u] : qs[((c * U + u) * 2u + 1u) * 64u + lane];
                x[c][0] = mfma16(kf.x[0][u], hi, x[c][0]);
                x[c][1] = mfma16(kf.x[1][u], hi, x[c][1]);
                if constexpr (!PK) {
                    x[c][0] = mfma16(kf.x[0][u], lo, x[c][0]);
                    x[c][1] = mfma16(kf.x[1][u], lo, x[c][1]);
                }
            }
        }
        if constexpr (AHEAD)
            kf.template load<ONCE>(ku, i, q);
        else
            vf.template load<ONCE>(vu, i, q);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (PK) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[0][e / 4][e % 4] += dpp<0x128>(x[0][e / 4][e % 4]);   // row_ror:8
        }
        const uint32_t slot0 = (q < 2u ? w0 : w1) + 8u * (q % 2u);   // the lane's first position
        if (edge) {
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const uint32_t last = limit(c);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c][e / 4][e % 4] = slot0 + e > last ? -INFINITY : x[c][e / 4][e % 4];
                saw[c] = saw[c] || slot0 <= last;
            }
        }
        whole = whole || !edge;
        float top[NT];
        bool moves = false;
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            top[c] = x[c][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top[c] = fmaxf(top[c], x[c][e / 4][e % 4]);
            top[c] *= factor[c];
            moves = moves || top[c] - m[c] > kMost;
        }
        if (__builtin_expect(__any(moves), 0)) {
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const float s = row_max(top[c]), mn = s - m[c] > kMost ? s - kRaise : m[c];
                const float alpha = mn == m[c] ? 1.f : __builtin_amdgcn_exp2f(m[c] - mn);
                m[c] = mn;
                l[c] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[c][dt] *= alpha;
            }
        }
        h8 ph[NT], pl[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            // A row that attends to nothing of the chunks so far has no reference yet; any serves.
            const float ref = m[c] == -INFINITY ? 0.f : m[c];
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[c][e / 4][e % 4], factor[c], -ref));
                l[c] += v[e];
            }
            two_terms(v, minus, ph[c], pl[c]);   // of PK the term of the lane's column, by `minus`
        }
        __builtin_amdgcn_sched_barrier(0);
        if (edge) {
            // Slots behind the last position may hold anything: their values count as zero, as do
            // infinities and NaN among those that some row does not attend to, which `odd` notes.
            const U4 keep = halves_below(last_pos + 1u > slot0 ? last_pos + 1u - slot0 : 0u);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) vf.x[dt] = __builtin_bit_cast(h8, __builtin_bit_cast(U4, vf.x[dt]) & keep);
            if (partly) {
                const U4 own = ~halves_below(sees_all + 1u > slot0 ? sees_all + 1u - slot0 : 0u);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const U4 x = __builtin_bit_cast(U4, vf.x[dt]);
                    const U4 top = ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u;   // of each half whose exponent is all ones
                    const U4 bad = (top | (top - (top >> 15))) & own;
                    found |= (bad[0] | bad[1]) | (bad[2] | bad[3]);
                    vf.x[dt] = __builtin_bit_cast(h8, x & ~bad);
                }
            }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
            for (int c = 0; c < NT; ++c) o[c][dt] = mfma16(vf.x[dt], PK ? pl[c] : ph[c], o[c][dt]);
            if constexpr (!PK) {
#pragma unroll
                for (int c = 0; c < NT; ++c) o[c][dt] = mfma16(vf.x[dt], pl[c], o[c][dt]);
            }
        }
        if constexpr (AHEAD) vf.template load<ONCE>(vnext, i, q);
    };
    for (uint32_t j = 0; j < mine; ++j) {
        const uint32_t w0 = where_is(j, 0), w1 = where_is(j, 1);
        step(j, w0, w1, max(w0, w1) + kPagedUnit - 1u > sees_all);
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        l[c] = row_sum(l[c]);
        if (!whole && row_max(saw[c] ? 1.f : 0.f) == 0.f) l[c] = -1.f;   // nothing to add
        if (q == 0) ms[w][16 * c + i] = m[c], ls[w][16 * c + i] = l[c];
    }
    // Infinities in K and V have no two terms to be multiplied by, and some of V were taken as zero: where a sum
    // is not finite or such a value was found, the chunks are gone through again (rare).
    float zero = found ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) zero = __builtin_fmaf(o[c][dt][e], 0.f, zero);
    const bool finite_here = __all(zero == 0.f), as_listed = !LISTED || (__ballot(tabled != early) & pages_in & ((1ull << kPagedListed / W) - 1ull)) == 0u;
    if (lane == 0) odd_in[w] = (finite_here ? 0u : 1u) | (as_listed ? 0u : 2u);
    __syncthreads();   // the queries in LDS have been read, every wave's m and l are there
    uint32_t odds = 0;
#pragma unroll
    for (int v = 0; v < W; ++v) odds |= odd_in[v];
    const bool any_odd = odds != 0u;
    if (__builtin_expect(any_odd, 0)) {
        if (by_formula<HD, RT, W, MODE>(odds & 2u, &endless)) return;
        for (uint32_t j = 0; j < mine; ++j) {
            if ((j & 31u) == 0) {
                look_up(j, std::false_type{});
                start = j;
            }
            const uint32_t w0 = where_is(j, 0), w1 = where_is(j, 1);
            const uint32_t slot0 = (q < 2u ? w0 : w1) + 8u * (q % 2u);
            const uint8_t *const at = vc + unit_of(j, q >= 2u) + (q % 2u) * (HD * 16u) + i * 16u;
#pragma unroll 1
            for (int dt = 0; dt < DT; ++dt) {
                const h8 x = *reinterpret_cast<const h8 *>(at + dt * 256);
                uint32_t up = ~0u, down = ~0u;
#pragma unroll
                for (int e = 7; e >= 0; --e) {
                    const bool counts = !finite(x[e]) && slot0 + e <= last_pos;
                    up = counts && !(x[e] < 0.f16) ? slot0 + e : up;
                    down = counts && !(x[e] > 0.f16) ? slot0 + e : down;
                }
                if (up != ~0u) atomicMin(&odd[0][16 * dt + i], up);
                if (down != ~0u) atomicMin(&odd[1][16 * dt + i], down);
            }
        }
    }

    // A wave's sums are taken to the row's largest reference. One without keys has nothing
    // to give; one whose every score is NaN has no reference but a NaN sum.
    auto *const os = reinterpret_cast<float (*)[R][OROW]>(lds);
    float sum[NT], top[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        // the waves' by the four lanes of a row
        float mv[W / 4], lv[W / 4];
#pragma unroll
        for (int v = 0; v < W / 4; ++v) mv[v] = ms[4 * v + q][16 * c + i], lv[v] = ls[4 * v + q][16 * c + i];
        top[c] = row_max(W > 4 ? fmaxf(mv[0], mv[W / 4 - 1]) : mv[0]);
        sum[c] = 0.f;
#pragma unroll
        for (int v = 0; v < W / 4; ++v)
            sum[c] += lv[v] < 0.f ? 0.f : mv[v] == -INFINITY ? lv[v] : lv[v] * __builtin_amdgcn_exp2f(mv[v] - top[c]);
        sum[c] = row_sum(sum[c]);
        if (row_max(lv[0] < 0.f && lv[W / 4 - 1] < 0.f ? 0.f : 1.f) == 0.f) sum[c] = -1.f;
        const float share = m[c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[c] - top[c]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[c][dt] *= share;
    }
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4 *>(&os[w][16 * c + i][16 * dt + 4 * q]) = o[c][dt];
    const bool alone = t.part == VX_PAGED_NONE;
    const size_t part = (size_t)head * p.parts + (alone ? 0u : t.part);
    if (w == 0 && q == 0) {   // the factors of the scores have been read, a barrier ago and more
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            fs[16 * c + i] = sum[c];
            if (alone || (PK && i >= 8u)) continue;
            p.ml[(part * RT + 16u * c + i) * 2u] = top[c];
            p.ml[(part * RT + 16u * c + i) * 2u + 1u] = sum[c];
        }
    }
    __syncthreads();
    constexpr int V = HD / 4;   // four dimensions a lane
    for (uint32_t k = tid; k < (uint32_t)RT * V; k += 64u * W) {
        const uint32_t r = k / V, c = 4u * (k % V), row = r0 + r;
        if (row >= rows) break;
        f4 v = *reinterpret_cast<const f4 *>(&os[0][r][c]);
#pragma unroll
        for (int u = 1; u < W; ++u) v += *reinterpret_cast<const f4 *>(&os[u][r][c]);
        if constexpr (PK) {
#pragma unroll
            for (int u = 0; u < W; ++u) v += *reinterpret_cast<const f4 *>(&os[u][r + 8u][c]);
        }
        const uint32_t k0 = token_of(p, row), j = row - k0 * p.group;
        if (any_odd) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool up = odd[0][c + e] <= t.base + k0, down = odd[1][c + e] <= t.base + k0;
                v[e] = up ? down ? __builtin_nanf("") : INFINITY : down ? -INFINITY : v[e];
            }
        }
        if (!alone) {
            *reinterpret_cast<f4 *>(p.acc + (part * RT + r) * HD + c) = v;
            continue;
        }
        v = fs[r] < 0.f ? f4{0.f, 0.f, 0.f, 0.f} : v * (1.0f / fs[r]);   // attends to nothing: 0
        float *const to = p.out + (size_t)(t.row + k0) * p.out_stride + (size_t)(head * p.group + j) * HD + c;
        __builtin_memcpy(to, &v, 16);   // at any multiple of four bytes
    }
}

// The parts of tiles' rows, joined: a workgroup takes every gridDim-th row, its lanes HD / 4 columns by
// as many parts at once as fit. What a row's parts hold is asked for as soon as it is known
// where they are. Bound by three loads that need each other: 128 parts of 8 rows of two heads 4.7 us, of
// which an empty launch takes 4.
template <int HD, bool SELECTED>
__global__ __launch_bounds__(256) void k_paged_join(AttnArgs p, uint32_t most, uint32_t heads) {
    constexpr int V = HD / 4, Y = 256 / V, E = 8;
    __shared__ float sc[kPagedMaxSplits], red[3][4];
    __shared__ __attribute__((aligned(16))) float os[Y][HD];
    const uint32_t tid = threadIdx.x, tile_rows = p.tile_rows, c = 4u * (tid % V), y = tid / V;
    const uint32_t all = SELECTED ? most : min(p.header[6] * tile_rows * heads, most), cap = p.table_width << p.shift;
    for (uint32_t k = blockIdx.x; k < all; k += gridDim.x) {
        const uint32_t head = k % heads, r = k / heads % tile_rows, index = k / heads / tile_rows;
        uint32_t step_row, row, first, n;   // the request's first row, its query row; the parts
        if constexpr (SELECTED) {
            step_row = index / p.tiles;
            row = index % p.tiles * tile_rows + r;
            first = index * p.splits;
            const uint32_t base = p.row_positions[step_row];
            if (p.row_requests[step_row] >= p.requests || base >= cap || row >= p.group) continue;
            const uint32_t chunks = ((min(p.budget, (base >> p.shift) + 1u) << p.shift) + 31u) / 32u;
            n = (chunks + p.per - 1u) / p.per;
        } else {
            const PagedJoin j = p.joins[index];
            const uint32_t rows = j.count * p.group;
            if (j.row >= p.max_rows || j.count > p.max_rows - j.row || j.base > cap || j.count > cap - j.base ||
                j.tile >= rows || j.tile + r >= rows || j.per == 0u || j.part >= p.parts)
                continue;
            step_row = j.row;
            row = j.tile + r;
            first = j.part;
            const uint32_t last = j.base + token_of(p, min(j.tile + tile_rows, rows) - 1u);
            n = min((last / 32u + j.per) / j.per, p.parts - first);   // of the tile's chunks
        }
        if (n <= 1u || n > kPagedMaxSplits) continue;
        const size_t at = ((size_t)head * p.parts + first) * tile_rows + r;   // the row's record in the first part
        f4 early[2 * E] = {};
        auto ask = [&](int e) { early[e] = *reinterpret_cast<const f4 *>(p.acc + (at + (size_t)min(y + e * Y, n - 1u) * tile_rows) * HD + c); };
#pragma unroll
        for (int e = 0; e < E; ++e) ask(e);
        if (n > (uint32_t)(E * Y)) {
#pragma unroll
            for (int e = E; e < 2 * E; ++e) ask(e);
        }
        float m = -INFINITY, l = -1.f;
        if (tid < n) {
            m = p.ml[(at + (size_t)tid * tile_rows) * 2u];
            l = p.ml[(at + (size_t)tid * tile_rows) * 2u + 1u];
        }
        float top = m, some = l < 0.f ? 0.f : 1.f;
#pragma unroll
        for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64)), some = fmaxf(some, __shfl_xor(some, d, 64));
        if ((tid & 63u) == 0) red[0][tid >> 6] = top, red[1][tid >> 6] = some;
        __syncthreads();
        top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        some = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
        // Not 0, which an infinite sum times would be NaN: a part's sums are below 2^59 (2^28 slots of weights up to 2^15 and
        // values below 2^16), so that with 2^-126 they are below 2^-67 where the row's own weights reach 1 and more.
        const float part = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top), mine = part == 0.f ? 0x1p-126f : part;
        if (tid < n) sc[tid] = mine;
        float sum = l < 0.f ? 0.f : l * mine;
#pragma unroll
        for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if ((tid & 63u) == 0) red[2][tid >> 6] = sum;
        __syncthreads();
        sum = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
        f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2 * E; ++e)
            if (y + e * Y < n) o += early[e] * sc[y + e * Y];
#pragma unroll 8
        for (uint32_t v = y + 2 * E * Y; v < n; v += Y)
            o += *reinterpret_cast<const f4 *>(p.acc + (at + (size_t)v * tile_rows) * HD + c) * sc[v];
        *reinterpret_cast<f4 *>(&os[y][c]) = o;
        __syncthreads();
        if (tid < (uint32_t)HD) {
            float x = os[0][tid];
#pragma unroll
            for (int u = 1; u < Y; ++u) x += os[u][tid];
            const uint32_t token = token_of(p, row), j = row - token * p.group;
            p.out[(size_t)(step_row + token) * p.out_stride + (size_t)(head * p.group + j) * HD + tid] = some == 0.f ? 0.f : x / sum;
        }
        __syncthreads();
    }
}

// Of a selection: tiles of a row, and how its list is divided: so that about as many workgroups
// come out as of a step without one, of least chunks or more.
void divide(const vx_paged_batch &b, const PagedShape &s, uint32_t budget, uint32_t *tiles, uint32_t *splits, uint32_t *per) {
    const uint32_t group = b.q_heads / b.geom.kv_heads;
    *tiles = (group + s.tile_rows - 1u) / s.tile_rows;
    const uint64_t chunks = ((uint64_t)std::min(budget, b.table_width) * b.geom.page_size + 31u) / 32u;
    const uint64_t units = (uint64_t)b.max_rows * b.geom.kv_heads * *tiles;
    uint64_t n = std::min<uint64_t>(std::max<uint64_t>((1u << s.workgroups) / units, 1u), kPagedMaxSplits);
    *per = (uint32_t)std::max<uint64_t>((chunks + n - 1u) / n, chunks <= kPagedWhole ? kPagedWhole : 2u * s.waves);
    *splits = (uint32_t)((chunks + *per - 1u) / *per);
}

// A selection is each row's own: its tiles are of a row's query heads, 16 at most.
PagedShape shape_of(vx_paged_batch b, uint32_t budget) {
    if (budget) b.max_count = 1;
    PagedShape s = paged_shape(b);
    if (budget && s.tile_rows > 16u) s.tile_rows = 16u, s.waves = 4u, s.workgroups = b.geom.head_dim < 256u ? 10u : 9u;
    return s;
}

uint64_t parts_of(const vx_paged_batch &b, const PagedShape &s, uint32_t budget) {
    if (!budget) return s.parts;
    uint32_t tiles, splits, per;
    divide(b, s, budget, &tiles, &splits, &per);
    return splits > 1u ? (uint64_t)b.max_rows * tiles * splits : 0u;
}

template <int HD>
void run(hipStream_t s, const AttnArgs &p, const PagedAttn &a, bool packed, dim3 g) {
    // K and V of a layer that the last-level cache (256 MB) cannot hold until the next step are read past
    // the caches, where each is read once (64 requests over up to 24000, 1.06 GB: 194 us, so 182; but 16
    // over 8000, 86 MB, which lie there still when they are read again: 16.6, so 18.5).
    const vx_paged_geom &m = a.b.geom;
    const bool once = a.b.max_count * p.group <= p.tile_rows &&
                      (uint64_t)m.pages * m.page_size * m.kv_heads * m.head_dim * 4u > 256u << 20;
    constexpr int WIDE = HD < 256 ? 8 : 4;
    if (a.selected && packed)
        k_paged_attn<HD, 1, 4, true, kSelected><<<g, 256, 0, s>>>(p);
    else if (a.selected)
        k_paged_attn<HD, 1, 4, false, kSelected><<<g, 256, 0, s>>>(p);
    else if (packed && once)
        k_paged_attn<HD, 1, 4, true, kOnce><<<g, 256, 0, s>>>(p);
    else if (packed)
        k_paged_attn<HD, 1, 4, true, kDense><<<g, 256, 0, s>>>(p);
    else if (p.tile_rows == 16u && once)
        k_paged_attn<HD, 1, 4, false, kOnce><<<g, 256, 0, s>>>(p);
    else if (p.tile_rows == 16u)
        k_paged_attn<HD, 1, 4, false, kDense><<<g, 256, 0, s>>>(p);
    else
        k_paged_attn<HD, 2, WIDE, false, kDense><<<g, 64 * WIDE, 0, s>>>(p);
}

template <int HD>
void join(hipStream_t s, const AttnArgs &p, const PagedAttn &a) {
    const uint32_t heads = a.b.geom.kv_heads;
    const uint32_t most = (uint32_t)((a.selected ? (uint64_t)a.b.max_rows * p.tiles : a.s.joins) * p.tile_rows * heads);
    const dim3 grid(std::min(most, 1024u));
    if (a.selected)
        k_paged_join<HD, true><<<grid, 256, 0, s>>>(p, most, heads);
    else
        k_paged_join<HD, false><<<grid, 256, 0, s>>>(p, most, heads);
}

}  // namespace

uint64_t paged_attn_scratch_bytes(const vx_paged_batch &b, uint32_t budget) {
    const PagedShape s = shape_of(b, budget);
    // never 0, which is what a batch that is not valid has
    return std::max<uint64_t>(parts_of(b, s, budget) * b.geom.kv_heads * s.tile_rows * (b.geom.head_dim + 2u) * 4u, 16u);
}

int launch_paged_attention(hipStream_t s, const PagedAttn &a) {
    AttnArgs p{};
    const vx_paged_geom &g = a.b.geom;
    const PagedShape shape = shape_of(a.b, a.budget);   // what lies where in the plan is in a.s
    if (a.selected) divide(a.b, shape, a.budget, &p.tiles, &p.splits, &p.per);
    p.items = reinterpret_cast<const PagedItem *>(a.plan + a.s.item_at);
    p.lists = a.selected ? a.selected : a.plan + a.s.page_at;
    p.header = a.plan;
    p.tables = a.tables;
    p.q = a.q;
    p.budget = a.budget;
    p.shift = paged_shift(g.page_size);
    p.table_width = a.b.table_width;
    p.requests = a.b.requests;
    p.max_rows = a.b.max_rows;
    p.pages = g.pages;
    auto inverse = [](uint32_t n) { return n > 1u ? (uint32_t)(((1ull << 32) + n - 1u) / n) : 0u; };
    p.group = a.b.q_heads / g.kv_heads;
    p.by_group = inverse(p.group);
    p.by_tiles = inverse(p.tiles);
    p.q_stride = a.q_stride;
    p.out_stride = a.out_stride;
    p.tile_rows = shape.tile_rows;
    p.parts = (uint32_t)parts_of(a.b, shape, a.budget);
    const size_t layer_at = (size_t)a.layer * g.pages * g.kv_heads * g.page_size * g.head_dim * 2u;
    p.kc = a.kc + layer_at;
    p.vc = a.vc + layer_at;
    p.out = a.out;
    p.acc = a.scratch;
    p.ml = a.scratch + (uint64_t)p.parts * g.kv_heads * p.tile_rows * g.head_dim;
    p.row_requests = a.plan + a.s.requests;
    p.row_positions = a.plan + a.s.positions;
    p.joins = reinterpret_cast<const PagedJoin *>(a.plan + a.s.join_at);
    const dim3 grid(a.selected ? a.b.max_rows * p.tiles : a.s.items, g.kv_heads, a.selected ? p.splits : 1u);
    switch (g.head_dim) {
        case 64: run<64>(s, p, a, shape.packed, grid); break;
        case 128: run<128>(s, p, a, shape.packed, grid); break;
        default: run<256>(s, p, a, shape.packed, grid); break;
    }
    VX_LAUNCHED("k_paged_attn");
    if (a.selected ? p.splits == 1u : a.s.joins == 0u) return VX_OK;   // nothing is divided
    switch (g.head_dim) {
        case 64: join<64>(s, p, a); break;
        case 128: join<128>(s, p, a); break;
        default: join<256>(s, p, a); break;
    }
    VX_LAUNCHED("k_paged_join");
    return VX_OK;
}

}  // namespace vx
