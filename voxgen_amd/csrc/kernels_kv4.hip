// The KV cache held in 4 bits: storing and reading rows, attention over the cache with
// its accumulated weights, and eviction by them (include/voxhip.h, vx_kv4_*, has the
// format). Slot counts are read from device memory, so that a captured step replays.
//
// A block of 32 slots is laid out for the matrix products that read it. With S^T =
// K . Q^T and O^T = V^T . P^T, a lane of v_mfma_f32_16x16x32_f16 holds as its A operand
// eight values along the summed axis of one row: of K, eight dimensions of a slot (one
// dword of codes); of V^T, eight slots of a dimension (one dword, V being stored
// transposed within the block). Which row of the product is which slot is free, so the
// slots of K's rows are taken in the order that leaves, in S^T, each lane with eight
// consecutive slots of its query row: the P^T operand of the second product, already in
// the lane's registers.
#include "kv4.h"

namespace vx {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kLimit = 61440.0f;   // inputs are clamped to this: o + 15 d then stays inside f16
constexpr float kLog2e = 1.4426950408889634f;

template <int HD>
struct Lay {
    static constexpr int G = HD / 32;          // groups of a row
    static constexpr int CODES = 16 * HD;      // bytes of a block's codes, its scales behind them
    static constexpr int BLOCK = 20 * HD;
};

__device__ __forceinline__ size_t plane_of(const vx_kv4_geom &g, uint32_t layer, uint32_t seq, uint32_t head) {
    return ((size_t)layer * g.sequences + seq) * g.kv_heads + head;
}
template <int HD>
__device__ __forceinline__ size_t plane_bytes(const vx_kv4_geom &g) {
    return (size_t)((g.context + 31u) / 32u) * Lay<HD>::BLOCK;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}

// The bit of element e of a dword of eight codes.
__device__ __forceinline__ constexpr int code_bit(int e) { return 4 * (e / 2) + 16 * (e % 2); }

// Eight codes as f16 pairs: 1024 + c and 64 + c are made by or-ing a nibble under the
// exponent for which its lowest bit counts one, and the difference is exact.
__device__ __forceinline__ void codes8(uint32_t w, h2 *c) {
    const h2 k1024 = {1024.f16, 1024.f16}, k64 = {64.f16, 64.f16};
    const uint32_t u = w >> 8;
    c[0] = __builtin_bit_cast(h2, (w & 0x000f000fu) | 0x64006400u) - k1024;
    c[1] = __builtin_bit_cast(h2, (w & 0x00f000f0u) | 0x54005400u) - k64;
    c[2] = __builtin_bit_cast(h2, (u & 0x000f000fu) | 0x64006400u) - k1024;
    c[3] = __builtin_bit_cast(h2, (u & 0x00f000f0u) | 0x54005400u) - k64;
}
// The values of eight codes: f16(o + d * c), one rounding; of one (d, o) or of eight.
__device__ __forceinline__ h8 values8(uint32_t w, h2 d, h2 o) {
    h2 c[4];
    codes8(w, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __builtin_elementwise_fma(c[i], d, o);
    return __builtin_shufflevector(__builtin_shufflevector(c[0], c[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(c[2], c[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ h8 values8(uint32_t w, h8 d, h8 o) {
    h2 c[4];
    codes8(w, c);
    c[0] = __builtin_elementwise_fma(c[0], __builtin_shufflevector(d, d, 0, 1), __builtin_shufflevector(o, o, 0, 1));
    c[1] = __builtin_elementwise_fma(c[1], __builtin_shufflevector(d, d, 2, 3), __builtin_shufflevector(o, o, 2, 3));
    c[2] = __builtin_elementwise_fma(c[2], __builtin_shufflevector(d, d, 4, 5), __builtin_shufflevector(o, o, 4, 5));
    c[3] = __builtin_elementwise_fma(c[3], __builtin_shufflevector(d, d, 6, 7), __builtin_shufflevector(o, o, 6, 7));
    return __builtin_shufflevector(__builtin_shufflevector(c[0], c[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(c[2], c[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// ------------------------------------------------------------------- rows
// Eight values of a row.
__device__ __forceinline__ void load8(const float *p, bool vec, float *x) {
    if (vec) {
        const f4 a = *reinterpret_cast<const f4 *>(p), b = *reinterpret_cast<const f4 *>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}

// Codes, step and offset of a lane's eight values, a quarter of their group: the quad of
// lanes 4i..4i+3 holds the group. The f32 operations are those of the format, each
// rounded once (division is correctly rounded in this build's default mode).
__device__ __forceinline__ uint32_t encode8(const float *x, _Float16 &d, _Float16 &o) {
    float lo = INFINITY, hi = -INFINITY, bad = 0.f, y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bad = x[i] != x[i] ? 1.f : bad;
        y[i] = fminf(fmaxf(x[i], -kLimit), kLimit);
        lo = fminf(lo, y[i]);
        hi = fmaxf(hi, y[i]);
    }
    lo = fminf(lo, dpp<0xb1>(lo)), hi = fmaxf(hi, dpp<0xb1>(hi)), bad = fmaxf(bad, dpp<0xb1>(bad));
    lo = fminf(lo, dpp<0x4e>(lo)), hi = fmaxf(hi, dpp<0x4e>(hi)), bad = fmaxf(bad, dpp<0x4e>(bad));
    d = (_Float16)((hi - lo) / 15.0f);
    o = (_Float16)lo;
    const float df = (float)d, of = (float)o;
    uint32_t w = 0;
    if (bad != 0.f) {
        d = 0.f16;
        o = __builtin_bit_cast(_Float16, (unsigned short)0x7e00);   // the group is NaN
    } else if (df > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w |= (uint32_t)fminf(fmaxf(rintf((y[i] - of) / df), 0.f), 15.f) << code_bit(i);
    }
    return w;
}

// A workgroup per octet of slots, KV head and sequence: eight rows of HD / 8 lanes code
// eight values each. K's codes go out as they are; V's are transposed through LDS, and a
// lane then owns one dimension's dword of the octet, which it merges with the codes of
// the octet's other slots (another call's): no dword has two writers.
template <int HD>
__global__ __launch_bounds__(HD) void k_kv4_store(Kv4Rows a) {
    using L = Lay<HD>;
    constexpr int W = HD / 8;
    __shared__ uint32_t vcodes[8 * W];
    const uint32_t tid = threadIdx.x, r = tid / W, c = tid % W, head = blockIdx.y, s = blockIdx.z, seq = a.first + s;
    const uint32_t base = a.slots[seq];
    if (base >= a.g.context) return;
    const uint32_t end = min(base + a.tokens, a.g.context);
    const uint32_t oct = base / 8u + blockIdx.x, slot = oct * 8u + r;
    if (oct * 8u >= end) return;
    const bool live = slot >= base && slot < end;
    const uint32_t t = live ? slot - base : 0u;
    const size_t row = (size_t)s * a.tokens + t, plane = plane_of(a.g, a.layer, seq, head);
    const uint32_t at = head * HD + c * 8u, in_block = oct % 4u;
    uint8_t *const kb = a.kc + plane * plane_bytes<HD>(a.g) + (size_t)(oct / 4u) * L::BLOCK;
    uint8_t *const vb = a.vc + plane * plane_bytes<HD>(a.g) + (size_t)(oct / 4u) * L::BLOCK;
    float x[8], y[8];
    load8(a.k + row * a.k_stride + at, a.vec, x);
    load8(a.v + row * a.v_stride + at, a.vec, y);
    uint32_t *const vw = reinterpret_cast<uint32_t *>(vb) + in_block * HD + tid;
    const uint32_t had = *vw;
    _Float16 d, o;
    uint32_t w = encode8(x, d, o);
    if (live) {
        reinterpret_cast<uint32_t *>(kb)[(slot % 32u) * W + c] = w;
        if (c % 4u == 0) {
            const h2 p = {d, o};
            reinterpret_cast<uint32_t *>(kb + L::CODES)[(slot % 32u) * L::G + c / 4u] = __builtin_bit_cast(uint32_t, p);
        }
        if (c == 0 && a.slot_positions)
            a.slot_positions[plane * a.g.context + slot] = (a.positions ? a.positions[seq] : base) + t;
    }
    w = encode8(y, d, o);
    vcodes[r * W + c] = w;
    if (live && c % 4u == 0) {
        _Float16 *const p = reinterpret_cast<_Float16 *>(vb + L::CODES) + (in_block * L::G + c / 4u) * 16u + r;
        p[0] = d;
        p[8] = o;
    }
    __syncthreads();
    // Dword tid of the octet: dimension 32 (tid % G) + tid / G.
    const uint32_t dim = tid % L::G * 32u + tid / L::G;
    uint32_t merged = had;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t code = vcodes[e * W + dim / 8u] >> (4u * (dim % 8u / 2u) + 16u * (dim % 2u)) & 15u;
        const uint32_t sl = oct * 8u + e;
        if (sl >= base && sl < end) merged = (merged & ~(15u << code_bit(e))) | code << code_bit(e);
    }
    *vw = merged;
}

template <int HD>
__global__ __launch_bounds__(HD) void k_kv4_load(Kv4Rows a) {
    using L = Lay<HD>;
    constexpr int W = HD / 8;
    const uint32_t tid = threadIdx.x, r = tid / W, c = tid % W, head = blockIdx.y, s = blockIdx.z, seq = a.first + s;
    const uint32_t base = a.slots[seq];
    if (base >= a.g.context) return;
    const uint32_t end = min(base + a.tokens, a.g.context);
    const uint32_t oct = base / 8u + blockIdx.x, slot = oct * 8u + r;
    if (oct * 8u >= end) return;
    const size_t plane = plane_of(a.g, a.layer, seq, head), first_row = (size_t)s * a.tokens;
    const size_t block = plane * plane_bytes<HD>(a.g) + (size_t)(oct / 4u) * L::BLOCK;
    if (a.k && slot >= base && slot < end) {
        const uint8_t *const kb = a.kc + block;
        const uint32_t w = reinterpret_cast<const uint32_t *>(kb)[(slot % 32u) * W + c];
        const h2 p = __builtin_bit_cast(h2, reinterpret_cast<const uint32_t *>(kb + L::CODES)[(slot % 32u) * L::G + c / 4u]);
        const h8 x = values8(w, h2{p[0], p[0]}, h2{p[1], p[1]});
        float *const to = a.k + (first_row + slot - base) * a.k_stride + head * HD + c * 8u;
        if (a.vec) {
            reinterpret_cast<f4 *>(to)[0] = f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
            reinterpret_cast<f4 *>(to)[1] = f4{(float)x[4], (float)x[5], (float)x[6], (float)x[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i] = (float)x[i];
        }
    }
    if (a.v) {   // dimension tid of the octet's slots
        const uint8_t *const vb = a.vc + block;
        const uint32_t w = reinterpret_cast<const uint32_t *>(vb)[((oct % 4u) * 32u + tid % 32u) * L::G + tid / 32u];
        const h8 *const sc = reinterpret_cast<const h8 *>(vb + L::CODES) + ((oct % 4u) * L::G + tid / 32u) * 2u;
        const h8 x = values8(w, sc[0], sc[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t sl = oct * 8u + e;
            if (sl >= base && sl < end) a.v[(first_row + sl - base) * a.v_stride + head * HD + tid] = (float)x[e];
        }
    }
}

__global__ __launch_bounds__(256) void k_kv4_advance(uint32_t *slots, uint32_t *positions, uint32_t n, uint32_t tokens,
                                                     uint32_t context) {
    const uint32_t s = blockIdx.x * 256u + threadIdx.x;
    if (s >= n) return;
    const uint32_t at = slots[s];
    if (at == VX_KV4_NO_SLOT) return;
    slots[s] = at >= context ? at : min(at + tokens, context);
    if (positions) positions[s] += tokens;
}

// ------------------------------------------------------------------- attention
constexpr uint32_t kRows = 16;       // query rows of a tile
constexpr uint32_t kWaves = 4;
constexpr float kLazy = 8.0f;        // a row's reference moves when a score exceeds it by this
constexpr float kRaise = 7.0f;       // weights are taken 2^7 up, so that their low f16 terms stay normal

struct AttnArgs {
    Kv4Attn a;
    uint32_t group, tiles, splits;   // query heads a KV head, tiles of 16 rows, key splits of the grid
    float *ml, *acc, *lse;           // [unit][split][16][2], [unit][split][16][HD], [unit][16]
};

// Keys of a tile's rows: `base` filled slots ahead of the call, rows r0.. of rows.
struct Span {
    uint32_t base, keys, blocks, per, active;   // blocks of the tile, blocks a split, splits in use
};
__device__ __forceinline__ Span span_of(const AttnArgs &p, uint32_t seq, uint32_t tile) {
    Span s;
    s.base = p.a.slots[seq];
    const uint32_t last = min((tile + 1u) * kRows, p.a.tokens * p.group) - 1u;   // last row of the tile
    s.keys = s.base >= p.a.g.context ? 0u : min(s.base + last / p.group + 1u, p.a.g.context);
    s.blocks = (s.keys + 31u) / 32u;
    s.per = max(kWaves, (s.blocks + p.splits - 1u) / p.splits);
    s.active = (s.blocks + s.per - 1u) / s.per;
    return s;
}

__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Over the four lanes l, l + 16, l + 32, l + 48 that share a query row.
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// A tile's query rows as the B operand: lane (i, q) holds row i, dimensions
// q HD / 4 + 8 u + 0..7 in step u, as two f16 terms of the row scaled to below 2^10 (the
// low term of a value down to 2^-13 of the row's largest is then still normal). Returns
// the factor of the scores: the row's scale, log2(e) and 1 / sqrt(HD).
template <int HD>
__device__ __forceinline__ float load_q(const AttnArgs &p, uint32_t s, uint32_t head, uint32_t row, bool valid, uint32_t q,
                                        h8 *qh, h8 *ql) {
    constexpr int U = HD / 32;
    float x[U][8];
    float top = 0.f;
    const uint32_t t = row / p.group, j = row - t * p.group;
    const float *src = p.a.q + ((size_t)s * p.a.tokens + t) * p.a.q_stride + (size_t)(head * p.group + j) * HD + q * (HD / 4);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (valid) {
            load8(src + 8 * u, p.a.qvec, x[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[u][i]));
    }
    top = row_max(top);
    int e = 0;
    if (top > 0.f && top < INFINITY) e = max(__builtin_amdgcn_frexp_expf(top), -100);
    const float up = ldexpf(1.0f, 10 - e);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = x[u][i] * up;
            qh[u][i] = (_Float16)v;
            ql[u][i] = (_Float16)(v - (float)qh[u][i]);
        }
    return ldexpf(kLog2e / sqrtf((float)HD), e - 10);
}

// S^T of a block's 32 slots with the tile's rows: lane (i, q) gets the scores of row i and
// slots 8 q + 0..7.
template <int HD>
__device__ __forceinline__ void scores(const uint8_t *kb, uint32_t i, uint32_t q, const h8 *qh, const h8 *ql, float *s) {
    using L = Lay<HD>;
    constexpr int U = HD / 32;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
        const uint32_t slot = 8u * (i / 4u) + 4u * tt + i % 4u;
        const uint32_t *const codes = reinterpret_cast<const uint32_t *>(kb + slot * (HD / 2) + q * (HD / 8));
        const uint32_t *const sc = reinterpret_cast<const uint32_t *>(kb + L::CODES) + slot * L::G;
        f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // dimensions q HD / 4 + 8 u..: group q HD / 128 + u / 4
            const h2 p = __builtin_bit_cast(h2, sc[HD == 64 ? q / 2u : q * (HD / 128) + u / 4]);
            const h8 k = values8(codes[u], h2{p[0], p[0]}, h2{p[1], p[1]});
            x = mfma16(k, qh[u], x);
            x = mfma16(k, ql[u], x);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * tt + r] = x[r];
    }
}

// One workgroup: a tile of 16 query rows (tokens x the KV head's query heads) of a
// sequence over one split of its blocks, which four waves take in turn, each with its own
// running maximum and sum; they join in LDS. A tile with one split in use is finished
// here, the others' partial sums go to scratch.
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_attn(AttnArgs p) {
    using L = Lay<HD>;
    constexpr int U = HD / 32, DT = HD / 16, OROW = HD + 4;
    __shared__ __attribute__((aligned(16))) float os[kWaves][kRows][OROW];
    __shared__ float ms[kWaves][kRows], ls[kWaves][kRows];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, i = lane & 15u, q = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t split = blockIdx.x / p.tiles, tile = p.tiles - 1u - blockIdx.x % p.tiles;
    const uint32_t head = blockIdx.y, s = blockIdx.z, seq = p.a.first + s;
    const Span sp = span_of(p, seq, tile);
    const uint32_t rows = p.a.tokens * p.group, r0 = tile * kRows;
    if (split >= sp.active && !(split == 0 && sp.active == 0)) return;
    const uint32_t b0 = split * sp.per, b1 = min(b0 + sp.per, sp.blocks);
    const uint32_t row = min(r0 + i, rows - 1u);
    const bool valid = r0 + i < rows;
    const uint32_t limit = sp.base + row / p.group;   // last slot the row attends to (sp.blocks == 0 where idle)
    const uint32_t sees_all = sp.base + r0 / p.group; // last slot that every row attends to

    h8 qh[U], ql[U];
    const float factor = load_q<HD>(p, s, head, row, valid, q, qh, ql);
    const size_t plane = plane_of(p.a.g, p.a.layer, seq, head) * plane_bytes<HD>(p.a.g);
    float m = -INFINITY, l = 0.f;
    f4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f4{0.f, 0.f, 0.f, 0.f};

    for (uint32_t b = b0 + w; b < b1; b += kWaves) {
        const uint8_t *const kb = p.a.kc + plane + (size_t)b * L::BLOCK, *const vb = p.a.vc + plane + (size_t)b * L::BLOCK;
        float x[8];
        scores<HD>(kb, i, q, qh, ql, x);
        const uint32_t slot0 = b * 32u + 8u * q;
        const bool edge = b * 32u + 31u > sees_all;   // some row's last slots, or the cache's
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] *= factor;
            if (edge && slot0 + e > limit) x[e] = -INFINITY;
            top = fmaxf(top, x[e]);
        }
        if (__any(top > m + kLazy)) {
            const float t = row_max(top), mn = t > m + kLazy ? t : m;
            const float alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }
        h8 ph, pl;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = __builtin_amdgcn_exp2f(x[e] - (m - kRaise));
            if (edge && slot0 + e > limit) v = 0.f;
            l += v;
            ph[e] = (_Float16)v;
            pl[e] = (_Float16)(v - (float)ph[e]);
        }
        // Slots past the tile's keys may hold anything: their values count as zero.
        const uint32_t some = edge ? min(max(sp.keys, slot0) - slot0, 8u) : 8u;
#pragma unroll
        for (int g = 0; g < L::G; ++g) {
            const h8 *const sc = reinterpret_cast<const h8 *>(vb + L::CODES) + (q * L::G + g) * 2u;
            h8 d = sc[0], off = sc[1];
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    d[e] = (uint32_t)e < some ? d[e] : 0.f16;
                    off[e] = (uint32_t)e < some ? off[e] : 0.f16;
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t code = reinterpret_cast<const uint32_t *>(vb)[(q * 32u + 16u * h + i) * L::G + g];
                const h8 v = values8(code, d, off);
                o[2 * g + h] = mfma16(v, ph, o[2 * g + h]);
                o[2 * g + h] = mfma16(v, pl, o[2 * g + h]);
            }
        }
    }
    l = row_sum(l);
    if (q == 0) ms[w][i] = m, ls[w][i] = l;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4 *>(&os[w][i][16 * dt + 4 * q]) = o[dt];
    __syncthreads();

    const size_t unit = ((size_t)s * p.a.g.kv_heads + head) * p.tiles + tile, part = unit * p.splits + split;
    constexpr int TPR = 256 / kRows, PER = HD / TPR;   // lanes a row, dimensions a lane
    const uint32_t orow = tid / TPR, c0 = tid % TPR;
    if (r0 + orow >= rows) return;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < (int)kWaves; ++v) top = fmaxf(top, ms[v][orow]);
    float sc[kWaves], sum = 0.f;
#pragma unroll
    for (int v = 0; v < (int)kWaves; ++v) {
        // a wave without keys has nothing to give; one whose every score is NaN has no maximum but a NaN sum
        sc[v] = ms[v][orow] == -INFINITY ? (ls[v][orow] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(ms[v][orow] - top);
        sum += ls[v][orow] * sc[v];
    }
    const bool alone = sp.active <= 1u;
    const uint32_t t = (r0 + orow) / p.group, j = (r0 + orow) - t * p.group;
    const bool attends = sp.base < p.a.g.context && sp.base + t < p.a.g.context;
    const float inv = !alone ? 1.f : attends ? 1.0f / sum : 0.f;
    float *const to = alone ? p.a.out + ((size_t)s * p.a.tokens + t) * p.a.out_stride + (size_t)(head * p.group + j) * HD
                            : p.acc + (part * kRows + orow) * HD;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t c = c0 + k * TPR;
        float v = 0.f;
#pragma unroll
        for (int u = 0; u < (int)kWaves; ++u) v += os[u][orow][c] * sc[u];
        to[c] = attends || !alone ? v * inv : 0.f;
    }
    if (c0 == 0) {
        if (alone) {
            p.lse[unit * kRows + orow] = (top - kRaise) + __builtin_amdgcn_logf(sum);
        } else {
            p.ml[(part * kRows + orow) * 2u] = top;
            p.ml[(part * kRows + orow) * 2u + 1u] = sum;
        }
    }
}

// The splits of a tile, joined.
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_join(AttnArgs p) {
    const uint32_t tile = blockIdx.x, head = blockIdx.y, s = blockIdx.z, seq = p.a.first + s;
    const Span sp = span_of(p, seq, tile);
    if (sp.active <= 1u) return;
    const uint32_t rows = p.a.tokens * p.group, r0 = tile * kRows;
    const size_t unit = ((size_t)s * p.a.g.kv_heads + head) * p.tiles + tile;
    constexpr int TPR = 256 / kRows, PER = HD / TPR;
    const uint32_t orow = threadIdx.x / TPR, c0 = threadIdx.x % TPR;
    if (r0 + orow >= rows) return;
    const float *const ml = p.ml + (unit * p.splits * kRows + orow) * 2u;
    const float *const acc = p.acc + (unit * p.splits * kRows + orow) * HD;
    float top = -INFINITY;
    for (uint32_t v = 0; v < sp.active; ++v) top = fmaxf(top, ml[(size_t)v * kRows * 2u]);
    float sum = 0.f, o[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = 0.f;
    for (uint32_t v = 0; v < sp.active; ++v) {
        const float m = ml[(size_t)v * kRows * 2u], l = ml[(size_t)v * kRows * 2u + 1u];
        const float sc = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - top);
        sum += l * sc;
#pragma unroll
        for (int k = 0; k < PER; ++k) o[k] += acc[(size_t)v * kRows * HD + c0 + k * TPR] * sc;
    }
    const uint32_t t = (r0 + orow) / p.group, j = (r0 + orow) - t * p.group;
    const bool attends = sp.base + t < p.a.g.context;
    float *const to = p.a.out + ((size_t)s * p.a.tokens + t) * p.a.out_stride + (size_t)(head * p.group + j) * HD;
#pragma unroll
    for (int k = 0; k < PER; ++k) to[c0 + k * TPR] = attends ? o[k] / sum : 0.f;
    if (c0 == 0) p.lse[unit * kRows + orow] = (top - kRaise) + __builtin_amdgcn_logf(sum);
}

// Accumulated weights: a wave per block of 32 slots takes the scores of every row that may
// attend to it again, and sums 2^(score - lse) over the rows.
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_weights(AttnArgs p) {
    using L = Lay<HD>;
    constexpr int U = HD / 32;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, i = lane & 15u, q = lane >> 4;
    const uint32_t b = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t head = blockIdx.y, s = blockIdx.z, seq = p.a.first + s;
    const uint32_t rows = p.a.tokens * p.group;
    const uint32_t base = p.a.slots[seq];
    if (base >= p.a.g.context) return;
    const uint32_t keys = min(base + p.a.tokens, p.a.g.context);
    if (b * 32u >= keys) return;
    const size_t plane = plane_of(p.a.g, p.a.layer, seq, head);
    const uint8_t *const kb = p.a.kc + plane * plane_bytes<HD>(p.a.g) + (size_t)b * L::BLOCK;
    const uint32_t slot0 = b * 32u + 8u * q;
    // the first token whose row attends to a slot of the block
    const uint32_t t0 = b * 32u > base ? b * 32u - base : 0u;
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    for (uint32_t tile = t0 * p.group / kRows; tile < p.tiles; ++tile) {
        const uint32_t row = min(tile * kRows + i, rows - 1u), t = row / p.group;
        const bool valid = tile * kRows + i < rows && base + t < p.a.g.context;
        h8 qh[U], ql[U];
        const float factor = load_q<HD>(p, s, head, row, true, q, qh, ql);
        const float lse = p.lse[(((size_t)s * p.a.g.kv_heads + head) * p.tiles + tile) * kRows + row % kRows];
        float x[8];
        scores<HD>(kb, i, q, qh, ql, x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (valid && slot0 + e <= base + t) sum[e] += __builtin_amdgcn_exp2f(x[e] * factor - lse);
    }
    float *const to = p.a.weights + plane * p.a.g.context;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v = sum[e];
        v += dpp<0xb1>(v);    // over the 16 lanes of the rows: quads, half rows, rows
        v += dpp<0x4e>(v);
        v += dpp<0x141>(v);
        v += dpp<0x140>(v);
        if (i == (uint32_t)e && slot0 + e < keys) {
            const bool fresh = slot0 + e >= base || p.a.decay == 0.f;
            to[slot0 + e] = fresh ? v : p.a.decay * to[slot0 + e] + v;
        }
    }
}

// ------------------------------------------------------------------- eviction
// An order of weights as integers: rising, NaN below all, both zeros alike.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0u;
    const uint32_t b = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr uint32_t kSelect = 1024;

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// A workgroup per plane. The keep-th largest weight is found a byte at a time from
// histograms; a pass over the slots in order then numbers those that leave below `keep`
// and those that stay above it.
__global__ __launch_bounds__(kSelect) void k_kv4_select(Kv4Evict a) {
    __shared__ uint32_t hist[256], part[3][kSelect / 64], found[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, w = tid >> 6;
    const uint32_t head = blockIdx.x, s = blockIdx.y, layer = blockIdx.z, seq = a.first + s;
    const size_t plane = plane_of(a.g, layer, seq, head);
    const float *const weights = a.weights + plane * a.g.context;
    const uint32_t *const positions = a.slot_positions + plane * a.g.context;
    uint32_t *const plan = a.plan + (((size_t)layer * a.n + s) * a.g.kv_heads + head) * a.moves * 2u;
    const uint32_t had = a.slots[seq], n = had == VX_KV4_NO_SLOT ? 0u : min(had, a.g.context), keep = a.keep;
    uint32_t moved = 0;
    if (n > keep) {
        uint32_t newest = 0;
        for (uint32_t j = tid; j < n; j += kSelect) newest = max(newest, positions[j]);
        newest = wave_max_u32(newest);
        if (lane == 0) part[0][w] = newest;
        __syncthreads();
        newest = wave_max_u32(part[0][lane % (kSelect / 64)]);
        auto order = [&](uint32_t j) {
            const uint32_t at = positions[j];
            return at < a.sinks || (uint64_t)at + a.recent > newest ? 0xFFFFFFFFu : order_of(weights[j]);
        };
        uint32_t prefix = 0, rest = keep;   // the threshold's bytes so far, slots still to take among its equals
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (uint32_t j = tid; j < n; j += kSelect) {
                const uint32_t v = order(j);
                if (shift == 24 || v >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[v >> shift & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t bin = 255, above = 0;
                while (bin > 0 && above + hist[bin] < rest) above += hist[bin--];
                found[0] = bin;
                found[1] = above;
            }
            __syncthreads();
            prefix |= found[0] << shift;
            rest -= found[1];
        }
        uint32_t ties = 0, holes = 0, sources = 0;   // so far
        for (uint32_t j0 = 0; j0 < n; j0 += kSelect) {
            const uint32_t j = j0 + tid;
            const uint32_t v = j < n ? order(j) : 0u;
            const bool tie = j < n && v == prefix;
            const uint64_t below = (1ull << lane) - 1u;
            const uint64_t tb = __ballot(tie);
            __syncthreads();
            if (lane == 0) part[0][w] = __popcll(tb);
            __syncthreads();
            uint32_t rank = ties + __popcll(tb & below), all = 0;
            for (uint32_t k = 0; k < kSelect / 64; ++k) {
                if (k < w) rank += part[0][k];
                all += part[0][k];
            }
            ties += all;
            const bool stays = j < n && (v > prefix || (tie && rank < rest));
            const bool hole = j < keep && !stays, source = j >= keep && stays;
            const uint64_t hb = __ballot(hole), sb = __ballot(source);
            if (lane == 0) part[1][w] = __popcll(hb), part[2][w] = __popcll(sb);
            __syncthreads();
            uint32_t hr = holes + __popcll(hb & below), sr = sources + __popcll(sb & below);
            for (uint32_t k = 0; k < kSelect / 64; ++k) {
                if (k < w) hr += part[1][k], sr += part[2][k];
                holes += part[1][k];
                sources += part[2][k];
            }
            if (hole && hr < a.moves) plan[2u * hr + 1u] = j;
            if (source && sr < a.moves) plan[2u * sr] = j;
        }
        moved = min(sources, a.moves);
    }
    for (uint32_t k = 2u * moved + tid; k < 2u * a.moves; k += kSelect) plan[k] = VX_KV4_NO_SLOT;
}

// Moves of a plan, a workgroup for kMoves of a plane's. V's codes of an octet share dwords,
// so that the run of moves into one octet (neighbours in the plan, whose targets rise) is
// made by the workgroup of its first.
constexpr uint32_t kMoves = 32;

template <int HD>
__global__ __launch_bounds__(HD) void k_kv4_compact(Kv4Evict a) {
    using L = Lay<HD>;
    constexpr int W = HD / 8;
    const uint32_t tid = threadIdx.x, head = blockIdx.y % a.g.kv_heads, s = blockIdx.y / a.g.kv_heads, layer = blockIdx.z;
    const uint32_t seq = a.first + s;
    if (blockIdx.x == 0 && layer == 0 && head == 0 && tid == 0) {
        const uint32_t n = a.slots[seq];
        if (n != VX_KV4_NO_SLOT && n > a.keep) a.slots[seq] = a.keep;
    }
    const size_t plane = plane_of(a.g, layer, seq, head);
    const uint32_t *const plan = a.plan_in + (((size_t)layer * a.n + s) * a.g.kv_heads + head) * a.moves * 2u;
    const uint32_t e0 = blockIdx.x * kMoves, e1 = min(e0 + kMoves, a.moves);
    auto move = [&](uint32_t e, uint32_t &from, uint32_t &to) {
        if (e >= a.moves) return false;
        from = plan[2u * e];
        to = plan[2u * e + 1u];
        return from >= a.keep && from < a.g.context && to < a.keep;
    };
    uint32_t from, to;
    if (!move(e0, from, to)) return;   // the moves come first in a plan
    for (uint32_t e = e0 + tid; e < e1; e += HD) {
        if (!move(e, from, to)) continue;
        const size_t base = plane * a.g.context;
        if (a.weights) a.weights[base + to] = a.weights[base + from];
        if (a.slot_positions) a.slot_positions[base + to] = a.slot_positions[base + from];
    }
    if (!a.kc) return;
    uint8_t *const kp = a.kc + plane * plane_bytes<HD>(a.g), *const vp = a.vc + plane * plane_bytes<HD>(a.g);
    for (uint32_t e = e0 + tid / W; e < e1; e += HD / W) {
        if (!move(e, from, to)) continue;
        uint8_t *const src = kp + (size_t)(from / 32u) * L::BLOCK, *const dst = kp + (size_t)(to / 32u) * L::BLOCK;
        const uint32_t c = tid % W;
        reinterpret_cast<uint32_t *>(dst)[(to % 32u) * W + c] = reinterpret_cast<const uint32_t *>(src)[(from % 32u) * W + c];
        if (c < (uint32_t)L::G)
            reinterpret_cast<uint32_t *>(dst + L::CODES)[(to % 32u) * L::G + c] =
                reinterpret_cast<const uint32_t *>(src + L::CODES)[(from % 32u) * L::G + c];
    }
    for (uint32_t e = e0; e < e1; ++e) {
        uint32_t before_from, before_to;
        if (!move(e, from, to)) continue;
        const uint32_t oct = to / 8u;
        if (e > 0 && move(e - 1u, before_from, before_to) && before_to / 8u == oct) continue;   // not the run's first
        uint8_t *const dst = vp + (size_t)(oct / 4u) * L::BLOCK;
        uint32_t *const word = reinterpret_cast<uint32_t *>(dst) + (oct % 4u) * HD + tid;
        uint32_t v = *word;
        for (uint32_t k = e; move(k, from, to) && to / 8u == oct && k < e + 8u; ++k) {
            const uint8_t *const src = vp + (size_t)(from / 32u) * L::BLOCK;
            const uint32_t oct_from = from / 8u % 4u, ef = from % 8u, et = to % 8u;
            const uint32_t code = reinterpret_cast<const uint32_t *>(src)[oct_from * HD + tid] >> (4u * (ef / 2u) + 16u * (ef % 2u)) & 15u;
            const uint32_t bit = 4u * (et / 2u) + 16u * (et % 2u);
            v = (v & ~(15u << bit)) | code << bit;
            if (tid < 2u * L::G) {   // d and o of every group
                const uint32_t g = tid / 2u, which = tid % 2u;
                reinterpret_cast<_Float16 *>(dst + L::CODES)[((oct % 4u) * L::G + g) * 16u + 8u * which + et] =
                    reinterpret_cast<const _Float16 *>(src + L::CODES)[(oct_from * L::G + g) * 16u + 8u * which + ef];
            }
        }
        *word = v;
    }
}

}  // namespace

#define KV4_HD(hd, call)                  \
    switch (hd) {                         \
        case 64: call(64); break;         \
        case 128: call(128); break;       \
        default: call(256); break;        \
    }

int launch_kv4_store(hipStream_t s, const Kv4Rows &a) {
    const dim3 grid((a.tokens + 14u) / 8u, a.g.kv_heads, a.n);
#define CALL(HD) k_kv4_store<HD><<<grid, HD, 0, s>>>(a)
    KV4_HD(a.g.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_kv4_store");
    return VX_OK;
}

int launch_kv4_load(hipStream_t s, const Kv4Rows &a) {
    const dim3 grid((a.tokens + 14u) / 8u, a.g.kv_heads, a.n);
#define CALL(HD) k_kv4_load<HD><<<grid, HD, 0, s>>>(a)
    KV4_HD(a.g.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_kv4_load");
    return VX_OK;
}

int launch_kv4_advance(hipStream_t s, uint32_t *slots, uint32_t *positions, uint32_t n, uint32_t tokens,
                       uint32_t context) {
    k_kv4_advance<<<(n + 255u) / 256u, 256, 0, s>>>(slots, positions, n, tokens, context);
    VX_LAUNCHED("k_kv4_advance");
    return VX_OK;
}

namespace {
// Splits of the key axis: enough workgroups for two on each of 256 CUs, none with less
// than a block a wave.
struct Shape {
    uint32_t group, tiles, splits;
    uint64_t units;
};
Shape shape_of(const Kv4Attn &a) {
    Shape h;
    h.group = a.q_heads / a.g.kv_heads;
    h.tiles = (a.tokens * h.group + kRows - 1u) / kRows;
    h.units = (uint64_t)h.tiles * a.g.kv_heads * a.n;
    const uint32_t blocks = (a.g.context + 31u) / 32u, most = (blocks + kWaves - 1u) / kWaves;
    const uint64_t want = (512u + h.units - 1u) / h.units;
    h.splits = (uint32_t)(want < most ? want : most);
    return h;
}
}  // namespace

uint64_t kv4_attn_scratch_bytes(const Kv4Attn &a, bool) {
    const Shape h = shape_of(a);
    return h.units * kRows * 4u + (h.splits > 1u ? h.units * h.splits * kRows * (2u + a.g.head_dim) * 4u : 0u);
}

int launch_kv4_attention(hipStream_t s, const Kv4Attn &a) {
    const Shape h = shape_of(a);
    AttnArgs p;
    p.a = a;
    p.group = h.group;
    p.tiles = h.tiles;
    p.splits = h.splits;
    p.acc = a.scratch;
    p.ml = p.acc + (h.splits > 1u ? h.units * h.splits * kRows * a.g.head_dim : 0u);
    p.lse = p.ml + (h.splits > 1u ? h.units * h.splits * kRows * 2u : 0u);
    const dim3 grid(h.tiles * h.splits, a.g.kv_heads, a.n);
#define CALL(HD) k_kv4_attn<HD><<<grid, 256, 0, s>>>(p)
    KV4_HD(a.g.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_kv4_attn");
    if (h.splits > 1u) {
        const dim3 jgrid(h.tiles, a.g.kv_heads, a.n);
#define CALL(HD) k_kv4_join<HD><<<jgrid, 256, 0, s>>>(p)
        KV4_HD(a.g.head_dim, CALL)
#undef CALL
        VX_LAUNCHED("k_kv4_join");
    }
    if (a.weights) {
        const dim3 wgrid(((a.g.context + 31u) / 32u + kWaves - 1u) / kWaves, a.g.kv_heads, a.n);
#define CALL(HD) k_kv4_weights<HD><<<wgrid, 256, 0, s>>>(p)
        KV4_HD(a.g.head_dim, CALL)
#undef CALL
        VX_LAUNCHED("k_kv4_weights");
    }
    return VX_OK;
}

int launch_kv4_select(hipStream_t s, const Kv4Evict &a) {
    k_kv4_select<<<dim3(a.g.kv_heads, a.n, a.g.layers), kSelect, 0, s>>>(a);
    VX_LAUNCHED("k_kv4_select");
    return VX_OK;
}

int launch_kv4_compact(hipStream_t s, const Kv4Evict &a) {
    const dim3 grid((a.moves + kMoves - 1u) / kMoves, a.g.kv_heads * a.n, a.g.layers);
#define CALL(HD) k_kv4_compact<HD><<<grid, HD, 0, s>>>(a)
    KV4_HD(a.g.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_kv4_compact");
    return VX_OK;
}

}  // namespace vx
