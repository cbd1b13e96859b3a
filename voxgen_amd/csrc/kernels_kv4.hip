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
#include <type_traits>

#include "kv4.h"

namespace vx {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
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
// exponent for which its lowest bit counts one, and the difference is exact. The masks are
// kept in registers, so that a pair takes one v_and_or_b32 (which takes no literals).
struct Masks {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, k1024 = 0x64006400u, k64 = 0x54005400u;
    __device__ __forceinline__ Masks() {
        asm("" : "+s"(low), "+s"(high));
        asm("" : "+v"(k1024), "+v"(k64));
    }
};
__device__ __forceinline__ void codes8(const Masks &k, uint32_t w, h2 *c) {
    const h2 k1024 = {1024.f16, 1024.f16}, k64 = {64.f16, 64.f16};
    const uint32_t u = w >> 8;
    c[0] = __builtin_bit_cast(h2, (w & k.low) | k.k1024) - k1024;
    c[1] = __builtin_bit_cast(h2, (w & k.high) | k.k64) - k64;
    c[2] = __builtin_bit_cast(h2, (u & k.low) | k.k1024) - k1024;
    c[3] = __builtin_bit_cast(h2, (u & k.high) | k.k64) - k64;
}
__device__ __forceinline__ h8 join8(const h2 *c) {
    return __builtin_shufflevector(__builtin_shufflevector(c[0], c[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(c[2], c[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
// The values of eight codes: f16(o + d * c), one rounding; of one (d, o) or of eight.
__device__ __forceinline__ h8 values8(const Masks &k, uint32_t w, h2 d, h2 o) {
    h2 c[4];
    codes8(k, w, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __builtin_elementwise_fma(c[i], d, o);
    return join8(c);
}
__device__ __forceinline__ h8 values8(const Masks &k, uint32_t w, h8 d, h8 o) {
    h2 c[4];
    codes8(k, w, c);
    c[0] = __builtin_elementwise_fma(c[0], __builtin_shufflevector(d, d, 0, 1), __builtin_shufflevector(o, o, 0, 1));
    c[1] = __builtin_elementwise_fma(c[1], __builtin_shufflevector(d, d, 2, 3), __builtin_shufflevector(o, o, 2, 3));
    c[2] = __builtin_elementwise_fma(c[2], __builtin_shufflevector(d, d, 4, 5), __builtin_shufflevector(o, o, 4, 5));
    c[3] = __builtin_elementwise_fma(c[3], __builtin_shufflevector(d, d, 6, 7), __builtin_shufflevector(o, o, 6, 7));
    return join8(c);
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
// the octet's other slots (another call's): no dword has two writers. Bound by one launch
// up to about a thousand tokens, then more and more by the bytes: 2.8 us for a token of 2 KV heads
// of 128, 4.6 for 1900 (4.5 MB, 1.0 TB/s), 5.8 in a graph for 8192 (19 MB, 3.3 TB/s).
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

// A workgroup per octet of slots, KV head and sequence, two lanes a dword of codes: K's rows
// go out as they are made, four values a lane; V's, made a dimension a lane, pass through LDS
// to be written the same way (2056 tokens of 2 heads of 128 3.4 us; stored a dimension a lane
// 3.8). Bound by one launch, then by the bytes written: 1.6 us for a token, 5.4 in a graph
// for 8192 (19 MB, 3.6 TB/s).
template <int HD>
__global__ __launch_bounds__(2 * HD) void k_kv4_load(Kv4Rows a) {
    using L = Lay<HD>;
    constexpr int W = HD / 8, Q = HD / 4, VROW = HD + 4;   // a row's dwords of codes and quads of values
    __shared__ __attribute__((aligned(16))) float vrows[8 * VROW];
    const uint32_t tid = threadIdx.x, head = blockIdx.y, s = blockIdx.z, seq = a.first + s;
    const uint32_t base = a.slots[seq];
    if (base >= a.g.context) return;
    const uint32_t end = min(base + a.tokens, a.g.context);
    const uint32_t oct = base / 8u + blockIdx.x;
    if (oct * 8u >= end) return;
    const size_t plane = plane_of(a.g, a.layer, seq, head), first_row = (size_t)s * a.tokens;
    const size_t block = plane * plane_bytes<HD>(a.g) + (size_t)(oct / 4u) * L::BLOCK;
    const uint32_t r = tid / Q, c = tid % Q, slot = oct * 8u + r;   // row of the octet, quad of the row
    const bool live = slot >= base && slot < end;
    auto put = [&](float *to, f4 v) {
        if (a.vec) {
            *reinterpret_cast<f4 *>(to) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = v[i];
        }
    };
    if (a.v && tid < (uint32_t)HD) {   // dimension tid of the octet's slots
        const uint8_t *const vb = a.vc + block;
        const uint32_t w = reinterpret_cast<const uint32_t *>(vb)[((oct % 4u) * 32u + tid % 32u) * L::G + tid / 32u];
        const h8 *const sc = reinterpret_cast<const h8 *>(vb + L::CODES) + ((oct % 4u) * L::G + tid / 32u) * 2u;
        const h8 x = values8(Masks(), w, sc[0], sc[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) vrows[e * VROW + tid] = (float)x[e];
    }
    if (a.k && live) {
        const uint8_t *const kb = a.kc + block;
        const uint32_t w = reinterpret_cast<const uint32_t *>(kb)[(slot % 32u) * W + c / 2u];
        const h2 p = __builtin_bit_cast(h2, reinterpret_cast<const uint32_t *>(kb + L::CODES)[(slot % 32u) * L::G + c / 8u]);
        const h8 x = values8(Masks(), w, h2{p[0], p[0]}, h2{p[1], p[1]});
        const bool upper = c % 2u;
        put(a.k + (first_row + slot - base) * a.k_stride + head * HD + c * 4u,
            f4{(float)(upper ? x[4] : x[0]), (float)(upper ? x[5] : x[1]), (float)(upper ? x[6] : x[2]), (float)(upper ? x[7] : x[3])});
    }
    if (!a.v) return;
    __syncthreads();
    if (live)
        put(a.v + (first_row + slot - base) * a.v_stride + head * HD + c * 4u, *reinterpret_cast<const f4 *>(&vrows[r * VROW + c * 4u]));
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
// Weights are taken as 2^(s - m), of a score s and the row's reference m. m moves to kRaise below
// a score that exceeds it by more than kMost: a weight is then at most 2^15, within f16, and the
// largest score's at least about 2^kRaise, so that the low f16 terms of lesser ones stay normal.
constexpr float kMost = 15.0f, kRaise = 7.0f;

constexpr uint32_t kMaxSplits = 256;

struct AttnArgs {
    Kv4Attn a;
    uint32_t group, rows, tiles;     // query heads a KV head, rows (tokens x group), tiles of them
    uint32_t by_group;               // 2^32 / group, rounded up; 0 where group is 1
    uint32_t tile_rows, splits, per; // rows of a tile, key splits of the grid, blocks of one
    bool eager;                      // a wave's first block is fetched before it is known whether slots fill it
    float *ml, *acc;                 // [unit][split][tile rows][2], [..][tile rows][HD]
    f2 *norm;                        // [sequence x KV head][rows]: see norm_of; left where weights are wanted
    // for the weights of prompts: the query rows as operands [sequence x KV head][16 rows][HD / 32][hi, lo][64],
    // the factors of their scores [sequence x KV head][rows], sums by row split [split][sequence x KV head][slots]
    h8 *qp;
    float *factors, *sums;
    uint32_t qtiles, row_splits, slots32;
};

// The token of a row. The product with 2^32 / group rounded up is exact for rows below 2^22
// and groups up to 2^10: it is over by less than 2^22 2^10 / 2^32 / group.
__device__ __forceinline__ uint32_t token_of(const AttnArgs &p, uint32_t row) {
    return p.by_group ? __umulhi(row, p.by_group) : row;
}

// Keys of a tile: all that its last row attends to. A split is `per` blocks
// whatever the sequence's length: sequences of unequal length then make splits of equal work.
struct Span {
    uint32_t base, keys, blocks, active;   // slots filled ahead of the call; blocks and splits of the tile
};
__device__ __forceinline__ Span span_of(const AttnArgs &p, uint32_t seq, uint32_t last_row) {
    Span s;
    s.base = p.a.slots[seq];
    s.keys = s.base >= p.a.g.context ? 0u : min(s.base + token_of(p, last_row) + 1u, p.a.g.context);
    s.blocks = (s.keys + 31u) / 32u;
    s.active = (s.blocks + p.per - 1u) / p.per;
    return s;
}

__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Over the four lanes l, l + 16, l + 32, l + 48 that share a query row: v_permlane16_swap
// and v_permlane32_swap put both partners' values into every lane.
__device__ __forceinline__ float row_max(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    u = __builtin_bit_cast(uint32_t, v);
    const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)t[0]), __builtin_bit_cast(float, (uint32_t)t[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    u = __builtin_bit_cast(uint32_t, v);
    const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)t[0]) + __builtin_bit_cast(float, (uint32_t)t[1]);
}

// A row's scale: below 2^10, the low f16 term of a value down to 2^-13 of the row's largest
// is still normal. The exponent of its largest magnitude; 0 where that is 0 or not finite.
__device__ __forceinline__ int scale_of(float top) {
    return top > 0.f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -100) : 0;
}
// Eight values times `up`, rounded to f32, as two f16 terms. The compiler must not see that v is a
// product: it makes hi of it once in one rounding (v_fma_mixlo_f16) and once in two, and where
// those differ, one value in 2^13, the low term belongs to another high one.
__device__ __forceinline__ void split8(const float *x, float up, h8 &hi, h8 &lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = x[i] * up;
        asm("" : "+v"(v));
        hi[i] = (_Float16)v;
        lo[i] = (_Float16)(v - (float)hi[i]);
    }
}
// Eight weights as two f16 terms; `minus` is -1 that the compiler cannot see, so that v - hi
// is one v_fma_mix_f32.
__device__ __forceinline__ void two_terms(const float *v, float minus, h8 &hi, h8 &lo) {
    h2 h[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = __builtin_convertvector((f2{v[2 * e], v[2 * e + 1]}), h2);
        r[e] = __builtin_convertvector((f2{__builtin_fmaf(minus, (float)h[e][0], v[2 * e]),
                                           __builtin_fmaf(minus, (float)h[e][1], v[2 * e + 1])}), h2);
    }
    hi = join8(h);
    lo = join8(r);
}

// What gives a row's softmax weight of a score s: 2^(s - m) / sum. Kept as the two, not as the
// logarithm of one number: that rounds to 2^-21 at the usual 8 to 16, v_log_f32 errs to one side
// by as much, and every weight of the row was 3e-7 to 6e-7 too large by it. A row that is NaN has
// that in m, so that a score of -inf still weighs nothing. The reciprocal is v_rcp_f32's, one
// step nearer (Newton): within 2^-24 as a division, which takes ten instructions.
__device__ __forceinline__ f2 norm_of(float m, float sum) {
    const float r = __builtin_amdgcn_rcpf(sum);
    return sum == sum ? f2{m, __builtin_fmaf(__builtin_fmaf(-sum, r, 1.0f), r, r)} : f2{__builtin_nanf(""), 1.0f};
}

// Sixteen query rows as the B operand: lane (i, q) holds row i, dimensions q HD / 4 + 8 u
// + 0..7 in step u; split() makes two f16 terms of the row, with log2(e) / sqrt(HD) in it and
// scaled, and returns the scale that is left to the scores. It is a power of two: products with it
// are exact, so that a score less the reference, an fma, is what it would be of rounded scores.
// (With the constant in the factor, large scores exceeded their own maximum by their rounding:
// from 2^28 on weights were infinite.)
template <int HD>
struct QRow {
    static constexpr int U = HD / 32;
    float x[U][8];
    __device__ __forceinline__ void load(const AttnArgs &p, uint32_t s, uint32_t head, uint32_t row, bool valid, uint32_t q) {
        const uint32_t t = token_of(p, row), j = row - t * p.group;
        const float *src = p.a.q + ((size_t)s * p.a.tokens + t) * p.a.q_stride + (size_t)(head * p.group + j) * HD + q * (HD / 4);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (valid) {
                load8(src + 8 * u, p.a.qvec, x[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
            }
        }
    }
    __device__ __forceinline__ float split(h8 *qh, h8 *ql) const {
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[u][i]));
        constexpr float c = kLog2e / (HD == 64 ? 8.0f : HD == 128 ? 11.3137085f : 16.0f);
        const int e = scale_of(row_max(top) * c);
        const float up = ldexpf(c, 10 - e);
#pragma unroll
        for (int u = 0; u < U; ++u) split8(x[u], up, qh[u], ql[u]);
        return ldexpf(1.0f, e - 10);
    }
};

// A lane's share of a block of K: for both of the product's row tiles tt, the codes of
// slot 8 (i / 4) + 4 tt + i % 4 in dimensions q HD / 4.. and their (d, o). Lane (i, q) of
// the product S^T then holds the scores of query row i and slots 8 q + 4 tt + r: eight
// consecutive ones.
template <int HD>
struct KFrag {
    static constexpr int U = HD / 32, SC = HD == 256 ? 2 : 1;
    uint32_t code[2][U], scale[2][SC];
    __device__ __forceinline__ void load(const uint8_t *kb, uint32_t i, uint32_t q) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const uint32_t slot = 8u * (i / 4u) + 4u * tt + i % 4u;
            __builtin_memcpy(code[tt], __builtin_assume_aligned(kb + slot * (HD / 2) + q * (HD / 8), HD == 64 ? 8 : 16), 4 * U);
            const uint32_t g = HD == 64 ? q / 2u : q * (HD / 128);
            __builtin_memcpy(scale[tt], __builtin_assume_aligned(kb + Lay<HD>::CODES + (slot * Lay<HD>::G + g) * 4u, 4 * SC), 4 * SC);
        }
    }
    __device__ __forceinline__ h8 value(const Masks &k, int tt, int u) const {
        const h2 p = __builtin_bit_cast(h2, scale[tt][u / 4]);
        return values8(k, code[tt][u], h2{p[0], p[0]}, h2{p[1], p[1]});
    }
};
// A lane's share of a block of V^T: octet q, dimensions 32 g + 16 h + i, and the (d, o) of
// the octet's slots in group g.
template <int HD>
struct VFrag {
    static constexpr int G = HD / 32;
    uint32_t code[2][G];
    __device__ __forceinline__ void load(const uint8_t *vb, uint32_t i, uint32_t q) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            __builtin_memcpy(code[h], __builtin_assume_aligned(vb + (q * 32u + 16u * h + i) * (4u * G), HD == 64 ? 8 : 16), 4 * G);
    }
};
struct VScale {
    h8 d, o;
    template <int HD>
    __device__ __forceinline__ void load(const uint8_t *vb, int g, uint32_t q) {
        const h8 *const sc = reinterpret_cast<const h8 *>(vb + Lay<HD>::CODES) + (q * Lay<HD>::G + g) * 2u;
        d = sc[0];
        o = sc[1];
    }
    // Slots from `some` on may hold anything: their values count as zero. A NaN offset becomes
    // the least one, unless that is NaN.
    __device__ __forceinline__ void keep(uint32_t some, _Float16 least) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            d[e] = (uint32_t)e < some ? d[e] : 0.f16;
            o[e] = (uint32_t)e < some ? o[e] : 0.f16;
        }
        d = __builtin_elementwise_max(d, (h8)(0.f16));
        o = __builtin_elementwise_max(o, (h8)(least));
    }
};

// One workgroup: a tile of 16 NT query rows (tokens x the KV head's query heads) of a
// sequence over one split of its blocks, which the waves take in turn, each with its own
// running maximum and sum; they join in LDS. A tile with one split in use is finished
// here, the others' partial sums go to scratch. A block's values are made once and meet
// all NT column tiles, whose query rows lie in LDS in the order of the operand (NT 1: in
// registers).
// PK, of at most eight rows: columns 0..7 of the products take the high terms of the rows,
// columns 8..15 the low ones, so that one product does for both; the scores of the two
// columns of a row are added, and so are its sums at the end.
// What bounds it (times of calls back to back, at the clock that the card then keeps; out of idle
// it is lower for the first hundred calls, which take a tenth longer; 16/2 heads of 128). For few
// rows over a short context, the instructions of one pass through the kernel at one wave a SIMD
// (4.2 us for a single block; 7.1 for 512 slots in one split). For few rows over a long one neither
// memory nor the VALU that makes the values is used up: 16 sequences over 32768 slots, 111 MB, take
// 34 us, 3.3 TB/s where reads reach 6.0, or 29 out of the last-level cache, with 0.62 of the VALU's
// issue slots at 3.4 waves a SIMD; a block's V is asked for at the block's start. For prompts, the
// issue of vector instructions: 1024 tokens over 8024 slots take 126 us, 1010 TFLOP/s of two-term
// products (a plain f16 product of 8192^3 on that card: 1056), in which products take 0.52 and the other vector
// instructions 0.47 of the SIMDs' cycles; with 1900 tokens (48 us) it is 0.29 and 0.44, the rest
// going to the start of each of 476 tiles and to its waves' wait and join, while nothing else is on
// the CU. Heads of 256 with one column tile of rows take 258 registers and more, one wave a SIMD
// (a token over 8001 slots of one KV head: 10 us); two have not been tried.
template <int HD, int NT, int W, bool PK>
__global__ __launch_bounds__(64 * W, NT > 1 || HD > 128 ? 1 : PK ? 4 : 3) void k_kv4_attn(AttnArgs p) {
    using L = Lay<HD>;
    constexpr int U = HD / 32, DT = HD / 16, OROW = HD + 4, R = 16 * NT, RT = PK ? 8 : R, B = W > 4 || NT > 2 ? W / 2 : W;
    constexpr int QLDS = NT > 1 ? R * HD : 0;   // floats: two f16 planes
    constexpr int LDS = B * R * OROW > QLDS ? B * R * OROW : QLDS;
    __shared__ __attribute__((aligned(16))) float lds[LDS];
    static_assert((!PK || NT == 1) && (W == 4 || W == 8), "one column tile of both terms; a wave or two a SIMD");
    __shared__ float ms[W][R], ls[W][R], fs[R];
    __shared__ uint32_t nan_at[W][L::G], nan_first[L::G];   // by groups, the first slot at the edge whose V is NaN
    const uint32_t tid = threadIdx.x, lane = tid & 63u, i = lane & 15u, q = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (lane < L::G) nan_at[w][lane] = ~0u;   // a wave's LDS accesses keep their order
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    // the tiles with the most keys first
    const uint32_t split = blockIdx.x / p.tiles, tile = p.tiles - 1u - blockIdx.x % p.tiles;
    const uint32_t head = blockIdx.y, s = blockIdx.z, seq = p.a.first + s;
    const uint32_t rows = p.rows, r0 = tile * RT, ri = PK ? i & 7u : i;
    const uint32_t b0 = split * p.per;
    const size_t plane = plane_of(p.a.g, p.a.layer, seq, head) * plane_bytes<HD>(p.a.g);
    const uint8_t *const kp = p.a.kc + plane, *const vp = p.a.vc + plane;
    KFrag<HD> kf;
    uint32_t b = b0 + w;
    auto load_first = [&](uint32_t end) {
        if (b < end) kf.load(kp + (size_t)b * L::BLOCK, i, q);
    };
    if (p.eager) load_first(min(b0 + p.per, (p.a.g.context + 31u) / 32u));
    QRow<HD> qr;
    if constexpr (NT == 1) qr.load(p, s, head, min(r0 + ri, rows - 1u), r0 + ri < rows, q);
    const Span sp = span_of(p, seq, min(r0 + RT, rows) - 1u);
    if (split != 0 && split >= sp.active) return;
    const uint32_t b1 = min(b0 + p.per, sp.blocks);
    if (!p.eager) load_first(b1);
    h8 qh[U], ql[U];
    float factor[NT];
    h8 *const qs = reinterpret_cast<h8 *>(lds);   // [NT][U][hi, lo][64]
    // The weights' kernel reads the operands again: a half of one of its tiles.
    auto leave = [&](uint32_t half, uint32_t row, float f) {
        const size_t pair = (size_t)s * p.a.g.kv_heads + head;
        h8 *const to = p.qp + (pair * p.qtiles * 2u + half) * U * 128u + lane;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            to[u * 128u] = qh[u];
            to[u * 128u + 64u] = ql[u];
        }
        if (q == 0 && row < rows) p.factors[pair * rows + row] = f;
    };
    if constexpr (NT == 1) {
        factor[0] = qr.split(qh, ql);
        if constexpr (PK) {
#pragma unroll
            for (int u = 0; u < U; ++u) qh[u] = i < 8u ? qh[u] : ql[u];
        } else if (p.qp && split == 0 && w == 0) {
            leave(tile, r0 + i, factor[0]);
        }
    } else {
        for (uint32_t c = w; c < NT; c += W) {
            const uint32_t row = r0 + 16u * c + i;
            qr.load(p, s, head, min(row, rows - 1u), row < rows, q);
            const float f = qr.split(qh, ql);
            if (q == 0) fs[16u * c + i] = f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                qs[((c * U + u) * 2u) * 64u + lane] = qh[u];
                qs[((c * U + u) * 2u + 1u) * 64u + lane] = ql[u];
            }
            if (p.qp && split == 0) leave(tile * NT + c, row, f);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NT; ++c) factor[c] = fs[16 * c + i];
    }
    // last slot that the lane's row of a column tile attends to
    auto limit = [&](int c) { return sp.base + token_of(p, min(r0 + 16u * c + ri, rows - 1u)); };
    const uint32_t sees_all = sp.base + token_of(p, r0);   // last slot that every row attends to

    float m[NT], l[NT];
    f4 o[NT][DT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        m[c] = -INFINITY;
        l[c] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[c][dt] = f4{0.f, 0.f, 0.f, 0.f};
    }

    const Masks masks;
    float minus = PK && i < 8u ? 0.0f : -1.0f;
    asm("" : "+v"(minus));
    // 0 x NaN would reach rows that do not attend to the NaN's slot. Tiles of several columns
    // are taken to have such rows, a constant for them: NT 4 with heads of 128 has every register
    // in use and three spilled, more of them without it.
    const bool partly = NT > 1 || sees_all + 1u < sp.keys;
    const _Float16 least = partly ? (_Float16)-kLimit : (_Float16)__builtin_nanf("");
    // A block; at the tile's edge, some row's last slots or the cache's.
    auto step = [&](auto at_edge) {
        constexpr bool edge = decltype(at_edge)::value;
        const uint8_t *const vb = vp + (size_t)b * L::BLOCK;
        VFrag<HD> vf;
        vf.load(vb, i, q);
        f4 x[NT][2];
#pragma unroll
        for (int c = 0; c < NT; ++c) x[c][0] = x[c][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const h8 k0 = kf.value(masks, 0, u), k1 = kf.value(masks, 1, u);
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const h8 hi = NT == 1 ? qh[u] : qs[((c * U + u) * 2u) * 64u + lane];
                const h8 lo = NT == 1 ? ql[u] : qs[((c * U + u) * 2u + 1u) * 64u + lane];
                x[c][0] = mfma16(k0, hi, x[c][0]);
                x[c][1] = mfma16(k1, hi, x[c][1]);
                if constexpr (!PK) {
                    x[c][0] = mfma16(k0, lo, x[c][0]);
                    x[c][1] = mfma16(k1, lo, x[c][1]);
                }
            }
        }
        if (b + W < b1) kf.load(kp + (size_t)(b + W) * L::BLOCK, i, q);
        VScale sc[2];
        sc[0].template load<HD>(vb, 0, q);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t slot0 = b * 32u + 8u * q;
        if constexpr (PK) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[0][e / 4][e % 4] += dpp<0x128>(x[0][e / 4][e % 4]);   // row_ror:8
        }
        if constexpr (edge) {
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const uint32_t last = limit(c);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c][e / 4][e % 4] = slot0 + e > last ? -INFINITY : x[c][e / 4][e % 4];
            }
        }
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
                const float t = row_max(top[c]), mn = t - m[c] > kMost ? t - kRaise : m[c];
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
            // A row that attends to nothing of the blocks so far has no reference yet; any serves.
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
        const uint32_t some = min(max(sp.keys, slot0) - slot0, 8u);
#pragma unroll
        for (int g = 0; g < L::G; ++g) {
            VScale &dc = sc[g % 2];
            if (g + 1 < L::G) sc[(g + 1) % 2].template load<HD>(vb, g + 1, q);
            if constexpr (edge) {
                dc.keep(some, least);
                __builtin_amdgcn_sched_barrier(0);   // without it the groups' selects mix, and registers spill
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const h8 v = values8(masks, vf.code[h][g], dc.d, dc.o);
#pragma unroll
                for (int c = 0; c < NT; ++c) o[c][2 * g + h] = mfma16(v, PK ? pl[c] : ph[c], o[c][2 * g + h]);
                if constexpr (!PK) {
#pragma unroll
                    for (int c = 0; c < NT; ++c) o[c][2 * g + h] = mfma16(v, pl[c], o[c][2 * g + h]);
                }
            }
        }
    };
    const uint32_t whole = min(b1, (sees_all + 1u) / 32u);   // blocks that every row attends to all of
    for (; b < whole; b += W) {
        // The older of a SIMD's two waves is served first and is done early, the other then runs
        // alone. Taking precedence in turns they end together: hd 64 and 256 3%, 128 1%.
        if (NT > 1 && b1 - b0 >= 32u) {
            if ((b / W ^ w / 4u) & 1u)
                __builtin_amdgcn_s_setprio(1);
            else
                __builtin_amdgcn_s_setprio(0);
        }
        step(std::false_type{});
    }
    if constexpr (NT > 1) __builtin_amdgcn_s_setprio(0);
    const uint32_t b_edge = b;
    while (b < b1) step(std::true_type{}), b += W;
    // Blocks at the edge took a NaN in V as finite. The first such slot is noted here: the rows
    // that attend to it have NaN in the group's dimensions.
    if (partly) {
        for (b = b_edge; b < b1; b += W) {
            const uint32_t slot0 = b * 32u + 8u * q;
#pragma unroll 1
            for (int g = 0; g < L::G; ++g) {
                VScale sc;
                sc.template load<HD>(vp + (size_t)b * L::BLOCK, g, q);
                uint32_t at = ~0u;
#pragma unroll
                for (int e = 7; e >= 0; --e) at = sc.o[e] != sc.o[e] ? slot0 + e : at;
                if (i == 0 && at < sp.keys) atomicMin(&nan_at[w][g], at);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        l[c] = row_sum(l[c]);
        if (q == 0) ms[w][16 * c + i] = m[c], ls[w][16 * c + i] = l[c];
    }
    __syncthreads();   // the queries in LDS have been read, every wave's m and l are there

    // A wave's sums are taken to the row's largest reference. One without keys has nothing
    // to give; one whose every score is NaN has no reference but a NaN sum.
    constexpr int PART = W > B ? R / 2 : R;   // rows of a wave's part
    auto *const os = reinterpret_cast<float (*)[PART][OROW]>(lds);
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
            sum[c] += mv[v] == -INFINITY ? lv[v] : lv[v] * __builtin_amdgcn_exp2f(mv[v] - top[c]);
        sum[c] = row_sum(sum[c]);
        const float mine = m[c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[c] - top[c]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[c][dt] *= mine;
    }
    if constexpr (W > B) {
        // Waves w and w + 4 exchange halves of their tiles, so that all write and read: each adds
        // the partner's half to its own, in the partner's part of LDS.
        constexpr int H = NT / 2;
        auto give = [&](auto upper) {
#pragma unroll
            for (int c = 0; c < H; ++c)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    *reinterpret_cast<f4 *>(&os[w][16 * c + i][16 * dt + 4 * q]) = o[decltype(upper)::value ? c : H + c][dt];
        };
        auto take = [&](auto upper) {
#pragma unroll
            for (int c = 0; c < H; ++c)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    f4 *const at = reinterpret_cast<f4 *>(&os[w ^ B][16 * c + i][16 * dt + 4 * q]);
                    *at = *at + o[decltype(upper)::value ? H + c : c][dt];
                }
        };
        if (w < B)
            give(std::false_type{});
        else
            give(std::true_type{});
        __syncthreads();
        if (w < B)
            take(std::false_type{});
        else
            take(std::true_type{});
    } else {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4 *>(&os[w][16 * c + i][16 * dt + 4 * q]) = o[c][dt];
    }
    const size_t unit = ((size_t)s * p.a.g.kv_heads + head) * p.tiles + tile, part = unit * p.splits + split;
    const bool alone = sp.active <= 1u;
    if (w == 0 && q == 0) {   // the factors of the scores have been read, a barrier ago and more
#pragma unroll
        for (int c = 0; c < NT; ++c) fs[16 * c + i] = sum[c];
    }
    if (tid < L::G) {
        uint32_t at = nan_at[0][tid];
#pragma unroll
        for (int v = 1; v < W; ++v) at = min(at, nan_at[v][tid]);
        nan_first[tid] = at;
    }
    if (w == 0 && q == 0) {
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const uint32_t row = r0 + 16u * c + i;
            if (row >= rows || (PK && i >= 8u)) continue;
            if (alone) {
                if (p.a.weights) p.norm[((size_t)s * p.a.g.kv_heads + head) * rows + row] = norm_of(top[c], sum[c]);
            } else {
                p.ml[(part * RT + 16u * c + i) * 2u] = top[c];
                p.ml[(part * RT + 16u * c + i) * 2u + 1u] = sum[c];
            }
        }
    }
    __syncthreads();
    constexpr int V = HD / 4;   // four dimensions a lane
    for (uint32_t k = tid; k < (uint32_t)RT * V; k += 64u * W) {
        const uint32_t r = k / V, c = 4u * (k % V), row = r0 + r;
        if (row >= rows) break;
        const uint32_t u0 = W > B && r < (uint32_t)PART ? B : 0u, at = r % (uint32_t)PART;   // a half's sums: in the other's parts
        f4 v = *reinterpret_cast<const f4 *>(&os[u0][at][c]);
#pragma unroll
        for (int u = 1; u < B; ++u) v += *reinterpret_cast<const f4 *>(&os[u0 + u][at][c]);
        if constexpr (PK) {
#pragma unroll
            for (int u = 0; u < B; ++u) v += *reinterpret_cast<const f4 *>(&os[u][r + 8u][c]);
        }
        const uint32_t t = token_of(p, row), j = row - t * p.group;
        if (nan_first[c / 32u] <= sp.base + t) v = v * __builtin_nanf("");
        if (!alone) {
            *reinterpret_cast<f4 *>(p.acc + (part * RT + r) * HD + c) = v;
            continue;
        }
        const bool attends = sp.base < p.a.g.context && sp.base + t < p.a.g.context;
        v = attends ? v * (1.0f / fs[r]) : f4{0.f, 0.f, 0.f, 0.f};
        float *const to = p.a.out + ((size_t)s * p.a.tokens + t) * p.a.out_stride + (size_t)(head * p.group + j) * HD + c;
        if (p.a.ovec) {
            *reinterpret_cast<f4 *>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = v[e];
        }
    }
}

// The weight of a slot from its rows' sum: added to what it had, unless the call's own
// tokens fill it or nothing is kept.
__device__ __forceinline__ void add_weight(float *to, uint32_t slot, uint32_t base, float decay, float v) {
    to[slot] = slot >= base || decay == 0.f ? v : decay * to[slot] + v;
}

// A lane's sum over the 16 lanes of its DPP row: quads, half rows, rows.
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0xb1>(v);
    v += dpp<0x4e>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}

// A barrier for what lies in LDS: __syncthreads waits for every global load too, which here
// are on their way for a later turn.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The splits of a row, joined: a workgroup a row, its lanes HD / 4 columns by as many
// splits at once as fit.
constexpr uint32_t kFewSplits = 8;
template <int HD>
__device__ __forceinline__ void join_row(const AttnArgs &p, uint32_t row, uint32_t head, uint32_t s) {
    constexpr int V = HD / 4, Y = 256 / V;
    __shared__ float sc[kMaxSplits], red[8];
    __shared__ __attribute__((aligned(16))) float os[Y][HD];
    const uint32_t tid = threadIdx.x, seq = p.a.first + s, tile_rows = p.tile_rows;
    const uint32_t tile = row / tile_rows, r = row - tile * tile_rows;
    const size_t unit = ((size_t)s * p.a.g.kv_heads + head) * p.tiles + tile;
    const size_t first = unit * p.splits * tile_rows + r;   // the row's record in split 0
    const uint32_t c = 4u * (tid % V), y = tid / V;
    const Span sp = span_of(p, seq, min((tile + 1u) * tile_rows, p.rows) - 1u);
    if (sp.active <= 1u) return;
    constexpr int E = 8;
    f4 early[E];   // on their way while the splits' weights are worked out
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const uint32_t v = min(y + k * Y, sp.active - 1u);
        early[k] = *reinterpret_cast<const f4 *>(p.acc + (first + (size_t)v * tile_rows) * HD + c);
    }
    float m = -INFINITY, l = 0.f;
    if (tid < sp.active) {
        m = p.ml[(first + (size_t)tid * tile_rows) * 2u];
        l = p.ml[(first + (size_t)tid * tile_rows) * 2u + 1u];
    }
    float top = m;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if ((tid & 63u) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mine = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
    if (tid < sp.active) sc[tid] = mine;
    float sum = l * mine;
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if ((tid & 63u) == 0) red[4 + (tid >> 6)] = sum;
    __syncthreads();
    sum = (red[4] + red[5]) + (red[6] + red[7]);
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < E; ++k)
        if (y + k * Y < sp.active) o += early[k] * sc[y + k * Y];
#pragma unroll 4
    for (uint32_t v = y + E * Y; v < sp.active; v += Y)
        o += *reinterpret_cast<const f4 *>(p.acc + (first + (size_t)v * tile_rows) * HD + c) * sc[v];
    *reinterpret_cast<f4 *>(&os[y][c]) = o;
    __syncthreads();
    const uint32_t t = token_of(p, row), j = row - t * p.group;
    const bool attends = sp.base + t < p.a.g.context;
    if (tid < (uint32_t)HD) {
        float x = os[0][tid];
#pragma unroll
        for (int u = 1; u < Y; ++u) x += os[u][tid];
        p.a.out[((size_t)s * p.a.tokens + t) * p.a.out_stride + (size_t)(head * p.group + j) * HD + tid] = attends ? x / sum : 0.f;
    }
    if (tid == 0 && p.a.weights) p.norm[((size_t)s * p.a.g.kv_heads + head) * p.rows + row] = norm_of(top, sum);
}

// The same of at most kFewSplits splits: HD / 4 lanes a row, whose splits they fetch at once,
// before it is known which are in use.
template <int HD>
__device__ __forceinline__ void join_rows(const AttnArgs &p, uint32_t group, uint32_t head, uint32_t s) {
    constexpr uint32_t V = HD / 4, Y = 256 / V;
    const uint32_t row = group * Y + threadIdx.x / V, c = 4u * (threadIdx.x % V), seq = p.a.first + s;
    if (row >= p.rows) return;
    const uint32_t tile = row / p.tile_rows, r = row - tile * p.tile_rows;
    const size_t pair = (size_t)s * p.a.g.kv_heads + head;
    const size_t first = (pair * p.tiles + tile) * p.splits * p.tile_rows + r;
    f4 part[kFewSplits];
    f2 ml[kFewSplits];
#pragma unroll
    for (uint32_t v = 0; v < kFewSplits; ++v)
        if (v < p.splits) {
            part[v] = *reinterpret_cast<const f4 *>(p.acc + (first + (size_t)v * p.tile_rows) * HD + c);
            ml[v] = *reinterpret_cast<const f2 *>(p.ml + (first + (size_t)v * p.tile_rows) * 2u);
        }
    const Span sp = span_of(p, seq, min((tile + 1u) * p.tile_rows, p.rows) - 1u);
    if (sp.active <= 1u) return;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (uint32_t v = 0; v < kFewSplits; ++v)
        if (v < sp.active) top = fmaxf(top, ml[v][0]);
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t v = 0; v < kFewSplits; ++v)
        if (v < sp.active) {
            const float scale = ml[v][0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[v][0] - top);
            sum += ml[v][1] * scale;
            o += part[v] * scale;
        }
    const uint32_t t = token_of(p, row), j = row - t * p.group;
    o = sp.base + t < p.a.g.context ? o * (1.0f / sum) : f4{0.f, 0.f, 0.f, 0.f};
    float *const to = p.a.out + ((size_t)s * p.a.tokens + t) * p.a.out_stride + (size_t)(head * p.group + j) * HD + c;
    if (p.a.ovec) {
        *reinterpret_cast<f4 *>(to) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = o[e];
    }
    if (c == 0 && p.a.weights) p.norm[pair * p.rows + row] = norm_of(top, sum);
}

// Accumulated weights of at most 16 rows: a wave per block of 32 slots takes the scores
// again, and sums their weights over the rows; a row's splits are joined here too, so that it
// need not wait for join_row.
template <int HD>
__device__ __forceinline__ void weigh(const AttnArgs &p, uint32_t group, uint32_t head, uint32_t s) {
    using L = Lay<HD>;
    constexpr int U = HD / 32;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, i = lane & 15u, q = lane >> 4, seq = p.a.first + s;
    const uint32_t b = group * 4u + __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t row = min(i, p.rows - 1u), t = token_of(p, row);
    const Span sp = span_of(p, seq, p.rows - 1u);   // one tile
    if (sp.base >= p.a.g.context || b >= sp.blocks) return;
    const size_t plane = plane_of(p.a.g, p.a.layer, seq, head), pair = (size_t)s * p.a.g.kv_heads + head;
    const Masks masks;
    KFrag<HD> kf;
    kf.load(p.a.kc + plane * plane_bytes<HD>(p.a.g) + (size_t)b * L::BLOCK, i, q);
    QRow<HD> qr;
    qr.load(p, s, head, row, true, q);
    // Lane (i, q), i < 8, stores the weight of slot 8 q + i.
    const uint32_t slot0 = b * 32u + 8u * q, mine = slot0 + (i & 7u);
    float *const to = p.a.weights + plane * p.a.g.context + mine;
    const bool stores = i < 8u && mine < sp.keys, adds = mine < sp.base && p.a.decay != 0.f;
    const float had = stores && adds ? *to : 0.f;
    f2 norm;
    if (sp.active <= 1u) {
        norm = p.norm[pair * p.rows + row];
    } else {
        // a lane's splits 16 at a time, so that their loads wait once
        float m = -INFINITY, l = 0.f;
        for (uint32_t v0 = q; v0 < sp.active; v0 += 64u) {
            f2 ml[16];
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k) {
                const uint32_t v = min(v0 + 4u * k, sp.active - 1u);
                ml[k] = *reinterpret_cast<const f2 *>(p.ml + ((pair * p.splits + v) * p.tile_rows + row) * 2u);
            }
            float top = m;
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k) {
                if (v0 + 4u * k >= sp.active) ml[k] = f2{-INFINITY, 0.f};
                top = fmaxf(top, ml[k][0]);
            }
            if (m != -INFINITY) l *= __builtin_amdgcn_exp2f(m - top);
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k)
                l += ml[k][0] == -INFINITY ? ml[k][1] : ml[k][1] * __builtin_amdgcn_exp2f(ml[k][0] - top);
            m = top;
        }
        const float top = row_max(m);
        norm = norm_of(top, row_sum(m == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - top)));
    }
    h8 qh[U], ql[U];
    const float factor = qr.split(qh, ql);
    const bool valid = i < p.rows && sp.base + t < p.a.g.context;
    // The scores to the bit: of up to eight rows the terms' products are summed apart (PK).
    f4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, y[2] = {x[0], x[1]};
    auto scores = [&](f4 *low) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const h8 k0 = kf.value(masks, 0, u), k1 = kf.value(masks, 1, u);
            x[0] = mfma16(k0, qh[u], x[0]);
            x[1] = mfma16(k1, qh[u], x[1]);
            low[0] = mfma16(k0, ql[u], low[0]);
            low[1] = mfma16(k1, ql[u], low[1]);
        }
    };
    if (p.rows <= 8u) {
        scores(y);
        x[0] += y[0], x[1] += y[1];
    } else {
        scores(x);
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool sees = valid && slot0 + e <= sp.base + t;
        const float v = sum16(sees ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[e / 4][e % 4], factor, -norm[0])) * norm[1] : 0.f);
        sum = i == (uint32_t)e ? v : sum;
    }
    if (stores) *to = adds ? p.a.decay * had + sum : sum;
}

// What follows the attention kernel, in one launch: workgroups 0..joins-1 join rows' splits,
// the others the weights of 128 slots each. Bound by launch and latency: 2.7 us (224 rows of 8
// splits), 4.7 (256 rows of 48), 4.8 with the weights of 8192 slots (as two launches 9.1).
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_finish(AttnArgs p, uint32_t joins) {
    if (blockIdx.x < joins) {
        if (p.splits <= kFewSplits)
            join_rows<HD>(p, blockIdx.x, blockIdx.y, blockIdx.z);
        else
            join_row<HD>(p, blockIdx.x, blockIdx.y, blockIdx.z);
    } else {
        weigh<HD>(p, blockIdx.x - joins, blockIdx.y, blockIdx.z);
    }
}

// Weights of more rows, from the scores once more: the sum over rows needs each row's final
// sum. The products are those of k_kv4_attn, operands and order alike, so that the scores are the
// very ones that the sum was made of: large ones round by more than their weights allow. A
// workgroup takes 256 slots, 64 a wave, whose values it makes once and keeps in registers, over
// every row_splits-th tile of 32 rows. The tiles' operands, left by the attention kernel, pass
// through LDS, the next on its way while one is multiplied. A lane sums its slots over its two
// rows of each tile; the sums over the row splits are added by k_kv4_add_weights, in order, so
// that they do not vary. Bound by the issue of vector instructions: 1024 tokens over 8024 slots
// take 57 us, 1115 TFLOP/s of products, in 0.59 of the SIMDs' cycles, the others taking 0.33.
template <int HD>
__global__ __launch_bounds__(256, 2) void k_kv4_weights_rows(AttnArgs p) {
    using L = Lay<HD>;
    constexpr int U = HD / 32, TILE = U * 256, PER = TILE / 256;   // h8 of a tile; a lane's share
    __shared__ __attribute__((aligned(16))) h8 qs[2][TILE];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, i = lane & 15u, q = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t chunk = blockIdx.x / p.row_splits, part = blockIdx.x % p.row_splits;
    const uint32_t head = blockIdx.y, s = blockIdx.z, seq = p.a.first + s;
    const uint32_t base = p.a.slots[seq];
    if (base >= p.a.g.context) return;
    const uint32_t keys = min(base + p.a.tokens, p.a.g.context);
    if (chunk * 256u >= keys) return;
    const size_t pair = (size_t)s * p.a.g.kv_heads + head;
    const uint32_t b0 = chunk * 8u + 2u * w, blocks = (keys + 31u) / 32u;
    const uint8_t *const kp = p.a.kc + plane_of(p.a.g, p.a.layer, seq, head) * plane_bytes<HD>(p.a.g);
    h8 k[2][2][U];   // of the wave's blocks; one behind the last: not stored below
    {
        const Masks masks;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            KFrag<HD> kf;
            kf.load(kp + (size_t)min(b0 + v, blocks - 1u) * L::BLOCK, i, q);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int u = 0; u < U; ++u) k[v][tt][u] = kf.value(masks, tt, u);
        }
    }
    // row tiles from the first that attends to a slot of the chunk
    const uint32_t t0 = chunk * 256u > base ? chunk * 256u - base : 0u;
    const uint32_t live = (keys - base) * p.group;   // rows whose slots the context holds; the others hold anything
    const uint32_t tiles = (live + 31u) / 32u;
    uint32_t tile = t0 * p.group / 32u + part;
    const h8 *const src = p.qp + pair * p.qtiles * TILE;
    const float *const factors = p.factors + pair * p.rows;
    const f2 *const norms = p.norm + pair * p.rows;
    h8 next[PER];
    float sum[2][8];   // of slots 8 q + e of the wave's blocks
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[0][e] = sum[1][e] = 0.f;
    auto fetch = [&](uint32_t from) {
#pragma unroll
        for (int n = 0; n < PER; ++n) next[n] = src[(size_t)from * TILE + n * 256u + tid];
    };
    if (tile < tiles) fetch(tile);
    for (uint32_t turn = 0; tile < tiles; tile += p.row_splits, turn ^= 1u) {
        // A buffer is written two turns after it was last read, with a barrier between.
#pragma unroll
        for (int n = 0; n < PER; ++n) qs[turn][n * 256u + tid] = next[n];
        if (tile + p.row_splits < tiles) fetch(tile + p.row_splits);
        uint32_t end[2];   // of the slots that the lane's rows attend to
        float factor[2];
        f2 norm[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t row = tile * 32u + 16u * c + i, at = min(row, live - 1u);
            end[c] = row < live ? base + token_of(p, row) + 1u : 0u;
            factor[c] = factors[at];
            norm[c] = norms[at];
        }
        const bool edge = (b0 + 2u) * 32u > base + token_of(p, tile * 32u) + 1u || tile * 32u + 32u > live;
        lds_barrier();
        const h8 *const from = qs[turn] + lane;
        f4 x[2][2][2];   // [column tile][block][row tile]
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int v = 0; v < 2; ++v) x[c][v][0] = x[c][v][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int term = 0; term < 2; ++term) {
                const h8 q0 = from[u * 128 + term * 64], q1 = from[(U + u) * 128 + term * 64];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) {
                        x[0][v][tt] = mfma16(k[v][tt][u], q0, x[0][v][tt]);
                        x[1][v][tt] = mfma16(k[v][tt][u], q1, x[1][v][tt]);
                    }
            }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[c][v][e / 4][e % 4] = __builtin_fmaf(x[c][v][e / 4][e % 4], factor[c], -norm[c][0]);
        // What a row does not attend to is 2^-inf whatever the row holds.
        if (edge) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[c][v][e / 4][e % 4] = (b0 + v) * 32u + 8u * q + e >= end[c] ? -INFINITY : x[c][v][e / 4][e % 4];
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    sum[v][e] = __builtin_fmaf(__builtin_amdgcn_exp2f(x[c][v][e / 4][e % 4]), norm[c][1], sum[v][e]);
    }
    // Lane (i, q) stores the sum of slot 8 q + i % 8 of block i / 8.
    float mine = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = sum16(sum[v][e]);
            mine = i == (uint32_t)(8 * v + e) ? y : mine;
        }
    const uint32_t slot = (b0 + i / 8u) * 32u + 8u * q + i % 8u;
    if (slot >= keys) return;
    if (p.row_splits > 1u)
        p.sums[((size_t)part * gridDim.y * gridDim.z + pair) * p.slots32 + slot] = mine;
    else
        add_weight(p.a.weights + plane_of(p.a.g, p.a.layer, seq, head) * p.a.g.context, slot, base, p.a.decay, mine);
}

__global__ __launch_bounds__(256) void k_kv4_add_weights(AttnArgs p) {
    const uint32_t slot = blockIdx.x * 256u + threadIdx.x, head = blockIdx.y, s = blockIdx.z, seq = p.a.first + s;
    const uint32_t base = p.a.slots[seq];
    if (base >= p.a.g.context || slot >= min(base + p.a.tokens, p.a.g.context)) return;
    const size_t pair = (size_t)s * p.a.g.kv_heads + head, pairs = (size_t)gridDim.y * gridDim.z;
    float v = 0.f;
    for (uint32_t k = 0; k < p.row_splits; ++k) v += p.sums[(k * pairs + pair) * p.slots32 + slot];
    add_weight(p.a.weights + plane_of(p.a.g, p.a.layer, seq, head) * p.a.g.context, slot, base, p.a.decay, v);
}

// ------------------------------------------------------------------- eviction
// An order of weights as integers: rising, NaN below all, both zeros alike.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, w), b = bits == 0x80000000u ? 0u : bits;
    return w != w ? 0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

constexpr uint32_t kSelect = 1024;                 // lanes of a plane's workgroup
constexpr uint32_t kSelectWaves = kSelect / 64;
constexpr uint32_t kSelectTurns = 16;              // 64 slots of a wave's run that a lane keeps in registers
constexpr uint32_t kBins = 2048, kCopies = 4;

// Over a wave, without LDS: lane l's sum over lanes 0..l (shifts within rows of 16, then the
// last lanes of rows and row pairs broadcast upwards), and the largest, which lane 63 ends up
// with.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += dpp_u32<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
    v += dpp_u32<0x112, 0xf>(v);
    v += dpp_u32<0x114, 0xf>(v);
    v += dpp_u32<0x118, 0xf>(v);
    v += dpp_u32<0x142, 0xa>(v);   // row_bcast 15, 31
    return v + dpp_u32<0x143, 0xc>(v);
}
// Of a value per wave, in lanes 0..15 of each 16: the sum of those before wave w.
__device__ __forceinline__ uint32_t before_wave(uint32_t v, uint32_t w) {
    v += dpp_u32<0x111, 0xf>(v);
    v += dpp_u32<0x112, 0xf>(v);
    v += dpp_u32<0x114, 0xf>(v);
    v += dpp_u32<0x118, 0xf>(v);
    return w ? (uint32_t)__builtin_amdgcn_readlane((int)v, (int)w - 1) : 0u;
}
// n and the lanes of `mask` below this one.
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask, uint32_t n) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, n));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max(v, dpp_u32<0x111, 0xf>(v));
    v = max(v, dpp_u32<0x112, 0xf>(v));
    v = max(v, dpp_u32<0x114, 0xf>(v));
    v = max(v, dpp_u32<0x118, 0xf>(v));
    v = max(v, dpp_u32<0x142, 0xa>(v));
    v = max(v, dpp_u32<0x143, 0xc>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// A workgroup per plane, a wave per run of slots. The keep-th largest order is found 11, 11
// and 10 bits at a time from histograms in LDS. With the waves' counts of orders above the
// threshold and of its equals, S(j), the slots below j that stay, follows; slot j < keep that
// leaves is then the (j - S(j))-th, slot j >= keep that stays the (S(j) - S(keep))-th. A lane
// keeps its slots' orders in registers; of more than 16384 slots it works them out in every
// pass. Four copies of the histogram, by lane: many weights are alike (zero, say), and
// additions to one word take turns. Bound by the latencies of its phases, one workgroup going
// through them all: 56 planes of 8192 slots 9.7 us, 64 of 2049 6.9. Of 32768 slots 61 us (0.3 TB/s
// of the 15 MB): every pass reads both tables anew.
template <bool KEPT>
__global__ __launch_bounds__(kSelect) void k_kv4_select(Kv4Evict a) {
    __shared__ uint32_t part[2][kSelectWaves], found[5];
    __shared__ __attribute__((aligned(16))) uint32_t hist[kBins * kCopies];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t head = blockIdx.x, s = blockIdx.y, layer = blockIdx.z, seq = a.first + s;
    const size_t plane = plane_of(a.g, layer, seq, head);
    const float *const weights = a.weights + plane * a.g.context;
    const uint32_t *const positions = a.slot_positions + plane * a.g.context;
    uint32_t *const plan = a.plan + (((size_t)layer * a.n + s) * a.g.kv_heads + head) * a.moves * 2u;
    const uint32_t had = a.slots[seq], n = had == VX_KV4_NO_SLOT ? 0u : min(had, a.g.context), keep = a.keep;
    // The moves, while `hist` is free again: at most 8192 pairs of slots below 16384.
    uint16_t *const pairs = reinterpret_cast<uint16_t *>(hist);
    uint32_t moved = 0;
    if (n > keep) {
        // Wave w's slots are [run w, run (w + 1)), 64 a turn. Lanes behind the last slot count as
        // slots of the least order: behind every other, they neither stay nor matter to those.
        const uint32_t run = (n + kSelect - 1u) / kSelect * 64u, jw = w * run, j0 = jw + lane;
        const uint32_t turns = jw < n ? (min(run, n - jw) + 63u) / 64u : 0u;
        constexpr uint32_t KEEP = KEPT ? kSelectTurns : 1;
        uint32_t kept[KEEP], newest = 0;
        // Positions that stay whatever they weigh: the first ones, and the last ones
        auto held = [&](uint32_t at) { return (at < a.sinks) | (a.recent > newest) | (at > newest - a.recent); };
        for (uint32_t k = 4u * tid; k < kBins * kCopies; k += 4u * kSelect)
            *reinterpret_cast<uint4 *>(&hist[k]) = make_uint4(0, 0, 0, 0);
        if constexpr (KEPT) {
            float wt[KEEP];
#pragma unroll
            for (uint32_t k = 0; k < KEEP; ++k)
                if (k < turns) {
                    const uint32_t j = min(j0 + 64u * k, n - 1u);
                    kept[k] = positions[j];
                    wt[k] = weights[j];
                }
#pragma unroll
            for (uint32_t k = 0; k < KEEP; ++k)
                if (k < turns) newest = max(newest, kept[k]);
            newest = wave_max_u32(newest);
            if (lane == 0) part[0][w] = newest;
            __syncthreads();
            newest = wave_max_u32(part[0][lane % kSelectWaves]);
#pragma unroll
            for (uint32_t k = 0; k < KEEP; ++k)
                if (k < turns)
                    kept[k] = j0 + 64u * k >= n ? 0u : held(kept[k]) ? 0xFFFFFFFFu : order_of(wt[k]);
        } else {
            for (uint32_t j = tid; j < n; j += kSelect) newest = max(newest, positions[j]);
            newest = wave_max_u32(newest);
            if (lane == 0) part[0][w] = newest;
            __syncthreads();
            newest = wave_max_u32(part[0][lane % kSelectWaves]);
        }
        // f(the turn's first slot, the order of the lane's) for the wave's slots, in order
        auto each = [&](auto f) {
            if constexpr (KEPT) {
#pragma unroll
                for (uint32_t k = 0; k < KEEP; ++k)
                    if (k < turns) f(jw + 64u * k, kept[k]);
            } else {
                for (uint32_t k = 0; k < turns; ++k) {
                    const uint32_t j = j0 + 64u * k, at = j < n ? positions[j] : 0u;
                    f(jw + 64u * k, j >= n ? 0u : held(at) ? 0xFFFFFFFFu : order_of(weights[j]));
                }
            }
        };
        uint32_t prefix = 0, rest = keep;   // the threshold's bits so far, slots still to take among its equals
        constexpr int kShift[3] = {21, 10, 0};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = kShift[pass], known = pass == 0 ? 0 : kShift[pass - 1];
            const uint32_t mask = pass == 2 ? 1023u : 2047u;
            each([&](uint32_t, uint32_t v) {
                if (pass == 0 || v >> known == prefix >> known)
                    atomicAdd(&hist[(v >> shift & mask) * kCopies + (tid & (kCopies - 1u))], 1u);
            });
            __syncthreads();
            // The bin that holds the rest-th from the top: each lane two bins, descending. Eight lanes
            // of sixteen read their second bin first: all of them meet different banks.
            const uint32_t b1 = kBins - 1u - 2u * tid;
            uint4 *const pair = reinterpret_cast<uint4 *>(hist + (b1 - 1u) * kCopies);
            const uint32_t turned = lane >> 3 & 1u;
            uint32_t h0 = 0, h1 = 0;
            if (pass < 2 || b1 < 1024u) {
                const uint4 n0 = pair[turned], n1 = pair[turned ^ 1u];
                h0 = n0.x + n0.y + n0.z + n0.w, h1 = n1.x + n1.y + n1.z + n1.w;
                if (turned) {
                    const uint32_t t = h0;
                    h0 = h1, h1 = t;
                }
                // for the next pass: only this lane reads them
                if (pass == 0 || (pass == 1 && b1 < 1024u)) pair[turned] = pair[turned ^ 1u] = make_uint4(0, 0, 0, 0);
            }
            uint32_t sum = wave_scan(h1 + h0);
            if (lane == 63) part[0][w] = sum;
            __syncthreads();
            sum += before_wave(part[0][lane % kSelectWaves], w);
            const uint32_t before = sum - h1 - h0;   // slots in the bins above this lane's
            if (before < rest && sum >= rest) {
                const bool upper = before + h1 >= rest;
                found[0] = upper ? b1 : b1 - 1u;
                found[1] = upper ? before : before + h1;
            }
            __syncthreads();
            prefix |= __builtin_amdgcn_readfirstlane(found[0]) << shift;
            rest -= __builtin_amdgcn_readfirstlane(found[1]);
        }
        // The waves' counts above the threshold and at it, and what the wave whose run holds slot
        // keep counts below that.
        uint32_t above = 0, ties = 0;
        each([&](uint32_t first, uint32_t v) {
            const uint64_t hb = __ballot(v > prefix), tb = __ballot(v == prefix);
            if (keep - first < 64u) {
                const uint64_t below = (1ull << (keep - first)) - 1u;
                found[2] = above + __popcll(hb & below);
                found[3] = ties + __popcll(tb & below);
                found[4] = w;
            }
            above += __popcll(hb);
            ties += __popcll(tb);
        });
        if (lane == 0) part[0][w] = above, part[1][w] = ties;
        __syncthreads();
        const uint32_t highs = part[0][lane % kSelectWaves], sames = part[1][lane % kSelectWaves];
        const uint32_t of = __builtin_amdgcn_readfirstlane(found[4]);
        const uint32_t low = before_wave(highs, of) + __builtin_amdgcn_readfirstlane(found[2]) +
                             min(before_wave(sames, of) + __builtin_amdgcn_readfirstlane(found[3]), rest);   // S(keep)
        uint32_t same = before_wave(sames, w), stayed = before_wave(highs, w) + min(same, rest);
        each([&](uint32_t first, uint32_t v) {
            uint64_t stay = __ballot(v > prefix);
            const uint64_t tb = __ballot(v == prefix);
            if (same < rest) {   // of the equals, the first ones
                const uint32_t equals = __popcll(tb);
                stay |= same + equals <= rest ? tb : __ballot(v == prefix && lanes_below(tb, same) < rest);
                same += equals;
            }
            const uint32_t j = first + lane, s_of = lanes_below(stay, stayed);
            const bool lower = j < keep, stays = __builtin_amdgcn_inverse_ballot_w64(stay);
            const uint32_t e = lower ? j - s_of : s_of - low, at = 2u * e + (lower ? 1u : 0u);
            if ((lower != stays) & (e < a.moves)) {
                if constexpr (KEPT)
                    pairs[at] = (uint16_t)j;
                else
                    plan[at] = j;
            }
            stayed += __popcll(stay);
        });
        moved = keep - low;
        moved = min(moved, a.moves);
    }
    if constexpr (KEPT) {
        __syncthreads();
#pragma unroll 4
        for (uint32_t k = tid; k < a.moves; k += kSelect) {
            const uint32_t none = VX_KV4_NO_SLOT;
            const uint32_t pair = reinterpret_cast<const uint32_t *>(pairs)[k];
            reinterpret_cast<uint2 *>(plan)[k] = k < moved ? make_uint2(pair & 0xffffu, pair >> 16) : make_uint2(none, none);
        }
    } else {
        for (uint32_t k = 2u * moved + tid; k < 2u * a.moves; k += kSelect) plan[k] = VX_KV4_NO_SLOT;
    }
}

// Moves of a plan, a workgroup of four waves for kMoves of a plane's: the first moves K and
// the tables, the others V; each issues all its reads before its writes. V's codes of an octet
// share dwords, so that the moves into one octet (within eight pairs of the plan, whose
// targets rise) are made by one wave, of the workgroup of the first: a workgroup looks at
// seven pairs before its own and seven behind. Bound by the bytes of V, of
// which a slot has a nibble in head_dim dwords: up to 2048 moves in each of 16 planes of 128, about
// 32 MB read and written, take 9.1 us (3.5 TB/s).
constexpr uint32_t kMoves = 16;

template <int HD>
__global__ __launch_bounds__(256) void k_kv4_compact(Kv4Evict a) {
    using L = Lay<HD>;
    constexpr uint32_t NONE = VX_KV4_NO_SLOT;
    __shared__ uint32_t froms[kMoves + 14], tos[kMoves + 14];   // of pairs e0 - 7 ..; NONE: no move
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t head = blockIdx.y % a.g.kv_heads, s = blockIdx.y / a.g.kv_heads, layer = blockIdx.z, seq = a.first + s;
    if (blockIdx.x == 0 && layer == 0 && head == 0 && tid == 0) {
        const uint32_t n = a.slots[seq];
        if (n != NONE && n > a.keep) a.slots[seq] = a.keep;
    }
    const size_t plane = plane_of(a.g, layer, seq, head);
    const uint32_t *const plan = a.plan_in + (((size_t)layer * a.n + s) * a.g.kv_heads + head) * a.moves * 2u;
    const uint32_t e0 = blockIdx.x * kMoves;
    if (tid < kMoves + 14u) {
        const uint32_t e = e0 + tid - 7u;   // before pair 0: past every move
        uint32_t from = NONE, to = NONE;
        if (e < a.moves) from = plan[2u * e], to = plan[2u * e + 1u];
        const bool fits = from >= a.keep && from < a.g.context && to < a.keep;
        froms[tid] = fits ? from : NONE;
        tos[tid] = fits ? to : NONE;
    }
    __syncthreads();
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (wave == 0) {
        // K: 16 bytes a lane of the codes, a dword of the (d, o)
        constexpr uint32_t C = HD / 32, NC = (kMoves * C + 63u) / 64u;   // lanes a row; turns
        uint8_t *const kp = a.kc + (a.kc ? plane * plane_bytes<HD>(a.g) : 0);
        uint4 codes[NC];
        uint32_t scales[NC];
        const uint32_t mine = lane < kMoves ? froms[lane + 7u] : NONE;
        float weight = 0.f;
        uint32_t position = 0;
        const size_t table = plane * a.g.context;
        if (mine != NONE && a.weights) weight = a.weights[table + mine];
        if (mine != NONE && a.slot_positions) position = a.slot_positions[table + mine];
#pragma unroll
        for (uint32_t n = 0; n < NC; ++n) {
            const uint32_t k = n * 64u + lane, e = k / C, c = k % C, from = e < kMoves ? froms[e + 7u] : NONE;
            if (from == NONE || !a.kc) continue;
            const uint8_t *const src = kp + (size_t)(from / 32u) * L::BLOCK;
            codes[n] = *reinterpret_cast<const uint4 *>(src + (from % 32u) * (HD / 2) + c * 16u);
            scales[n] = reinterpret_cast<const uint32_t *>(src + L::CODES)[(from % 32u) * L::G + c];
        }
#pragma unroll
        for (uint32_t n = 0; n < NC; ++n) {
            const uint32_t k = n * 64u + lane, e = k / C, c = k % C, to = e < kMoves ? tos[e + 7u] : NONE;
            if (to == NONE || !a.kc) continue;
            uint8_t *const dst = kp + (size_t)(to / 32u) * L::BLOCK;
            *reinterpret_cast<uint4 *>(dst + (to % 32u) * (HD / 2) + c * 16u) = codes[n];
            reinterpret_cast<uint32_t *>(dst + L::CODES)[(to % 32u) * L::G + c] = scales[n];
        }
        if (mine != NONE && a.weights) a.weights[table + tos[lane + 7u]] = weight;
        if (mine != NONE && a.slot_positions) a.slot_positions[table + tos[lane + 7u]] = position;
        return;
    }
    if (!a.kc) return;
    // V: the octets' first pairs, wave by wave.
    uint8_t *const vp = a.vc + plane * plane_bytes<HD>(a.g);
    bool first = false;
    if (lane < kMoves) {   // pair e0 + lane
        const uint32_t to = tos[lane + 7u];
        first = to != NONE;
#pragma unroll
        for (uint32_t k = 0; k < 7; ++k) first = first && tos[lane + k] / 8u != to / 8u;
    }
    uint64_t runs = __ballot(first);
    for (uint32_t turn = 0; runs; ++turn, runs &= runs - 1u) {
        if (turn % 3u != wave - 1u) continue;
        const uint32_t e = (uint32_t)__builtin_ctzll(runs) + 7u, oct = tos[e] / 8u;
        uint8_t *const dst = vp + (size_t)(oct / 4u) * L::BLOCK;
        bool in[8];
        uint32_t from[8], to[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            in[k] = tos[e + k] / 8u == oct;   // not so of NONE
            from[k] = froms[e + k];
            to[k] = tos[e + k] % 8u;
        }
        constexpr uint32_t ND = (HD + 63) / 64, NS = 8 * 2 * L::G / 64 ? 8 * 2 * L::G / 64 : 1;   // a lane's dwords, its d and o
        uint32_t *const word = reinterpret_cast<uint32_t *>(dst) + (oct % 4u) * HD + lane;
        uint32_t v[ND], got[ND][8];
#pragma unroll
        for (uint32_t n = 0; n < ND; ++n) {
            v[n] = word[64u * n];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (in[k]) got[n][k] = reinterpret_cast<const uint32_t *>(vp + (size_t)(from[k] / 32u) * L::BLOCK)[from[k] / 8u % 4u * HD + 64u * n + lane];
        }
        // d and o of every group: lane 2 G k + 2 g + which of pair e + k
        _Float16 scale[NS], *at[NS];
#pragma unroll
        for (uint32_t n = 0; n < NS; ++n) {
            const uint32_t x = n * 64u + lane, k = x / (2u * L::G), g = x / 2u % L::G, which = x % 2u;
            at[n] = nullptr;
            if (k >= 8u) continue;
            const uint32_t f = froms[e + k], t = tos[e + k];
            if (t / 8u != oct) continue;
            scale[n] = reinterpret_cast<const _Float16 *>(vp + (size_t)(f / 32u) * L::BLOCK + L::CODES)[(f / 8u % 4u * L::G + g) * 16u + 8u * which + f % 8u];
            at[n] = reinterpret_cast<_Float16 *>(dst + L::CODES) + ((oct % 4u) * L::G + g) * 16u + 8u * which + t % 8u;
        }
#pragma unroll
        for (uint32_t n = 0; n < ND; ++n) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (in[k]) {
                    const uint32_t code = got[n][k] >> (4u * (from[k] % 8u / 2u) + 16u * (from[k] % 2u)) & 15u;
                    const uint32_t bit = 4u * (to[k] / 2u) + 16u * (to[k] % 2u);
                    v[n] = (v[n] & ~(15u << bit)) | code << bit;
                }
            word[64u * n] = v[n];
        }
#pragma unroll
        for (uint32_t n = 0; n < NS; ++n)
            if (at[n]) *at[n] = scale[n];
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
#define CALL(HD) k_kv4_load<HD><<<grid, 2 * HD, 0, s>>>(a)
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
// Tiles of query rows and splits of the slots, by sizes alone (MI355X, us a call; 16/2 heads of
// 128 unless stated).
//
// Rows. Up to 8 take a tile whose columns hold both terms (PK; 16 sequences over 32768: 33.8
// against 37.4 as 16 rows). More take tiles of 16 by four waves while rows x planes x context x
// head_dim is within kSmallWork: a value is then made again for every 16 rows, but a workgroup
// starts and joins sooner (8 tokens over 508: 10.6, with 32-row tiles 13.2; 64 over 564: 12.0 and
// 14.3; beyond it 200 over 1200: 16.2 against 18). From there on tiles of 32 rows by eight waves,
// and of 64 where there are enough of those to fill the card: kWideTiles (1900 tokens: 49 against
// 59; 500 tokens, 126 such tiles: 18.5 against 12.6). One sequence's 32-row tiles of a long
// context take a second round over the 256 CUs as soon as there are more than 256 of them, so
// the wider ones then begin at kWideTilesLong (600 tokens over 4600: 66 against 81; over 600
// they lose, 19 against 17.5). Several sequences are taken to be of unequal length, which the
// device alone knows: those even the rounds out (300 tokens each at 4000 and 2000: 49 against 63
// in wide tiles; both at 4000, it is 81 against 63).
//
// Splits. As many as make kWideGrid workgroups of up to 16 rows (16 sequences over 32768: 33.8; 768:
// 35.2; 3000: 38.2), and 256 of more rows (512: 256 tokens over 4256 take 37.4 against 31), a
// workgroup having at least four blocks, and one of eight waves 16. A split costs the
// join's launch too: a context of at most 2048 / head_dim blocks is not split (448 slots: 7.7
// against 9.2) unless a launch for the weights follows anyway.
constexpr uint64_t kSmallWork = 1ull << 28;
constexpr uint32_t kWideTiles = 192, kWideTilesLong = 129, kLongContext = 1536;
constexpr uint32_t kWideGrid = 1536;
// Workgroups in so small a grid fetch their first block before they know the slot counts (512
// slots: 7.4 against 7.7 us; of larger grids it is no matter, and idle splits would read for
// nothing).
constexpr uint32_t kEagerGroups = 256;
struct Shape {
    uint32_t group, rows, nt, tile_rows, tiles, splits, per;
    uint64_t units;
    bool eager;
};
Shape shape_of(const Kv4Attn &a, bool with_weights) {
    Shape h;
    h.group = a.q_heads / a.g.kv_heads;
    h.rows = a.tokens * h.group;
    const uint64_t pairs = (uint64_t)a.g.kv_heads * a.n;
    const uint32_t blocks = (a.g.context + 31u) / 32u;
    // rows < 2^22 and a cache below 2^47 bytes: no overflow
    const bool small = h.rows <= 16u || h.rows * pairs * a.g.context <= kSmallWork / a.g.head_dim;
    const uint32_t wide = a.n == 1u && a.g.context >= kLongContext ? kWideTilesLong : kWideTiles;
    h.nt = small ? 1 : a.g.head_dim < 256u && (h.rows + 63u) / 64u * pairs >= wide ? 4 : 2;
    h.tile_rows = h.rows <= 8u ? 8u : 16u * h.nt;
    h.tiles = (h.rows + h.tile_rows - 1u) / h.tile_rows;
    h.units = h.tiles * pairs;
    const uint64_t grid = h.rows <= 16u ? kWideGrid : 256u, want = grid > h.units ? grid / h.units : 1u;
    uint32_t splits = h.nt == 1 ? (blocks + 3u) / 4u : blocks < 32u ? 1u : blocks / 16u;
    if (h.nt == 1 && blocks * a.g.head_dim <= 2048u && !(with_weights && h.rows <= 16u)) splits = 1;
    if (splits > want) splits = (uint32_t)want;
    if (splits > kMaxSplits) splits = kMaxSplits;
    h.per = (blocks + splits - 1u) / splits;
    h.splits = (blocks + h.per - 1u) / h.per;
    h.eager = h.units * h.splits <= kEagerGroups;
    return h;
}
}  // namespace

namespace {
// The parts of a call's scratch, in floats from its start; `end` is its size.
struct Parts {
    uint64_t acc, ml, qp, norm, factors, sums, end;
    uint32_t qtiles, row_splits, slots32;
};
Parts parts_of(const Kv4Attn &a, const Shape &h, bool with_weights) {
    Parts t;
    const uint64_t pairs = (uint64_t)a.g.kv_heads * a.n;
    const uint64_t records = h.splits > 1u ? h.units * h.splits * h.tile_rows : 0u;
    const bool rows = with_weights && h.rows > 16u;   // the weights of prompts
    t.qtiles = (h.tiles * h.tile_rows + 31u) / 32u;
    t.slots32 = (a.g.context + 31u) / 32u * 32u;
    // about 512 workgroups of 256 slots, at least two row tiles each; three and four row tiles one,
    // which saves the launch that adds the splits (16 tokens of 16 query heads to 2 over 4000: 20.3 ->
    // 19.9 us a call, over 500 18.7 -> 17.6), from 5 tiles on that costs more (24 tokens: 23.5 against
    // 22.2)
    const uint64_t chunks = (a.g.context + 255u) / 256u * pairs, most = h.rows <= 128u ? 1u : (h.rows + 63u) / 64u;
    uint64_t splits = (512u + chunks - 1u) / chunks;
    if (splits > most) splits = most;
    t.row_splits = (uint32_t)splits;
    t.acc = 0;
    t.ml = t.acc + records * a.g.head_dim;
    t.qp = t.ml + records * 2u;
    t.norm = t.qp + (rows ? pairs * t.qtiles * 32u * a.g.head_dim : 0u);
    t.factors = t.norm + (pairs * h.rows + 1u) / 2u * 4u;
    t.sums = t.factors + (rows ? (pairs * h.rows + 3u) / 4u * 4u : 0u);
    t.end = t.sums + (rows && t.row_splits > 1u ? (uint64_t)t.row_splits * pairs * t.slots32 : 0u);
    return t;
}
}  // namespace

uint64_t kv4_attn_scratch_bytes(const Kv4Attn &a, bool with_weights) {
    return parts_of(a, shape_of(a, with_weights), with_weights).end * 4u;
}

template <int HD>
static int attention(hipStream_t s, const Kv4Attn &a) {
    const Shape h = shape_of(a, a.weights != nullptr);
    const Parts t = parts_of(a, h, a.weights != nullptr);
    const bool rows = a.weights && h.rows > 16u;
    AttnArgs p;
    p.a = a;
    p.group = h.group;
    p.by_group = h.group == 1u ? 0u : (uint32_t)((0x100000000ull + h.group - 1u) / h.group);
    p.rows = h.rows;
    p.tiles = h.tiles;
    p.tile_rows = h.tile_rows;
    p.splits = h.splits;
    p.per = h.per;
    p.eager = h.eager;
    p.acc = a.scratch + t.acc;
    p.ml = a.scratch + t.ml;
    p.norm = reinterpret_cast<f2 *>(a.scratch + t.norm);
    p.qp = rows ? reinterpret_cast<h8 *>(a.scratch + t.qp) : nullptr;
    p.factors = a.scratch + t.factors;
    p.sums = a.scratch + t.sums;
    p.qtiles = t.qtiles;
    p.row_splits = t.row_splits;
    p.slots32 = t.slots32;
    const dim3 grid(h.tiles * h.splits, a.g.kv_heads, a.n);
    if (h.rows <= 8u) {
        k_kv4_attn<HD, 1, 4, true><<<grid, 256, 0, s>>>(p);
    } else if (h.nt == 1) {
        k_kv4_attn<HD, 1, 4, false><<<grid, 256, 0, s>>>(p);
    } else if (h.nt == 2) {
        k_kv4_attn<HD, 2, 8, false><<<grid, 512, 0, s>>>(p);
    } else if constexpr (HD < 256) {
        k_kv4_attn<HD, 4, 8, false><<<grid, 512, 0, s>>>(p);
    }
    VX_LAUNCHED("k_kv4_attn");
    const uint32_t per_join = h.splits <= kFewSplits ? 1024u / HD : 1u;   // rows
    const uint32_t joins = h.splits > 1u ? (h.rows + per_join - 1u) / per_join : 0u;
    const uint32_t groups = a.weights && !rows ? ((a.g.context + 31u) / 32u + 3u) / 4u : 0u;
    if (joins + groups) {
        k_kv4_finish<HD><<<dim3(joins + groups, a.g.kv_heads, a.n), 256, 0, s>>>(p, joins);
        VX_LAUNCHED("k_kv4_finish");
    }
    if (rows) {
        const uint32_t chunks = (a.g.context + 255u) / 256u;
        k_kv4_weights_rows<HD><<<dim3(chunks * t.row_splits, a.g.kv_heads, a.n), 256, 0, s>>>(p);
        VX_LAUNCHED("k_kv4_weights_rows");
        if (t.row_splits > 1u) {
            k_kv4_add_weights<<<dim3(chunks, a.g.kv_heads, a.n), 256, 0, s>>>(p);
            VX_LAUNCHED("k_kv4_add_weights");
        }
    }
    return VX_OK;
}

int launch_kv4_attention(hipStream_t s, const Kv4Attn &a) {
    return a.g.head_dim == 64u ? attention<64>(s, a) : a.g.head_dim == 128u ? attention<128>(s, a) : attention<256>(s, a);
}

int launch_kv4_select(hipStream_t s, const Kv4Evict &a) {
    const dim3 grid(a.g.kv_heads, a.n, a.g.layers);
    if (a.g.context <= kSelect * kSelectTurns)
        k_kv4_select<true><<<grid, kSelect, 0, s>>>(a);
    else
        k_kv4_select<false><<<grid, kSelect, 0, s>>>(a);
    VX_LAUNCHED("k_kv4_select");
    return VX_OK;
}

int launch_kv4_compact(hipStream_t s, const Kv4Evict &a) {
    const dim3 grid((a.moves + kMoves - 1u) / kMoves, a.g.kv_heads * a.n, a.g.layers);
#define CALL(HD) k_kv4_compact<HD><<<grid, 256, 0, s>>>(a)
    KV4_HD(a.g.head_dim, CALL)
#undef CALL
    VX_LAUNCHED("k_kv4_compact");
    return VX_OK;
}

}  // namespace vx
