// The 4-bit KV cache (include/voxhip.h, vx_kv4_*): launch descriptions shared by the
// C ABI checks (kv4.cpp) and the kernels (kernels_kv4.hip).
#pragma once

#include "vx_internal.h"

namespace vx {

constexpr uint32_t kKv4Block = 32;        // slots of a block
constexpr uint32_t kKv4MaxContext = 1u << 28;   // these keep every grid below 2^32 threads a dimension
constexpr uint32_t kKv4MaxRows = 1u << 22;      // tokens of a sequence, times the query heads of a KV head

inline uint64_t kv4_block_bytes(uint32_t head_dim) { return 20ull * head_dim; }
inline uint64_t kv4_plane_bytes(const vx_kv4_geom &g) {
    return (g.context + kKv4Block - 1u) / kKv4Block * kv4_block_bytes(g.head_dim);
}

struct Kv4Rows {
    vx_kv4_geom g;
    uint32_t layer = 0, first = 0, n = 0, tokens = 0;
    uint32_t k_stride = 0, v_stride = 0;
    float *k = nullptr, *v = nullptr;       // at the push's base; store only reads them
    uint8_t *kc = nullptr, *vc = nullptr;
    const uint32_t *slots = nullptr, *positions = nullptr;
    uint32_t *slot_positions = nullptr;
    bool vec = false;                       // every row's address is 16-byte aligned
};
int launch_kv4_store(hipStream_t s, const Kv4Rows &a);
int launch_kv4_load(hipStream_t s, const Kv4Rows &a);
int launch_kv4_advance(hipStream_t s, uint32_t *slots, uint32_t *positions, uint32_t n, uint32_t tokens,
                       uint32_t context);

struct Kv4Attn {
    vx_kv4_geom g;
    uint32_t layer = 0, first = 0, n = 0, tokens = 0, q_heads = 0;
    uint32_t q_stride = 0, out_stride = 0;
    float decay = 1.0f;
    const float *q = nullptr;
    const uint8_t *kc = nullptr, *vc = nullptr;
    float *out = nullptr;
    float *weights = nullptr;               // nullable
    const uint32_t *slots = nullptr;
    float *scratch = nullptr;
    bool qvec = false, ovec = false;        // rows 16-byte aligned
};
uint64_t kv4_attn_scratch_bytes(const Kv4Attn &a, bool with_weights);
int launch_kv4_attention(hipStream_t s, const Kv4Attn &a);

struct Kv4Evict {
    vx_kv4_geom g;
    uint32_t first = 0, n = 0, keep = 0, sinks = 0, recent = 0, moves = 0;
    const uint32_t *plan_in = nullptr;
    uint32_t *plan = nullptr;
    uint8_t *kc = nullptr, *vc = nullptr;
    float *weights = nullptr;
    uint32_t *slot_positions = nullptr;
    uint32_t *slots = nullptr;
};
int launch_kv4_select(hipStream_t s, const Kv4Evict &a);
int launch_kv4_compact(hipStream_t s, const Kv4Evict &a);

}  // namespace vx
