// A KV cache held at a budget by accumulated attention weight: cutting a prompt to it, and the decode step over it
// (eviction.hip, heavy_hitter.hip).
#pragma once

#include "common.hpp"

namespace eco {

// The cache of one layer: C slots per row and KV head. Slots [0, count[b, h]) are filled; position is the token a slot
// holds, score the attention weight it has received, length[b] the tokens the row has seen. All contiguous.
struct BudgetCache {
    uint16_t *keys, *values;     // [B, Hkv, C, D]
    float* score;                // [B, Hkv, C]
    int32_t *position, *count;   // [B, Hkv, C], [B, Hkv]
    int32_t* length;             // [B]
    int batch, kv_heads, slots, head_dim;
    int recent, first;           // the newest and the first tokens, never evicted
};

struct EvictParams {
    BudgetCache cache;
    const uint16_t *k, *v;
    int64_t sk_t, sk_h, sv_t, sv_h;
    const float* mass;
    int64_t sm_h;
    const int32_t *begin, *end;  // rows of sequence b (one per cache row)
    int64_t rows;
};

int evict_prompt(const EvictParams& p, int max_tokens, hipStream_t stream);

struct HeavyParams {
    BudgetCache cache;
    const uint16_t* q;  // [B, Hq, D]
    int64_t sq_b, sq_h;
    const uint16_t *k, *v;  // the new token's [B, Hkv, D]
    int64_t sk_b, sk_h, sv_b, sv_h;
    const float* sinks;
    uint16_t* out;  // [B, Hq, D]
    int64_t so_b, so_h;
    int q_heads, groups;
    int splits, span;  // parts a row's slots are cut into, slots of a part
    float scale, softcap;
    int chosen;      // whether a launch before chose the slots (else every workgroup chooses)
    int pitch;       // slots of a row of `logits`: C in whole fours
    float* logits;   // workspace: [B, Hkv, G, pitch]
    float* partial;  // [B, Hkv, splits, G, D]
    float* stats;    // [B, Hkv, splits, G, 2]: maximum and sum
    int32_t* plan;   // [B, Hkv, 4]: the slot written, filled slots, position
};

size_t heavy_hitter_workspace(int batch, int q_heads, int kv_heads, int slots, int head_dim);
int heavy_hitter_decode(HeavyParams p, int format, void* workspace, size_t workspace_bytes, hipStream_t stream);

// Order of scores as unsigned integers: a NaN below everything, -0 equal to 0.
__device__ __forceinline__ uint32_t score_rank(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    return (b >> 31) ? ~b : (b | 0x80000000u);
}

}  // namespace eco
