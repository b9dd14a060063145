// Attention over packed prompts and the attention weight its keys receive: parameters and host entry points
// (prompt_attention.hip, attention_mass.hip).
#pragma once

#include "common.hpp"

namespace eco {

// Sequence s of a packed call: queries [q_begin[s], q_end[s]) of q_rows rows, keys [k_begin[s], k_end[s]) of k_rows
// (clamped to the rows there are, so that malformed bounds read and write inside the tensors). Query i of a sequence
// of nq queries and nk keys sees its keys j <= i + nk - nq.
struct PackedRows {
    const int32_t *q_begin, *q_end, *k_begin, *k_end;
    int sequences;
    int64_t q_rows, k_rows;
};

struct PromptParams {
    const uint16_t *q, *k, *v;
    int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;  // element strides of tokens and heads
    PackedRows rows;
    const float* sinks;  // [Hq] or null
    uint16_t* out;
    int64_t so_t, so_h;
    float* lse;  // [Hq, sl_h] or null
    int64_t sl_h;
    int fill;                          // rows of no sequence: out 0 and lse -inf (1), or left as they are (0)
    int q_heads, kv_heads, groups, head_dim;
    int tiles;      // row tiles a launch holds per sequence and KV head (longer sequences loop over them)
    float scale, softcap;
};

int prompt_attention(const PromptParams& p, int format, int max_queries, int max_keys, void* workspace,
                     size_t workspace_bytes, hipStream_t stream);
size_t prompt_attention_workspace(int sequences, int max_queries, int max_keys, int q_heads, int kv_heads,
                                  int head_dim);

struct MassParams {
    const uint16_t *q, *k;
    int64_t sq_t, sq_h, sk_t, sk_h;
    PackedRows rows;
    const float* lse;  // [Hq, sl_h]
    int64_t sl_h;
    float* mass;  // [Hkv, sm_h]
    int64_t sm_h;
    int fill;    // keys of no sequence: 0 (1), or left as they are (0)
    int window;  // only the last `window` queries of a sequence count
    int q_heads, kv_heads, groups, head_dim;
    int tiles;  // key tiles a launch holds per sequence and KV head (longer sequences loop over them)
    float scale, softcap;
};

int attention_mass(const MassParams& p, int format, int max_keys, hipStream_t stream);

}  // namespace eco
