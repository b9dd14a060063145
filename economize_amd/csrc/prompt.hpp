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

// x / by for 0 <= x < 2^31 - by through one product: 2^32 over `by` rounded up gives the quotient or one more.
struct Divisor {
    uint32_t by, inverse;
    Divisor() = default;
    explicit Divisor(int64_t d) : by(static_cast<uint32_t>(d)), inverse(static_cast<uint32_t>((0x100000000ull + d - 1) / d)) {}
    __host__ __device__ __forceinline__ int operator()(int x) const {
        const int q = static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * inverse >> 32);
        return by == 1 ? x : q - (q * static_cast<int>(by) > x ? 1 : 0);
    }
};

// Workgroups that look after the rows of no sequence, where a call asks for it.
constexpr int FILLERS = 128;

// Up to so many sequences are taken by their work, the most first.
constexpr int SORTED = 8;

// Which (sequence, KV head) pair and which of its tiles a workgroup takes. The tiles of a pair read the same rows, so
// they run close together: the pairs in `group` at a time, their longest tiles first. Workgroups go to the eight XCDs
// in turn, each with an L2 of its own: with `pin` a pair stays on one.
struct WorkOrder {
    int pairs, tiles, group, pin;
    Divisor whole, full_width, last_width;  // workgroups of a group of pairs; pairs in a group, and in the last one
    int per_xcd() const { return (pairs + 7) / 8; }
    int64_t blocks() const { return static_cast<int64_t>(tiles) * (pin ? 8 * per_xcd() : pairs); }
};

// `tiles` of `parts` workgroups each per pair, whose rows read by all of them take `bytes`: as many pairs at a time as
// three quarters of an L2 hold. Pinned where that leaves the XCDs about the same work: with KV heads in eights each
// gets every sequence, otherwise many sequences even out (6 sequences of different lengths with 4 KV heads, pinned:
// half of the CUs' time idle).
inline WorkOrder work_order(int sequences, int kv_heads, int64_t tiles, int parts, int64_t bytes) {
    const int64_t pairs = static_cast<int64_t>(sequences) * kv_heads;
    const int64_t most_tiles = (1 << 23) / (pairs * parts);  // (a launch holds fewer than 2^32 threads)
    tiles = tiles < most_tiles ? tiles : most_tiles;
    WorkOrder o;
    o.pairs = static_cast<int>(pairs);
    o.tiles = static_cast<int>(tiles < 1 ? 1 : tiles) * parts;
    o.pin = kv_heads % 8 == 0 || pairs >= 128;
    const int64_t fit = (3 << 20) / (bytes < 1 ? 1 : bytes);
    const int64_t most = o.pin ? o.per_xcd() : pairs;
    // (an odd number: workgroups in turn go to the four shader engines of an XCD, and where only every other pair has
    // tiles left, two of the engines would be idle)
    o.group = static_cast<int>(fit < 1 ? 1 : fit > most ? most : fit - (fit % 2 == 0));
    o.whole = Divisor(static_cast<int64_t>(o.tiles) * o.group);
    o.full_width = Divisor(o.group);
    o.last_width = Divisor((most - 1) % o.group + 1);
    return o;
}

struct PromptParams {
    const uint16_t *q, *k, *v;
    int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;  // element strides of tokens and heads
    PackedRows rows;
    const float* sinks;  // [Hq] or null
    uint16_t* out;
    int64_t so_t, so_h;
    float* lse;  // [Hq, sl_h] or null
    int64_t sl_h;
    int fill;  // FILLERS workgroups give rows of no sequence out 0 and lse -inf (0: they are left as they are)
    int q_heads, kv_heads, groups, head_dim;
    Divisor per_group, per_kv, per_part;  // over the groups, the KV heads, the row tiles of a part
    WorkOrder order;  // (sequences of more row tiles than the launch holds loop over them)
    int parts, part_shift;         // a row tile's keys are cut into up to so many, of 1 << part_shift tiles or more
    float *part_out, *part_stats;  // [parts, q_rows, Hq, D] and [.., 2], of the row tiles that were cut
    float scale, softcap;
};

int prompt_attention(PromptParams p, int format, int max_queries, int max_keys, void* workspace, size_t workspace_bytes,
                     hipStream_t stream);
size_t prompt_attention_workspace(int sequences, int64_t q_rows, int max_queries, int max_keys, int q_heads, int kv_heads,
                                  int head_dim);

struct MassParams {
    const uint16_t *q, *k;
    int64_t sq_t, sq_h, sk_t, sk_h;
    PackedRows rows;
    const float* lse;  // [Hq, sl_h]
    int64_t sl_h;
    float* mass;  // [Hkv, sm_h]
    int64_t sm_h;
    int fill;    // FILLERS workgroups give keys of no sequence 0 (0: they are left as they are)
    int window;  // only the last `window` queries of a sequence count
    int q_heads, kv_heads, groups, head_dim;
    Divisor per_kv, per_part;
    WorkOrder order;  // (sequences of more key tiles than the launch holds loop over them)
    int parts;       // a key tile's query heads are cut into so many parts (1, or one per head)
    float* partial;  // [parts, Hkv, k_rows] where parts > 1
    float scale, softcap;
};

int attention_mass(MassParams p, int format, int max_queries, int max_keys, void* workspace, size_t workspace_bytes,
                   hipStream_t stream);
size_t attention_mass_workspace(int max_queries, int64_t k_rows, bool windowed, int q_heads, int kv_heads);

}  // namespace eco
