// extern "C" entry points of packed prompts and of caches held at a budget (declared in include/economize_amd.h):
// argument checks around prompt_attention.hip, attention_mass.hip, eviction.hip and heavy_hitter.hip.

#include <cmath>

#include "../../include/economize_amd.h"
#include "eviction.hpp"
#include "prompt.hpp"

namespace eco {

namespace {

constexpr int64_t MOST_ROWS = 0x7fff0000;  // (a tile past the last row is still a 32-bit index)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_shape(const char* what, int format, int q_heads, int kv_heads, int head_dim, float scale, float softcap) {
    const std::string w = what;
    if (format != BF16 && format != FP16) return fail(w + ": queries, keys and values must be bf16 or fp16");
    if (q_heads <= 0 || kv_heads <= 0) return fail(w + ": sizes must be positive");
    if (q_heads % kv_heads) return fail(w + ": the query heads are not a multiple of the KV heads");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(w + ": head dim must be 64, 128 or 256");
    if (!(scale > 0.0f) || std::isinf(scale)) return fail(w + ": scale must be positive and finite");
    if (!(softcap >= 0.0f) || std::isinf(softcap)) return fail(w + ": softcap must be 0 (none) or positive and finite");
    return 0;
}

// Strides of 16-bit elements whose rows start on 16 bytes; `most` bounds the distance of a tile's rows to 32 bits.
int check_rows(const char* what, const void* p, std::initializer_list<int64_t> strides) {
    if (!aligned16(p)) return fail(std::string(what) + " must be 16-byte aligned");
    for (int64_t s : strides)
        if (s % 8 || s < 0 || s >= (1 << 24))
            return fail(std::string(what) + " need strides that are multiples of 16 bytes, from 0 to below 2^24 elements");
    return 0;
}

int check_packed(const char* what, const PackedRows& r) {
    const std::string w = what;
    if (!r.q_begin || !r.q_end || !r.k_begin || !r.k_end) return fail(w + ": null sequence bounds");
    if (r.sequences <= 0) return fail(w + ": need at least one sequence");
    if (r.q_rows < 0 || r.k_rows < 0 || r.q_rows > MOST_ROWS || r.k_rows > MOST_ROWS)
        return fail(w + ": rows must be from 0 to 2^31 - 2^16");
    return 0;
}

// Outputs [rows, heads, D] of these strides hold no element twice.
int check_apart(const char* what, int64_t rows, int64_t heads, int64_t s_row, int64_t s_head, int head_dim) {
    const bool heads_within = s_head <= s_row;
    const int64_t inner = heads_within ? s_head : s_row, outer = heads_within ? s_row : s_head;
    const int64_t n = heads_within ? heads : rows, m = heads_within ? rows : heads;
    if ((n > 1 && inner < head_dim) || (m > 1 && outer < (n > 1 ? (n - 1) * inner : 0) + head_dim))
        return fail(std::string(what) + ": the outputs overlap each other");
    return 0;
}

int check_cache(const char* what, const BudgetCache& c) {
    const std::string w = what;
    if (!c.keys || !c.values || !c.score || !c.position || !c.count || !c.length) return fail(w + ": null cache");
    if (!aligned16(c.keys) || !aligned16(c.values)) return fail(w + ": the cache must be 16-byte aligned");
    if (c.batch <= 0 || c.kv_heads <= 0 || c.slots <= 0) return fail(w + ": sizes must be positive");
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return fail(w + ": head dim must be 64, 128 or 256");
    if (c.recent < 1 || c.first < 0 || static_cast<int64_t>(c.recent) + c.first > c.slots)
        return fail(w + ": need recent >= 1, first >= 0 and recent + first <= slots");
    if (static_cast<int64_t>(c.batch) * c.kv_heads > 65535) return fail(w + ": the cache has too many rows for one call");
    if (c.slots > (1 << 25) || static_cast<int64_t>(c.batch) * c.kv_heads > 0x3fffffff / c.slots)
        return fail(w + ": the cache has too many slots for one call");
    return 0;
}

}  // namespace

}  // namespace eco

using namespace eco;

extern "C" {

size_t eco_prompt_attention_workspace_size(int32_t sequences, int64_t q_rows, int32_t max_queries, int32_t max_keys,
                                           int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    if (sequences <= 0 || q_rows < 0 || max_queries < 0 || max_keys < 0 || q_heads <= 0 || kv_heads <= 0 ||
        q_heads % kv_heads)
        return 0;
    return prompt_attention_workspace(sequences, q_rows, max_queries, max_keys, q_heads, kv_heads, head_dim);
}

int eco_prompt_attention(const void* q, int32_t format, int64_t sq_t, int64_t sq_h, const void* k, const void* v,
                         int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h, const int32_t* q_begin,
                         const int32_t* q_end, const int32_t* k_begin, const int32_t* k_end, int32_t sequences,
                         int64_t q_rows, int64_t k_rows, int32_t max_queries, int32_t max_keys, const float* sinks,
                         void* out, int64_t so_t, int64_t so_h, float* lse, int64_t sl_h, int32_t fill, int32_t q_heads,
                         int32_t kv_heads, int32_t head_dim, float scale, float softcap, void* workspace,
                         size_t workspace_bytes, void* stream) {
    const char* what = "prompt attention";
    if (q_rows == 0) return 0;
    if (!q || !out || (k_rows > 0 && (!k || !v))) return fail("prompt attention: null pointer");
    if (int rc = check_shape(what, format, q_heads, kv_heads, head_dim, scale, softcap)) return rc;
    const PackedRows rows{q_begin, q_end, k_begin, k_end, sequences, q_rows, k_rows};
    if (int rc = check_packed(what, rows)) return rc;
    if (int rc = check_rows("prompt attention: queries", q, {sq_t, sq_h})) return rc;
    if (int rc = check_rows("prompt attention: keys", k, {sk_t, sk_h})) return rc;
    if (int rc = check_rows("prompt attention: values", v, {sv_t, sv_h})) return rc;
    if (int rc = check_rows("prompt attention: outputs", out, {so_t, so_h})) return rc;
    if (int rc = check_apart(what, q_rows, q_heads, so_t, so_h, head_dim)) return rc;
    if (lse && sl_h < q_rows) return fail("prompt attention: lse rows are shorter than the queries");
    if (max_queries < 0 || max_keys < 0) return fail("prompt attention: sizes must not be negative");
    if (static_cast<int64_t>(sequences) * kv_heads > 65535) return fail("prompt attention: too many sequences");
    if (q_rows > MOST_ROWS / (q_heads / kv_heads)) return fail("prompt attention: too many queries for one call");
    PromptParams p{};
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.sq_t = sq_t, p.sq_h = sq_h, p.sk_t = sk_t, p.sk_h = sk_h, p.sv_t = sv_t, p.sv_h = sv_h;
    p.rows = rows;
    p.sinks = sinks;
    p.out = static_cast<uint16_t*>(out);
    p.so_t = so_t, p.so_h = so_h;
    p.lse = lse, p.sl_h = sl_h;
    p.fill = fill;
    p.q_heads = q_heads, p.kv_heads = kv_heads, p.groups = q_heads / kv_heads, p.head_dim = head_dim;
    p.scale = scale, p.softcap = softcap;
    if (!aligned16(workspace)) return fail("prompt attention: the workspace must be 16-byte aligned");
    return prompt_attention(p, format, max_queries, max_keys, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

size_t eco_attention_mass_workspace_size(int32_t max_queries, int64_t k_rows, int32_t window, int32_t q_heads,
                                         int32_t kv_heads) {
    if (max_queries < 0 || k_rows < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return 0;
    return attention_mass_workspace(window > 0 && window < max_queries ? window : max_queries, k_rows, window > 0, q_heads,
                                    kv_heads);
}

int eco_attention_mass(const void* q, int32_t format, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t,
                       int64_t sk_h, const float* lse, int64_t sl_h, const int32_t* q_begin, const int32_t* q_end,
                       const int32_t* k_begin, const int32_t* k_end, int32_t sequences, int64_t q_rows, int64_t k_rows,
                       int32_t max_queries, int32_t max_keys, int32_t window, float* mass, int64_t sm_h, int32_t fill,
                       int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale, float softcap, void* workspace,
                       size_t workspace_bytes, void* stream) {
    const char* what = "attention mass";
    if (k_rows == 0) return 0;
    if (!k || !mass || (q_rows > 0 && (!q || !lse))) return fail("attention mass: null pointer");
    if (int rc = check_shape(what, format, q_heads, kv_heads, head_dim, scale, softcap)) return rc;
    const PackedRows rows{q_begin, q_end, k_begin, k_end, sequences, q_rows, k_rows};
    if (int rc = check_packed(what, rows)) return rc;
    if (int rc = check_rows("attention mass: queries", q, {sq_t, sq_h})) return rc;
    if (int rc = check_rows("attention mass: keys", k, {sk_t, sk_h})) return rc;
    if (sl_h < q_rows) return fail("attention mass: lse rows are shorter than the queries");
    if (sm_h < k_rows) return fail("attention mass: mass rows are shorter than the keys");
    if (q_rows > MOST_ROWS / (q_heads / kv_heads)) return fail("attention mass: too many queries for one call");
    if (window < 0 || max_queries < 0 || max_keys < 0) return fail("attention mass: sizes must not be negative");
    if (static_cast<int64_t>(sequences) * kv_heads > 65535) return fail("attention mass: too many sequences");
    MassParams p{};
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.sq_t = sq_t, p.sq_h = sq_h, p.sk_t = sk_t, p.sk_h = sk_h;
    p.rows = rows;
    p.lse = lse, p.sl_h = sl_h;
    p.mass = mass, p.sm_h = sm_h;
    p.fill = fill, p.window = window;
    p.q_heads = q_heads, p.kv_heads = kv_heads, p.groups = q_heads / kv_heads, p.head_dim = head_dim;
    p.scale = scale, p.softcap = softcap;
    const int counted = window > 0 && window < max_queries ? window : max_queries;
    return attention_mass(p, format, counted, max_keys, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

int eco_evict_prompt(const void* k, const void* v, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h,
                     const float* mass, int64_t sm_h, const int32_t* begin, const int32_t* end, int64_t rows,
                     int32_t max_tokens, void* keys, void* values, float* score, int32_t* position, int32_t* count,
                     int32_t* length, int32_t batch, int32_t kv_heads, int32_t slots, int32_t head_dim, int32_t recent,
                     int32_t first, void* stream) {
    const char* what = "prompt eviction";
    if (!k || !v || !mass || !begin || !end) return fail("prompt eviction: null pointer");
    EvictParams p{};
    p.cache = BudgetCache{static_cast<uint16_t*>(keys), static_cast<uint16_t*>(values), score, position, count, length,
                          batch, kv_heads, slots, head_dim, recent, first};
    if (int rc = check_cache(what, p.cache)) return rc;
    if (int rc = check_rows("prompt eviction: keys", k, {sk_t, sk_h})) return rc;
    if (int rc = check_rows("prompt eviction: values", v, {sv_t, sv_h})) return rc;
    if (rows < 0 || rows > MOST_ROWS || max_tokens < 0) return fail("prompt eviction: rows must be from 0 to 2^31 - 2^16");
    if (sm_h < rows) return fail("prompt eviction: mass rows are shorter than the keys");
    // (tokens are copied in any order: a slot may be written before the token it held is read)
    const int64_t cells = static_cast<int64_t>(batch) * kv_heads * slots;
    struct Span {
        uintptr_t at;
        int64_t bytes;
    };
    const Span to[] = {{reinterpret_cast<uintptr_t>(keys), cells * head_dim * 2},
                       {reinterpret_cast<uintptr_t>(values), cells * head_dim * 2},
                       {reinterpret_cast<uintptr_t>(score), cells * 4},
                       {reinterpret_cast<uintptr_t>(position), cells * 4}};
    const Span from[] = {{reinterpret_cast<uintptr_t>(k), ((rows - 1) * sk_t + (kv_heads - 1) * sk_h + head_dim) * 2},
                         {reinterpret_cast<uintptr_t>(v), ((rows - 1) * sv_t + (kv_heads - 1) * sv_h + head_dim) * 2},
                         {reinterpret_cast<uintptr_t>(mass), ((kv_heads - 1) * sm_h + rows) * 4}};
    for (const Span& a : from)
        for (const Span& b : to)
            if (rows > 0 && a.at < b.at + b.bytes && b.at < a.at + a.bytes)
                return fail("prompt eviction: the prompt must be in memory apart from the cache's");
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.sk_t = sk_t, p.sk_h = sk_h, p.sv_t = sv_t, p.sv_h = sv_h;
    p.mass = mass, p.sm_h = sm_h;
    p.begin = begin, p.end = end;
    p.rows = rows;
    return evict_prompt(p, max_tokens, static_cast<hipStream_t>(stream));
}

size_t eco_heavy_hitter_workspace_size(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t slots,
                                       int32_t head_dim) {
    if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || slots <= 0 || q_heads % kv_heads) return 0;
    return heavy_hitter_workspace(batch, q_heads, kv_heads, slots, head_dim);
}

int eco_heavy_hitter_decode(const void* q, int32_t format, int64_t sq_b, int64_t sq_h, const void* k, const void* v,
                            int64_t sk_b, int64_t sk_h, int64_t sv_b, int64_t sv_h, const float* sinks, void* keys,
                            void* values, float* score, int32_t* position, int32_t* count, int32_t* length, void* out,
                            int64_t so_b, int64_t so_h, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t slots,
                            int32_t head_dim, int32_t recent, int32_t first, float scale, float softcap,
                            void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "heavy-hitter decode";
    if (!q || !k || !v || !out || !workspace) return fail("heavy-hitter decode: null pointer");
    if (int rc = check_shape(what, format, q_heads, kv_heads, head_dim, scale, softcap)) return rc;
    HeavyParams p{};
    p.cache = BudgetCache{static_cast<uint16_t*>(keys), static_cast<uint16_t*>(values), score, position, count, length,
                          batch, kv_heads, slots, head_dim, recent, first};
    if (int rc = check_cache(what, p.cache)) return rc;
    if (q_heads / kv_heads > 64) return fail("heavy-hitter decode: at most 64 query heads per KV head");
    if (!aligned16(workspace)) return fail("heavy-hitter decode: the workspace must be 16-byte aligned");
    if (int rc = check_rows("heavy-hitter decode: queries", q, {sq_b, sq_h})) return rc;
    if (int rc = check_rows("heavy-hitter decode: keys", k, {sk_b, sk_h})) return rc;
    if (int rc = check_rows("heavy-hitter decode: values", v, {sv_b, sv_h})) return rc;
    if (int rc = check_rows("heavy-hitter decode: outputs", out, {so_b, so_h})) return rc;
    if (int rc = check_apart(what, batch, q_heads, so_b, so_h, head_dim)) return rc;
    p.q = static_cast<const uint16_t*>(q);
    p.sq_b = sq_b, p.sq_h = sq_h;
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.sk_b = sk_b, p.sk_h = sk_h, p.sv_b = sv_b, p.sv_h = sv_h;
    p.sinks = sinks;
    p.out = static_cast<uint16_t*>(out);
    p.so_b = so_b, p.so_h = so_h;
    p.q_heads = q_heads, p.groups = q_heads / kv_heads;
    p.scale = scale, p.softcap = softcap;
    return heavy_hitter_decode(p, format, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
