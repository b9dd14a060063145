// Attention over packed prompts: every sequence's queries attend causally over its own keys.
//
// With x_ij = scale q_i . k_j (soft-capped or not), query i gives o_i = sum_j exp(x_ij - lse_i) v_j over the keys it
// sees, lse_i = log(sum_j exp(x_ij) + exp(sink)). One pass over the keys with a running maximum and sum (both fp32).
//
// A workgroup holds 128 rows of one (sequence, KV head): row r is query r / G of head r % G of the group, so the G
// heads of a group share every K/V tile and a tile's rows span few queries (little of the causal diagonal is wasted). A
// wave holds 32 rows as columns: S^T = K Q^T puts one query in each lane (l % 32) with 16 of 32 keys in its registers,
// so the softmax needs one exchange with lane l ^ 32 and P^T is already the second product's operand: its eight keys
// per lane are {4 h .. 4 h + 3, 8 + 4 h ..} of 16 (h = l / 32), the order the transposed value reads deliver. O^T keeps
// the query in the lane, so rescaling is one multiplier per lane. Keys and values come straight into LDS, two tiles of
// 64 each, one step ahead; the scores of a tile are computed under the exponentials of the one before.
//
// Long sequences are bound by the matrix instructions and the power they draw: 32768 tokens, 32 heads of 128 on 8, take
// 8.1 ms, 1.08 PFLOP/s (a large library product reaches 1.31; on zeros, which draw less, a build of 8.5 ms took 6.4).
// Short ones are bound by a row tile's chain of bounds, keys, products and outputs (6 us beside 1.3 us a tile of keys):
// 24 prompts of 1 to 2047 tokens take 370 us, 0.76 PFLOP/s. Heads of 64 are bound by the exponentials (8 x 4000 tokens:
// 0.80 PFLOP/s), heads of 256 by registers, which leave one wave to a SIMD (0.59). 64 rows to a wave read LDS half as
// often but left no registers to overlap products and exponentials (32768 tokens 10 ms where 32 rows took 8.5).

#include "prompt_tile.hpp"

namespace eco {

namespace {

constexpr int WAVES = 4, THREADS = WAVES * 64;
constexpr int ROWS = WAVES * 32;  // rows of a tile

constexpr float NEVER = -1e30f;  // running maximum before the first key (log2 units)

// The parts of a row tile that sees so many tiles of keys, and the first tile of a part.
__device__ __forceinline__ int parts_of(const PromptParams& p, int key_tiles) {
    const int n = key_tiles >> p.part_shift;
    return n < 1 ? 1 : n < p.parts ? n : p.parts;
}

__device__ __forceinline__ int part_begin(int key_tiles, int part, int parts) {
    return static_cast<int>(static_cast<int64_t>(key_tiles) * part / parts);
}

template <int D, int FMT, bool CAP>
__global__ __launch_bounds__(THREADS, D == 256 ? 1 : D == 128 ? 2 : 3) void prompt_attention_kernel(PromptParams p) {
    typedef Tile<D> T;
    constexpr int KS = D / 16;  // 16-channel steps of the first product
    constexpr int DT = D / 32;  // 32-channel blocks of the output
    __shared__ __align__(256) uint8_t lds[4][T::BYTES];
    __shared__ int unseen;  // an infinity or a NaN was taken out of the values of a tile that not every row sees

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, half = lane >> 5;
    const int work = gridDim.x - p.fill;
    if (static_cast<int>(blockIdx.x) >= work) {  // the last workgroups: rows of no sequence
        for_gaps(p.rows.q_begin, p.rows.q_end, p.rows.sequences, p.rows.q_rows, blockIdx.x - work,
                 [&](int64_t from, int64_t to, int worker, int workers) {
            const int64_t chunks = (to - from) * p.q_heads * (D / 8);
            for (int64_t c = static_cast<int64_t>(worker) * THREADS + tid; c < chunks; c += static_cast<int64_t>(workers) * THREADS) {
                const int64_t row = c / (D / 8);
                const int64_t t = from + row / p.q_heads;
                const int h = static_cast<int>(row % p.q_heads);
                *reinterpret_cast<uint4*>(p.out + t * p.so_t + h * p.so_h + (c % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
                if (p.lse && c % (D / 8) == 0) p.lse[h * p.sl_h + t] = -INFINITY;
            }
        });
        return;
    }
    int pair, slot;
    if (!work_of(p.order, blockIdx.x, pair, slot)) return;
    // (parts outermost: workgroups without work come last, where they leave no shader engine without any)
    const int stride = p.per_part.by, part = p.per_part(slot), first = slot - part * stride;
    const int s = p.per_kv(pair), kvh = pair - s * p.kv_heads;
    const Sequence seq = ranked_sequence(p.rows, s);
    const int total = seq.nq * p.groups;  // (below 2^31: the host checks)
    const int tiles = (total + ROWS - 1) / ROWS;
    const int offset = seq.nk - seq.nq;  // query i sees keys <= i + offset
    const uint16_t* kbase = p.k + seq.k0 * p.sk_t + kvh * p.sk_h;
    const uint16_t* vbase = p.v + seq.k0 * p.sv_t + kvh * p.sv_h;
    auto over_groups = [&](int r) { return p.per_group(r); };
    const float cc = CAP ? 1.0f : p.scale * kLog2e;
    const TileCopy<D, THREADS> kcopy(tid, p.sk_t, true), vcopy(tid, p.sv_t, false);
    // Fragment places in a tile: keys row l % 32, 8 channels from 8 (l / 32); values transposed, rows 4 (l / 32) + l %
    // 16 / 4, channels 16 (l / 16 % 2) + 4 (l % 4). The swizzles are exclusive-ors of the chunk, so the place of
    // channel step i is the first one's with 32 i (values: 64 d) flipped, and further rows are a constant away.
    const int vrow = 4 * half + ((lane & 15) >> 2);
    const uint32_t kplace = col * (D * 2) + T::key_chunk(col, half) * 16;
    const uint32_t vplace = vrow * (D * 2) + T::value_chunk(vrow, ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;

    for (int t = first; t < tiles; t += stride) {
        const int low_row = (tiles - 1 - t) * ROWS;  // the longest rows first
        const int row0 = low_row + wave * 32;
        const int last = over_groups(low_row + ROWS - 1 < total ? low_row + ROWS - 1 : total - 1) + offset;
        const int full = over_groups(low_row) + offset;  // every row of the tile sees keys <= full, some keys <= last
        const int wave_full = over_groups(row0 < total ? row0 : total - 1) + offset;
        // The part's tiles of keys: from `from` up to key_tiles, of the row tile's all_tiles
        const int all_tiles = last < 0 ? 0 : (last >> 6) + 1;
        const int parts = parts_of(p, all_tiles);
        if (part >= parts) continue;
        const int from = part_begin(all_tiles, part, parts), key_tiles = part_begin(all_tiles, part + 1, parts);

        auto keys = [&](int j) { kcopy.start(lds[j & 1], kbase, p.sk_t, 64 * j, seq.nk); };
        auto values = [&](int j) { vcopy.start(lds[2 + (j & 1)], vbase, p.sv_t, 64 * j, seq.nk); };
        if (t != first) tile_barrier();  // the previous row tile's reads are done
        if (tid == 0) unseen = 0;
        if (key_tiles > from) {
            keys(from);
            values(from);
            if (key_tiles > from + 1) keys(from + 1);
        }
        const bool live = row0 + col < total;  // the lane's row
        const int row_at = live ? row0 + col : total - 1;
        const int qi = over_groups(row_at), head = row_at - qi * p.groups;
        const int limit = live ? qi + offset : -1;
        uint4 qf[KS];
        const uint16_t* qp = p.q + (seq.q0 + qi) * p.sq_t + (kvh * p.groups + head) * p.sq_h + half * 8;
#pragma unroll
        for (int i = 0; i < KS; ++i) qf[i] = *reinterpret_cast<const uint4*>(qp + 16 * i);

        f32x16 acc[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
        float m = NEVER, l0 = 0.0f, l1 = 0.0f;
        f32x16 sa[2], sb[2];

        // S^T of tile j
        auto scores = [&](int j, f32x16 (&x)[2]) {
            uint32_t at = lds_address(lds[j & 1]) + kplace;
            asm volatile("" : "+v"(at));  // (computed here: held for every channel step and buffer it would not fit)
#pragma unroll
            for (int b = 0; b < 2; ++b) x[b] = f32x16{};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint4 kf = lds_read16((at ^ (32 * i)) + 32 * b * (D * 2));
                    x[b] = mfma32<FMT>(kf, qf[i], x[b]);
                }
        };
        auto hide = [&](int j, f32x16 (&x)[2]) {  // soft cap, and what the lane's query does not see
            if constexpr (CAP) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        x[b][i] = soft_cap_log2(x[b][i] * p.scale, p.softcap, 1.0f / p.softcap);
            }
            if (64 * j + 63 > wave_full) {
                const int seen = limit - 64 * j - 4 * half;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (32 * b + 8 * (i >> 2) + (i & 3) > seen) x[b][i] = -INFINITY;
            }
        };
        // The maximum moves only when it grows by more than 2^8: weights stay below 2^8.
        auto raise = [&](const f32x16 (&x)[2]) {
            float mx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i] = max_nan(x[0][i], x[1][i]);
#pragma unroll
            for (int i = 4; i < 16; ++i) mx[i & 3] = max_nan(max_nan(mx[i & 3], x[0][i]), x[1][i]);
            const float mn = swap_max(max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]))) * cc;
            if (__ballot(mn > m + 8.0f)) {
                const float to = mn > m ? mn : m;
                const float a = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l0 *= a;
                l1 *= a;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] *= a;
            }
        };
        auto weights = [&](const f32x16 (&x)[2], uint32_t (&pf)[16]) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][i], cc, -m));
                    const float z = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][i + 1], cc, -m));
                    l0 += y;
                    l1 += z;
                    pf[8 * b + (i >> 1)] = pack_pair<FMT>(y, z);
                }
        };
        auto products = [&](int j, const uint32_t (&pf)[16]) {
            uint32_t at = lds_address(lds[2 + (j & 1)]) + vplace;
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    uint2 w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) w[e] = lds_read_transposed((at ^ (64 * d)) + (16 * b + 8 * e) * (D * 2));
                    const uint4 vf = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
                    acc[d] = mfma32<FMT>(vf, make_uint4(pf[4 * b], pf[4 * b + 1], pf[4 * b + 2], pf[4 * b + 3]), acc[d]);
                }
        };
        // Tile j's values have arrived and are about to be used. A weight of 0 times an infinity or a NaN would be a
        // NaN: in the tiles that some rows do not see whole such values become 0, and are added at the end to the rows
        // that see them.
        auto clean = [&](int j) {
            if (64 * j + 63 > full) {
                if (clean_values<D, FMT, THREADS>(lds[2 + (j & 1)], tid)) unseen = 1;
                __syncthreads();
            }
        };
        auto arrive = [&](int j) {
            tile_barrier();  // keys j + 1 and values j are there, keys j and values j - 1 used up
            if (j + 2 < key_tiles) keys(j + 2);
            if (j + 1 < key_tiles) values(j + 1);
            clean(j);
        };
        // One tile: its weights while the next tile's scores are computed, then its products.
        auto step = [&](int j, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
            arrive(j);
            uint32_t pf[16];
            scores(j + 1, nxt);
            weights(cur, pf);
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, (112 + 2 * KS - 1) / (2 * KS), 0);
            }
            // (the weights belong here: left to itself the compiler moves them behind the masks)
            asm volatile("" : "+v"(pf[0]), "+v"(pf[1]), "+v"(pf[2]), "+v"(pf[3]), "+v"(pf[4]), "+v"(pf[5]), "+v"(pf[6]),
                         "+v"(pf[7]), "+v"(pf[8]), "+v"(pf[9]), "+v"(pf[10]), "+v"(pf[11]), "+v"(pf[12]), "+v"(pf[13]),
                         "+v"(pf[14]), "+v"(pf[15]), "+v"(l0), "+v"(l1));
            hide(j + 1, nxt);
            products(j, pf);
            raise(nxt);
        };

        if (key_tiles > from) {
            tile_barrier();
            scores(from, sa);
            hide(from, sa);
            raise(sa);
        }
        int j = from;
        for (; j + 2 < key_tiles; j += 2) {
            step(j, sa, sb);
            step(j + 1, sb, sa);
        }
        if (j + 1 < key_tiles) {
            step(j++, sa, sb);
            sa[0] = sb[0];
            sa[1] = sb[1];
        }
        if (j < key_tiles) {
            uint32_t pf[16];
            arrive(j);
            weights(sa, pf);
            products(j, pf);
        }
        __syncthreads();
        if (unseen) {
            const int unseen_from = (full + 1) & ~63, upto = last < 64 * key_tiles - 1 ? last : 64 * key_tiles - 1;
            for (int key = unseen_from > 64 * from ? unseen_from : 64 * from; key <= upto; ++key) {
                const uint16_t* vp = vbase + key * p.sv_t + 4 * half;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t x = vp[32 * d + 8 * (i >> 2) + (i & 3)];
                        float v, none;
                        unpack_pair<FMT>(x, v, none);
                        if (key <= limit && (x & 0x7FFFu) >= (FMT == BF16 ? 0x7F80u : 0x7C00u)) acc[d][i] += v;
                    }
            }
        }
        // The wave's 32 rows through LDS (the tiles are used up), so that whole rows are written
        constexpr int PITCH = D * 2 + 16;
        static_assert(WAVES * 32 * PITCH <= sizeof(lds), "the rows fit the tiles");
        uint8_t* mine = &lds[0][0] + wave * 32 * PITCH;
        const float sum = swap_sum(l0 + l1);
        const int h = kvh * p.groups + head;
        const int64_t token = seq.q0 + qi;
        if (parts > 1) {  // the part's maximum, sum and products, joined with the others by prompt_join_kernel
            if (row0 + col < total) {
                const int64_t row = (static_cast<int64_t>(part) * p.rows.q_rows + token) * p.q_heads + h;
                if (half == 0) *reinterpret_cast<float2*>(p.part_stats + 2 * row) = make_float2(m, sum);
                float* to = p.part_out + row * D + 4 * half;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(to + 32 * d + 8 * i) =
                            make_float4(acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]);
            }
            continue;
        }
        float scale = 1.0f, den = sum, top = m;
        if (p.sinks) {
            const float sink = p.sinks[h] * kLog2e;
            top = sink > m ? sink : m;
            scale = __builtin_amdgcn_exp2f(m - top);
            den = sum * scale + __builtin_amdgcn_exp2f(sink - top);
        }
        const float inv = den == 0.0f ? 0.0f : scale / den;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint2*>(mine + col * PITCH + (32 * d + 8 * i + 4 * half) * 2) =
                    make_uint2(pack_pair<FMT>(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv),
                               pack_pair<FMT>(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv));
        if (p.lse && half == 0 && row0 + col < total)
            p.lse[h * p.sl_h + token] = (top + __builtin_amdgcn_logf(den)) * 0.6931471805599453f;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 32 * T::CHUNKS / 64; ++i) {
            const int row = (lane + 64 * i) / T::CHUNKS, chunk = (lane + 64 * i) % T::CHUNKS;
            const int r = row0 + row;
            if (r >= total) continue;
            const int q = over_groups(r);
            *reinterpret_cast<uint4*>(p.out + (seq.q0 + q) * p.so_t + (kvh * p.groups + r - q * p.groups) * p.so_h +
                                      chunk * 8) = *reinterpret_cast<const uint4*>(mine + row * PITCH + chunk * 16);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The parts of the rows whose keys were cut (6 prompt chunks of 100 to 612 tokens in two parts: 8 us of 134): four
// channels to a lane, JOINED rows of a row tile to a workgroup.
constexpr int JOINED = 32;

template <int D, int FMT>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptParams p) {
    int pair, first;
    if (!work_of(p.order, blockIdx.x, pair, first)) return;
    const int kvh = pair % p.kv_heads;
    const Sequence seq = sequence_of(p.rows, pair / p.kv_heads);
    const int total = seq.nq * p.groups, tiles = (total + ROWS - 1) / ROWS, offset = seq.nk - seq.nq;
    constexpr int LANES = D / 4;  // to a row
    const int sub = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    for (int t = first; t < tiles; t += p.order.tiles) {
        const int top = (t + 1) * ROWS - 1 < total ? (t + 1) * ROWS - 1 : total - 1;
        const int last = top / p.groups + offset, all_tiles = last < 0 ? 0 : (last >> 6) + 1;
        const int parts = parts_of(p, all_tiles);
        if (parts == 1) continue;
        for (int r = t * ROWS + blockIdx.y * JOINED + sub; r <= top && r < t * ROWS + (blockIdx.y + 1) * JOINED;
             r += 256 / LANES) {
            const int qi = r / p.groups, h = kvh * p.groups + r - qi * p.groups;
            const int64_t token = seq.q0 + qi, row = token * p.q_heads + h, step = p.rows.q_rows * p.q_heads;
            float most = NEVER, den = 0.0f;
            if (p.sinks && p.sinks[h] * kLog2e > NEVER) {
                most = p.sinks[h] * kLog2e;
                den = 1.0f;
            }
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int c0 = 0; c0 < parts; c0 += 4) {  // four parts' loads in flight
                float2 st[4];
                float4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t at = row + (c0 + i < parts ? c0 + i : parts - 1) * step;
                    st[i] = *reinterpret_cast<const float2*>(p.part_stats + 2 * at);
                    x[i] = *reinterpret_cast<const float4*>(p.part_out + at * D + 4 * lane);
                }
                float top4 = most;
#pragma unroll
                for (int i = 0; i < 4; ++i) top4 = st[i].x > top4 ? st[i].x : top4;
                const float a = __builtin_amdgcn_exp2f(most - top4);
                most = top4;
                den *= a;
                y.x *= a;
                y.y *= a;
                y.z *= a;
                y.w *= a;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (c0 + i >= parts) continue;
                    const float w = __builtin_amdgcn_exp2f(st[i].x - most);
                    den += st[i].y * w;
                    y.x += x[i].x * w;
                    y.y += x[i].y * w;
                    y.z += x[i].z * w;
                    y.w += x[i].w * w;
                }
            }
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;
            *reinterpret_cast<uint2*>(p.out + token * p.so_t + h * p.so_h + 4 * lane) =
                make_uint2(pack_pair<FMT>(y.x * inv, y.y * inv), pack_pair<FMT>(y.z * inv, y.w * inv));
            if (p.lse && lane == 0) p.lse[h * p.sl_h + token] = (most + __builtin_amdgcn_logf(den)) * 0.6931471805599453f;
        }
    }
}

size_t part_bytes(int parts, int64_t q_rows, int q_heads, int floats) {
    return static_cast<size_t>(parts) * q_rows * q_heads * floats * sizeof(float);
}

// The parts' workspace has a place for every row, also where a few rows of a large buffer are sequences.
constexpr int64_t MOST_PART_BYTES = 1 << 29;

// Where there are fewer row tiles than workgroups resident at once (two to a CU; one at head dim 256, whose tiles fill
// the LDS), their keys are cut into up to so many parts. With twice the workgroups and with these, 32 heads of 128 on 8:
// a prompt of 4000 tokens 178 and 146 us, 512 tokens behind 8000 98 and 89, 128 behind 16000 82 and 63; 16 heads of 256:
// a prompt of 2000 tokens 111 and 98, 512 behind 30000 410 and 376.
//
// A part holds at least eight tiles of 64 keys, since its rows' sums are written and read once more, or four where the
// row tiles are an eighth of those workgroups or less (with eight and four: one token behind 1000 keys 27 and 17 us, 16
// behind 1000 in 4 sequences 28 and 22, but a prompt of 1000 tokens 29 and 35).
struct Cut {
    int parts, shift;  // up to so many parts, of at least 1 << shift tiles
};

Cut cut_of(int sequences, int64_t q_rows, int max_queries, int max_keys, int q_heads, int kv_heads, int head_dim) {
    if (q_rows == 0) return {1, 0};
    const int64_t groups = q_heads / kv_heads;
    const int64_t by_longest = (max_queries * groups + ROWS - 1) / ROWS * sequences;
    const int64_t by_rows = q_rows * groups / ROWS + sequences;
    const int64_t row_tiles = (by_longest < by_rows ? by_longest : by_rows) * kv_heads;
    const int64_t resident = head_dim == 256 ? 256 : 512;
    const int shift = 8 * row_tiles <= resident ? 2 : 3;
    int64_t most = static_cast<int64_t>(max_keys) / (64 << shift);
    const int64_t fit = MOST_PART_BYTES / static_cast<int64_t>(part_bytes(1, q_rows, q_heads, head_dim + 2));
    most = most < fit ? most : fit;
    const int64_t parts = row_tiles > 0 ? (resident + row_tiles - 1) / row_tiles : 1;
    return {static_cast<int>(parts < 1 || most < 1 ? 1 : parts < most ? parts : most), shift};
}

template <int D, int FMT>
int launch(PromptParams p, int max_queries, int max_keys, hipStream_t stream) {
    const int64_t tiles = (static_cast<int64_t>(max_queries) * p.groups + ROWS - 1) / ROWS;
    // (twice the average where the longest is not known: 24 prompts, 24572 keys: 369 us, 381 as if each had them all)
    const int64_t twice = 2 * p.rows.k_rows / p.rows.sequences, bytes = (twice < max_keys ? twice : max_keys) * D * 4;
    p.order = work_order(p.rows.sequences, p.kv_heads, tiles, p.parts, bytes);
    p.per_group = Divisor(p.groups);
    p.per_kv = Divisor(p.kv_heads);
    p.per_part = Divisor(p.order.tiles / p.parts);
    p.fill = p.fill ? FILLERS : 0;
    const dim3 grid(static_cast<uint32_t>(p.order.blocks() + p.fill));
    if (p.softcap > 0.0f)
        hipLaunchKernelGGL((prompt_attention_kernel<D, FMT, true>), grid, dim3(THREADS), 0, stream, p);
    else
        hipLaunchKernelGGL((prompt_attention_kernel<D, FMT, false>), grid, dim3(THREADS), 0, stream, p);
    if (int rc = check_launch("prompt_attention_kernel")) return rc;
    if (p.parts == 1) return 0;
    p.order = work_order(p.rows.sequences, p.kv_heads, tiles, 1, bytes);
    hipLaunchKernelGGL((prompt_join_kernel<D, FMT>), dim3(static_cast<uint32_t>(p.order.blocks()), ROWS / JOINED),
                       dim3(256), 0, stream, p);
    return check_launch("prompt_join_kernel");
}

template <int FMT>
int launch_dim(const PromptParams& p, int max_queries, int max_keys, hipStream_t stream) {
    if (p.head_dim == 64) return launch<64, FMT>(p, max_queries, max_keys, stream);
    if (p.head_dim == 128) return launch<128, FMT>(p, max_queries, max_keys, stream);
    return launch<256, FMT>(p, max_queries, max_keys, stream);
}

}  // namespace

size_t prompt_attention_workspace(int sequences, int64_t q_rows, int max_queries, int max_keys, int q_heads, int kv_heads,
                                  int head_dim) {
    const int parts = cut_of(sequences, q_rows, max_queries, max_keys, q_heads, kv_heads, head_dim).parts;
    return parts == 1 ? 0 : part_bytes(parts, q_rows, q_heads, head_dim + 2);
}

int prompt_attention(PromptParams p, int format, int max_queries, int max_keys, void* workspace, size_t workspace_bytes,
                     hipStream_t stream) {
    const Cut cut = cut_of(p.rows.sequences, p.rows.q_rows, max_queries, max_keys, p.q_heads, p.kv_heads, p.head_dim);
    p.parts = cut.parts;
    p.part_shift = cut.shift;
    if (p.parts > 1 && (!workspace || workspace_bytes < part_bytes(p.parts, p.rows.q_rows, p.q_heads, p.head_dim + 2)))
        return fail("prompt attention: the workspace is too small");
    p.part_out = static_cast<float*>(workspace);
    p.part_stats = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                            part_bytes(p.parts, p.rows.q_rows, p.q_heads, p.head_dim));
    return format == BF16 ? launch_dim<BF16>(p, max_queries, max_keys, stream)
                          : launch_dim<FP16>(p, max_queries, max_keys, stream);
}

}  // namespace eco
