// Attention over packed prompts: every sequence's queries attend causally over its own keys.
//
// With x_ij = scale q_i . k_j (soft-capped or not), query i gives o_i = sum_j exp(x_ij - lse_i) v_j over the keys it sees,
// lse_i = log(sum_j exp(x_ij) + exp(sink)). One pass over the keys with a running maximum and sum (both fp32).
//
// A workgroup holds 128 QT rows of one (sequence, KV head): row r is query r / G of head r % G of the group, so the G
// heads of a group share every K/V tile and a tile's rows span few queries (little of the causal diagonal is wasted).
// A wave holds 32 QT rows as columns: S^T = K Q^T puts one query in each lane (l % 32) with 16 of 32 keys in its
// registers, so the softmax needs one exchange with lane l ^ 32 and P^T is already the second product's operand: its eight
// keys per lane are {4 h .. 4 h + 3, 8 + 4 h ..} of 16 (h = l / 32), the order the transposed value reads deliver.
// O^T keeps the query in the lane, so rescaling is one multiplier per lane.

#include "prompt_tile.hpp"

namespace eco {

namespace {

constexpr int WAVES = 4;
constexpr int THREADS = WAVES * 64;
constexpr float NEVER = -1e30f;  // running maximum before the first key (log2 units)

template <int D, int FMT, bool CAP>
__global__ __launch_bounds__(THREADS, (D == 256 ? 1 : 2)) void prompt_attention_kernel(PromptParams p) {
    typedef Tile<D> T;
    constexpr int KS = D / 16;  // 16-channel steps of the first product
    constexpr int DT = D / 32;  // 32-channel blocks of the output
    constexpr int ROWS = WAVES * 32;
    __shared__ __align__(16) uint8_t lds_k[2][T::BYTES];
    __shared__ __align__(16) uint8_t lds_v[2][T::BYTES];
    __shared__ int unseen;  // an infinity or a NaN was taken out of the values of a tile that not every row sees

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, half = lane >> 5;
    const int pairs = p.rows.sequences * p.kv_heads;
    const int per_tile = pairs;
    int id = blockIdx.x;
    if (id >= per_tile * p.tiles) {  // the last workgroups: rows of no sequence
        const int workers = gridDim.x - per_tile * p.tiles, me = id - per_tile * p.tiles;
        for (int g = 0; g <= p.rows.sequences; ++g) {
            int64_t from = g == 0 ? 0 : p.rows.q_end[g - 1];
            int64_t to = g == p.rows.sequences ? p.rows.q_rows : p.rows.q_begin[g];
            from = from < 0 ? 0 : from;
            to = to > p.rows.q_rows ? p.rows.q_rows : to;
            if (to <= from) continue;
            const int64_t chunks = (to - from) * p.q_heads * (D / 8);
            for (int64_t c = static_cast<int64_t>(me) * THREADS + tid; c < chunks; c += static_cast<int64_t>(workers) * THREADS) {
                const int64_t row = c / (D / 8);
                const int64_t t = from + row / p.q_heads;
                const int h = static_cast<int>(row % p.q_heads);
                *reinterpret_cast<uint4*>(p.out + t * p.so_t + h * p.so_h + (c % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
                if (p.lse && c % (D / 8) == 0) p.lse[h * p.sl_h + t] = -INFINITY;
            }
        }
        return;
    }
    const int pair = id % pairs, first = id / pairs;
    const int s = pair / p.kv_heads, kvh = pair % p.kv_heads;
    const Sequence seq = sequence_of(p.rows, s);
    const int64_t total = static_cast<int64_t>(seq.nq) * p.groups;
    const int tiles = static_cast<int>((total + ROWS - 1) / ROWS);
    const int offset = seq.nk - seq.nq;  // query i sees keys <= i + offset
    const uint16_t* kbase = p.k + seq.k0 * p.sk_t + kvh * p.sk_h;
    const uint16_t* vbase = p.v + seq.k0 * p.sv_t + kvh * p.sv_h;
    const float cc = CAP ? 1.0f : p.scale * kLog2e;
    const TileCopy<D> kcopy(tid, p.sk_t, true), vcopy(tid, p.sv_t, false);
    // Fragment places in a tile: keys row l % 32, 8 channels from 8 (l / 32); values transposed, rows 4 (l / 32) + l % 16 / 4,
    // channels 16 (l / 16 % 2) + 4 (l % 4). The swizzles are exclusive-ors of the chunk, so the place of channel step i is the
    // first one's with 32 i (values: 64 d) flipped, and further rows are a constant away.
    const int vrow = 4 * half + ((lane & 15) >> 2);
    const uint32_t kplace = col * (D * 2) + T::key_chunk(col, half) * 16;
    const uint32_t vplace = vrow * (D * 2) + T::value_chunk(vrow, ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;

    for (int t = first; t < tiles; t += p.tiles) {
        const int64_t low_row = static_cast<int64_t>(tiles - 1 - t) * ROWS;  // the longest rows first
        const int64_t row0 = low_row + wave * 32;
        const int64_t r = row0 + col;
        const bool there = r < total;
        const int qi = static_cast<int>((there ? r : total - 1) / p.groups);
        const int head = static_cast<int>((there ? r : total - 1) - static_cast<int64_t>(qi) * p.groups);
        const int limit = there ? qi + offset : -1;
        uint4 qf[KS];
        {
            const uint16_t* qp = p.q + (seq.q0 + qi) * p.sq_t + (kvh * p.groups + head) * p.sq_h + half * 8;
#pragma unroll
            for (int i = 0; i < KS; ++i) qf[i] = *reinterpret_cast<const uint4*>(qp + 16 * i);
        }
        const int64_t top_row = low_row + ROWS - 1 < total ? low_row + ROWS - 1 : total - 1;
        const int last = static_cast<int>(top_row / p.groups) + offset;  // the last key any row of the tile sees
        const int full = static_cast<int>(low_row / p.groups) + offset;  // the last key every row sees
        const int wave_full = static_cast<int>((row0 < total ? row0 : total - 1) / p.groups) + offset;
        const int key_tiles = last < 0 ? 0 : (last >> 6) + 1;

        f32x16 acc[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
        float m = NEVER, l0 = 0.0f, l1 = 0.0f;
        f32x16 sa[2], sb[2];

        auto keys = [&](int j) { kcopy.start(lds_k[j & 1], kbase, p.sk_t, 64 * j, seq.nk); };
        auto values = [&](int j) { vcopy.start(lds_v[j & 1], vbase, p.sv_t, 64 * j, seq.nk); };
        // S^T of tile j
        auto scores = [&](int j, f32x16 (&x)[2]) {
            uint32_t at = lds_address(lds_k[j & 1]) + kplace;
            asm volatile("" : "+v"(at));  // (computed here: held for every channel step and buffer it would not fit)
#pragma unroll
            for (int b = 0; b < 2; ++b) x[b] = f32x16{};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int b = 0; b < 2; ++b) x[b] = mfma32<FMT>(lds_read16((at ^ (32 * i)) + 32 * b * (D * 2)), qf[i], x[b]);
        };
        auto hide = [&](int j, f32x16 (&x)[2]) {  // soft cap, and what the lane's query does not see
            if constexpr (CAP) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[b][i] = soft_cap_log2(x[b][i] * p.scale, p.softcap, 1.0f / p.softcap);
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
        auto top_of = [&](const f32x16 (&x)[2]) {
            float mx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i] = max_nan(x[0][i], x[1][i]);
#pragma unroll
            for (int i = 4; i < 16; ++i) mx[i & 3] = max_nan(max_nan(mx[i & 3], x[0][i]), x[1][i]);
            return max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
        };
        // The maximum moves only when it grows by more than 2^8: weights stay below 2^8.
        auto raise = [&](float mx) {
            const float mn = swap_max(mx) * cc;
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
            uint32_t at = lds_address(lds_v[j & 1]) + vplace;
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    uint2 w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) w[e] = lds_read_transposed((at ^ (64 * d)) + (16 * b + 8 * e) * (D * 2));
                    acc[d] = mfma32<FMT>(make_uint4(w[0].x, w[0].y, w[1].x, w[1].y),
                                         make_uint4(pf[4 * b], pf[4 * b + 1], pf[4 * b + 2], pf[4 * b + 3]), acc[d]);
                }
        };
        // Tile j's values have arrived and are about to be used. A weight of 0 times an infinity or a NaN would be a NaN: in
        // the tiles that some rows do not see whole such values become 0, and are added at the end to the rows that see them.
        auto clean = [&](int j) {
            if (64 * j + 63 > full) {
                if (clean_values<D, FMT>(lds_v[j & 1], tid)) unseen = 1;
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
            raise(top_of(nxt));
        };

        tile_barrier();  // the previous row tile's reads are done
        if (tid == 0) unseen = 0;
        if (key_tiles > 0) {
            keys(0);
            values(0);
            if (key_tiles > 1) keys(1);
            tile_barrier();
            scores(0, sa);
            hide(0, sa);
            raise(top_of(sa));
        }
        int j = 0;
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
            for (int key = (full + 1) & ~63; key <= last; ++key) {
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
        const float sum = swap_sum(l0 + l1);
        if (!there) continue;
        const int h = kvh * p.groups + head;
        const int64_t token = seq.q0 + qi;
        float scale = 1.0f, den = sum, top = m;
        if (p.sinks) {
            const float sink = p.sinks[h] * kLog2e;
            top = sink > m ? sink : m;
            scale = __builtin_amdgcn_exp2f(m - top);
            den = sum * scale + __builtin_amdgcn_exp2f(sink - top);
        }
        const float inv = den == 0.0f ? 0.0f : scale / den;
        uint16_t* op = p.out + token * p.so_t + h * p.so_h + 4 * half;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint2*>(op + 32 * d + 8 * i) =
                    make_uint2(pack_pair<FMT>(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv),
                               pack_pair<FMT>(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv));
        if (p.lse && half == 0) p.lse[h * p.sl_h + token] = (top + __builtin_amdgcn_logf(den)) * 0.6931471805599453f;
    }
}

template <int D, int FMT>
int launch(PromptParams p, int max_queries, hipStream_t stream) {
    constexpr int ROWS = WAVES * 32;
    const int64_t rows = static_cast<int64_t>(max_queries) * p.groups;
    int64_t tiles = (rows + ROWS - 1) / ROWS;
    const int64_t pairs = static_cast<int64_t>(p.rows.sequences) * p.kv_heads;
    if (tiles * pairs > (1 << 28)) tiles = (1 << 28) / pairs;
    if (tiles < 1) tiles = 1;
    p.tiles = static_cast<int>(tiles);
    const int fill = p.fill ? 32 : 0;
    const dim3 grid(static_cast<uint32_t>(tiles * pairs + fill));
    if (p.softcap > 0.0f)
        hipLaunchKernelGGL((prompt_attention_kernel<D, FMT, true>), grid, dim3(THREADS), 0, stream, p);
    else
        hipLaunchKernelGGL((prompt_attention_kernel<D, FMT, false>), grid, dim3(THREADS), 0, stream, p);
    return check_launch("prompt_attention_kernel");
}

template <int FMT>
int launch_dim(const PromptParams& p, int max_queries, hipStream_t stream) {
    if (p.head_dim == 64) return launch<64, FMT>(p, max_queries, stream);
    if (p.head_dim == 128) return launch<128, FMT>(p, max_queries, stream);
    return launch<256, FMT>(p, max_queries, stream);
}

}  // namespace

size_t prompt_attention_workspace(int, int, int, int, int, int) { return 0; }

int prompt_attention(const PromptParams& p, int format, int max_queries, int max_keys, void*, size_t,
                     hipStream_t stream) {
    (void)max_keys;
    return format == BF16 ? launch_dim<BF16>(p, max_queries, stream) : launch_dim<FP16>(p, max_queries, stream);
}

}  // namespace eco
