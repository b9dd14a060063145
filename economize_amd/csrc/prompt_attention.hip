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

template <int D, int FMT, int QT, bool CAP>
__global__ __launch_bounds__(THREADS, (QT * D >= 256 ? 1 : 2)) void prompt_attention_kernel(PromptParams p) {
    constexpr int KS = D / 16;  // 16-channel steps of the first product
    constexpr int DT = D / 32;  // 32-channel blocks of the output
    constexpr int ROWS = WAVES * 32 * QT;
    __shared__ __align__(16) uint8_t lds[2][2][Tile<D>::BYTES];
    __shared__ int unseen;  // an infinity or a NaN was taken out of the values of a tile that not every row sees

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 31, half = lane >> 5;
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
    const float c2 = p.scale * kLog2e;

    for (int t = first; t < tiles; t += p.tiles) {
        const int64_t row0 = static_cast<int64_t>(tiles - 1 - t) * ROWS + wave * 32 * QT;  // the longest rows first
        int qi[QT], head[QT], limit[QT];
        uint4 qf[QT][KS];
        int wave_last = -1, wave_full = 0x7fffffff;
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            int64_t r = row0 + 32 * u + col;
            const bool there = r < total;
            if (!there) r = total - 1;
            qi[u] = static_cast<int>(r / p.groups);
            head[u] = static_cast<int>(r - static_cast<int64_t>(qi[u]) * p.groups);
            limit[u] = there ? qi[u] + offset : -1;
            const uint16_t* qp = p.q + (seq.q0 + qi[u]) * p.sq_t + (kvh * p.groups + head[u]) * p.sq_h + half * 8;
#pragma unroll
            for (int i = 0; i < KS; ++i) qf[u][i] = *reinterpret_cast<const uint4*>(qp + 16 * i);
        }
        {  // the wave's rows: the last key any sees, the last key all see
            const int64_t lo = row0 < total ? row0 : total - 1;
            const int64_t hi = row0 + 32 * QT - 1 < total ? row0 + 32 * QT - 1 : total - 1;
            wave_last = row0 < total ? static_cast<int>(hi / p.groups) + offset : -1;
            wave_full = static_cast<int>(lo / p.groups) + offset;
        }
        const int64_t top_row = static_cast<int64_t>(tiles - t) * ROWS - 1;
        const int last = static_cast<int>((top_row < total ? top_row : total - 1) / p.groups) + offset;
        const int key_tiles = last < 0 ? 0 : (last >> 6) + 1;
        const int64_t low_row = static_cast<int64_t>(tiles - 1 - t) * ROWS;
        const int full = static_cast<int>(low_row / p.groups) + offset;  // every row of the tile sees keys <= full
        // A weight of 0 times an infinity or a NaN would be a NaN: in the tiles that some rows do not see whole such values
        // are stored as 0, and added at the end to the rows that see them.
        auto put = [&](int j, TileLoad<D, THREADS>& kt, TileLoad<D, THREADS>& vt) {
            kt.template store<true>(lds[j & 1][0], tid);
            if (64 * j + 63 > full && vt.template drop_non_finite<FMT>()) unseen = 1;
            vt.template store<false>(lds[j & 1][1], tid);
        };

        f32x16 acc[QT][DT];
        float m[QT], l[QT];
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            m[u] = NEVER;
            l[u] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[u][d] = f32x16{};
        }

        TileLoad<D, THREADS> kt, vt;
        if (key_tiles > 0) {
            kt.load(kbase, p.sk_t, 0, seq.nk, tid);
            vt.load(vbase, p.sv_t, 0, seq.nk, tid);
        }
        __syncthreads();  // the previous row tile's reads are done
        if (tid == 0) unseen = 0;
        __syncthreads();
        if (key_tiles > 0) put(0, kt, vt);
        if (key_tiles > 1) {
            kt.load(kbase, p.sk_t, 64, seq.nk, tid);
            vt.load(vbase, p.sv_t, 64, seq.nk, tid);
        }
        __syncthreads();
        for (int j = 0; j < key_tiles; ++j) {
            const uint8_t *kl = lds[j & 1][0], *vl = lds[j & 1][1];
            if (j + 1 < key_tiles) {  // the next tile: its registers into the other buffer, the one after it on its way
                put(j + 1, kt, vt);
                if (j + 2 < key_tiles) {
                    kt.load(kbase, p.sk_t, 64 * (j + 2), seq.nk, tid);
                    vt.load(vbase, p.sv_t, 64 * (j + 2), seq.nk, tid);
                }
            }
            const int key0 = 64 * j;
            if (key0 <= wave_last) {
                f32x16 sc[QT][2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = 32 * b + col;
#pragma unroll
                    for (int u = 0; u < QT; ++u) sc[u][b] = f32x16{};
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        const uint4 kf = *reinterpret_cast<const uint4*>(
                            kl + row * (D * 2) + Tile<D>::key_chunk(row, 2 * i + half) * 16);
#pragma unroll
                        for (int u = 0; u < QT; ++u) sc[u][b] = mfma32<FMT>(kf, qf[u][i], sc[u][b]);
                    }
                }
                const bool masked = key0 + 63 > wave_full;
                uint32_t pf[QT][16];
#pragma unroll
                for (int u = 0; u < QT; ++u) {
                    if constexpr (CAP) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                sc[u][b][r] = soft_cap_log2(sc[u][b][r] * p.scale, p.softcap, 1.0f / p.softcap);
                    }
                    if (masked) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (key0 + 32 * b + 8 * (r >> 2) + 4 * half + (r & 3) > limit[u]) sc[u][b][r] = -INFINITY;
                    }
                    float mx = sc[u][0][0];
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) mx = max_nan(mx, sc[u][b][r]);
                    mx = swap_max(mx);
                    const float cc = CAP ? 1.0f : c2;
                    const float mn = mx * cc;
                    // the maximum moves only when it grows by more than 2^8: weights stay below 2^8 of it
                    if (__ballot(mn > m[u] + 8.0f)) {
                        const float to = mn > m[u] ? mn : m[u];
                        const float a = __builtin_amdgcn_exp2f(m[u] - to);
                        m[u] = to;
                        l[u] *= a;
#pragma unroll
                        for (int d = 0; d < DT; ++d) acc[u][d] *= a;
                    }
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
#pragma unroll
                        for (int r = 0; r < 16; r += 2) {
                            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][b][r], cc, -m[u]));
                            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][b][r + 1], cc, -m[u]));
                            l[u] += x;
                            l[u] += y;
                            pf[u][8 * b + (r >> 1)] = pack_pair<FMT>(x, y);
                        }
                    }
                }
                // values: rows 16 b + 8 w + 4 half + (lane % 16) / 4, channels 32 d + 16 (lane / 16 % 2) + 4 (lane % 4)
                const int vrow = 4 * half + ((lane & 15) >> 2);
                const int vcol = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), vsub = (lane & 1) * 8;
                auto value = [&](int b, int d) {
                    typedef short i16x4 __attribute__((ext_vector_type(4)));
                    uint2 w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = 16 * b + 8 * e + vrow;
                        const uint8_t* at = vl + row * (D * 2) + Tile<D>::value_chunk(row, 4 * d + vcol) * 16 + vsub;
                        w[e] = __builtin_bit_cast(
                            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(at)));
                    }
                    return make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
                };
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const uint4 w = value(b, d);
#pragma unroll
                        for (int u = 0; u < QT; ++u)
                            acc[u][d] = mfma32<FMT>(w, make_uint4(pf[u][4 * b], pf[u][4 * b + 1], pf[u][4 * b + 2],
                                                                  pf[u][4 * b + 3]), acc[u][d]);
                    }
            }
            __syncthreads();
        }
        if (unseen) {
            for (int key = (full + 1) & ~63; key <= last; ++key) {
                const uint16_t* vp = vbase + key * p.sv_t + 4 * half;
#pragma unroll
                for (int u = 0; u < QT; ++u)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const uint32_t x = vp[32 * d + 8 * (r >> 2) + (r & 3)];
                            float v, none;
                            unpack_pair<FMT>(x, v, none);
                            if (key <= limit[u] && (x & 0x7FFFu) >= (FMT == BF16 ? 0x7F80u : 0x7C00u)) acc[u][d][r] += v;
                        }
            }
        }
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            const float sum = swap_sum(l[u]);
            const int64_t r = row0 + 32 * u + col;
            if (r >= total) continue;
            const int h = kvh * p.groups + head[u];
            const int64_t token = seq.q0 + qi[u];
            float scale = 1.0f, den = sum, top = m[u];
            if (p.sinks) {
                const float sink = p.sinks[h] * kLog2e;
                top = sink > m[u] ? sink : m[u];
                scale = __builtin_amdgcn_exp2f(m[u] - top);
                den = sum * scale + __builtin_amdgcn_exp2f(sink - top);
            }
            const float inv = den == 0.0f ? 0.0f : scale / den;
            uint16_t* op = p.out + token * p.so_t + h * p.so_h + 4 * half;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint2*>(op + 32 * d + 8 * i) =
                        make_uint2(pack_pair<FMT>(acc[u][d][4 * i] * inv, acc[u][d][4 * i + 1] * inv),
                                   pack_pair<FMT>(acc[u][d][4 * i + 2] * inv, acc[u][d][4 * i + 3] * inv));
            if (p.lse && half == 0) p.lse[h * p.sl_h + token] = (top + __builtin_amdgcn_logf(den)) * 0.6931471805599453f;
        }
    }
}

template <int D, int FMT, int QT>
int launch(PromptParams p, int max_queries, hipStream_t stream) {
    constexpr int ROWS = WAVES * 32 * QT;
    const int64_t rows = static_cast<int64_t>(max_queries) * p.groups;
    int64_t tiles = (rows + ROWS - 1) / ROWS;
    const int64_t pairs = static_cast<int64_t>(p.rows.sequences) * p.kv_heads;
    if (tiles * pairs > (1 << 28)) tiles = (1 << 28) / pairs;
    if (tiles < 1) tiles = 1;
    p.tiles = static_cast<int>(tiles);
    const int fill = p.fill ? 32 : 0;
    const dim3 grid(static_cast<uint32_t>(tiles * pairs + fill));
    if (p.softcap > 0.0f)
        hipLaunchKernelGGL((prompt_attention_kernel<D, FMT, QT, true>), grid, dim3(THREADS), 0, stream, p);
    else
        hipLaunchKernelGGL((prompt_attention_kernel<D, FMT, QT, false>), grid, dim3(THREADS), 0, stream, p);
    return check_launch("prompt_attention_kernel");
}

template <int FMT>
int launch_dim(const PromptParams& p, int max_queries, hipStream_t stream) {
    if (p.head_dim == 64) return launch<64, FMT, 1>(p, max_queries, stream);
    if (p.head_dim == 128) return launch<128, FMT, 1>(p, max_queries, stream);
    return launch<256, FMT, 1>(p, max_queries, stream);
}

}  // namespace

size_t prompt_attention_workspace(int, int, int, int, int, int) { return 0; }

int prompt_attention(const PromptParams& p, int format, int max_queries, int max_keys, void*, size_t,
                     hipStream_t stream) {
    (void)max_keys;
    return format == BF16 ? launch_dim<BF16>(p, max_queries, stream) : launch_dim<FP16>(p, max_queries, stream);
}

}  // namespace eco
