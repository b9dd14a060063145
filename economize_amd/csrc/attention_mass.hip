// The attention weight every key of packed prompts receives: mass[h, j] = sum over the queries i that see key j (all,
// or the last `window` of its sequence) and the query heads of KV head h of exp(x_ij - lse_i), from the softmax
// statistics lse_i the attention left: one product, no running maximum.
//
// A wave holds 32 KT keys as columns in registers and streams the queries of the group's heads through LDS, 64 at a
// time: S = Q K^T puts one key in each lane with 16 of 32 queries in its registers, so a weight is added where it is
// computed, in fp32 and in a fixed order: no atomics, the same bits every time. The products of 32 queries run while
// the weights of the 32 before are computed. All tiles of a (sequence, KV head) walk the queries from the last down, so
// they read the same ones at the same time. Long walks are cut by heads, each a workgroup of its own, summed by
// mass_sum_kernel.
//
// Bound by the matrix instructions and the exponentials together: 32768 tokens, 32 heads of 128 on 8, take 4.0 ms, 1.10
// PFLOP/s (1.31 in a large library product); 4 prompts of 1000 to 8192 tokens 465 us, 1.00. The last 64 queries of 16
// prompts of 501 to 8000 tokens (16 heads of 64 on 4) take 29 us, four times their keys' HBM time: four steps to a
// walk, whose fetches and barriers a workgroup waits for.

#include "prompt_tile.hpp"

namespace eco {

namespace {

constexpr int WAVES = 4;
constexpr int THREADS = WAVES * 64;

template <int D, int FMT, int KT, bool CAP>
__global__ __launch_bounds__(THREADS, KT == 2 || D == 256 ? 2 : D == 128 ? 4 : 5) void attention_mass_kernel(MassParams p) {
    typedef Tile<D> T;
    constexpr int KS = D / 16;
    constexpr int KEYS = WAVES * 32 * KT;
    __shared__ __align__(256) uint8_t lds[2][T::BYTES];
    __shared__ __align__(16) float stat[4][64];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, half = lane >> 5;
    const int work = gridDim.x - p.fill;
    if (static_cast<int>(blockIdx.x) >= work) {  // the last workgroups: keys of no sequence
        for_gaps(p.rows.k_begin, p.rows.k_end, p.rows.sequences, p.rows.k_rows, blockIdx.x - work,
                 [&](int64_t from, int64_t to, int worker, int workers) {
            for (int64_t t = from + worker * THREADS + tid; t < to; t += static_cast<int64_t>(workers) * THREADS)
                for (int h = 0; h < p.kv_heads; ++h) p.mass[h * p.sm_h + t] = 0.0f;
        });
        return;
    }
    int pair, slot;
    if (!work_of(p.order, blockIdx.x, pair, slot)) return;
    const int first = p.per_part(slot), part = slot - first * p.parts, stride = p.order.tiles / p.parts;
    const int s = p.per_kv(pair), kvh = pair - s * p.kv_heads;
    const Sequence seq = ranked_sequence(p.rows, s);
    const int tiles = (seq.nk + KEYS - 1) / KEYS;
    const int offset = seq.nk - seq.nq;
    const int window_begin = p.window > 0 && p.window < seq.nq ? seq.nq - p.window : 0;
    const int heads = p.groups / p.parts;
    const float cc = CAP ? 1.0f : p.scale * kLog2e;
    const TileCopy<D, THREADS> copy(tid, p.sq_t, true);
    const uint32_t place = col * (D * 2) + T::key_chunk(col, half) * 16;

    for (int t = first; t < tiles; t += stride) {  // the first keys are seen by most queries: the longest work first
        int begin = t * KEYS - offset;  // the first query that counts and sees one of the tile's keys
        if (begin < window_begin) begin = window_begin;
        const int per_head = begin < seq.nq ? (seq.nq - begin + 63) / 64 : 0;
        const int steps = per_head * heads;  // of 64 queries, from the last down to `begin`, heads innermost
        const int key0 = t * KEYS + wave * 32 * KT;
        uint4 kf[KT][KS];
        float sum[KT];
#pragma unroll
        for (int u = 0; u < KT; ++u) {
            const int key = key0 + 32 * u + col;
            const uint16_t* kp = p.k + (seq.k0 + (key < seq.nk ? key : seq.nk - 1)) * p.sk_t + kvh * p.sk_h + half * 8;
#pragma unroll
            for (int i = 0; i < KS; ++i) kf[u][i] = *reinterpret_cast<const uint4*>(kp + 16 * i);
            sum[u] = 0.0f;
        }
        float st = 0.0f;  // the next step's statistics, on their way (the first wave's)
        // The step under way (its first query) and the one fetched next (its first query and head).
        int now = 0, next = begin + 64 * (per_head - 1), next_head = 0;
        const uint16_t* qbase = p.q + seq.q0 * p.sq_t + (kvh * p.groups + part * heads) * p.sq_h;
        const float* lbase = p.lse + (kvh * p.groups + part * heads) * p.sl_h + seq.q0;
        auto fetch = [&](int step) {
            copy.start(lds[step & 1], qbase + next_head * p.sq_h, p.sq_t, next, seq.nq);
            if (wave == 0) {
                const int i = next + lane < seq.nq ? next + lane : seq.nq - 1;
                st = lbase[next_head * p.sl_h + i];
            }
        };
        auto arrive = [&](int step) {  // step's queries and statistics are there
            if (wave == 0) stat[step & 3][lane] = st * kLog2e;
            tile_barrier();
            now = next;
            if (++next_head == heads) {
                next_head = 0;
                next -= 64;
            }
            if (step + 1 < steps) fetch(step + 1);
        };
        auto scores = [&](int step, int b, f32x16 (&x)[KT]) {
            uint32_t at = lds_address(lds[step & 1]) + place + b * 32 * (D * 2);
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int u = 0; u < KT; ++u) x[u] = f32x16{};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint4 qf = lds_read16(at ^ (32 * i));
#pragma unroll
                for (int u = 0; u < KT; ++u) x[u] = mfma32<FMT>(qf, kf[u][i], x[u]);
            }
        };
        auto hide = [&](int b, f32x16 (&x)[KT]) {  // soft cap, and the queries that do not see the lane's key
            if constexpr (CAP) {
#pragma unroll
                for (int u = 0; u < KT; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[u][i] = soft_cap_log2(x[u][i] * p.scale, p.softcap, 1.0f / p.softcap);
            }
            const int i0 = now + 32 * b;
            if (key0 + 32 * KT - 1 > i0 + offset || i0 + 31 >= seq.nq) {
#pragma unroll
                for (int u = 0; u < KT; ++u) {
                    const int lo = key0 + 32 * u + col - offset - i0 - 4 * half, hi = seq.nq - i0 - 4 * half;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = 8 * (i >> 2) + (i & 3);
                        if (e < lo || e >= hi) x[u][i] = -INFINITY;
                    }
                }
            }
        };
        auto weights = [&](int step, int b, const f32x16 (&x)[KT]) {
            float4 ls[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                ls[i] = *reinterpret_cast<const float4*>(&stat[step & 3][32 * b + 8 * i + 4 * half]);
#pragma unroll
            for (int u = 0; u < KT; ++u) {
                float part4[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // short sums first: their rounding stays small
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float4 f = ls[i >> 2];
                    const float l = (i & 3) == 0 ? f.x : (i & 3) == 1 ? f.y : (i & 3) == 2 ? f.z : f.w;
                    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], cc, -l));
                    part4[i & 3] = i < 4 ? y : part4[i & 3] + y;
                }
                sum[u] += (part4[0] + part4[1]) + (part4[2] + part4[3]);
            }
        };
        // The products of half b of a step into nxt, under the weights of the half before, in cur.
        auto both = [&](int step, int b, f32x16 (&nxt)[KT], const f32x16 (&cur)[KT]) {
            scores(step, b, nxt);
            weights(b ? step : step - 1, b ^ 1, cur);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, KT, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, (52 * KT + KS - 1) / KS, 0);
            }
#pragma unroll
            for (int u = 0; u < KT; ++u) asm volatile("" : "+v"(sum[u]));  // (the weights belong before the masks)
            hide(b, nxt);
        };
        f32x16 xa[KT], xb[KT];
        tile_barrier();  // the previous tile's reads are done
        if (steps > 0) {
            fetch(0);
            arrive(0);
            scores(0, 0, xa);
            hide(0, xa);
            int step = 0;
            for (; step + 1 < steps; ++step) {
                both(step, 1, xb, xa);
                arrive(step + 1);
                both(step + 1, 0, xa, xb);
            }
            both(step, 1, xb, xa);
            weights(step, 1, xb);
        }
        float* to = p.parts == 1 ? p.mass + kvh * p.sm_h
                                 : p.partial + (static_cast<int64_t>(part) * p.kv_heads + kvh) * p.rows.k_rows;
#pragma unroll
        for (int u = 0; u < KT; ++u) {
            const float all = swap_sum(sum[u]);
            const int key = key0 + 32 * u + col;
            if (half == 0 && key < seq.nk) to[seq.k0 + key] = all;
        }
    }
}

// The parts, in order.
__global__ __launch_bounds__(256) void mass_sum_kernel(MassParams p) {
    const int s = blockIdx.y / p.kv_heads, kvh = blockIdx.y % p.kv_heads;
    const Sequence seq = sequence_of(p.rows, s);
    for (int key = blockIdx.x * 256 + threadIdx.x; key < seq.nk; key += gridDim.x * 256) {
        float sum = 0.0f;
        for (int c = 0; c < p.parts; ++c)
            sum += p.partial[(static_cast<int64_t>(c) * p.kv_heads + kvh) * p.rows.k_rows + seq.k0 + key];
        p.mass[kvh * p.sm_h + seq.k0 + key] = sum;
    }
}

// Long walks are cut by heads: their lengths differ up to the whole, and shorter ones even out (one prompt of 500
// tokens, 32 heads of 128 on 8: 40 us whole, 16 us cut). A window's walks are as long as each other and only gain from
// being many (window 256 over 16 x 4200 keys: 151 us whole, 167 cut; window 512 over 30000: 151 and 135).
int parts_of(int max_queries, bool windowed, int groups) {
    const int64_t steps = (static_cast<int64_t>(max_queries) + 63) / 64 * groups;
    return steps >= (windowed ? 32 : 12) ? groups : 1;
}

template <int D, int FMT, int KT>
int launch(MassParams p, int max_queries, int max_keys, hipStream_t stream) {
    constexpr int KEYS = WAVES * 32 * KT;
    const int64_t pairs = static_cast<int64_t>(p.rows.sequences) * p.kv_heads;
    const int64_t tiles = (static_cast<int64_t>(max_keys) + KEYS - 1) / KEYS;
    const int64_t bytes = static_cast<int64_t>(max_queries) * p.groups * D * 2;
    p.order = work_order(p.rows.sequences, p.kv_heads, tiles, p.parts, bytes);
    p.per_kv = Divisor(p.kv_heads);
    p.per_part = Divisor(p.parts);
    p.fill = p.fill ? FILLERS : 0;
    const dim3 grid(static_cast<uint32_t>(p.order.blocks() + p.fill));
    if (p.softcap > 0.0f)
        hipLaunchKernelGGL((attention_mass_kernel<D, FMT, KT, true>), grid, dim3(THREADS), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_mass_kernel<D, FMT, KT, false>), grid, dim3(THREADS), 0, stream, p);
    if (int rc = check_launch("attention_mass_kernel")) return rc;
    if (p.parts == 1) return 0;
    const int64_t blocks = (static_cast<int64_t>(max_keys) + 255) / 256;
    hipLaunchKernelGGL(mass_sum_kernel, dim3(static_cast<uint32_t>(blocks < 1 ? 1 : blocks), static_cast<uint32_t>(pairs)),
                       dim3(256), 0, stream, p);
    return check_launch("mass_sum_kernel");
}

// Keys to a wave: 32, or 64 of 128 channels, for which every query fragment read from LDS feeds two products, where six
// workgroups to a CU are left. With 32 and 64: 1 x 4000 tokens, 32 heads on 8: 91 and 113 us; 8 x 1000: 55 and 65; 8 x
// 4000: 586 and 566; 1 x 16000: 1045 and 982. Heads of 64 channels are bound by the exponentials, and more waves hide
// more of the rest (1 x 16000 tokens, 16 heads on 4: 407 and 474 us); 256 channels leave no registers for more.
template <int FMT>
int launch_dim(const MassParams& p, int max_queries, int max_keys, hipStream_t stream) {
    if (p.head_dim == 64) return launch<64, FMT, 1>(p, max_queries, max_keys, stream);
    if (p.head_dim == 256) return launch<256, FMT, 1>(p, max_queries, max_keys, stream);
    constexpr int KEYS = WAVES * 64;
    const int64_t by_longest = (static_cast<int64_t>(max_keys) + KEYS - 1) / KEYS * p.rows.sequences;
    const int64_t by_rows = p.rows.k_rows / KEYS + p.rows.sequences;
    const int64_t workgroups = (by_longest < by_rows ? by_longest : by_rows) * p.kv_heads * p.parts;
    return workgroups >= 6 * 256 ? launch<128, FMT, 2>(p, max_queries, max_keys, stream)
                                 : launch<128, FMT, 1>(p, max_queries, max_keys, stream);
}

}  // namespace

size_t attention_mass_workspace(int max_queries, int64_t k_rows, bool windowed, int q_heads, int kv_heads) {
    const int parts = parts_of(max_queries, windowed, q_heads / kv_heads);
    return parts == 1 ? 0 : static_cast<size_t>(parts) * kv_heads * k_rows * sizeof(float);
}

int attention_mass(MassParams p, int format, int max_queries, int max_keys, void* workspace, size_t workspace_bytes,
                   hipStream_t stream) {
    p.parts = parts_of(max_queries, p.window > 0, p.groups);
    const size_t need = attention_mass_workspace(max_queries, p.rows.k_rows, p.window > 0, p.q_heads, p.kv_heads);
    if (need > 0 && (!workspace || workspace_bytes < need)) return fail("attention mass: the workspace is too small");
    p.partial = static_cast<float*>(workspace);
    return format == BF16 ? launch_dim<BF16>(p, max_queries, max_keys, stream)
                          : launch_dim<FP16>(p, max_queries, max_keys, stream);
}

}  // namespace eco
