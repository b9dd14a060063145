// The attention weight every key of packed prompts receives: mass[h, j] = sum over the queries i that see key j (all, or
// the last `window` of its sequence) and the query heads of KV head h of exp(x_ij - lse_i), from the softmax statistics
// lse_i the attention left. No running maximum is needed and no query is read twice by a workgroup.
//
// A wave holds 64 keys as columns in registers and streams the queries of the group's heads through LDS: S = Q K^T puts
// one key in each lane with 16 of 32 queries in its registers, so a weight is added where it is computed, in fp32 and in
// a fixed order: no atomics, the same bits every time.

#include "prompt_tile.hpp"

namespace eco {

namespace {

constexpr int WAVES = 4;
constexpr int THREADS = WAVES * 64;

template <int D, int FMT, int KT, bool CAP>
__global__ __launch_bounds__(THREADS, 2) void attention_mass_kernel(MassParams p) {
    constexpr int KS = D / 16;
    constexpr int KEYS = WAVES * 32 * KT;
    __shared__ __align__(16) uint8_t lds[2][Tile<D>::BYTES];
    __shared__ __align__(16) float stat[2][64];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int work = gridDim.x - p.fill;
    if (static_cast<int>(blockIdx.x) >= work) {  // the last workgroups: keys of no sequence
        const int workers = p.fill, me = blockIdx.x - work;
        for (int g = 0; g <= p.rows.sequences; ++g) {
            int64_t from = g == 0 ? 0 : p.rows.k_end[g - 1];
            int64_t to = g == p.rows.sequences ? p.rows.k_rows : p.rows.k_begin[g];
            from = from < 0 ? 0 : from;
            to = to > p.rows.k_rows ? p.rows.k_rows : to;
            for (int64_t t = from + me * THREADS + tid; t < to; t += static_cast<int64_t>(workers) * THREADS)
                for (int h = 0; h < p.kv_heads; ++h) p.mass[h * p.sm_h + t] = 0.0f;
        }
        return;
    }
    int pair, first;
    if (!work_of(p.order, blockIdx.x, pair, first)) return;
    const int s = pair / p.kv_heads, kvh = pair % p.kv_heads;
    const Sequence seq = sequence_of(p.rows, s);
    const int tiles = (seq.nk + KEYS - 1) / KEYS;
    const int offset = seq.nk - seq.nq;
    const int window_begin = p.window > 0 && p.window < seq.nq ? seq.nq - p.window : 0;
    const float c2 = p.scale * kLog2e, cc = CAP ? 1.0f : c2;

    for (int t = first; t < tiles; t += p.order.tiles) {  // the first keys are seen by most queries: the longest work first
        const int wg0 = t * KEYS;
        const int key0 = wg0 + wave * 32 * KT;
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
        int begin = wg0 - offset;
        if (begin < window_begin) begin = window_begin;
        const int per_head = begin < seq.nq ? (seq.nq - begin + 63) / 64 : 0;
        const int steps = per_head * p.groups;
        TileLoad<D, THREADS> qt;
        float st = 0.0f;
        auto load = [&](int step) {
            const int g = step % p.groups, i0 = begin + 64 * (per_head - 1 - step / p.groups);
            const int head = kvh * p.groups + g;
            qt.load(p.q + seq.q0 * p.sq_t + head * p.sq_h, p.sq_t, i0, seq.nq, tid);
            if (tid < 64)
                st = i0 + tid < seq.nq ? p.lse[head * p.sl_h + seq.q0 + i0 + tid] * kLog2e : INFINITY;
        };
        auto put = [&](int buf) {
            qt.template store<true>(lds[buf], tid);
            if (tid < 64) stat[buf][tid] = st;
        };
        if (steps > 0) load(0);
        __syncthreads();
        if (steps > 0) put(0);
        if (steps > 1) load(1);
        __syncthreads();
        for (int step = 0; step < steps; ++step) {
            const int buf = step & 1;
            if (step + 1 < steps) {
                put(buf ^ 1);
                if (step + 2 < steps) load(step + 2);
            }
            const int i0 = begin + 64 * (per_head - 1 - step / p.groups);
            if (key0 <= i0 + 63 + offset && key0 < seq.nk) {
                const bool masked = key0 + 32 * KT - 1 > i0 + offset || i0 + 63 >= seq.nq;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    f32x16 x[KT];
#pragma unroll
                    for (int u = 0; u < KT; ++u) x[u] = f32x16{};
                    const int row = 32 * b + col;
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        const uint4 qf = *reinterpret_cast<const uint4*>(
                            lds[buf] + row * (D * 2) + Tile<D>::key_chunk(row, 2 * i + half) * 16);
#pragma unroll
                        for (int u = 0; u < KT; ++u) x[u] = mfma32<FMT>(qf, kf[u][i], x[u]);
                    }
                    float4 ls[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        ls[i] = *reinterpret_cast<const float4*>(&stat[buf][32 * b + 8 * i + 4 * half]);
#pragma unroll
                    for (int u = 0; u < KT; ++u) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float4 four = ls[r >> 2];
                            const float l = (r & 3) == 0 ? four.x : (r & 3) == 1 ? four.y : (r & 3) == 2 ? four.z : four.w;
                            float y = x[u][r];
                            if constexpr (CAP) y = soft_cap_log2(y * p.scale, p.softcap, 1.0f / p.softcap);
                            x[u][r] = __builtin_fmaf(y, cc, -l);
                        }
                        if (masked) {
                            asm volatile("" ::: );  // (a branch of its own: as selects the masks would cost every tile)
                            const int key = key0 + 32 * u + col;
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const int i = i0 + 32 * b + 8 * (r >> 2) + 4 * half + (r & 3);
                                if (key > i + offset || i >= seq.nq) x[u][r] = -INFINITY;
                            }
                        }
                        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // short sums first: their rounding stays small
#pragma unroll
                        for (int r = 0; r < 16; ++r) part[r & 3] += __builtin_amdgcn_exp2f(x[u][r]);
                        sum[u] += (part[0] + part[1]) + (part[2] + part[3]);
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < KT; ++u) {
            const float total = swap_sum(sum[u]);
            const int key = key0 + 32 * u + col;
            if (half == 0 && key < seq.nk) p.mass[kvh * p.sm_h + seq.k0 + key] = total;
        }
    }
}

template <int D, int FMT, int KT>
int launch(MassParams p, int max_queries, int max_keys, hipStream_t stream) {
    constexpr int KEYS = WAVES * 32 * KT;
    p.order = work_order(static_cast<int64_t>(p.rows.sequences) * p.kv_heads, (static_cast<int64_t>(max_keys) + KEYS - 1) / KEYS,
                         static_cast<int64_t>(max_queries) * p.groups * D * 2);
    p.fill = p.fill ? 8 : 0;
    const dim3 grid(static_cast<uint32_t>(p.order.blocks() + p.fill));
    if (p.softcap > 0.0f)
        hipLaunchKernelGGL((attention_mass_kernel<D, FMT, KT, true>), grid, dim3(THREADS), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_mass_kernel<D, FMT, KT, false>), grid, dim3(THREADS), 0, stream, p);
    return check_launch("attention_mass_kernel");
}

template <int FMT>
int launch_dim(const MassParams& p, int max_queries, int max_keys, hipStream_t stream) {
    if (p.head_dim == 64) return launch<64, FMT, 2>(p, max_queries, max_keys, stream);
    if (p.head_dim == 128) return launch<128, FMT, 2>(p, max_queries, max_keys, stream);
    return launch<256, FMT, 1>(p, max_queries, max_keys, stream);
}

}  // namespace

int attention_mass(const MassParams& p, int format, int max_queries, int max_keys, hipStream_t stream) {
    return format == BF16 ? launch_dim<BF16>(p, max_queries, max_keys, stream) : launch_dim<FP16>(p, max_queries, max_keys, stream);
}

}  // namespace eco
