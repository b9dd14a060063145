// One decode step over a cache held at a budget. The row's new token takes the next free slot, or, when all C are
// filled, the slot of lowest score among those whose token is neither one of the first nor one of the newest (equal
// scores: the lower slot). The token's query heads attend over every filled slot, and each slot's score grows by the
// weight it received, summed over the heads of its KV head.
//
// heavy_attend_kernel: a row's slots are cut into parts, one workgroup each; a wave takes 32 slots at a time, its 16
// query heads as columns (S^T = K Q^T, v_mfma_f32_16x16x32: one head per lane), so P^T is the second product's operand
// with values read transposed from LDS. The scaled scores go to the workspace with the part's maximum, sum and outputs.
// heavy_merge_kernel: the parts' join, and the weights from the scores kept, added to the slots' scores. Every sum has
// a fixed order: no atomics. (The join by the last part of a row to finish, in the same launch, took as long for 2048
// slots of 4 heads, 57.6 us against 55.0, and twice as long for one row of 8192, 83 against 44.)
//
// Bound by HBM: 32 rows of 8 heads and up to 2048 slots of 128 channels take 42 us in the first kernel (5.4 TB/s) and 5
// in the second, 58 us a call; 16 rows of 16 heads and 4096 slots of 256 channels 169 us (6.3 TB/s) and 5. One row of a
// small model (8 heads of 64 on 2, 512 slots) takes 7 and 3 us on the GPU, 15 us a call with the host's part.

#include "eviction.hpp"

namespace eco {

namespace {

constexpr int WAVES = 4;
constexpr int THREADS = WAVES * 64;
constexpr float NEVER = -1e30f;

template <int FMT>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    if constexpr (FMT == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

template <int FMT>
__device__ __forceinline__ uint32_t pair16(float a, float b) {
    if constexpr (FMT == BF16) {
        bf16x2 r;
        r[0] = static_cast<__bf16>(a);
        r[1] = static_cast<__bf16>(b);
        return __builtin_bit_cast(uint32_t, r);
    } else {
        f16x2 r;
        r[0] = static_cast<_Float16>(a);
        r[1] = static_cast<_Float16>(b);
        return __builtin_bit_cast(uint32_t, r);
    }
}

// The slot the new token takes (the same in every workgroup of the row and head).
template <int THREADS>
__device__ __forceinline__ int choose_slot(const BudgetCache& c, int bh, int filled, int token, uint64_t* scratch) {
    if (filled < c.slots) return filled;
    const float* score = c.score + static_cast<int64_t>(bh) * c.slots;
    const int32_t* position = c.position + static_cast<int64_t>(bh) * c.slots;
    uint64_t best = ~0ull;
    constexpr int AT_ONCE = 8;  // slots per thread whose loads are in flight together
    for (int i0 = threadIdx.x; i0 < c.slots; i0 += AT_ONCE * THREADS) {
        int pos[AT_ONCE];
        float sc[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = i0 + j * THREADS < c.slots ? i0 + j * THREADS : c.slots - 1;
            pos[j] = position[i];
            sc[j] = score[i];
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = i0 + j * THREADS < c.slots ? i0 + j * THREADS : c.slots - 1;
            const bool free = pos[j] >= c.first && pos[j] <= token - c.recent;
            const uint64_t key = static_cast<uint64_t>(free ? score_rank(sc[j]) : 0xFFFFFFFFu) << 32 | static_cast<uint32_t>(i);
            best = key < best ? key : best;
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor(best, d);
        best = o < best ? o : best;
    }
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) best = scratch[w] < best ? scratch[w] : best;
    return static_cast<int>(static_cast<uint32_t>(best));
}

constexpr int CHOOSERS = 1024;

__global__ __launch_bounds__(CHOOSERS) void heavy_choose_kernel(HeavyParams p) {
    __shared__ uint64_t scratch[CHOOSERS / 64];
    const int bh = blockIdx.x;
    int filled = p.cache.count[bh];
    filled = filled < 0 ? 0 : (filled > p.cache.slots ? p.cache.slots : filled);
    const int to = choose_slot<CHOOSERS>(p.cache, bh, filled, p.cache.length[bh / p.cache.kv_heads], scratch);
    if (threadIdx.x == 0) p.plan[4 * static_cast<int64_t>(bh)] = to;
}

// 32 slots of one wave in LDS, in chunks of 16 bytes; the swizzles spread the rows of one fragment read (16 rows of 16
// bytes per 16 lanes; transposed: 8 rows of 32 bytes per 32 lanes) over all banks.
template <int D>
struct SlotTile {
    static constexpr int CHUNKS = D / 8;
    static constexpr int BYTES = 32 * D * 2;
    static constexpr int N = 32 * CHUNKS / 64;  // chunks per lane
    static __device__ __forceinline__ int key_at(int row, int chunk) {
        const int c = CHUNKS == 8 ? chunk ^ ((row >> 1) & 7) : chunk ^ (row & 15);
        return row * (D * 2) + c * 16;
    }
    static __device__ __forceinline__ int value_at(int row, int chunk) {
        const int c = CHUNKS == 8 ? chunk ^ (((row >> 1) & 3) << 1) : chunk ^ ((row & 7) << 1);
        return row * (D * 2) + c * 16;
    }
};

template <int D, int FMT>
__global__ __launch_bounds__(THREADS, (D == 256 ? 1 : 2)) void heavy_attend_kernel(HeavyParams p) {
    typedef SlotTile<D> T;
    constexpr int KS = D / 32;  // 32-channel steps of the first product
    constexpr int DT = D / 16;  // 16-channel blocks of the output
    __shared__ __align__(16) uint8_t tiles[WAVES][2][T::BYTES];
    __shared__ uint64_t scratch[WAVES];
    __shared__ float wm[WAVES][16], wl[WAVES][16];

    const BudgetCache& c = p.cache;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, grp = lane >> 4;
    const int bh = blockIdx.x, b = bh / c.kv_heads, h = bh % c.kv_heads;
    const int split = blockIdx.y, block = blockIdx.z;
    uint16_t* keys = c.keys + static_cast<int64_t>(bh) * c.slots * D;
    uint16_t* values = c.values + static_cast<int64_t>(bh) * c.slots * D;
    const int s0 = split * p.span, end = s0 + p.span < c.slots ? s0 + p.span : c.slots;

    // A tile's slots on their way; those past the row's last slot are read from it (any slot may be read: only what is
    // filled is used).
    uint4 kr[T::N], vr[T::N];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < T::N; ++i) {
            const int at = lane + 64 * i;
            int slot = k0 + at / T::CHUNKS;
            slot = slot < end ? slot : end - 1;
            kr[i] = stream_load16(keys + static_cast<int64_t>(slot) * D + at % T::CHUNKS * 8);
            vr[i] = stream_load16(values + static_cast<int64_t>(slot) * D + at % T::CHUNKS * 8);
        }
    };
    const int first_slot = s0 + 32 * wave;
    if (first_slot < end) load(first_slot);  // before anything of the row is known: its slot is chosen meanwhile

    int filled = c.count[bh];
    filled = filled < 0 ? 0 : (filled > c.slots ? c.slots : filled);
    const int token = c.length[b];
    const int head = block * 16 + col;
    const bool head_there = head < p.groups;
    const uint16_t* qp = p.q + b * p.sq_b + (h * p.groups + (head_there ? head : p.groups - 1)) * p.sq_h + grp * 8;
    uint4 qf[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *reinterpret_cast<const uint4*>(qp + 32 * i);
    const uint16_t* new_k = p.k + b * p.sk_b + h * p.sk_h;
    const uint16_t* new_v = p.v + b * p.sv_b + h * p.sv_h;
    int32_t* plan = p.plan + 4 * static_cast<int64_t>(bh);
    const int to = p.chosen ? plan[0] : choose_slot<THREADS>(c, bh, filled, token, scratch);
    const int n = filled < c.slots ? filled + 1 : c.slots;
    if (split == 0 && block == 0 && tid == 0) {
        if (!p.chosen) plan[0] = to;
        plan[1] = n;
        plan[2] = token;
    }
    const int s1 = end < n ? end : n;
    float* logits = p.logits + (static_cast<int64_t>(bh) * p.groups + head) * p.pitch;

    f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{};
    float m = NEVER, l = 0.0f;
    const float c2 = p.scale * kLog2e;
    uint8_t *kl = tiles[wave][0], *vl = tiles[wave][1];
    for (int k0 = first_slot; k0 < s1; k0 += 32 * WAVES) {
#pragma unroll
        for (int i = 0; i < T::N; ++i) {
            const int at = lane + 64 * i, row = at / T::CHUNKS, chunk = at % T::CHUNKS;
            *reinterpret_cast<uint4*>(kl + T::key_at(row, chunk)) = kr[i];
            // (a weight of 0 times what an unfilled slot holds must be 0)
            *reinterpret_cast<uint4*>(vl + T::value_at(row, chunk)) = k0 + row < s1 ? vr[i] : make_uint4(0, 0, 0, 0);
        }
        if (k0 + 32 * WAVES < s1) load(k0 + 32 * WAVES);
        __builtin_amdgcn_wave_barrier();
        if (to >= k0 && to < k0 + 32 && lane < T::CHUNKS) {  // the new token over the one it replaces
            *reinterpret_cast<uint4*>(kl + T::key_at(to - k0, lane)) = reinterpret_cast<const uint4*>(new_k)[lane];
            *reinterpret_cast<uint4*>(vl + T::value_at(to - k0, lane)) = reinterpret_cast<const uint4*>(new_v)[lane];
        }
        __builtin_amdgcn_wave_barrier();
        f32x4 x[2] = {f32x4{}, f32x4{}};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int v = 0; v < 2; ++v)
                x[v] = mfma16<FMT>(*reinterpret_cast<const uint4*>(kl + T::key_at(16 * v + col, 4 * i + grp)), qf[i], x[v]);
        float mx = NEVER;
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int slot = k0 + 16 * v + 4 * grp + r;
                float y = p.softcap > 0.0f ? soft_cap_log2(x[v][r] * p.scale, p.softcap, 1.0f / p.softcap) : x[v][r] * c2;
                if (slot >= s1) y = -INFINITY;
                x[v][r] = y;
                mx = max_nan(mx, y);
            }
#pragma unroll
        for (int v = 0; v < 2; ++v) {  // (rows of the workspace are whole fours)
            const int slot = k0 + 16 * v + 4 * grp;
            if (!head_there || slot >= s1) continue;
            *reinterpret_cast<float4*>(logits + slot) = make_float4(x[v][0], x[v][1], x[v][2], x[v][3]);
        }
        mx = group_max(mx);
        const float mn = mx > m ? mx : m;
        const float a = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= a;
        uint32_t pw[4];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                e[r] = __builtin_amdgcn_exp2f(x[v][r] - m);
                l += e[r];
            }
            pw[2 * v] = pair16<FMT>(e[0], e[1]);
            pw[2 * v + 1] = pair16<FMT>(e[2], e[3]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            typedef short i16x4 __attribute__((ext_vector_type(4)));
            uint2 w[2];
#pragma unroll
            for (int v = 0; v < 2; ++v)
                w[v] = __builtin_bit_cast(
                    uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
                               vl + T::value_at(16 * v + 4 * grp + (col >> 2), 2 * d + ((col & 3) >> 1)) + 8 * (col & 1))));
            acc[d] = mfma16<FMT>(make_uint4(w[0].x, w[0].y, w[1].x, w[1].y), make_uint4(pw[0], pw[1], pw[2], pw[3]),
                                 acc[d]);
        }
        __builtin_amdgcn_wave_barrier();
    }
    // the new token's row, by the part that holds its slot
    if (to >= s0 && to < s1 && block == 0) {
        __syncthreads();  // every wave's reads of the part are done
        for (int i = tid; i < D / 8; i += THREADS) {
            reinterpret_cast<uint4*>(keys + static_cast<int64_t>(to) * D)[i] = reinterpret_cast<const uint4*>(new_k)[i];
            reinterpret_cast<uint4*>(values + static_cast<int64_t>(to) * D)[i] = reinterpret_cast<const uint4*>(new_v)[i];
        }
    }
    // the four waves' join
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (grp == 0) {
        wm[wave][col] = m;
        wl[wave][col] = l;
    }
    __syncthreads();
    float top = wm[0][col];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = wm[w][col] > top ? wm[w][col] : top;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += wl[w][col] * __builtin_amdgcn_exp2f(wm[w][col] - top);
    const float a = __builtin_amdgcn_exp2f(m - top);
    float* joined = reinterpret_cast<float*>(&tiles[0][0][0]);  // [WAVES][16][D + 4]: the slots in it are used up
    constexpr int JP = D + 4;
    static_assert(WAVES * 16 * JP * 4 <= sizeof(tiles), "the join fits the tiles");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        float4 y = make_float4(acc[d][0] * a, acc[d][1] * a, acc[d][2] * a, acc[d][3] * a);
        *reinterpret_cast<float4*>(joined + (wave * 16 + col) * JP + 16 * d + 4 * grp) = y;
    }
    __syncthreads();
    const int heads = p.groups - block * 16 < 16 ? p.groups - block * 16 : 16;
    const int64_t at = (static_cast<int64_t>(bh) * p.splits + split) * p.groups + block * 16;
    for (int i = tid; i < heads * D; i += THREADS) {
        const int g = i / D, d = i % D;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) y += joined[(w * 16 + g) * JP + d];
        p.partial[(at + g) * D + d] = y;
    }
    if (tid < heads) *reinterpret_cast<float2*>(p.stats + 2 * (at + tid)) = make_float2(top, sum);
}

// The maximum and the sum of a head over its parts' (and its sink), by one wave.
__device__ __forceinline__ float2 head_stats(const HeavyParams& p, int bh, int g, int lane) {
    const float2* st = reinterpret_cast<const float2*>(p.stats) + static_cast<int64_t>(bh) * p.splits * p.groups + g;
    float top = NEVER, sum = 0.0f;
    for (int s = lane; s < p.splits; s += 64) {
        const float2 x = st[static_cast<int64_t>(s) * p.groups];
        const float to = x.x > top ? x.x : top;
        sum = sum * __builtin_amdgcn_exp2f(top - to) + x.y * __builtin_amdgcn_exp2f(x.x - to);
        top = to;
    }
    float most = top;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float o = __shfl_xor(most, d);
        most = o > most ? o : most;
    }
    const float sink = p.sinks ? p.sinks[bh % p.cache.kv_heads * p.groups + g] * kLog2e : NEVER;
    most = sink > most ? sink : most;
    sum *= __builtin_amdgcn_exp2f(top - most);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if (p.sinks) sum += __builtin_amdgcn_exp2f(sink - most);
    return make_float2(most, sum);
}

// The parts' join: the first p.groups workgroups of a row and KV head give one head's output each, the others the
// scores of 4 THREADS slots each.
template <int D, int FMT>
__global__ __launch_bounds__(THREADS) void heavy_merge_kernel(HeavyParams p) {
    const BudgetCache& c = p.cache;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int bh = blockIdx.x, b = bh / c.kv_heads, h = bh % c.kv_heads;
    const int32_t* plan = p.plan + 4 * static_cast<int64_t>(bh);
    const int to = plan[0], n = plan[1], token = plan[2];
    if (static_cast<int>(blockIdx.y) < p.groups) {
        constexpr int SHARES = THREADS / D;  // threads to a channel, each a share of the parts
        __shared__ float shares[THREADS];
        const int g = blockIdx.y, d = tid % D, share = tid / D;
        const float2 st = head_stats(p, bh, g, lane);
        const float2* stats = reinterpret_cast<const float2*>(p.stats) + static_cast<int64_t>(bh) * p.splits * p.groups + g;
        const float* x = p.partial + (static_cast<int64_t>(bh) * p.splits * p.groups + g) * D + d;
        float y = 0.0f;
        for (int s0 = share; s0 < p.splits; s0 += 8 * SHARES) {  // eight parts' loads in flight
            float m[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int s = s0 + i * SHARES < p.splits ? s0 + i * SHARES : s0;
                m[i] = stats[static_cast<int64_t>(s) * p.groups].x;
                v[i] = x[static_cast<int64_t>(s) * p.groups * D];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (s0 + i * SHARES < p.splits) y += v[i] * __builtin_amdgcn_exp2f(m[i] - st.x);
        }
        if constexpr (SHARES > 1) {
            shares[tid] = y;
            __syncthreads();
            if (share > 0) return;
            y = 0.0f;
#pragma unroll
            for (int i = 0; i < SHARES; ++i) y += shares[i * D + d];
        }
        p.out[b * p.so_b + (h * p.groups + g) * p.so_h + d] =
            static_cast<uint16_t>(pair16<FMT>(y / st.y, 0.0f) & 0xFFFFu);
        return;
    }
    __shared__ float lse[64];
    for (int g = wave; g < p.groups; g += WAVES) {
        const float2 st = head_stats(p, bh, g, lane);
        if (lane == 0) lse[g] = st.x + __builtin_amdgcn_logf(st.y);
    }
    __syncthreads();
    const int s0 = (blockIdx.y - p.groups) * 4 * THREADS;
    const float* x = p.logits + static_cast<int64_t>(bh) * p.groups * p.pitch;
    float* score = c.score + static_cast<int64_t>(bh) * c.slots;
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f}, old[4];
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        at[i] = s0 + tid + i * THREADS;
        at[i] = at[i] < n ? at[i] : n - 1;
        old[i] = score[at[i]];
    }
#pragma unroll 4
    for (int g = 0; g < p.groups; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(x[static_cast<int64_t>(g) * p.pitch + at[i]] - lse[g]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (s0 + tid + i * THREADS < n) score[at[i]] = (at[i] == to ? 0.0f : old[i]) + w[i];
    if (s0 == 0 && tid == 0) {
        c.position[static_cast<int64_t>(bh) * c.slots + to] = token;
        c.count[bh] = n;
        if (h == 0) c.length[b] = token + 1;
    }
}

struct Plan {
    int splits, span, pitch;
    size_t logits, partial, stats, plan;
    size_t total() const { return logits + partial + stats + plan; }
};

Plan make_plan(int batch, int q_heads, int kv_heads, int slots, int head_dim) {
    Plan r;
    const int64_t groups = q_heads / kv_heads, rows = static_cast<int64_t>(batch) * kv_heads;
    // as many workgroups as are resident at once on 256 CUs: one per CU at head dim 256 (its tiles fill the LDS), two
    // below (16 rows of 16 heads and 4096 slots of 256 channels: 177 us at one, 182 at two, 198 at four; 32 rows of 8
    // heads and 2048 of 128: 59 at one, 58 at two, 61 at four, 66 at six), but at least 128 slots (a step of the four
    // waves) to each
    const int64_t per_cu = head_dim == 256 ? 1 : 2;
    int64_t splits = (per_cu * 256 + rows - 1) / rows;
    const int64_t most = (slots + 127) / 128;
    splits = splits > most ? most : splits;
    r.span = static_cast<int>(((slots + splits - 1) / splits + 127) / 128 * 128);
    r.splits = (slots + r.span - 1) / r.span;
    r.pitch = (slots + 3) / 4 * 4;
    auto align = [](size_t x) { return (x + 255) / 256 * 256; };
    r.logits = align(sizeof(float) * rows * groups * r.pitch);
    r.partial = align(sizeof(float) * rows * r.splits * groups * head_dim);
    r.stats = align(sizeof(float) * rows * r.splits * groups * 2);
    r.plan = align(sizeof(int32_t) * rows * 4);
    return r;
}

template <int D, int FMT>
int launch(const HeavyParams& p, hipStream_t stream) {
    const BudgetCache& c = p.cache;
    const dim3 grid(c.batch * c.kv_heads, p.splits, ceil_div(p.groups, 16));
    if (p.chosen) {
        hipLaunchKernelGGL(heavy_choose_kernel, dim3(grid.x), dim3(CHOOSERS), 0, stream, p);
        if (int rc = check_launch("heavy_choose_kernel")) return rc;
    }
    hipLaunchKernelGGL((heavy_attend_kernel<D, FMT>), grid, dim3(THREADS), 0, stream, p);
    if (int rc = check_launch("heavy_attend_kernel")) return rc;
    hipLaunchKernelGGL((heavy_merge_kernel<D, FMT>), dim3(grid.x, p.groups + ceil_div(c.slots, 4 * THREADS)), dim3(THREADS),
                       0, stream, p);
    return check_launch("heavy_merge_kernel");
}

template <int FMT>
int launch_dim(const HeavyParams& p, hipStream_t stream) {
    if (p.cache.head_dim == 64) return launch<64, FMT>(p, stream);
    if (p.cache.head_dim == 128) return launch<128, FMT>(p, stream);
    return launch<256, FMT>(p, stream);
}

}  // namespace

size_t heavy_hitter_workspace(int batch, int q_heads, int kv_heads, int slots, int head_dim) {
    return make_plan(batch, q_heads, kv_heads, slots, head_dim).total();
}

int heavy_hitter_decode(HeavyParams p, int format, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const BudgetCache& c = p.cache;
    const Plan r = make_plan(c.batch, p.q_heads, c.kv_heads, c.slots, c.head_dim);
    if (workspace_bytes < r.total()) return fail("heavy-hitter decode: the workspace is too small");
    uint8_t* w = static_cast<uint8_t*>(workspace);
    p.logits = reinterpret_cast<float*>(w);
    p.partial = reinterpret_cast<float*>(w + r.logits);
    p.stats = reinterpret_cast<float*>(w + r.logits + r.partial);
    p.plan = reinterpret_cast<int32_t*>(w + r.logits + r.partial + r.stats);
    p.splits = r.splits;
    p.span = r.span;
    p.pitch = r.pitch;
    // Every workgroup reading all scores and positions of its row costs less than a launch until there are many of both
    // (one row of 8 heads: 8192 slots 17 us either way, 32768 slots 36 us against 40, 131072 slots 129 against 158; 32
    // rows of 2048 slots 60 against 57).
    p.chosen = c.slots >= 16384;
    return format == BF16 ? launch_dim<BF16>(p, stream) : launch_dim<FP16>(p, stream);
}

}  // namespace eco
