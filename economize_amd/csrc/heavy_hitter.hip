// One decode step over a cache held at a budget. The row's new token takes the next free slot, or, when all C are filled,
// the slot of lowest score among those whose token is neither one of the first nor one of the newest (equal scores: the
// lower slot). The token's query heads attend over every filled slot, and each slot's score grows by the weight it
// received, summed over the heads of its KV head.
//
// heavy_attend_kernel: a row's slots are cut into parts, one workgroup each; a wave takes 32 slots at a time, its 16 query
// heads as columns (S^T = K Q^T, v_mfma_f32_16x16x32: one head per lane), so P^T is the second product's operand with
// values read transposed from LDS. The scaled scores go to the workspace with the part's maximum, sum and outputs.
// heavy_merge_kernel: the parts' join, and the weights from the scores kept, added to the slots' scores. Every sum has a
// fixed order: no atomics.

#include <cstdlib>
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
    for (int w = 0; w < WAVES; ++w) best = scratch[w] < best ? scratch[w] : best;
    return static_cast<int>(static_cast<uint32_t>(best));
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
    const int to = choose_slot(c, bh, filled, token, scratch);
    const int n = filled < c.slots ? filled + 1 : c.slots;
    if (split == 0 && block == 0 && tid == 0) {
        int32_t* plan = p.plan + 4 * static_cast<int64_t>(bh);
        plan[0] = to;
        plan[1] = n;
        plan[2] = token;
    }
    const int s1 = end < n ? end : n;
    float* logits = p.logits + (static_cast<int64_t>(bh) * p.groups + head) * c.slots;

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
                if (slot < s1) {
                    if (head_there) logits[slot] = y;
                } else {
                    y = -INFINITY;
                }
                x[v][r] = y;
                mx = max_nan(mx, y);
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
    float* part = p.partial + ((static_cast<int64_t>(bh) * p.splits + split) * p.groups + block * 16) * (D + 2);
    for (int i = tid; i < heads * D; i += THREADS) {
        const int g = i / D, d = i % D;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) y += joined[(w * 16 + g) * JP + d];
        part[g * (D + 2) + 2 + d] = y;
    }
    if (tid < heads) {
        part[tid * (D + 2)] = top;
        part[tid * (D + 2) + 1] = sum;
    }
}

template <int D, int FMT>
__global__ __launch_bounds__(THREADS) void heavy_merge_kernel(HeavyParams p) {
    __shared__ float lse[64], weight[64];
    const BudgetCache& c = p.cache;
    const int tid = threadIdx.x;
    const int bh = blockIdx.x, b = bh / c.kv_heads, h = bh % c.kv_heads;
    const int32_t* plan = p.plan + 4 * static_cast<int64_t>(bh);
    const int to = plan[0], n = plan[1], token = plan[2];
    const int64_t step = static_cast<int64_t>(p.groups) * (D + 2);
    const float* part = p.partial + static_cast<int64_t>(bh) * p.splits * step;
    if (tid < p.groups) {
        float top = NEVER;
        for (int s = 0; s < p.splits; ++s) {
            const float m = part[s * step + tid * (D + 2)];
            top = m > top ? m : top;
        }
        if (p.sinks) {
            const float sink = p.sinks[h * p.groups + tid] * kLog2e;
            top = sink > top ? sink : top;
        }
        float sum = 0.0f;
        for (int s = 0; s < p.splits; ++s)
            sum += part[s * step + tid * (D + 2) + 1] * __builtin_amdgcn_exp2f(part[s * step + tid * (D + 2)] - top);
        if (p.sinks) sum += __builtin_amdgcn_exp2f(p.sinks[h * p.groups + tid] * kLog2e - top);
        lse[tid] = top + __builtin_amdgcn_logf(sum);
        weight[tid] = 1.0f / sum;
        // (the parts' weights are taken relative to `top` again below)
    }
    __syncthreads();
    if (blockIdx.y == 0) {
        for (int i = tid; i < p.groups * D; i += THREADS) {
            const int g = i / D, d = i % D;
            float top = NEVER, y = 0.0f;
            for (int s = 0; s < p.splits; ++s) {
                const float m = part[s * step + g * (D + 2)];
                top = m > top ? m : top;
            }
            if (p.sinks) {
                const float sink = p.sinks[h * p.groups + g] * kLog2e;
                top = sink > top ? sink : top;
            }
            for (int s = 0; s < p.splits; ++s)
                y += part[s * step + g * (D + 2) + 2 + d] * __builtin_amdgcn_exp2f(part[s * step + g * (D + 2)] - top);
            p.out[b * p.so_b + (h * p.groups + g) * p.so_h + d] =
                static_cast<uint16_t>(pair16<FMT>(y * weight[g], 0.0f) & 0xFFFFu);
        }
        if (tid == 0) {
            c.position[static_cast<int64_t>(bh) * c.slots + to] = token;
            c.count[bh] = n;
            if (h == 0) c.length[b] = token + 1;
        }
    }
    const int slot = blockIdx.y * THREADS + tid;
    if (slot < n) {
        const float* x = p.logits + static_cast<int64_t>(bh) * p.groups * c.slots + slot;
        float w = 0.0f;
        for (int g = 0; g < p.groups; ++g) w += __builtin_amdgcn_exp2f(x[static_cast<int64_t>(g) * c.slots] - lse[g]);
        float* score = c.score + static_cast<int64_t>(bh) * c.slots + slot;
        *score = (slot == to ? 0.0f : *score) + w;
    }
}

struct Plan {
    int splits, span;
    size_t logits, partial, plan;
};

Plan make_plan(int batch, int q_heads, int kv_heads, int slots, int head_dim, int cus) {
    Plan r;
    const int groups = q_heads / kv_heads;
    const int64_t rows = static_cast<int64_t>(batch) * kv_heads;
    static const int per = getenv("ECO_HH") ? atoi(getenv("ECO_HH")) : 2;
    int64_t splits = (per * static_cast<int64_t>(cus) + rows - 1) / rows;
    const int64_t most = (slots + 127) / 128;
    splits = splits > most ? most : splits;
    r.span = static_cast<int>(((slots + splits - 1) / splits + 127) / 128 * 128);
    r.splits = (slots + r.span - 1) / r.span;
    auto align = [](size_t x) { return (x + 255) / 256 * 256; };
    r.logits = align(sizeof(float) * rows * groups * slots);
    r.partial = align(sizeof(float) * rows * r.splits * groups * (head_dim + 2));
    r.plan = align(sizeof(int32_t) * rows * 4);
    return r;
}

template <int D, int FMT>
int launch(const HeavyParams& p, hipStream_t stream) {
    const BudgetCache& c = p.cache;
    const int rows = c.batch * c.kv_heads;
    hipLaunchKernelGGL((heavy_attend_kernel<D, FMT>), dim3(rows, p.splits, ceil_div(p.groups, 16)), dim3(THREADS), 0,
                       stream, p);
    if (int rc = check_launch("heavy_attend_kernel")) return rc;
    hipLaunchKernelGGL((heavy_merge_kernel<D, FMT>), dim3(rows, ceil_div(c.slots, THREADS)), dim3(THREADS), 0, stream,
                       p);
    return check_launch("heavy_merge_kernel");
}

template <int FMT>
int launch_dim(const HeavyParams& p, hipStream_t stream) {
    if (p.cache.head_dim == 64) return launch<64, FMT>(p, stream);
    if (p.cache.head_dim == 128) return launch<128, FMT>(p, stream);
    return launch<256, FMT>(p, stream);
}

}  // namespace

size_t heavy_hitter_workspace(int batch, int q_heads, int kv_heads, int slots, int head_dim, int cus) {
    const Plan r = make_plan(batch, q_heads, kv_heads, slots, head_dim, cus);
    return r.logits + r.partial + r.plan;
}

int heavy_hitter_decode(HeavyParams p, int format, void* workspace, size_t workspace_bytes, int cus,
                        hipStream_t stream) {
    const BudgetCache& c = p.cache;
    const Plan r = make_plan(c.batch, p.q_heads, c.kv_heads, c.slots, c.head_dim, cus);
    if (workspace_bytes < r.logits + r.partial + r.plan) return fail("heavy-hitter decode: the workspace is too small");
    uint8_t* w = static_cast<uint8_t*>(workspace);
    p.logits = reinterpret_cast<float*>(w);
    p.partial = reinterpret_cast<float*>(w + r.logits);
    p.plan = reinterpret_cast<int32_t*>(w + r.logits + r.partial);
    p.splits = r.splits;
    p.span = r.span;
    return format == BF16 ? launch_dim<BF16>(p, stream) : launch_dim<FP16>(p, stream);
}

}  // namespace eco
