// Cutting packed prompts to a cache's budget: of the n tokens of a row, every KV head keeps all if they fit C slots, else
// the first `first`, the newest `recent` and the C - first - recent of greatest mass among the rest (equal masses: the
// lower index), in token order.

#include "eviction.hpp"

namespace eco {

namespace {

constexpr int THREADS = 1024;
constexpr int WAVES = THREADS / 64;

// One workgroup per (row, KV head): the mass of the last token to keep by a radix selection over its 32 bits (digits of
// 11, 11 and 10 bits, histograms in LDS), then the kept tokens' positions and masses in order.
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictParams p) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t wave_sum[2][WAVES];
    __shared__ uint32_t digit, above;
    const BudgetCache& c = p.cache;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int b = blockIdx.x / c.kv_heads, h = blockIdx.x % c.kv_heads;
    int64_t from = p.begin[b], to = p.end[b];
    from = from < 0 ? 0 : (from > p.rows ? p.rows : from);
    to = to > p.rows ? p.rows : to;
    const int n = to > from ? static_cast<int>(to - from) : 0;
    const float* mass = p.mass + h * p.sm_h + from;
    float* score = c.score + static_cast<int64_t>(blockIdx.x) * c.slots;
    int32_t* position = c.position + static_cast<int64_t>(blockIdx.x) * c.slots;
    if (tid == 0) {
        c.count[blockIdx.x] = n < c.slots ? n : c.slots;
        if (h == 0) c.length[b] = n;
    }
    if (n <= c.slots) {
        for (int j = tid; j < n; j += THREADS) {
            score[j] = mass[j];
            position[j] = j;
        }
        return;
    }
    const int lo = c.first, hi = n - c.recent;  // candidates [lo, hi)
    uint32_t need = c.slots - c.first - c.recent;  // how many of them stay (< hi - lo)
    uint32_t prefix = 0, mask = 0;
    if (need > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            const uint32_t bins = 1u << bits;
            for (uint32_t i = tid; i < bins; i += THREADS) hist[i] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += THREADS) {
                const uint32_t r = score_rank(mass[j]);
                if ((r & mask) == prefix) atomicAdd(&hist[(r >> shift) & (bins - 1)], 1u);
            }
            __syncthreads();
            // the digit whose tokens take the count past `need`: suffix sums over two bins per thread
            const uint32_t top = bins - 1 - 2 * tid;
            uint32_t mine0 = 0, mine1 = 0;
            if (2 * tid < bins) {
                mine0 = hist[top];
                mine1 = hist[top - 1];
            }
            uint32_t run = mine0 + mine1;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t x = __shfl_up(run, d);
                if (lane >= d) run += x;
            }
            if (lane == 63) wave_sum[0][wave] = run;
            __syncthreads();
            uint32_t before = run - mine0 - mine1;
            for (int w = 0; w < wave; ++w) before += wave_sum[0][w];
            if (2 * tid < bins) {
                if (before < need && need <= before + mine0) {
                    digit = top;
                    above = before;
                } else if (before + mine0 < need && need <= before + mine0 + mine1) {
                    digit = top - 1;
                    above = before + mine0;
                }
            }
            __syncthreads();
            prefix |= digit << shift;
            mask |= (bins - 1) << shift;
            need -= above;
            __syncthreads();
        }
    } else {
        prefix = 0xFFFFFFFFu;  // no candidate stays: none is above, and none of the equal ones is taken
    }
    // tokens above `prefix` stay, and the first `need` of those equal to it
    uint32_t kept = 0, equal = 0;
    for (int j0 = 0; j0 < n; j0 += 4 * THREADS) {
        float x[4];
        uint32_t over = 0, same = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + 4 * tid + i;
            if (j >= n) continue;
            x[i] = mass[j];
            const uint32_t r = score_rank(x[i]);
            if (j < lo || j >= hi || r > prefix) over |= 1u << i;
            else if (r == prefix) same |= 1u << i;
        }
        const uint32_t mine = __popc(over) | __popc(same) << 16;
        uint32_t run = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(run, d);
            if (lane >= d) run += y;
        }
        const int buf = (j0 / (4 * THREADS)) & 1;
        if (lane == 63) wave_sum[buf][wave] = run;
        __syncthreads();
        uint32_t before = run - mine, all = 0;
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += wave_sum[buf][w];
            all += wave_sum[buf][w];
        }
        uint32_t eq = equal + (before >> 16), at = kept + (before & 0xFFFFu) + (eq < need ? eq : need);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = (over >> i & 1) || ((same >> i & 1) && eq < need);
            if (same >> i & 1) ++eq;
            if (in && at < static_cast<uint32_t>(c.slots)) {
                score[at] = x[i];
                position[at] = j0 + 4 * tid + i;
                ++at;
            }
        }
        kept += all & 0xFFFFu;
        equal += all >> 16;
    }
}

// The kept tokens' keys and values: one 16-byte chunk per thread.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictParams p) {
    const BudgetCache& c = p.cache;
    const int chunks = c.head_dim / 8;
    const int bh = blockIdx.y, b = bh / c.kv_heads, h = bh % c.kv_heads;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int slot = static_cast<int>(at / chunks), chunk = static_cast<int>(at % chunks);
    if (slot >= c.count[bh] || slot >= c.slots) return;
    int64_t from = p.begin[b];
    from = from < 0 ? 0 : from;
    int64_t row = from + c.position[static_cast<int64_t>(bh) * c.slots + slot];
    const int64_t to = (static_cast<int64_t>(bh) * c.slots + slot) * c.head_dim + chunk * 8;
    *reinterpret_cast<uint4*>(c.keys + to) = *reinterpret_cast<const uint4*>(p.k + row * p.sk_t + h * p.sk_h + chunk * 8);
    *reinterpret_cast<uint4*>(c.values + to) =
        *reinterpret_cast<const uint4*>(p.v + row * p.sv_t + h * p.sv_h + chunk * 8);
}

}  // namespace

int evict_prompt(const EvictParams& p, int max_tokens, hipStream_t stream) {
    (void)max_tokens;
    const BudgetCache& c = p.cache;
    hipLaunchKernelGGL(evict_select_kernel, dim3(c.batch * c.kv_heads), dim3(THREADS), 0, stream, p);
    if (int rc = check_launch("evict_select_kernel")) return rc;
    const int64_t chunks = static_cast<int64_t>(c.slots) * (c.head_dim / 8);
    hipLaunchKernelGGL(evict_copy_kernel, dim3(static_cast<uint32_t>((chunks + 255) / 256), c.batch * c.kv_heads),
                       dim3(256), 0, stream, p);
    return check_launch("evict_copy_kernel");
}

}  // namespace eco
