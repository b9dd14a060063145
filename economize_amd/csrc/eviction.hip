// Cutting packed prompts to a cache's budget: of the n tokens of a row, every KV head keeps all if they fit C slots,
// else the first `first`, the newest `recent` and the C - first - recent of greatest mass among the rest (equal masses:
// the lower index), in token order.

#include "eviction.hpp"

namespace eco {

namespace {

constexpr int THREADS = 1024;
constexpr int WAVES = THREADS / 64;
constexpr int HELD = 16;    // masses a thread holds in registers
constexpr int COPIES = 4;   // of the histogram: lanes of equal digits would queue at one counter
constexpr int BINS = 2048, COPY = BINS + 4;  // (a bin's copies lie in different banks)

// One workgroup per (row, KV head): the mass of the last token to keep by a radix selection over its 32 bits (digits of
// 11, 11 and 10 bits, histograms in LDS), then the kept tokens' positions and masses in order. Up to HELD THREADS
// tokens are read once; longer rows once per digit and once more for the kept ones. Bound by its dependent rounds, not
// by the 4 bytes a token: 16 rows of 8 heads of 6000 to 8192 tokens take 15 us (one histogram and one load at a time:
// 18 us), a row of 1021 tokens 7. It ends with the first digit whose tokens all stay (a call over 32000 tokens of 8
// heads 42 -> 36 us).
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictParams p) {
    __shared__ __align__(16) uint32_t hist[COPY * COPIES];
    __shared__ uint32_t counts[HELD][WAVES];  // tokens above the last one to keep, and equal to it << 16
    __shared__ uint32_t wave_sum[WAVES], totals;
    __shared__ uint32_t digit, above, inside;  // the digit that holds it, tokens above that digit's and of it
    const BudgetCache& c = p.cache;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
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
    float x[HELD];  // tokens base + tid + i THREADS
    auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int j = base + tid + i * THREADS;
            if (base + i * THREADS < n) x[i] = mass[j < n ? j : n - 1];
        }
    };
    constexpr int SPAN = HELD * THREADS;
    load(0);
    uint32_t prefix = 0, mask = 0;
    if (need > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            const uint32_t bins = 1u << bits;
            for (uint32_t i = tid; i < COPY * COPIES / 4; i += THREADS)
                reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (int base = 0; base < hi; base += SPAN) {
                if (n > SPAN) load(base);
#pragma unroll
                for (int i = 0; i < HELD; ++i) {
                    if (base + i * THREADS >= hi) break;
                    const int j = base + tid + i * THREADS;
                    const uint32_t r = score_rank(x[i]);
                    if (j >= lo && j < hi && (r & mask) == prefix)
                        atomicAdd(&hist[(lane & (COPIES - 1)) * COPY + ((r >> shift) & (bins - 1))], 1u);
                }
            }
            __syncthreads();
            // the digit whose tokens take the count past `need`: suffix sums over two bins per thread
            const uint32_t top = bins - 1 - 2 * tid;
            uint32_t mine0 = 0, mine1 = 0;
            if (2 * tid < bins) {
#pragma unroll
                for (int i = 0; i < COPIES; ++i) {
                    mine0 += hist[i * COPY + top];
                    mine1 += hist[i * COPY + top - 1];
                }
            }
            uint32_t run = mine0 + mine1;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t y = __shfl_up(run, d);
                if (lane >= d) run += y;
            }
            if (lane == 63) wave_sum[wave] = run;
            __syncthreads();
            uint32_t before = run - mine0 - mine1;
            for (int w = 0; w < wave; ++w) before += wave_sum[w];
            if (2 * tid < bins) {
                if (before < need && need <= before + mine0) {
                    digit = top;
                    above = before;
                    inside = mine0;
                } else if (before + mine0 < need && need <= before + mine0 + mine1) {
                    digit = top - 1;
                    above = before + mine0;
                    inside = mine1;
                }
            }
            __syncthreads();
            prefix |= digit << shift;
            mask |= (bins - 1) << shift;
            need -= above;
            if (inside == need && prefix > 0) {  // all of the digit stay (mostly one token, by the second digit)
                prefix -= 1;
                need = 0;
                break;
            }
        }
    } else {
        prefix = 0xFFFFFFFFu;  // no candidate stays: none is above, and none of the equal ones is taken
    }
    // tokens above `prefix` stay, and the first `need` of those equal to it
    uint32_t kept = 0, equal = 0;
    for (int base = 0; base < n; base += SPAN) {
        if (n > SPAN) load(base);
        uint32_t over = 0, same = 0;  // this lane's tokens, a bit each
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (base + i * THREADS >= n) {
                if (lane == 0) counts[i][wave] = 0;
                continue;
            }
            const int j = base + tid + i * THREADS;
            const uint32_t r = score_rank(x[i]);
            const bool o = j < n && (j < lo || j >= hi || r > prefix), e = j >= lo && j < hi && r == prefix;
            over |= (o ? 1u : 0u) << i;
            same |= (e ? 1u : 0u) << i;
            const uint32_t packed = __popcll(__ballot(o)) | __popcll(__ballot(e)) << 16;
            if (lane == 0) counts[i][wave] = packed;
        }
        __syncthreads();
        if (wave == 0) {  // their running sums in token order: four entries a lane
            uint32_t* e = &counts[0][0] + 4 * lane;
            uint32_t v[4], run = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = run;
                run += e[i];
            }
            uint32_t upto = run;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t y = __shfl_up(upto, d);
                if (lane >= d) upto += y;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = v[i] + upto - run;
            if (lane == 63) totals = upto;
        }
        __syncthreads();
        const uint64_t below = (1ull << lane) - 1;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (base + i * THREADS >= n) break;
            const bool o = over >> i & 1, e = same >> i & 1;
            const uint64_t os = __ballot(o), es = __ballot(e);
            const uint32_t first = counts[i][wave];
            const uint32_t eq = equal + (first >> 16) + __popcll(es & below);
            const uint32_t at = kept + (first & 0xFFFFu) + __popcll(os & below) + (eq < need ? eq : need);
            if ((o || (e && eq < need)) && at < static_cast<uint32_t>(c.slots)) {
                score[at] = x[i];
                position[at] = base + tid + i * THREADS;
            }
        }
        kept += totals & 0xFFFFu;
        equal += totals >> 16;
        __syncthreads();
    }
}

// The kept tokens' keys and values: one 16-byte chunk per thread, where the launch holds the longest row. Bound by HBM
// (16 rows of 8 heads, 1024 kept of 128 channels: 27 us for 135 MB, 5.0 TB/s); the 15 us of the selection come before
// it.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictParams p) {
    const BudgetCache& c = p.cache;
    const int chunks = c.head_dim / 8;
    const int bh = blockIdx.y, b = bh / c.kv_heads, h = bh % c.kv_heads;
    const int64_t kept = static_cast<int64_t>(c.count[bh]) * chunks;
    int64_t from = p.begin[b];
    from = from < 0 ? 0 : from;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < kept; at += static_cast<int64_t>(gridDim.x) * 256) {
        const int slot = static_cast<int>(at / chunks), chunk = static_cast<int>(at % chunks);
        const int64_t row = from + c.position[static_cast<int64_t>(bh) * c.slots + slot];
        const int64_t to = (static_cast<int64_t>(bh) * c.slots + slot) * c.head_dim + chunk * 8;
        *reinterpret_cast<uint4*>(c.keys + to) =
            *reinterpret_cast<const uint4*>(p.k + row * p.sk_t + h * p.sk_h + chunk * 8);
        *reinterpret_cast<uint4*>(c.values + to) =
            *reinterpret_cast<const uint4*>(p.v + row * p.sv_t + h * p.sv_h + chunk * 8);
    }
}

}  // namespace

int evict_prompt(const EvictParams& p, int max_tokens, hipStream_t stream) {
    const BudgetCache& c = p.cache;
    hipLaunchKernelGGL(evict_select_kernel, dim3(c.batch * c.kv_heads), dim3(THREADS), 0, stream, p);
    if (int rc = check_launch("evict_select_kernel")) return rc;
    const int64_t chunks = static_cast<int64_t>(max_tokens < c.slots ? max_tokens : c.slots) * (c.head_dim / 8);
    const uint32_t blocks = static_cast<uint32_t>(chunks > 256 ? (chunks + 255) / 256 : 1);
    hipLaunchKernelGGL(evict_copy_kernel, dim3(blocks, c.batch * c.kv_heads), dim3(256), 0, stream, p);
    return check_launch("evict_copy_kernel");
}

}  // namespace eco
