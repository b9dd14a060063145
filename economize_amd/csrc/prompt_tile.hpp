// Device pieces shared by the packed-prompt kernels: 32x32x16 products, K/V tiles in LDS, the rows of a sequence.
#pragma once

#include "prompt.hpp"

namespace eco {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int FMT>
__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (FMT == BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// Two floats as a pair of bf16 or fp16, rounded to nearest even.
template <int FMT>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
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

__device__ __forceinline__ float swap_max(float x) {  // the larger of lanes l and l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float swap_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The bounds of one sequence, clamped to the rows of the tensors.
struct Sequence {
    int64_t q0, k0;
    int nq, nk;
};

__device__ __forceinline__ Sequence sequence_of(const PackedRows& r, int s) {
    auto clamp = [](int64_t x, int64_t hi) { return x < 0 ? 0 : (x > hi ? hi : x); };
    Sequence q;
    q.q0 = clamp(r.q_begin[s], r.q_rows);
    q.nq = static_cast<int>(clamp(r.q_end[s], r.q_rows) - q.q0);
    q.k0 = clamp(r.k_begin[s], r.k_rows);
    q.nk = static_cast<int>(clamp(r.k_end[s], r.k_rows) - q.k0);
    if (q.nq < 0) q.nq = 0;
    if (q.nk < 0) q.nk = 0;
    return q;
}

// The sequence of this rank by work, the most first, where there are few: the last workgroups are then short ones (6
// prompt chunks 143 -> 131 us, the masses of 4 prompts 500 -> 460 us). Many even out in any order and lose by it (24
// packed prompts 376 -> 389 us, the last queries of 16 29.4 -> 30.5). Every lane holds one sequence's bounds and counts
// those before it.
__device__ __forceinline__ Sequence ranked_sequence(const PackedRows& r, int rank) {
    if (r.sequences == 1 || r.sequences > SORTED) return sequence_of(r, rank);
    const int lane = threadIdx.x & 63;
    static_assert(SORTED <= 64, "a lane to each");
    const Sequence mine = sequence_of(r, lane < r.sequences ? lane : r.sequences - 1);
    const float work = static_cast<float>(mine.nq) * (2.0f * static_cast<float>(mine.nk) - static_cast<float>(mine.nq));
    int before = 0;
    for (int j = 0; j < r.sequences; ++j) {
        const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(work), j));
        before += other > work || (other == work && j < lane) ? 1 : 0;
    }
    const int from = __builtin_amdgcn_readfirstlane(__ffsll(__ballot(lane < r.sequences && before == rank)) - 1);
    Sequence q;
    q.q0 = __builtin_amdgcn_readlane(static_cast<int>(mine.q0), from);  // (rows are below 2^31)
    q.k0 = __builtin_amdgcn_readlane(static_cast<int>(mine.k0), from);
    q.nq = __builtin_amdgcn_readlane(mine.nq, from);
    q.nk = __builtin_amdgcn_readlane(mine.nk, from);
    return q;
}

// The pair and the tile (0 the longest) of workgroup id; false where there is none.
__device__ __forceinline__ bool work_of(const WorkOrder& o, int id, int& pair, int& tile) {
    const int total = o.pin ? (o.pairs + 7) / 8 : o.pairs;
    const int k = o.pin ? id >> 3 : id;
    const int group = o.whole(k), first = group * o.group, within = k - group * static_cast<int>(o.whole.by);
    const bool last = total - first < o.group;
    tile = last ? o.last_width(within) : o.full_width(within);
    const int p = first + within - tile * static_cast<int>(last ? o.last_width.by : o.full_width.by);
    pair = o.pin ? p * 8 + (id & 7) : p;
    return pair < o.pairs;
}

// The rows of no sequence, by FILLERS workgroups, of which this is `me`: visit(from, to, worker, workers) for its share
// of the gaps before, between and behind the sequences. (Gaps side by side: one after the other each costs a chain of
// two loads.)
template <typename Visit>
__device__ __forceinline__ void for_gaps(const int32_t* begin, const int32_t* end, int sequences, int64_t rows, int me, Visit visit) {
    const int gaps = sequences + 1, at_once = gaps < 32 ? gaps : 32;
    const int worker = me / at_once, workers = FILLERS / at_once;
    if (worker >= workers) return;
    for (int g = me - worker * at_once; g < gaps; g += at_once) {
        int64_t from = g == 0 ? 0 : end[g - 1];
        int64_t to = g == sequences ? rows : begin[g];
        from = from < 0 ? 0 : from;
        to = to > rows ? rows : to;
        if (from < to) visit(from, to, worker, workers);
    }
}

// A tile of 64 rows of D 16-bit channels in LDS, in chunks of 16 bytes. Keys are read as MFMA operands of 32 rows by 16
// channels (ds_read_b128, lane l row l % 32), values transposed (ds_read_b64_tr_b16, 4 rows by 64 bytes for 32 lanes);
// the two swizzles spread the rows of one such read over all 64 banks.
template <int D>
struct Tile {
    static constexpr int CHUNKS = D / 8;
    static constexpr int BYTES = 64 * D * 2;
    static __device__ __forceinline__ int key_chunk(int row, int chunk) {
        return CHUNKS == 8 ? chunk ^ ((row >> 1) & 7) : chunk ^ (row & 15);
    }
    static __device__ __forceinline__ int value_chunk(int row, int chunk) {
        return CHUNKS == 8 ? chunk ^ (((row >> 1) & 1) << 2) : chunk ^ ((row & 3) << 2);
    }
};

// Every wave's copies have arrived and its LDS accesses are done, in all waves of the workgroup.
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

typedef __attribute__((address_space(3))) uint8_t lds_byte;

__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_byte*)p));
}

__device__ __forceinline__ uint4 lds_read16(uint32_t at) {
    return __builtin_bit_cast(
        uint4, *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>((lds_byte*)static_cast<uintptr_t>(at)));
}

// ds_read_b64_tr_b16: the 16 lanes of a group name four rows of 16 elements, lane 4 k + q the eight bytes of row k's
// elements 4 q .. 4 q + 3; lane i receives element i of the four rows.
__device__ __forceinline__ uint2 lds_read_transposed(uint32_t at) {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) i16x4*)static_cast<uintptr_t>(at)));
}

// Copies of 64-row tiles straight into LDS (buffer_load_dwordx4 ... lds: 64 lanes' 16 bytes in a row from the address
// in M0), by a workgroup of THREADS. A lane's place in LDS is fixed, so it fetches the chunk the swizzle puts there.
// Rows past the sequence's end are outside the buffer resource (the whole offset is the lane's: the scalar one is no
// part of the check). The copies of a tile complete at the workgroup's next tile_barrier.
template <int D, int THREADS>
struct TileCopy {
    static constexpr int CHUNKS = D / 8, N = 64 * CHUNKS / THREADS, ROWS = THREADS / CHUNKS;  // rows per instruction
    static constexpr int KINDS = ROWS < 16 ? 16 / ROWS : 1;  // the swizzle repeats every 16 rows
    uint32_t from[KINDS];
    int wave;

    __device__ __forceinline__ TileCopy(int tid, int64_t stride, bool keys) {
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
        for (int i = 0; i < KINDS; ++i) {
            const int row = tid / CHUNKS + i * ROWS, at = tid % CHUNKS;
            const int chunk = keys ? Tile<D>::key_chunk(row, at) : Tile<D>::value_chunk(row, at);
            from[i] = static_cast<uint32_t>(tid / CHUNKS) * static_cast<uint32_t>(stride * 2) + chunk * 16u;
        }
    }

    __device__ __forceinline__ void start(uint8_t* lds, const uint16_t* base, int64_t stride, int row0, int rows) const {
        const int left = rows - row0;
        const int n = left < 64 ? left : 64;
        const uint32_t bytes = n <= 0 ? 0u : static_cast<uint32_t>((n - 1) * stride * 2 + D * 2);
        const uint64_t at = reinterpret_cast<uint64_t>(base + static_cast<int64_t>(row0) * stride);
        typedef int i32x4 __attribute__((ext_vector_type(4)));
        i32x4 rsrc;
        rsrc[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(at));
        rsrc[1] = __builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32) & 0xFFFF);
        rsrc[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
        rsrc[3] = 0x00020000;
        const uint32_t to = lds_address(lds) + wave * 1024u;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t m0 = __builtin_amdgcn_readfirstlane(to + i * (THREADS * 16u));
            uint32_t skip = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(i * ROWS) * static_cast<uint32_t>(stride * 2));
            asm volatile("" : "+s"(skip));  // (added here: the sums held over the loop cost a wave of every SIMD)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :: "s"(m0), "v"(from[i % KINDS] + skip), "s"(rsrc) : "memory");
        }
    }
};

// Infinities and NaN of a tile of values in LDS to 0, by THREADS; whether this thread found one.
template <int D, int FMT, int THREADS>
__device__ __forceinline__ bool clean_values(uint8_t* lds, int tid) {
    constexpr uint32_t LIMIT = FMT == BF16 ? 0x7F80u : 0x7C00u;
    // (a thread's eight chunks together at head dim 256: 8 x 600 tokens of 16 heads 86 -> 82 us; at 128 the longer code slows
    // the loop around it, 8 x 4000 tokens of 32 heads on 8 1071 -> 1084 us)
    constexpr int AT_ONCE = D == 256 ? 8 : 1;
    bool found = false;
#pragma unroll 1
    for (int i0 = tid; i0 < 64 * D / 8; i0 += AT_ONCE * THREADS) {
        uint4 x[AT_ONCE];
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) x[i] = *reinterpret_cast<const uint4*>(lds + (i0 + i * THREADS) * 16);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const uint32_t m = max_magnitude8(x[i]);
            big = m > big ? m : big;
        }
        if (big < LIMIT) continue;
        auto clean = [](uint32_t w) {
            return ((w & 0x7FFFu) >= LIMIT ? 0u : w & 0xFFFFu) | ((w >> 16 & 0x7FFFu) >= LIMIT ? 0u : w & 0xFFFF0000u);
        };
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            *reinterpret_cast<uint4*>(lds + (i0 + i * THREADS) * 16) =
                make_uint4(clean(x[i].x), clean(x[i].y), clean(x[i].z), clean(x[i].w));
        found = true;
    }
    return found;
}

}  // namespace eco
