// k_row_groups.hip -- rows by group: a stable counting sort of one small index per row.
//
//   offsets[g] = how many rows have an index below g          order = the rows, group by group, each group's ascending
//   positions[order[p]] = p, or -1 for a row of no group      (those stand behind the last group)
//
// No atomic decides an order: a wave takes its rows 64 at a time, the lanes of one index find each other with one ballot
// per bit of it, and the rows of earlier lanes, waves and blocks are counted before.  Up to SMALL_ROWS rows it is one
// launch of one block; beyond that two (counts per block and group; the placing, each block of which adds up what the blocks
// before it have), or, where that would be many counts to read for every block, three (their prefix along the blocks between).
// What bounds it: the small form is latency (a load, two passes over LDS counters, a store); the large one the
// launches, each of which moves a few megabytes (1 048 576 indices of 64 bits in 256 groups: 20 us, of which counting 4.7, prefixes
// 4.7 and placing 11, 0.84 TB/s together; 33.5 million in 64 groups: 370 us, 2.2 TB/s; 256 rows in 128 groups: 3.5 us).
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "ragged_api.hpp"

namespace tfh {
namespace ragged {
namespace {

constexpr int WAVES = 16, THREADS = WAVES * 64;
constexpr int ROUNDS = 8;                              // 64 rows each, a wave's share of a block
constexpr int FEW_ROUNDS = 4;                          // the same where a block's counters are few (FEW_BINS): twice the blocks (1 M rows
                                                       // of 256 groups: 21 us; with four times the blocks 24)
constexpr int FEW_BINS = 320;
constexpr int SMALL_ROWS = WAVES * 64 * ROUNDS;        // 8192
// Counts that every placing block reads by itself: 64 blocks of 129 take 16 us so in all and 19 with the prefixes' launch, 256
// blocks of 257 take 40 and 21.
constexpr int64_t JOINED_COUNTS = 1 << 14;
constexpr int rounds_for(int64_t bins) { return bins <= FEW_BINS ? FEW_ROUNDS : ROUNDS; }

__device__ __forceinline__ int key_of(const GroupArgs& a, int i) {
    const int64_t at = a.inner == 1 ? (int64_t)i * a.s_outer : (int64_t)(i / a.inner) * a.s_outer + (int64_t)(i % a.inner) * a.s_inner;
    const int64_t id = a.id64 ? ((const int64_t*)a.ids)[at] : (int64_t)((const int32_t*)a.ids)[at];
    return id >= 0 && id < a.n_groups ? (int)id : a.n_groups;
}

// Exclusive prefix over `bins` counters in LDS by the whole block; `sums`: 16 words of LDS.
__device__ void prefix(int* v, int bins, int* sums) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (bins + THREADS - 1) / THREADS, from = tid * per;
    int mine = 0;
    for (int i = from; i < from + per && i < bins; ++i) mine += v[i];
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int before = upto - mine;
    for (int w = 0; w < wave; ++w) before += sums[w];
    for (int i = from; i < from + per && i < bins; ++i) {
        const int c = v[i];
        v[i] = before;
        before += c;
    }
    __syncthreads();
}

template <int R> __global__ __launch_bounds__(THREADS) void group_count_kernel(const GroupArgs a) {
    extern __shared__ int lds_i[];
    const int bins = a.n_groups + 1;
    const int64_t from = (int64_t)blockIdx.x * THREADS * R + threadIdx.x;
    int key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = from + r * THREADS < a.n_rows ? key_of(a, (int)(from + r * THREADS)) : -1;
    for (int b = threadIdx.x; b < bins; b += THREADS) lds_i[b] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (key[r] >= 0) atomicAdd(&lds_i[key[r]], 1);   // whole numbers: any order, one result
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += THREADS) a.counts[(int64_t)blockIdx.x * bins + b] = lds_i[b];
}
// counts[block][bin] -> how many rows of the bin the earlier blocks have; the bins' totals behind the last block's.  A lane a
// bin; the blocks are shared out to the waves.
__global__ __launch_bounds__(THREADS) void group_prefix_kernel(const GroupArgs a) {
    __shared__ int sums[WAVES][64];
    const int bins = a.n_groups + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.x * 64 + lane;
    const int per = (a.blocks + WAVES - 1) / WAVES, from = wave * per, to = from + per < a.blocks ? from + per : a.blocks;
    int mine = 0;
    if (b < bins)
#pragma unroll 8
        for (int k = from; k < to; ++k) mine += a.counts[(int64_t)k * bins + b];
    sums[wave][lane] = mine;
    __syncthreads();
    if (b >= bins) return;
    int before = 0;
    for (int w = 0; w < wave; ++w) before += sums[w][lane];
#pragma unroll 8
    for (int k = from; k < to; ++k) {
        const int c = a.counts[(int64_t)k * bins + b];
        a.counts[(int64_t)k * bins + b] = before;
        before += c;
    }
    if (wave == WAVES - 1) a.counts[(int64_t)a.blocks * bins + b] = before;
}

enum Counted { NONE = 0, JOINED = 1, PREFIXED = 2 };   // one block; counts to add up; their prefixes
template <int COUNTED, int R>
__global__ __launch_bounds__(THREADS) void group_place_kernel(const GroupArgs a) {
    extern __shared__ int lds_i[];   // [bins] first places, [16], [waves][bins] counters, [bins] what earlier blocks have (not NONE)
    const int bins = a.n_groups + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* const start = lds_i;
    int* const sums = lds_i + bins;
    int* const count = lds_i + bins + 16 + wave * bins;
    int* const counts = lds_i + bins + 16;
    int bits = 32 - __builtin_clz(a.n_groups);
    const int64_t first = (int64_t)blockIdx.x * THREADS * R + wave * (64 * R);
    int key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t i = first + r * 64 + lane;
        key[r] = i < a.n_rows ? key_of(a, (int)i) : -1;
    }
    int* const before = counts + WAVES * bins;
    for (int i = tid; i < bins * WAVES; i += THREADS) counts[i] = 0;
    if constexpr (COUNTED == JOINED)
        for (int b = tid; b < bins; b += THREADS) start[b] = before[b] = 0;
    if constexpr (COUNTED == PREFIXED)
        for (int b = tid; b < bins; b += THREADS)
            start[b] = a.counts[(int64_t)a.blocks * bins + b], before[b] = a.counts[(int64_t)blockIdx.x * bins + b];
    __syncthreads();
    if constexpr (COUNTED == JOINED) {
        // the blocks' counts, bins next to each other: (THREADS / P) bins at a time
        const int width = bins <= 64 ? 64 : bins <= 128 ? 128 : 256, part = tid / width, parts = THREADS / width;
        for (int b = tid % width; b < bins; b += width) {
            int earlier = 0, later = 0;
#pragma unroll 16
            for (int k = part; k < a.blocks; k += parts) {
                const int c = a.counts[(int64_t)k * bins + b];
                if (k < (int)blockIdx.x) earlier += c;
                else later += c;
            }
            atomicAdd(&before[b], earlier);
            atomicAdd(&start[b], earlier + later);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (key[r] >= 0) atomicAdd(&count[key[r]], 1);
    __syncthreads();
    // per bin: this block's first place in it, and each wave's
    for (int b = tid; b < bins; b += THREADS) {
        int n = 0;
        for (int w = 0; w < WAVES; ++w) {
            const int c = counts[w * bins + b];
            counts[w * bins + b] = n;
            n += c;
        }
        if (COUNTED == NONE) start[b] = n;
    }
    __syncthreads();
    prefix(start, bins, sums);
    if (blockIdx.x == 0)
        for (int b = tid; b < bins; b += THREADS) a.offsets[b] = start[b];
    for (int b = lane; b < bins; b += 64) count[b] += start[b] + (COUNTED == NONE ? 0 : before[b]);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (first + r * 64 >= a.n_rows) break;
        const bool here = key[r] >= 0;
        uint64_t same = __ballot(here);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((key[r] >> b) & 1);
            same &= (key[r] >> b) & 1 ? set : ~set;
        }
        if (here) {
            const int rank = __popcll(same & ((1ull << lane) - 1)), i = (int)(first + r * 64 + lane);
            const int place = count[key[r]] + rank;
            __builtin_amdgcn_wave_barrier();
            if (rank == 0) count[key[r]] = place + __popcll(same);
            a.order[place] = i;
            if (a.positions) a.positions[i] = key[r] < a.n_groups ? place : -1;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

}  // namespace

size_t group_rows_workspace(int64_t n_rows, int32_t n_groups) {
    if (n_rows <= SMALL_ROWS) return 0;
    const int64_t each = THREADS * rounds_for(n_groups + 1), blocks = (n_rows + each - 1) / each;
    return (size_t)(n_groups + 1) * (blocks + 1) * sizeof(int32_t);
}

namespace {
template <int COUNTED, int R> void launch_place(const GroupArgs& a, hipStream_t st) {
    const int bins = a.n_groups + 1, lds = (bins * (WAVES + 1 + (COUNTED != NONE)) + 16) * (int)sizeof(int);
    if (lds > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&group_place_kernel<COUNTED, R>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    TFH_LAUNCH_NAMED("(group_place_kernel)", (group_place_kernel<COUNTED, R>), dim3((unsigned)a.blocks), dim3(THREADS), lds, st, a);
}
template <int R> void launch_large(const GroupArgs& a, hipStream_t st) {
    const int bins = a.n_groups + 1;
    hipLaunchKernelGGL(group_count_kernel<R>, dim3((unsigned)a.blocks), dim3(THREADS), bins * sizeof(int), st, a);
    if (bins * a.blocks <= JOINED_COUNTS) return launch_place<JOINED, R>(a, st);
    hipLaunchKernelGGL(group_prefix_kernel, dim3((bins + 63) / 64), dim3(THREADS), 0, st, a);
    launch_place<PREFIXED, R>(a, st);
}
}  // namespace

int32_t launch_group_rows(GroupArgs a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    const int rounds = rounds_for(a.n_groups + 1), each = THREADS * rounds;
    a.blocks = a.n_rows <= SMALL_ROWS ? 1 : (a.n_rows + each - 1) / each;
    if (a.n_rows <= THREADS) launch_place<NONE, 1>(a, st);
    else if (a.n_rows <= SMALL_ROWS) launch_place<NONE, ROUNDS>(a, st);
    else if (rounds == ROUNDS) launch_large<ROUNDS>(a, st);
    else launch_large<FEW_ROUNDS>(a, st);
    return hip_check(hipGetLastError(), "row grouping launch");
}

}  // namespace ragged
}  // namespace tfh
