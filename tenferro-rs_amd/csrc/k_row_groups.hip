// k_row_groups.hip -- rows by group: a stable counting sort of one small index per row.
//
//   offsets[g] = how many rows have an index below g          order = the rows, group by group, each group's ascending
//   positions[order[p]] = p, or -1 for a row of no group      (those stand behind the last group)
//
// No atomic decides an order: a wave takes its rows 64 at a time, the lanes of one index find each other with one ballot
// per bit of it, and the rows of earlier lanes, waves and blocks are counted before.  Up to SMALL_ROWS rows it is one
// launch of one block; beyond that three (counts per block and group, their prefix along the blocks, the placing).
// What bounds it: the small form is latency (a load, two passes over LDS counters, a store); the large one the three
// launches, each of which moves a few megabytes.
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "ragged_api.hpp"

namespace tfh {
namespace ragged {
namespace {

constexpr int WAVES = 16, THREADS = WAVES * 64;
constexpr int ROUNDS = 8;                              // 64 rows each, a wave's share of a block
constexpr int BLOCK_ROWS = WAVES * 64 * ROUNDS;        // 8192
constexpr int SMALL_ROWS = BLOCK_ROWS;

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

// counts[bin][block] -> how many rows of the bin the earlier blocks have; the bin's total behind them at [bins][...].
__global__ __launch_bounds__(256) void group_count_kernel(const GroupArgs a) {
    extern __shared__ int lds_i[];
    const int bins = a.n_groups + 1;
    for (int b = threadIdx.x; b < bins; b += 256) lds_i[b] = 0;
    __syncthreads();
    const int64_t from = (int64_t)blockIdx.x * BLOCK_ROWS;
#pragma unroll 4
    for (int r = threadIdx.x; r < BLOCK_ROWS; r += 256)
        if (from + r < a.n_rows) atomicAdd(&lds_i[key_of(a, (int)(from + r))], 1);   // whole numbers: any order, one result
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256) a.counts[(int64_t)b * a.blocks + blockIdx.x] = lds_i[b];
}
__global__ __launch_bounds__(64) void group_prefix_kernel(const GroupArgs a) {
    int* const row = a.counts + (int64_t)blockIdx.x * a.blocks;
    const int lane = threadIdx.x;
    int before = 0;
    for (int b0 = 0; b0 < a.blocks; b0 += 64) {
        const int c = b0 + lane < a.blocks ? row[b0 + lane] : 0;
        int upto = c;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d, 64);
            if (lane >= d) upto += o;
        }
        if (b0 + lane < a.blocks) row[b0 + lane] = before + upto - c;
        before += __shfl(upto, 63, 64);
    }
    if (lane == 0) a.counts[(int64_t)(a.n_groups + 1) * a.blocks + blockIdx.x] = before;
}

template <bool SMALL>
__global__ __launch_bounds__(THREADS) void group_place_kernel(const GroupArgs a) {
    extern __shared__ int lds_i[];   // [bins] first places, [16], then [waves][bins] counters
    const int bins = a.n_groups + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* const start = lds_i;
    int* const sums = lds_i + bins;
    int* const count = lds_i + bins + 16 + wave * bins;
    int* const counts = lds_i + bins + 16;
    int bits = 32 - __builtin_clz(a.n_groups);
    const int64_t first = (int64_t)blockIdx.x * BLOCK_ROWS + wave * (64 * ROUNDS);
    int key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = first + r * 64 + lane;
        key[r] = i < a.n_rows ? key_of(a, (int)i) : -1;
    }
    for (int i = tid; i < bins * WAVES; i += THREADS) counts[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
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
        start[b] = SMALL ? n : a.counts[(int64_t)bins * a.blocks + b];
    }
    __syncthreads();
    prefix(start, bins, sums);
    if (blockIdx.x == 0)
        for (int b = tid; b < bins; b += THREADS) a.offsets[b] = start[b];
    for (int b = lane; b < bins; b += 64) count[b] += start[b] + (SMALL ? 0 : a.counts[(int64_t)b * a.blocks + blockIdx.x]);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
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
    const int64_t blocks = (n_rows + BLOCK_ROWS - 1) / BLOCK_ROWS;
    return (size_t)(n_groups + 1) * (blocks + 1) * sizeof(int32_t);
}

int32_t launch_group_rows(GroupArgs a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    const int bins = a.n_groups + 1;
    a.blocks = a.n_rows > 0 ? (a.n_rows + BLOCK_ROWS - 1) / BLOCK_ROWS : 1;
    const int lds = (bins * (WAVES + 1) + 16) * (int)sizeof(int);
    if (lds > 64 * 1024) {
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&group_place_kernel<true>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&group_place_kernel<false>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    }
    if (a.n_rows <= SMALL_ROWS) {
        TFH_LAUNCH_TIMED(group_place_kernel<true>, dim3(1), dim3(THREADS), lds, st, a);
    } else {
        hipLaunchKernelGGL(group_count_kernel, dim3(a.blocks), dim3(256), bins * sizeof(int), st, a);
        hipLaunchKernelGGL(group_prefix_kernel, dim3(bins), dim3(64), 0, st, a);
        TFH_LAUNCH_TIMED(group_place_kernel<false>, dim3(a.blocks), dim3(THREADS), lds, st, a);
    }
    return hip_check(hipGetLastError(), "row grouping launch");
}

}  // namespace ragged
}  // namespace tfh
