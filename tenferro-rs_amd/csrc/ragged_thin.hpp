// ragged_thin.hpp -- the adapters' middle product V[p, :] = scale * X[src(p), :] . F[g] for 16-bit operands: a long k and
// few columns (r <= 128), so that one pass over X is what it costs and the matrix cores are idle most of the time.
//
// A block has 32 rows of one group and all r columns; its waves share out k, 64 of it at a time, each with tiles of its own
// in LDS that its own loads fill some steps ahead -- whole lines of every row, which loads in operand position would ask for
// in four pieces -- and no barrier until their sums meet.  64 rows by 4096 k's, rank 16: 9 us, bound by the loads' latency; 8192
// rows, rank 32: 14 us from caches (4.8 TB/s), 25 from HBM.
#pragma once
#include "ragged_fast.hpp"

namespace tfh {
namespace ragged {

constexpr int THIN_ROWS = 32;
// Steps that a wave has in LDS or on their way, by what 32 YT columns leave room for.
template <int YT> constexpr int thin_ahead() { return YT == 2 ? 3 : 2; }
template <int YT, int WAVES> constexpr int thin_lds() { return WAVES * thin_ahead<YT>() * (THIN_ROWS + 32 * YT) * 128; }

// V's row p as a pair of numbers of the operands' type, v = up (hi + lo): 16 bits of it in bf16, 22 in f16, so that it is
// no rounding of its own beside the result's.  f16 alone has a short exponent: its rows' largest elements are brought to [2^14, 2^15)
// first, the top of it, so that the others have their 22 bits down to 2^-18 of that, and half of them, as many as a result, to 2^-29.
// `v`: this lane's columns lane, lane + 64.
template <class T>
__device__ __forceinline__ void store_pair(const Args& a, int64_t p, const float (&v)[2], int lane) {
    float down = 1.0f;
    if constexpr (__is_same(T, _Float16)) {
        float most = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float m = __builtin_fabsf(v[i]);
            if (m > most && m < __builtin_inff()) most = m;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
        int e = 0;
        if (most > 0) {
            (void)frexpf(most, &e);
            e = 15 - e;
            e = e > 120 ? 120 : e < -120 ? -120 : e;
        }
        down = ldexpf(1.0f, e);
        if (lane == 0) a.up[p] = ldexpf(1.0f, -e);
    }
    T* const row = (T*)a.C + p * a.c_row;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = lane + 64 * i;
        if (c >= a.pad) continue;
        const float s = c < a.N ? v[i] * down : 0.0f;
        const T hi = (T)s;
        row[c] = hi;
        row[c + a.pad] = __builtin_isfinite((float)hi) ? (T)(s - (float)hi) : (T)0.0f;   // infinity - infinity is no number
    }
}

template <class T, bool BKFAST, int YT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 1) void ragged_thin_kernel(const Args a) {
    constexpr int TN = 32 * YT, RB = TN / 8, AHEAD = thin_ahead<YT>();   // RB: chunks of a row of k of F
    constexpr int SLOT = (THIN_ROWS + TN) * 128, LOADS = 4 + 4 * YT;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    char* const lds = (char*)smem_raw;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Tile t;
    if (!find_tile(a, THIN_ROWS, 1, block_of(a), t)) return;
    const int row = lane & 31, half = lane >> 5;
    const u32x4 A = buffer_of(a.A, (uint32_t)((a.a_rows - 1) * a.a_row * 2 + a.K * 2));
    const u32x4 B = buffer_of((const char*)a.B + t.group * a.b_group * 2, (uint32_t)(BKFAST ? (a.N - 1) * a.b_n * 2 + a.K * 2 : (a.K - 1) * a.b_k * 2 + a.N * 2));
    // k-fast: a load has 8 rows, lane l the chunk (l ^ row) % 8 of row l / 8
    const int cr = lane >> 3, kc = ((lane ^ cr) & 7) * 8;
    uint32_t va[4], vb[4 * YT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + cr;
        const int64_t s = r < t.rows ? source_row(a, t.first + r) : -1;
        va[i] = s >= 0 ? (uint32_t)(s * a.a_row * 2) + kc * 2 : NOWHERE;
    }
#pragma unroll
    for (int i = 0; i < 4 * YT; ++i) {
        if constexpr (BKFAST) {
            vb[i] = 8 * i + cr < a.N ? (uint32_t)((8 * i + cr) * a.b_n * 2) + kc * 2 : NOWHERE;
        } else {
            const int id = lane + 64 * i, k = id / RB, n = ((id % RB) ^ (rowfast_swizzle<T>(k) & (RB - 1))) * 8;
            vb[i] = n < a.N ? (uint32_t)(k * a.b_k * 2) + n * 2 : NOWHERE;
        }
    }
    f32x16 acc[YT];
#pragma unroll
    for (int y = 0; y < YT; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[y][r] = 0;
    const int steps = (a.K + 63) / 64, mine = steps > wave ? (steps - wave + WAVES - 1) / WAVES : 0;   // of this wave
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + wave * (AHEAD * SLOT);
    auto issue = [&](int step, int slot) {   // (behind the last step: nothing)
        const bool there = step < mine;
        const int k0 = (step * WAVES + wave) * 64;
        const uint32_t oa = scalar_of(there ? k0 * 2 : 0), ob = scalar_of(!there ? 0 : BKFAST ? k0 * 2 : (uint32_t)(k0 * a.b_k * 2)), to = scalar_of(lds0 + slot * SLOT);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_to_lds(A, there && k0 + kc < a.K ? va[i] : NOWHERE, oa, to + i * 1024);
#pragma unroll
        for (int i = 0; i < 4 * YT; ++i) {
            const int k = k0 + (BKFAST ? kc : (lane + 64 * i) / RB);
            load_to_lds(B, there && k < a.K ? vb[i] : NOWHERE, ob, to + THIN_ROWS * 128 + i * 1024);
        }
    };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) issue(d, d);
    int slot = 0;
    for (int s = 0; s < mine; ++s) {
        const char* const tile = lds + wave * (AHEAD * SLOT) + slot * SLOT;
        wait_loads<(AHEAD - 1) * LOADS>();
        u32x4 fa[4], fb[4 * YT];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            fa[h] = fragment32<T, THIN_ROWS, true>(tile, 0, h, lane);
#pragma unroll
            for (int y = 0; y < YT; ++y) fb[h * YT + y] = fragment32<T, TN, BKFAST>(tile + THIN_ROWS * 128, y * 32, h, lane);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read, before the slot is filled again
        __builtin_amdgcn_sched_barrier(0);
        issue(s + AHEAD, slot);
        slot = slot + 1 < AHEAD ? slot + 1 : 0;
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int y = 0; y < YT; ++y) acc[y] = mma32<T>(fb[h * YT + y], fa[h], acc[y]);
    }
    wait_loads<0>();
    // the waves' sums, in the order of the waves
    __syncthreads();
    constexpr int PART = THIN_ROWS * TN * 4;
#pragma unroll
    for (int y = 0; y < YT; ++y)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int chunk = (y * 8 + 2 * g + half) ^ (row & 7);
            const f32x4 v = {acc[y][4 * g], acc[y][4 * g + 1], acc[y][4 * g + 2], acc[y][4 * g + 3]};
            *(f32x4*)(lds + wave * PART + row * (TN * 4) + chunk * 16) = v;
        }
    __syncthreads();
    const float scale = (float)a.alpha * (a.scales ? ((const float*)a.scales)[t.group] : 1.0f);
    for (int r = wave; r < t.rows; r += WAVES) {
        float v[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = lane + 64 * i;
            if (c < TN) {
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v[i] += *(const float*)(lds + w * PART + r * (TN * 4) + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4);
                v[i] *= scale;
            }
        }
        const int64_t p = t.first + r;
        if (a.pad > 0) {
            store_pair<T>(a, p, v, lane);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (lane + 64 * i < a.N) ((float*)a.C)[p * a.c_row + lane + 64 * i] = v[i];
        }
    }
}

// Whether it can take a call: as the fast kernel, with at most 128 columns (of a contiguous row of results).
inline bool thin_takes(const Args& a, bool bkfast) {
    if (a.N > 128 || a.c_n != 1 || a.use_beta || a.scatter || a.zero_rest || a.b_group % 8) return false;
    return fast_rows(a.A, a.a_rows, a.a_row, a.a_col, a.K) && (bkfast ? fast_rows(a.B, a.N, a.b_n, a.b_k, a.K) : fast_rows(a.B, a.K, a.b_k, a.b_n, a.N));
}

}  // namespace ragged
}  // namespace tfh
