// ragged_thin.hpp -- the adapters' middle product V[p, :] = scale * X[src(p), :] . F[g] for 16-bit operands: a long k and
// few columns (r <= 128), so that one pass over X is what it costs and the matrix cores are idle most of the time.
//
// A block has 32 rows of one group and all r columns; its eight waves share out k (64 of it at a time), each with the
// operands straight from memory in registers, a step ahead, and add their sums up in LDS.  (Tiles through LDS with every
// wave on the same k would have a few kilobytes in flight per CU; this has 64.)
#pragma once
#include "ragged_fast.hpp"

namespace tfh {
namespace ragged {

constexpr int THIN_WAVES = 8, THIN_ROWS = 32;

// V's row p as a pair of numbers of the operands' type, v = up (hi + lo): 16 bits of it in bf16, 22 in f16, so that it is
// no rounding of its own beside the result's.  f16 alone has a short exponent: its rows are brought to [2^7, 2^8) first.
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
            e = 8 - e;
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

template <class T, bool BKFAST, int YT> constexpr int thin_lds() { return THIN_WAVES * THIN_ROWS * 32 * YT * 4; }

template <class T, bool BKFAST, int YT>
__global__ __launch_bounds__(64 * THIN_WAVES, 1) void ragged_thin_kernel(const Args a) {
    constexpr int TN = 32 * YT, RB = TN / 8;   // RB: chunks of a row of k of F
    extern __shared__ __align__(16) unsigned char smem_raw[];
    char* const lds = (char*)smem_raw;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Tile t;
    if (!find_tile(a, THIN_ROWS, 1, blockIdx.x, t)) return;
    const int row = lane & 31, half = lane >> 5;
    const int64_t s = row < t.rows ? source_row(a, t.first + row) : -1;
    const auto A = __builtin_amdgcn_make_buffer_rsrc((void*)a.A, 0, (int)(uint32_t)((a.a_rows - 1) * a.a_row * 2 + a.K * 2), 0x00020000);
    const auto B = __builtin_amdgcn_make_buffer_rsrc((char*)a.B + t.group * a.b_group * 2, 0,
                                                     (int)(uint32_t)(BKFAST ? (a.N - 1) * a.b_n * 2 + a.K * 2 : (a.K - 1) * a.b_k * 2 + a.N * 2), 0x00020000);
    const uint32_t va = s >= 0 ? (uint32_t)(s * a.a_row * 2) : NOWHERE;
    uint32_t vb[YT];
#pragma unroll
    for (int y = 0; y < YT; ++y) vb[y] = y * 32 + row < a.N ? (uint32_t)((y * 32 + row) * a.b_n * 2) : NOWHERE;
    f32x16 acc[YT];
#pragma unroll
    for (int y = 0; y < YT; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[y][r] = 0;
    // a step: 64 k's, 16 for each h; lane (row, half) has chunk 2 h + half of its row
    constexpr int AHEAD = YT == 1 ? 4 : YT == 2 ? 2 : 1;   // steps whose loads are in flight, by the registers they take
    u32x4 na[AHEAD][4], nb[AHEAD][4 * YT];
    auto load = [&](int k0, u32x4 (&la)[4], u32x4 (&lb)[4 * YT]) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int k = k0 + 16 * h + 8 * half;
            la[h] = __builtin_amdgcn_raw_buffer_load_b128(A, k < a.K && va != NOWHERE ? va + k * 2 : NOWHERE, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4 * YT; ++i) {
            uint32_t v;
            if constexpr (BKFAST) {
                const int k = k0 + 16 * (i / YT) + 8 * half;
                v = k < a.K && vb[i % YT] != NOWHERE ? vb[i % YT] + k * 2 : NOWHERE;
            } else {
                const int id = lane + 64 * i, k = k0 + id / RB, n = (id % RB) * 8;
                v = k < a.K && n < a.N ? (uint32_t)(k * a.b_k * 2) + n * 2 : NOWHERE;
            }
            lb[i] = __builtin_amdgcn_raw_buffer_load_b128(B, v, 0, 0);
        }
    };
    char* const mine = lds + wave * (64 * TN * 2);   // row-fast F: this wave's own tile, to be read across
    constexpr int STRIDE = 64 * THIN_WAVES;
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) load(wave * 64 + d * STRIDE, na[d], nb[d]);   // (beyond K: zeros)
    for (int k0 = wave * 64; k0 < a.K; k0 += AHEAD * STRIDE) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            u32x4 fa[4], fb[4 * YT];
#pragma unroll
            for (int h = 0; h < 4; ++h) fa[h] = na[d][h];
#pragma unroll
            for (int i = 0; i < 4 * YT; ++i) fb[i] = nb[d][i];
            load(k0 + (d + AHEAD) * STRIDE, na[d], nb[d]);
            if constexpr (!BKFAST) {
#pragma unroll
                for (int i = 0; i < 4 * YT; ++i) {
                    const int id = lane + 64 * i;
                    *(u32x4*)(mine + rowfast_at<T, TN>(id / RB, id % RB)) = fb[i];
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 4 * YT; ++i) fb[i] = fragment32<T, TN, false>(mine, (i % YT) * 32, i / YT, lane);
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int y = 0; y < YT; ++y) acc[y] = mma32<T>(fb[h * YT + y], fa[h], acc[y]);
        }
    }
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
    for (int r = wave; r < t.rows; r += THIN_WAVES) {
        float v[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = lane + 64 * i;
            if (c < TN) {
#pragma unroll
                for (int w = 0; w < THIN_WAVES; ++w) v[i] += *(const float*)(lds + w * PART + r * (TN * 4) + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4);
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
