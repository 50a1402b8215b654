// ragged_few.hpp -- products of few rows with matrices that are read from memory for them alone (a decoding step): 16-bit
// operands, both contiguous along k.
//
// Bound by how fast the matrices arrive, so a block takes 16 columns only -- 256 blocks for 4096 of them -- and its eight
// waves share k: each asks for its whole share (up to 512 k's, 16 KB) before it multiplies the first of it, straight into
// registers in operand position, and the waves' sums meet in LDS.  The rows come from L2 in every block.
#pragma once
#include "ragged_fast.hpp"

namespace tfh {
namespace ragged {

constexpr int FEW_WAVES = 8;

// TR: blocks of 16 rows.  STEPS: steps of 32 k's that a wave has in flight (4 where its share is no longer, else 16).  rows mode: tiles of a group; shared mode: all rows, the low-rank part group by group.
template <class T, int MODE, int TR, int STEPS>
__global__ __launch_bounds__(64 * FEW_WAVES, 1) void ragged_few_kernel(const Args a) {
    typedef Num<T> NT;
    constexpr int TM = 16 * TR;
    __shared__ __align__(16) float sums[FEW_WAVES][TM][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4, j = lane & 15;
    const int tiles_n = (a.N + 15) / 16;
    Tile t;
    if constexpr (MODE == ROWS) {
        if (!find_tile(a, TM, tiles_n, blockIdx.x, t)) return;
    } else {
        t.group = 0;
        t.tile_n = blockIdx.x % tiles_n;
        t.first = (blockIdx.x / tiles_n) * TM;
        t.rows = a.n_rows - t.first < TM ? (int)(a.n_rows - t.first) : TM;
    }
    const bool real = MODE != ROWS || t.group < a.n_groups;
    const int n0 = t.tile_n * 16, kend = real ? a.K : 0;
    const auto A = __builtin_amdgcn_make_buffer_rsrc((void*)a.A, 0, (int)(uint32_t)((a.a_rows - 1) * a.a_row * 2 + a.K * 2), 0x00020000);
    const auto B = __builtin_amdgcn_make_buffer_rsrc((char*)a.B + (MODE == ROWS && real ? t.group * a.b_group * 2 : 0), 0,
                                                     (int)(uint32_t)((a.N - 1) * a.b_n * 2 + a.K * 2), 0x00020000);
    const uint32_t vb = n0 + j < a.N ? (uint32_t)((n0 + j) * a.b_n * 2) + q * 16 : NOWHERE;
    uint32_t va[TR];
    f32x4 acc[TR], low[TR];
#pragma unroll
    for (int x = 0; x < TR; ++x) {
        const int64_t s = x * 16 + j < t.rows && real ? source_row(a, t.first + x * 16 + j) : -1;
        va[x] = s >= 0 ? (uint32_t)(s * a.a_row * 2) + q * 16 : NOWHERE;
        acc[x] = low[x] = (f32x4){0, 0, 0, 0};
    }
    auto at = [&](uint32_t v, int k) { return v != NOWHERE && k + q * 8 < kend ? v + k * 2 : NOWHERE; };
    // shares of whole steps, as even as they come
    const int steps = (kend + 31) / 32, each = (steps + FEW_WAVES - 1) / FEW_WAVES;
    const int from = wave * each, to = from + each < steps ? from + each : steps;
    constexpr int SUB = TR <= 2 ? 4 : TR <= 4 ? 2 : 1;   // steps whose rows are asked for together, one such lot ahead
    for (int s0 = from; s0 < to; s0 += STEPS) {           // (beyond the share: zeros)
        u32x4 b[STEPS], x0[2][SUB][TR];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) b[s] = __builtin_amdgcn_raw_buffer_load_b128(B, s0 + s < to ? at(vb, (s0 + s) * 32) : NOWHERE, 0, 0);
        auto rows = [&](int set, int s) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int x = 0; x < TR; ++x)
                    x0[set][u][x] = __builtin_amdgcn_raw_buffer_load_b128(A, s0 + s + u < to ? at(va[x], (s0 + s + u) * 32) : NOWHERE, 0, 0);
        };
        rows(0, 0);
#pragma unroll
        for (int s = 0; s < STEPS; s += SUB) {
            if (s + SUB < STEPS) rows((s / SUB + 1) & 1, s + SUB);
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int x = 0; x < TR; ++x) acc[x] = NT::mma(b[s + u], x0[(s / SUB) & 1][u][x], acc[x]);
        }
    }
    if constexpr (MODE == SHARED) {
        // The groups of the rows are dealt to the waves; a row takes its own group's products only.
        const auto V = __builtin_amdgcn_make_buffer_rsrc((char*)a.V + (int64_t)t.first * a.v_row * 2, 0, (int)(uint32_t)(t.rows * a.v_row * 2), 0x00020000);
        constexpr int AT_ONCE = 4;   // groups whose factors are asked for together
        for (int k0 = 0; k0 < a.pad; k0 += 32) {
            const int rank = k0 + q * 8;
            u32x4 hi[TR], lo[TR];
#pragma unroll
            for (int x = 0; x < TR; ++x) {
                const uint32_t v = x * 16 + j < t.rows ? (uint32_t)((x * 16 + j) * a.v_row * 2) + rank * 2 : NOWHERE;
                hi[x] = __builtin_amdgcn_raw_buffer_load_b128(V, v, 0, 0);
                lo[x] = __builtin_amdgcn_raw_buffer_load_b128(V, v == NOWHERE ? NOWHERE : v + a.pad * 2, 0, 0);
            }
            int turn = 0, mine = 0, froms[AT_ONCE], tos[AT_ONCE];
            u32x4 factor[AT_ONCE];
            auto multiply = [&](int count) {
#pragma unroll
                for (int c = 0; c < AT_ONCE; ++c) {
                    if (c >= count) break;
#pragma unroll
                    for (int x = 0; x < TR; ++x) {
                        const int r = x * 16 + j;
                        if (tos[c] <= x * 16 || froms[c] >= x * 16 + 16) continue;
                        const f32x4 sum = NT::mma(factor[c], lo[x], NT::mma(factor[c], hi[x], low[x]));
#pragma unroll
                        for (int i = 0; i < 4; ++i) low[x][i] = r >= froms[c] && r < tos[c] ? sum[i] : low[x][i];
                    }
                }
            };
            each_group(a, t.first, t.first + t.rows - 1, [&](int g, int f, int e) {
                if (turn++ % FEW_WAVES != wave) return;
                const auto F = __builtin_amdgcn_make_buffer_rsrc((char*)a.E + g * a.e_group * 2, 0, (int)(uint32_t)((a.N - 1) * a.e_n * 2 + a.r * 2), 0x00020000);
                const u32x4 b = __builtin_amdgcn_raw_buffer_load_b128(F, rank < a.r && n0 + j < a.N ? (uint32_t)((n0 + j) * a.e_n * 2) + rank * 2 : NOWHERE, 0, 0);
#pragma unroll
                for (int c = 0; c < AT_ONCE; ++c)
                    if (c == mine) factor[c] = b, froms[c] = f - t.first, tos[c] = e - t.first;
                if (++mine == AT_ONCE) {
                    multiply(AT_ONCE);
                    mine = 0;
                }
            });
            multiply(mine);
        }
        const int first_of = clamp_row(a.offsets[0], a.n_rows), end_of = clamp_row(a.offsets[a.n_groups], a.n_rows);
#pragma unroll
        for (int x = 0; x < TR; ++x) {
            const int p = t.first + x * 16 + j;
            const float up = a.up && p >= first_of && p < end_of ? a.up[p] : 1.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[x][i] += up * low[x][i];
        }
    }
#pragma unroll
    for (int x = 0; x < TR; ++x) *(f32x4*)&sums[wave][x * 16 + j][4 * q] = acc[x];
    __syncthreads();
    const float alpha = (float)a.alpha * (MODE == ROWS && a.scales && real ? ((const float*)a.scales)[t.group] : 1.0f), beta = (float)a.beta;
    for (int id = tid; id < t.rows * 16; id += 64 * FEW_WAVES) {
        const int r = id >> 4, n = id & 15;
        if (n0 + n >= a.N) continue;
        float v = 0;
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) v += sums[w][r][n];
        v *= alpha;
        int64_t row = t.first + r;
        if (a.scatter && a.order) {
            row = a.order[row];
            if (row < 0 || row >= a.n_rows) continue;
        }
        T* const c = (T*)a.C + row * a.c_row + (n0 + n) * a.c_n;
        if (a.use_beta && real) v += beta * (float)*c;
        *c = (T)(real ? v : 0.0f);
    }
}

// Whether it can take a call.
template <int MODE> inline bool few_takes(const Args& a) {
    if (a.b_group % 8 || !fast_rows(a.A, a.a_rows, a.a_row, a.a_col, a.K) || !fast_rows(a.B, a.N, a.b_n, a.b_k, a.K)) return false;
    return MODE != SHARED || (a.pad > 0 && a.e_group % 8 == 0 && fast_rows(a.E, a.N, a.e_n, a.e_k, a.r));
}

}  // namespace ragged
}  // namespace tfh
