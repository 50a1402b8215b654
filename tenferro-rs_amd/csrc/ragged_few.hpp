// ragged_few.hpp -- products of few rows with matrices that are read from memory for them alone (a decoding step): 16-bit
// operands, both contiguous along k.
//
// Bound by how fast the matrices arrive, so a block takes 16 columns only -- 256 blocks for 4096 of them -- and its waves
// share k, each with tiles of its own in LDS that its own loads fill some steps of 64 k's ahead, whole lines of every row
// (in operand position a load has 64 bytes of 16 rows, whose power-of-two distance then evicts them from L1 before their
// other halves are asked for: 64 rows took 32 us so, against 11 for one).  The rows come from L2 in every block.  The waves'
// sums meet in LDS.  The low-rank part has waves of its own, whose chain of dependent loads (offsets, factors) would
// otherwise come before or after all of that.
#pragma once
#include "ragged_fast.hpp"

namespace tfh {
namespace ragged {

constexpr int FEW_WAVES = 8;
template <int MODE> constexpr int few_low_waves() { return MODE == SHARED ? 4 : 0; }
template <int TR> constexpr int few_ahead() { return TR == 1 ? 4 : TR == 2 ? 3 : 2; }   // what LDS leaves room for
template <int TR> constexpr int few_lds() { return FEW_WAVES * few_ahead<TR>() * (16 * TR + 16) * 128; }
template <int MODE> constexpr int few_threads() { return 64 * (FEW_WAVES + few_low_waves<MODE>()); }

// TR: blocks of 16 rows.  rows mode: tiles of a group; shared mode: all rows, the low-rank part group by group.
template <class T, int MODE, int TR>
__global__ __launch_bounds__((few_threads<MODE>()), 1) void ragged_few_kernel(const Args a) {
    typedef Num<T> NT;
    constexpr int TM = 16 * TR, LOW = few_low_waves<MODE>(), ALL = FEW_WAVES + LOW;
    constexpr int AHEAD = few_ahead<TR>(), SLOT = (TM + 16) * 128, LOADS = 2 * TR + 2;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    char* const lds = (char*)smem_raw;
    float(*const sums)[TM][16] = (float(*)[TM][16])smem_raw;   // [ALL], when the tiles have been used
    static_assert(ALL * TM * 16 * 4 <= few_lds<TR>(), "the sums fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4, j = lane & 15;
    const int tiles_n = (a.N + 15) / 16;
    Tile t;
    if constexpr (MODE == ROWS) {
        if (!find_tile(a, TM, tiles_n, block_of(a), t)) return;
    } else {
        const uint32_t block = block_of(a);
        if (block >= (uint32_t)((a.n_rows + TM - 1) / TM) * (uint32_t)tiles_n) return;
        t.group = 0;
        t.tile_n = block % tiles_n;
        t.first = (block / tiles_n) * TM;
        t.rows = a.n_rows - t.first < TM ? (int)(a.n_rows - t.first) : TM;
    }
    const bool real = MODE != ROWS || t.group < a.n_groups;
    const int n0 = t.tile_n * 16, kend = real ? a.K : 0;
    f32x4 acc[TR];
#pragma unroll
    for (int x = 0; x < TR; ++x) acc[x] = (f32x4){0, 0, 0, 0};
    if (MODE != SHARED || wave < FEW_WAVES) {
        const u32x4 A = buffer_of(a.A, (uint32_t)((a.a_rows - 1) * a.a_row * 2 + a.K * 2));
        const u32x4 B = buffer_of((const char*)a.B + (MODE == ROWS && real ? t.group * a.b_group * 2 : 0), (uint32_t)((a.N - 1) * a.b_n * 2 + a.K * 2));
        const int cr = lane >> 3, kc = ((lane ^ cr) & 7) * 8;   // a load has 8 rows, lane l the chunk (l ^ row) % 8 of row l / 8
        uint32_t va[2 * TR], vb[2];
#pragma unroll
        for (int i = 0; i < 2 * TR; ++i) {
            const int r = 8 * i + cr;
            const int64_t s = r < t.rows && real ? source_row(a, t.first + r) : -1;
            va[i] = s >= 0 ? (uint32_t)(s * a.a_row * 2) + kc * 2 : NOWHERE;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) vb[i] = n0 + 8 * i + cr < a.N ? (uint32_t)((n0 + 8 * i + cr) * a.b_n * 2) + kc * 2 : NOWHERE;
        // shares of whole steps, as even as they come
        const int steps = (kend + 63) / 64, each = (steps + FEW_WAVES - 1) / FEW_WAVES;
        const int from = wave * each, mine = from < steps ? (from + each < steps ? each : steps - from) : 0;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + wave * (AHEAD * SLOT);
        auto issue = [&](int step, int slot) {   // (behind the last step: nothing)
            const bool there = step < mine;
            const int k0 = (from + step) * 64;
            const uint32_t o = scalar_of(there ? k0 * 2 : 0), to = scalar_of(lds0 + slot * SLOT);
            const bool in = there && k0 + kc < kend;
#pragma unroll
            for (int i = 0; i < 2; ++i) load_to_lds(B, in ? vb[i] : NOWHERE, o, to + i * 1024);
#pragma unroll
            for (int i = 0; i < 2 * TR; ++i) load_to_lds(A, in ? va[i] : NOWHERE, o, to + 2048 + i * 1024);
        };
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) issue(d, d);
        int slot = 0;
        for (int s = 0; s < mine; ++s) {
            const char* const tile = lds + wave * (AHEAD * SLOT) + slot * SLOT;
            wait_loads<(AHEAD - 1) * LOADS>();
            u32x4 fb[2], fa[2][TR];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                fb[h] = fragment<T, 16, true>(tile, 0, h, lane);
#pragma unroll
                for (int x = 0; x < TR; ++x) fa[h][x] = fragment<T, TM, true>(tile + 2048, x * 16, h, lane);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read, before the slot is filled again
            __builtin_amdgcn_sched_barrier(0);
            issue(s + AHEAD, slot);
            slot = slot + 1 < AHEAD ? slot + 1 : 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int x = 0; x < TR; ++x) acc[x] = NT::mma(fb[h], fa[h][x], acc[x]);
        }
        wait_loads<0>();
    } else if constexpr (MODE == SHARED) {
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
                unrolled<AT_ONCE>([&](auto item) {
                    constexpr int c = decltype(item)::value;
                    if (c >= count) return;
                    const u32x4 lower = finite_only<T>(factor[c]);
#pragma unroll
                    for (int x = 0; x < TR; ++x) {
                        const int r = x * 16 + j;
                        if (tos[c] <= x * 16 || froms[c] >= x * 16 + 16) continue;
                        const f32x4 sum = NT::mma(lower, lo[x], NT::mma(factor[c], hi[x], acc[x]));
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[x][i] = r >= froms[c] && r < tos[c] ? sum[i] : acc[x][i];
                    }
                });
            };
            each_group(a, t.first, t.first + t.rows - 1, [&](int g, int f, int e) {
                if (turn++ % LOW != wave - FEW_WAVES) return;
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
            for (int i = 0; i < 4; ++i) acc[x][i] *= up;
        }
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < TR; ++x) *(f32x4*)&sums[wave][x * 16 + j][4 * q] = acc[x];
    __syncthreads();
    const float alpha = (float)a.alpha * (MODE == ROWS && a.scales && real ? ((const float*)a.scales)[t.group] : 1.0f), beta = (float)a.beta;
    for (int id = tid; id < t.rows * 16; id += 64 * ALL) {
        const int r = id >> 4, n = id & 15;
        if (n0 + n >= a.N) continue;
        float v = 0;
#pragma unroll
        for (int w = 0; w < ALL; ++w) v += sums[w][r][n];
        v *= alpha;
        int64_t row = t.first + r;
        if (a.scatter && a.order) {
            row = a.order[row];
            if (row < 0 || row >= a.n_rows) continue;
        }
        if (MODE == ROWS && a.wide) {
            ((float*)a.C)[row * a.c_row + (n0 + n) * a.c_n] = real ? v : 0.0f;
            continue;
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
