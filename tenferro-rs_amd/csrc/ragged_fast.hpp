// ragged_fast.hpp -- products over rows in groups for 16-bit operands whose rows start 16-byte aligned: the same tiles in
// LDS as ragged.hpp, but written there by the memory system itself (buffer loads with LDS as their destination, 16 bytes a
// lane, no registers in between), double-buffered, and a register pipeline in front of the matrix cores.
//
// Per stage (128 bytes of k of every row, two halves of 64) and wave:
//   first half's products   while the second half's fragments are read from LDS
//   wait: the fragments are here, the next stage's loads have landed; barrier: so they have for every wave, and this
//         stage's buffer has been read by all
//   second half's products  while the loads of the stage after the next are issued into this stage's buffer and the next
//                           stage's first fragments are read
// so a load has most of a stage's products to arrive in, a fragment half a stage, and there is one barrier per stage.
#pragma once
#include "ragged.hpp"

namespace tfh {
namespace ragged {

// A buffer of `bytes` bytes from `base`: a load whose offset lies beyond reads zeros.
__device__ __forceinline__ u32x4 buffer_of(const void* base, uint32_t bytes) {
    const uint64_t p = (uint64_t)base;
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((uint32_t)p);
    r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32) & 0xffff);
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00020000;
    return r;
}
constexpr uint32_t NOWHERE = 0xfffffff0u;   // an offset beyond every buffer (spans are under MOST_SPAN)
constexpr int64_t MOST_SPAN = 0xffff0000ll;

// 16 bytes a lane from buffer + offset + scalar into LDS at `to` + 16 * lane.  The compiler does not count these loads:
// wait_loads() does, before anything they write is read.
__device__ __forceinline__ void load_to_lds(u32x4 buffer, uint32_t offset, uint32_t scalar, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(offset), "s"(buffer), "s"(scalar) : "memory");
}
template <int LEFT> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void wait_fragments_and_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 32 x 32 x 16 products: lane l = 32 p + j holds row j and k = 8 p .. 8 p + 7 of either operand; register r of the result
// is row 8 (r / 4) + 4 p + r % 4 of the first operand and column j, a row of the second.  (The 16 x 16 form needs twice
// the instructions, and its 256 accumulators in pieces of 4 made the compiler move a third of them in every stage.)
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <class T> __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// The 16 k's h = 0 .. 3 of a stage for 32 rows from `row`.
template <class T, int TM, bool KFAST>
__device__ __forceinline__ u32x4 fragment32(const char* tile, int row, int h, int lane) {
    if constexpr (KFAST) {
        return *(const u32x4*)(tile + kfast_at<T>(row + (lane & 31), 2 * h + (lane >> 5)));
    } else {
        typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
        const int j = lane & 15, k = 16 * h + 8 * (lane >> 5) + (j >> 2), col = row + (lane & 16) + 4 * (j & 3);
        const uint32_t within = (col * 2) & 15, chunk = (col * 2) >> 4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(tile + rowfast_at<T, TM>(k, chunk) + within));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(tile + rowfast_at<T, TM>(k + 4, chunk) + within));
        struct { s16x4 a, b; } both = {lo, hi};
        return __builtin_bit_cast(u32x4, both);
    }
}

// The shape of a block: WM x WN = 4 waves of 32 XT x 32 YT results.
template <int WM_, int WN_, int XT_, int YT_> struct Shape {
    static_assert(WM_ * WN_ == 4, "four waves");
    static constexpr int WM = WM_, WN = WN_, XT = XT_, YT = YT_, TM = 32 * WM * XT, TN = 32 * WN * YT;
    static constexpr int STAGE = (TM + TN) * 128, LDS = 2 * STAGE;
    static constexpr bool BY_GROUP = TM > 128;
    static constexpr int BLOCKS = XT * YT > 8 ? 1 : 2;   // of a CU: registers and LDS leave room for so many
};

// One tile: its k loop and its results.  BY_GROUP: its rows are of one group (of none: t.group == a.n_groups).
template <class T, int MODE, bool BKFAST, class S, bool BY_GROUP>
__device__ __forceinline__ void fast_tile(const Args& a, const Tile& t, char* lds) {
    static_assert(sizeof(T) == 2, "16-bit operands");
    constexpr int XT = S::XT, YT = S::YT, TM = S::TM, TN = S::TN, BK = 64, STAGE = S::STAGE;
    constexpr int CA = TM / 32, CB = TN / 32;      // chunks of each operand per thread and stage
    constexpr bool OUT = MODE == OUTER || MODE == PAIR, AKFAST = !OUT;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % S::WM, wn = wave / S::WM;
    const bool real = MODE != ROWS || t.group < a.n_groups;
    const int n0 = t.tile_n * TN, m0 = t.tile_m * TM;
    f32x16 acc[XT][YT];
#pragma unroll
    for (int x = 0; x < XT; ++x)
#pragma unroll
        for (int y = 0; y < YT; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0;

    // (shared mode's low-rank part comes first, see below)
    // This thread's chunks.  k-fast: the chunk (tid ^ row) % 8 of rows tid / 8 + 32 i; row-fast: chunk (tid + 256 i) % RX of
    // k = (tid + 256 i) / RX, its place swizzled; either way a wave's 64 lanes fill 1024 consecutive bytes of LDS.
    const int cr = tid >> 3, kc = ((tid ^ cr) & 7) * 8;
    constexpr int RA = TM / 8, RB = TN / 8;        // chunks of a row of k in a row-fast tile
    const int kend = OUT ? t.rows : real ? a.K : 0;
    uint32_t va[CA], vb[CB];
    u32x4 A, B;
    uint32_t step_a = BK * 2, step_b = BK * 2;     // bytes from a stage to the next
    int32_t next_row = -1;                         // outer, gathered: lane l holds the row of A for the next stage's l-th k
    auto look_up = [&](int k0) {
        if constexpr (!AKFAST)
            if (a.gather && a.order) next_row = k0 + lane < kend ? (int)source_row(a, t.first + k0 + lane) : -1;
    };
    if constexpr (AKFAST) {
        A = buffer_of(a.A, (uint32_t)((a.a_rows - 1) * a.a_row * 2 + a.K * 2));
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            const int64_t s = cr + 32 * i < t.rows && real ? source_row(a, t.first + cr + 32 * i) : -1;
            va[i] = s >= 0 ? (uint32_t)(s * a.a_row * 2) + kc * 2 : NOWHERE;
        }
    } else {
        // rows of k are rows of the group; a gathered A's are looked up stage by stage
        const bool gather = a.gather && a.order;
        const int64_t first = gather ? 0 : t.first, rows = gather ? a.a_rows : kend;
        A = buffer_of((const char*)a.A + first * a.a_row * 2, rows > 0 ? (uint32_t)((rows - 1) * a.a_row * 2 + a.M * 2) : 0);
        step_a = gather ? 0 : BK * (uint32_t)a.a_row * 2;
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            const int id = tid + 256 * i, k = id / RA, m = m0 + ((id % RA) ^ (rowfast_swizzle<T>(k) & (RA - 1))) * 8;
            va[i] = m < a.M ? (gather ? 0 : (uint32_t)(k * a.a_row * 2)) + m * 2 : NOWHERE;
        }
        look_up(0);
    }
    if constexpr (BKFAST) {
        B = buffer_of((const char*)a.B + (MODE == ROWS && real ? t.group * a.b_group * 2 : 0), (uint32_t)((a.N - 1) * a.b_n * 2 + a.K * 2));
#pragma unroll
        for (int i = 0; i < CB; ++i) vb[i] = n0 + cr + 32 * i < a.N ? (uint32_t)((n0 + cr + 32 * i) * a.b_n * 2) + kc * 2 : NOWHERE;
    } else {
        const int64_t first = OUT ? t.first * a.b_k : MODE == ROWS && real ? t.group * a.b_group : 0;
        B = buffer_of((const char*)a.B + first * 2, kend > 0 ? (uint32_t)((kend - 1) * a.b_k * 2 + a.N * 2) : 0);
        step_b = BK * (uint32_t)a.b_k * 2;
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int id = tid + 256 * i, k = id / RB, n = n0 + ((id % RB) ^ (rowfast_swizzle<T>(k) & (RB - 1))) * 8;
            vb[i] = n < a.N ? (uint32_t)(k * a.b_k * 2) + n * 2 : NOWHERE;
        }
    }
    // Large shared tiles: the low-rank part is the first stages of the loop, V[p, :] as A's and E[g] as B's.
    constexpr bool EXT = MODE == SHARED && BY_GROUP;
    u32x4 V = A, F = B;
    uint32_t ve = 0, fe = 0;
    int ext = 0;
    if constexpr (EXT) {
        if (t.group < a.n_groups) {
            ext = 2 * a.pad / BK;
            V = buffer_of((const char*)a.V + (int64_t)t.first * a.v_row * 2, (uint32_t)((t.rows - 1) * a.v_row * 2 + 2 * a.pad * 2));
            F = buffer_of((const char*)a.E + t.group * a.e_group * 2, (uint32_t)(BKFAST ? (a.N - 1) * a.e_n * 2 + a.r * 2 : (a.r - 1) * a.e_k * 2 + a.N * 2));
            ve = (uint32_t)(cr * a.v_row * 2) + kc * 2;
            fe = BKFAST ? (uint32_t)((n0 + cr) * a.e_n * 2) : 0;
        }
    }
    const int stages = ext + (kend + BK - 1) / BK;
    struct Stage {
        bool low;              // of the low-rank part
        int k0;                // first k in its part
        uint32_t oa, ob;       // scalar offsets
    };
    auto stage_of = [&](int s) {   // (behind the last one every chunk is beyond kend)
        Stage g;
        g.low = EXT && s < ext;
        g.k0 = (g.low ? s : s - ext) * BK;
        const bool there = s < stages;
        g.oa = !there ? 0 : g.low ? g.k0 * 2 : (uint32_t)(s - ext) * step_a;
        g.ob = !there || g.low ? 0 : (uint32_t)(s - ext) * step_b;
        return g;
    };
    auto pick = [](bool first, u32x4 x, u32x4 y) { return (u32x4){first ? x[0] : y[0], first ? x[1] : y[1], first ? x[2] : y[2], y[3]}; };
    // chunk i of the two operands for a stage, into buffer `to`
    auto issue_a = [&](int i, const Stage& g, uint32_t to) {
        uint32_t v = va[i];
        if constexpr (AKFAST) {
            v = g.k0 + kc < kend ? v : NOWHERE;
            if constexpr (EXT) {
                const uint32_t low = cr + 32 * i < t.rows ? ve + i * 32 * (uint32_t)(a.v_row * 2) : NOWHERE;
                v = g.low ? low : v;
            }
        } else {
            const int k = (tid + 256 * i) / RA;
            if (a.gather && a.order) {
                const int s = __shfl(next_row, k, 64);   // (-1 behind the group's last row)
                v = s >= 0 && v != NOWHERE ? v + (uint32_t)s * (uint32_t)(a.a_row * 2) : NOWHERE;
            } else
                v = g.k0 + k < kend ? v : NOWHERE;
        }
        load_to_lds(EXT ? pick(g.low, V, A) : A, v, g.oa, to + i * 4096 + wave * 1024);
    };
    auto issue_b = [&](int i, const Stage& g, uint32_t to) {
        uint32_t v = vb[i];
        if constexpr (BKFAST) v = g.k0 + kc < kend ? v : NOWHERE;
        else v = g.k0 + (tid + 256 * i) / RB < kend ? v : NOWHERE;
        if constexpr (EXT) {
            uint32_t low;
            if constexpr (BKFAST) {
                int rank = g.k0 + kc;
                rank = rank >= a.pad ? rank - a.pad : rank;
                low = rank < a.r && vb[i] != NOWHERE ? fe + i * 32 * (uint32_t)(a.e_n * 2) + rank * 2 : NOWHERE;
            } else {
                const int id = tid + 256 * i, kk = id / RB;
                int rank = g.k0 + kk;
                rank = rank >= a.pad ? rank - a.pad : rank;
                low = rank < a.r && vb[i] != NOWHERE ? (uint32_t)rank * (uint32_t)(a.e_k * 2) + vb[i] - (uint32_t)(kk * a.b_k * 2) : NOWHERE;
            }
            v = g.low ? low : v;
        }
        load_to_lds(EXT ? pick(g.low, F, B) : B, v, g.ob, to + TM * 128 + i * 4096 + wave * 1024);
    };
    u32x4 fa[2][XT], fb[2][YT];
    auto read = [&](int set, int i, const char* stage, int h) {
        if (i < XT) fa[set][i] = fragment32<T, TM, AKFAST>(stage, (wm * XT + i) * 32, h, lane);
        else fb[set][i - XT] = fragment32<T, TN, BKFAST>(stage + TM * 128, (wn * YT + i - XT) * 32, h, lane);
    };
    constexpr int FRAGS = XT + YT, CHUNKS = CA + CB;
    if constexpr (MODE == SHARED && !BY_GROUP) {
        // V . E[g] for the groups that the tile's rows belong to, before the accumulators hold anything else: in f16 a row's
        // V is scaled by a power of two, which is undone here.  The pair's halves are 2 pad k's against E twice.  Rows of
        // another group keep what they have -- selected, not multiplied by zero, which infinite factors would survive.
        const u32x4 V = buffer_of((const char*)a.V + (int64_t)t.first * a.v_row * 2, (uint32_t)((t.rows - 1) * a.v_row * 2 + 2 * a.pad * 2));
        const int last = t.first + t.rows - 1;
        for (int g = __builtin_amdgcn_readfirstlane(group_of(a, t.first)); g < a.n_groups; ++g) {
            const int from = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[g], a.n_rows)) - t.first;
            const int to = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[g + 1], a.n_rows)) - t.first;
            if (from + t.first > last) break;
            if (to <= from || to <= 0) continue;
            const u32x4 E = buffer_of((const char*)a.E + g * a.e_group * 2, (uint32_t)(BKFAST ? (a.N - 1) * a.e_n * 2 + a.r * 2 : (a.r - 1) * a.e_k * 2 + a.N * 2));
            for (int k0 = 0; k0 < 2 * a.pad; k0 += BK) {
                __syncthreads();   // the last stage has been read
#pragma unroll
                for (int i = 0; i < CA; ++i)
                    load_to_lds(V, cr + 32 * i < t.rows ? (uint32_t)((cr + 32 * i) * a.v_row * 2) + (k0 + kc) * 2 : NOWHERE, 0, lds0 + i * 4096 + wave * 1024);
#pragma unroll
                for (int i = 0; i < CB; ++i) {
                    uint32_t v;
                    if constexpr (BKFAST) {
                        const int k = k0 + kc, rank = k >= a.pad ? k - a.pad : k, n = n0 + cr + 32 * i;
                        v = n < a.N && rank < a.r ? (uint32_t)(n * a.e_n * 2) + rank * 2 : NOWHERE;
                    } else {
                        const int id = tid + 256 * i, kk = id / RB, k = k0 + kk, rank = k >= a.pad ? k - a.pad : k;
                        const int n = n0 + ((id % RB) ^ (rowfast_swizzle<T>(kk) & (RB - 1))) * 8;
                        v = n < a.N && rank < a.r ? (uint32_t)(rank * a.e_k * 2) + n * 2 : NOWHERE;
                    }
                    load_to_lds(E, v, 0, lds0 + TM * 128 + i * 4096 + wave * 1024);
                }
                wait_loads<0>();
                wait_fragments_and_barrier();
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    u32x4 eb[YT];
#pragma unroll
                    for (int y = 0; y < YT; ++y) eb[y] = fragment32<T, TN, BKFAST>(lds + TM * 128, (wn * YT + y) * 32, h, lane);
#pragma unroll
                    for (int x = 0; x < XT; ++x) {
                        const int r0 = (wm * XT + x) * 32, r = r0 + (lane & 31);
                        if (to <= r0 || from >= r0 + 32) continue;
                        const u32x4 ea = fragment32<T, TM, true>(lds, r0, h, lane);
                        const bool all = from <= r0 && to >= r0 + 32, mine = r >= from && r < to;
#pragma unroll
                        for (int y = 0; y < YT; ++y) {
                            const f32x16 v = mma32<T>(eb[y], ea, acc[x][y]);
                            if (all) acc[x][y] = v;
                            else
#pragma unroll
                                for (int i = 0; i < 16; ++i) acc[x][y][i] = mine ? v[i] : acc[x][y][i];
                        }
                    }
                }
            }
        }
        __syncthreads();
        if (a.up) {
            const int first_of = clamp_row(a.offsets[0], a.n_rows), end_of = clamp_row(a.offsets[a.n_groups], a.n_rows);
#pragma unroll
            for (int x = 0; x < XT; ++x) {
                const int p = t.first + (wm * XT + x) * 32 + (lane & 31);
                const float up = p >= first_of && p < end_of ? a.up[p] : 1.0f;   // a row of no group has none
#pragma unroll
                for (int y = 0; y < YT; ++y)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[x][y][i] *= up;
            }
        }
    }
    if (stages > 0) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const Stage g = stage_of(s);
#pragma unroll
            for (int i = 0; i < CA; ++i) issue_a(i, g, lds0 + s * STAGE);
#pragma unroll
            for (int i = 0; i < CB; ++i) issue_b(i, g, lds0 + s * STAGE);
            look_up((s + 1) * BK);
        }
        wait_loads<CHUNKS>();
        wait_fragments_and_barrier();
#pragma unroll
        for (int i = 0; i < FRAGS; ++i) read(0, i, lds, 0);
        int at = 0;
        for (int s = 0; s < stages; ++s) {
            // (behind the last stage the loads go nowhere and the fragments that are read are not used: no branch in the loop)
            const Stage g = stage_of(s + 2);
            const uint32_t to = lds0 + at;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                if (h == 3) {
                    wait_loads<0>();
                    wait_fragments_and_barrier();
                }
                constexpr int EACH = (FRAGS + XT - 1) / XT, LOADS = (CHUNKS + XT - 1) / XT;
#pragma unroll
                for (int x = 0; x < XT; ++x) {
                    if (h == 3)
#pragma unroll
                        for (int i = x * LOADS; i < (x + 1) * LOADS && i < CHUNKS; ++i) {
                            if (i < CA) issue_a(i, g, to);
                            else issue_b(i - CA, g, to);
                        }
#pragma unroll
                    for (int i = x * EACH; i < (x + 1) * EACH && i < FRAGS; ++i) read((h + 1) & 1, i, lds + (h == 3 ? at ^ STAGE : at), (h + 1) & 3);
#pragma unroll
                    for (int y = 0; y < YT; ++y) acc[x][y] = mma32<T>(fb[h & 1][y], fa[h & 1][x], acc[x][y]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            look_up((s + 3) * BK);
            at ^= STAGE;
        }
        wait_loads<0>();
    }

    // Results leave through LDS, so that a wave stores whole runs of a row: 16-byte chunks, the chunk index XORed with the
    // row because the 32 rows of a register would meet in one bank otherwise.  (Straight from the registers a store would
    // touch 32 rows with 16 bytes each.)
    const float alpha = (float)a.alpha * (MODE == ROWS && a.scales && real ? ((const float*)a.scales)[t.group] : 1.0f), beta = (float)a.beta;
    if constexpr (MODE == PAIR) {
        // B's columns are a pair, hi and lo `pad` apart: their sums are added here, in f32
        static_assert(TM * TN * 4 <= S::LDS && TN % 64 == 0, "the sums fit the two stages");
        __syncthreads();
#pragma unroll
        for (int x = 0; x < XT; ++x) {
            const int r = (wm * XT + x) * 32 + (lane & 31);
#pragma unroll
            for (int y = 0; y < YT; ++y)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int chunk = (wn * YT + y) * 8 + 2 * g + (lane >> 5);
                    const f32x4 v = {acc[x][y][4 * g], acc[x][y][4 * g + 1], acc[x][y][4 * g + 2], acc[x][y][4 * g + 3]};
                    *(f32x4*)(lds + r * (TN * 4) + ((chunk ^ (r & 15)) << 4)) = v;
                }
        }
        __syncthreads();
        const int rows = a.M - m0 < TM ? a.M - m0 : TM;
        const bool down = a.c_row == 1;   // the direction in which the result is contiguous goes along the lanes
        auto at = [&](int r, int c) { return *(const float*)(lds + r * (TN * 4) + (((c >> 2) ^ (r & 15)) << 4) + (c & 3) * 4); };
        for (int id = tid; id < rows * a.r; id += 256) {
            const int r = down ? id % rows : id / a.r, c = down ? id / rows : id % a.r;
            ((T*)a.C)[t.group * a.c_group + (m0 + r) * a.c_row + c * a.c_n] = (T)(alpha * (at(r, c) + at(r, c + a.pad)));
        }
        return;
    }
    if (a.use_beta && real) {   // the sum is rounded once: nothing in between
#pragma unroll
        for (int x = 0; x < XT; ++x) {
            const int r = (wm * XT + x) * 32 + (lane & 31);
            if (OUT ? m0 + r >= a.M : r >= t.rows) continue;
            int64_t row = OUT ? m0 + r : t.first + r;
            if constexpr (!OUT)
                if (a.scatter && a.order) {
                    row = a.order[row];
                    if (row < 0 || row >= a.n_rows) continue;
                }
            T* const c = (T*)a.C + (OUT ? t.group * a.c_group : 0) + row * a.c_row;
#pragma unroll
            for (int y = 0; y < YT; ++y)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = n0 + (wn * YT + y) * 32 + 8 * g + 4 * (lane >> 5);
                    if (n >= a.N) continue;
                    T out[4];
                    __builtin_memcpy(out, c + n, 8);
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = (T)(alpha * acc[x][y][4 * g + i] + beta * (float)out[i]);
                    __builtin_memcpy(c + n, out, 8);
                }
        }
        return;
    }
    constexpr int CHUNKS_N = TN / 8;
    static_assert(TM * TN * 2 <= S::LDS, "the results fit the two stages");
    __syncthreads();
#pragma unroll
    for (int x = 0; x < XT; ++x) {
        const int r = (wm * XT + x) * 32 + (lane & 31);
#pragma unroll
        for (int y = 0; y < YT; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = (wn * YT + y) * 32 + 8 * g + 4 * (lane >> 5);
                T out[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = (T)(alpha * acc[x][y][4 * g + i]);
                __builtin_memcpy(lds + r * (TN * 2) + (((n >> 3) ^ (r & (CHUNKS_N - 1))) << 4) + (n & 4) * 2, out, 8);
            }
    }
    __syncthreads();
    const int most_n = a.N - n0 < TN ? a.N - n0 : TN, rows = OUT ? (a.M - m0 < TM ? a.M - m0 : TM) : t.rows;
    for (int id = tid; id < rows * CHUNKS_N; id += 256) {
        const int r = id / CHUNKS_N, n = (id % CHUNKS_N) * 8;
        if (n >= most_n) continue;
        int64_t row = OUT ? m0 + r : t.first + r;
        if constexpr (!OUT)
            if (a.scatter && a.order) {
                row = a.order[row];
                if (row < 0 || row >= a.n_rows) continue;
            }
        T* const c = (T*)a.C + (OUT ? t.group * a.c_group : 0) + row * a.c_row + n0 + n;
        const u32x4 v = *(const u32x4*)(lds + r * (TN * 2) + (((n >> 3) ^ (r & (CHUNKS_N - 1))) << 4));
        if (most_n - n >= 8) __builtin_memcpy(c, &v, 16);
        else __builtin_memcpy(c, &v, 8);
    }
}

template <class T, int MODE, bool BKFAST, class S>
__global__ __launch_bounds__(256, S::BLOCKS) void ragged_fast_kernel(const Args a) {
    // shared mode: large tiles belong to one group each (the host sets zero_rest: the rows of no group are one more), small
    // ones span as many as their rows are of, so that few rows of many groups do not read W once for each
    constexpr bool BY_GROUP = MODE == ROWS || (MODE == SHARED && S::BY_GROUP);
    constexpr int TM = S::TM, TN = S::TN;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    char* const lds = (char*)smem_raw;
    const int tiles_n = (a.N + TN - 1) / TN;
    Tile t;
    if constexpr (BY_GROUP) {
        if (!find_tile(a, TM, tiles_n, blockIdx.x, t)) return;
        if constexpr (TM == 256) {
            // a group's last tile is seldom full: half or a quarter of the rows in half or 0.4 of the time
            typedef Shape<1, 4, 2, 2> Quarter;
            typedef Shape<2, 2, 2, 4> Half;
            static_assert(Quarter::TN == TN && Half::TN == TN && Half::LDS <= S::LDS, "the same columns");
            if (t.rows <= 64) {
                fast_tile<T, MODE, BKFAST, Quarter, true>(a, t, lds);
                return;
            }
            if (t.rows <= 128) {
                fast_tile<T, MODE, BKFAST, Half, true>(a, t, lds);
                return;
            }
        }
    } else if constexpr (MODE == OUTER || MODE == PAIR) {
        const int tiles_m = (a.M + TM - 1) / TM;
        const uint32_t id = (uint32_t)gemm::logical_block(blockIdx.x, gridDim.x), each = (uint32_t)tiles_m * tiles_n;
        t.group = (int)(id / each);
        gemm::tile_of(id % each, tiles_m, tiles_n, t.tile_m, t.tile_n);
        t.first = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[t.group], a.n_rows));
        const int to = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[t.group + 1], a.n_rows));
        t.rows = to > t.first ? to - t.first : 0;
    } else {
        const int tiles_m = (int)((a.n_rows + TM - 1) / TM);
        gemm::tile_of((uint32_t)gemm::logical_block(blockIdx.x, gridDim.x), tiles_m, tiles_n, t.tile_m, t.tile_n);
        t.group = 0;
        t.first = t.tile_m * TM;
        t.rows = a.n_rows - t.first < TM ? (int)(a.n_rows - t.first) : TM;
    }
    fast_tile<T, MODE, BKFAST, S, BY_GROUP>(a, t, lds);
}

// Whether the kernel can take a call: rows that start 16-byte aligned and end with a chunk, spans that 32 bits address.
inline bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
inline bool fast_rows(const void* p, int64_t rows, int64_t stride, int64_t inner_stride, int64_t inner) {
    return aligned(p, 16) && inner_stride == 1 && inner % 8 == 0 && stride % 8 == 0 && stride > 0 && (rows - 1) * stride * 2 + inner * 2 < MOST_SPAN;
}
template <int MODE> inline bool fast_takes(const Args& a, bool bkfast) {
    if (MODE == PAIR) return a.pad > 0 && a.pad <= 64 && !a.use_beta && fast_rows(a.A, a.a_rows, a.a_row, a.a_col, a.M) && fast_rows(a.B, a.b_rows, a.b_k, a.b_n, 2 * a.pad);
    if (a.c_n != 1 || a.c_row % 4 || a.N % 4 || !aligned(a.C, 8)) return false;
    if (MODE == OUTER) {
        if (a.c_group % 4) return false;
        return fast_rows(a.A, a.a_rows, a.a_row, a.a_col, a.M) && fast_rows(a.B, a.b_rows, a.b_k, a.b_n, a.N);
    }
    if (MODE == SHARED) {
        if (a.pad <= 0 || a.e_group % 8 || !(bkfast ? fast_rows(a.E, a.N, a.e_n, a.e_k, a.r) : fast_rows(a.E, a.r, a.e_k, a.e_n, a.N))) return false;
    }
    if (a.b_group % 8) return false;
    return fast_rows(a.A, a.a_rows, a.a_row, a.a_col, a.K) && (bkfast ? fast_rows(a.B, a.N, a.b_n, a.b_k, a.K) : fast_rows(a.B, a.K, a.b_k, a.b_n, a.N));
}

}  // namespace ragged
}  // namespace tfh
