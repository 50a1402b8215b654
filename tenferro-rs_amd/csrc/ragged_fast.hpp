// ragged_fast.hpp -- products over rows in groups for 16-bit operands whose rows start 16-byte aligned: the same tiles in
// LDS as ragged.hpp, but written there by the memory system itself (buffer loads with LDS as their destination, 16 bytes a
// lane, no registers in between), double-buffered, and a register pipeline in front of the matrix cores.
//
// Per stage (64 or 128 bytes of k of every row) and wave, 16 k's at a time:
//   their products          while the fragments of the next 16 are read from LDS
//   before the last 16:     wait until those fragments are here and the next stage's loads have landed; barrier: so they
//                           have for every wave, and this stage's slot has been read by all
//   the last 16's products  while a later stage's loads are issued into this stage's slot and the next stage's first
//                           fragments are read
// so a fragment has 16 k's products to arrive in, a load those of all slots but one, and there is one barrier per stage.
//
// Bound by the matrix cores, and by their power with random numbers.  Reached, bf16: one group of 16 384 rows, 8192 x 4096: 1250
// TFLOP/s (a library product: 1490); 65 536 gathered rows of 64 uneven groups, 2048 x 2048: 590 us, 930 TFLOP/s, the matrix cores 45 %
// busy at 1.8 GHz -- a tile of 32 stages starts and ends with a tenth of its time, the groups' last tiles and the last round cost as
// much, and LDS is read and written three quarters of the time; gradients of 32 768 rows of 32 uneven groups, 2048 x 1024: 186 us, 740, with their rows
// looked up; the rows' gradients there, kept in f32: 203 us (178 in bf16); adapters' shared product, 16 384 x 4096 x 4096: 530 us, 1040.
#pragma once
#include <utility>

#include "ragged.hpp"

namespace tfh {
namespace ragged {

// A scalar operand of the loads below.  A vector instruction's write of a scalar register (readfirstlane is one) must lie
// five wait states before a load that reads it; the compiler sees to that for its own loads, not for those in asm.  Moved
// here by the scalar unit, which waits for it, the value is one that a load may read at once.  (A spilled scalar register
// comes back through a vector instruction, wherever the compiler puts it: the loads' own s_nop 4 makes up for that one.)
__device__ __forceinline__ uint32_t scalar_of(uint32_t v) {
    uint32_t s;
    asm("s_mov_b32 %0, %1" : "=s"(s) : "s"(__builtin_amdgcn_readfirstlane(v)));
    return s;
}
// A buffer of `bytes` bytes from `base`: a load whose offset lies beyond reads zeros.
__device__ __forceinline__ u32x4 buffer_of(const void* base, uint32_t bytes) {
    const uint64_t p = (uint64_t)base;
    u32x4 r;
    r[0] = scalar_of((uint32_t)p);
    r[1] = scalar_of((uint32_t)(p >> 32) & 0xffff);
    r[2] = scalar_of(bytes);
    r[3] = 0x00020000;
    return r;
}
constexpr uint32_t NOWHERE = 0xfffffff0u;   // an offset beyond every buffer (spans are under MOST_SPAN)
constexpr int64_t MOST_SPAN = 0xffff0000ll;

// 16 bytes a lane from buffer + offset + scalar into LDS at `to` + AT + 16 * lane.  The compiler does not count these loads:
// wait_loads() does, before anything they write is read.  Where a load goes is in m0, which is written and read within one
// statement.  (The compiler reserves that register: it writes it for its own instructions that read it only, of which LDS accesses and
// products are none.)
template <int AT = 0> __device__ __forceinline__ void load_to_lds(u32x4 buffer, uint32_t offset, uint32_t scalar, uint32_t to) {
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds" ::"s"(to), "n"(AT), "v"(offset), "s"(buffer), "s"(scalar) : "memory", "scc");
}
template <class F, int... I> __device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F> __device__ __forceinline__ void unrolled(F f) { each_of(std::make_integer_sequence<int, N>{}, f); }
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
// A fragment with zeros for infinities and what is no number: what the lower half of a pair is multiplied by.  The upper half has met
// them already, and the lower one, a zero or of the other sign, would make no number of that infinity.
template <class T> __device__ __forceinline__ u32x4 finite_only(u32x4 v) {
    constexpr uint32_t EXPONENT = __is_same(T, __bf16) ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t low = (v[i] & EXPONENT) == EXPONENT ? 0 : v[i] & 0xffff;
        v[i] = (v[i] & EXPONENT << 16) == EXPONENT << 16 ? low : (v[i] & 0xffff0000) | low;
    }
    return v;
}
// A k-fast tile with KB = 64 or 128 bytes of k for each row: where a chunk lies, so that any eight consecutive rows' same
// chunk fills the banks once.
template <int KB> __device__ __forceinline__ uint32_t turn(uint32_t row) { return KB == 128 ? row & 7 : (row >> 1) & 3; }
template <int KB> __device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t chunk) { return row * KB + ((chunk ^ turn<KB>(row)) << 4); }
// The 16 k's h of a stage for 32 rows from `row`.
template <class T, int TM, bool KFAST, int KB = 128>
__device__ __forceinline__ u32x4 fragment32(const char* tile, int row, int h, int lane) {
    if constexpr (KFAST) {
        return *(const u32x4*)(tile + chunk_at<KB>(row + (lane & 31), 2 * h + (lane >> 5)));
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

// The shape of a block: WM x WN = 4 waves of 32 XT x 32 YT results; KB bytes of k of each row are a stage, SA stages of the
// first operand and SB of the second are in LDS or on their way to it.
//
// A k-fast tile wants KB = 128: its loads then ask for whole lines, and 64-byte pieces cost L2 as much each (256 x 256 tiles
// need 13 TB/s of it).  That leaves room in LDS for five tiles, three of one operand and two of the other; the other's loads
// go first after the barrier.  256 x 128 tiles, two to a compute unit, take KB = 64, three stages of both; outer products, whose
// tiles are row-fast and ask for whole rows of columns anyway, lose nothing by that.
template <int WM_, int WN_, int XT_, int YT_, int KB_ = 128, int SA_ = 2, int SB_ = 2> struct Shape {
    static_assert(WM_ * WN_ == 4, "four waves");
    static_assert(SB_ >= 2 && (SA_ == SB_ || SA_ == SB_ + 1), "the waits below count on it");
    static constexpr int WM = WM_, WN = WN_, XT = XT_, YT = YT_, TM = 32 * WM * XT, TN = 32 * WN * YT, KB = KB_, SA = SA_, SB = SB_;
    static constexpr int TILE_A = TM * KB, TILE_B = TN * KB, LDS = SA * TILE_A + SB * TILE_B;
    static constexpr int BLOCKS = XT * YT > 8 ? 1 : 2;   // of a CU: registers and LDS leave room for so many
};

// One tile: its k loop and its results.  Its rows are of one group (of none: t.group == a.n_groups), but in shared mode of any.
template <class T, int MODE, bool BKFAST, class S>
__device__ __forceinline__ void fast_tile(const Args& a, const Tile& t, char* lds) {
    static_assert(sizeof(T) == 2, "16-bit operands");
    constexpr int XT = S::XT, YT = S::YT, TM = S::TM, TN = S::TN, KB = S::KB, BK = KB / 2, SA = S::SA, SB = S::SB;
    constexpr int TILE_A = S::TILE_A, TILE_B = S::TILE_B, BASE_B = SA * TILE_A;   // LDS: the first operand's slots, then the second's
    constexpr int CPR = KB / 16, RPI = 256 / CPR;            // k-fast: chunks of a row, rows that 256 threads fetch at once
    constexpr int CA = TM / RPI, CB = TN / RPI, H = BK / 16;   // chunks of each operand per thread and stage; 16 k's of a stage
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

    // This thread's chunks.  k-fast: of rows tid / CPR + RPI i, its place in the row turned; row-fast: chunk (tid + 256 i) % RX
    // of k = (tid + 256 i) / RX, turned as well; either way a wave's 64 lanes fill 1024 consecutive bytes of LDS.
    const int cr = tid / CPR, kc = (int)((tid ^ turn<KB>(cr)) & (CPR - 1)) * 8;
    constexpr int RA = TM / 8, RB = TN / 8;        // chunks of a row of k in a row-fast tile
    const int kend = OUT ? t.rows : real ? a.K : 0;
    uint32_t va[CA], vb[CB];
    u32x4 A, B;
    uint32_t step_a = BK * 2, step_b = BK * 2;     // bytes from a stage to the next
    // Outer, gathered: where the rows of A for the stages to come start, in bytes (NOWHERE: there is none), 64 a register, the next ones in the first.  The compiler's wait for
    // what is looked up here waits for the loads into LDS too, so it is LOOK x 64 rows at once and seldom.
    constexpr int LOOK = 4;
    uint32_t next_rows[LOOK];
    auto look_up = [&](int k0) {
#pragma unroll
        for (int i = 0; i < LOOK; ++i) {
            const int k = k0 + 64 * i + lane;
            const int row = k < kend ? (int)source_row(a, t.first + k) : -1;
            next_rows[i] = row >= 0 ? (uint32_t)row * (uint32_t)(a.a_row * 2) : NOWHERE;
        }
    };
    if constexpr (AKFAST) {
        A = buffer_of(a.A, (uint32_t)((a.a_rows - 1) * a.a_row * 2 + a.K * 2));
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            const int64_t s = cr + RPI * i < t.rows && real ? source_row(a, t.first + cr + RPI * i) : -1;
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
    }
    if constexpr (BKFAST) {
        B = buffer_of((const char*)a.B + (MODE == ROWS && real ? t.group * a.b_group * 2 : 0), (uint32_t)((a.N - 1) * a.b_n * 2 + a.K * 2));
#pragma unroll
        for (int i = 0; i < CB; ++i) vb[i] = n0 + cr + RPI * i < a.N ? (uint32_t)((n0 + cr + RPI * i) * a.b_n * 2) + kc * 2 : NOWHERE;
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
    const int stages = (kend + BK - 1) / BK;

    // What the loads of a stage are: buffers, the chunks' offsets in them, and scalar offsets that go on from stage to stage.
    // Offsets change at the ends of the parts only, by a branch that is seldom taken, and the loop's loads take them as they are.
    struct {
        u32x4 A, B;
        uint32_t va[CA], vb[CB], oa, ob;
    } now;
    auto stage_a = [&](int s) {   // s one more than before
        now.oa += step_a;
        if (s == 0) {
            now.A = A, now.oa = 0;
#pragma unroll
            for (int i = 0; i < CA; ++i) now.va[i] = va[i];
        }
        if constexpr (!AKFAST) {
            if (a.gather && a.order && s < stages) {
                const int k0 = s * BK;
                if (k0 % (64 * LOOK) == 0) {
                    look_up(k0);
                } else if (k0 % 64 == 0) {
#pragma unroll
                    for (int i = 0; i + 1 < LOOK; ++i) next_rows[i] = next_rows[i + 1];
                }
#pragma unroll
                for (int i = 0; i < CA; ++i) {
                    uint32_t row;   // (a wave's chunks are of two or four rows)
                    if constexpr (RA == 32) {
                        const int k = k0 % 64 + 2 * wave + 8 * i;
                        const uint32_t r0 = __builtin_amdgcn_readlane(next_rows[0], k), r1 = __builtin_amdgcn_readlane(next_rows[0], k + 1);
                        row = lane < 32 ? r0 : r1;
                    } else {
                        row = __shfl(next_rows[0], k0 % 64 + (tid + 256 * i) / RA, 64);
                    }
                    now.va[i] = __builtin_elementwise_add_sat(va[i], row);   // what is nowhere stays there
                }
            }
        }
        if (s >= stages - 1) {
            const bool gone = s >= stages;   // behind the last stage: nothing; in it: nothing beyond the last k
            const int k0 = s * BK;
            if (gone) now.oa = 0;
#pragma unroll
            for (int i = 0; i < CA; ++i) {
                const int k = k0 + (AKFAST ? kc : (tid + 256 * i) / RA);
                now.va[i] = gone || k >= kend ? NOWHERE : now.va[i];
            }
        }
        now.oa = scalar_of(now.oa);
    };
    auto stage_b = [&](int s) {
        now.ob += step_b;
        if (s == 0) {
            now.B = B, now.ob = 0;
#pragma unroll
            for (int i = 0; i < CB; ++i) now.vb[i] = vb[i];
        }
        if (s >= stages - 1) {
            const bool gone = s >= stages;
            const int k0 = s * BK;
            if (gone) now.ob = 0;
#pragma unroll
            for (int i = 0; i < CB; ++i) {
                const int k = k0 + (BKFAST ? kc : (tid + 256 * i) / RB);
                now.vb[i] = gone || k >= kend ? NOWHERE : now.vb[i];
            }
        }
        now.ob = scalar_of(now.ob);
    };
    u32x4 fa[2][XT], fb[2][YT];
    auto read = [&](int set, int i, int slot_a, int slot_b, int h) {   // in the order in which the products ask for them
        if (i >= YT) fa[set][i - YT] = fragment32<T, TM, AKFAST, KB>(lds + slot_a, (wm * XT + i - YT) * 32, h, lane);
        else fb[set][i] = fragment32<T, TN, BKFAST, KB>(lds + slot_b, (wn * YT + i) * 32, h, lane);
    };
    constexpr int FRAGS = XT + YT, CHUNKS = CA + CB;
    if constexpr (MODE == SHARED) {
        // V . E[g] for the groups that the tile's rows belong to, before the accumulators hold anything else: in f16 a row's
        // V is scaled by a power of two, which is undone here.  The pair's halves are 2 pad k's against E twice.  Rows of
        // another group keep what they have -- selected, not multiplied by zero, which infinite factors would survive.
        const u32x4 V = buffer_of((const char*)a.V + (int64_t)t.first * a.v_row * 2, (uint32_t)((t.rows - 1) * a.v_row * 2 + 2 * a.pad * 2));
        each_group(a, t.first, t.first + t.rows - 1, [&](int g, int from, int to) {
            from -= t.first, to -= t.first;
            const u32x4 E = buffer_of((const char*)a.E + g * a.e_group * 2, (uint32_t)(BKFAST ? (a.N - 1) * a.e_n * 2 + a.r * 2 : (a.r - 1) * a.e_k * 2 + a.N * 2));
            for (int k0 = 0; k0 < 2 * a.pad; k0 += BK) {
                __syncthreads();   // the last stage has been read
#pragma unroll
                for (int i = 0; i < CA; ++i)
                    load_to_lds(V, cr + RPI * i < t.rows ? (uint32_t)((cr + RPI * i) * a.v_row * 2) + (k0 + kc) * 2 : NOWHERE, 0, lds0 + i * 4096 + wave * 1024);
#pragma unroll
                for (int i = 0; i < CB; ++i) {
                    uint32_t v;
                    if constexpr (BKFAST) {
                        const int k = k0 + kc, rank = k >= a.pad ? k - a.pad : k, n = n0 + cr + RPI * i;
                        v = n < a.N && rank < a.r ? (uint32_t)(n * a.e_n * 2) + rank * 2 : NOWHERE;
                    } else {
                        const int id = tid + 256 * i, kk = id / RB, k = k0 + kk, rank = k >= a.pad ? k - a.pad : k;
                        const int n = n0 + ((id % RB) ^ (rowfast_swizzle<T>(kk) & (RB - 1))) * 8;
                        v = n < a.N && rank < a.r ? (uint32_t)(rank * a.e_k * 2) + n * 2 : NOWHERE;
                    }
                    load_to_lds(E, v, 0, lds0 + BASE_B + i * 4096 + wave * 1024);
                }
                wait_loads<0>();
                wait_fragments_and_barrier();
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    u32x4 eb[YT];
#pragma unroll
                    for (int y = 0; y < YT; ++y) {
                        eb[y] = fragment32<T, TN, BKFAST, KB>(lds + BASE_B, (wn * YT + y) * 32, h, lane);
                        if (k0 + 16 * h >= a.pad) eb[y] = finite_only<T>(eb[y]);
                    }
#pragma unroll
                    for (int x = 0; x < XT; ++x) {
                        const int r0 = (wm * XT + x) * 32, r = r0 + (lane & 31);
                        if (to <= r0 || from >= r0 + 32) continue;
                        const u32x4 ea = fragment32<T, TM, true, KB>(lds, r0, h, lane);
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
        });
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
        // Between two barriers lie H M products, and the loads of a stage of each operand into the slots that the first of them
        // frees: item c beside product place(c).  Evenly, because loads in a row wait for one
        // another and hold the products up; with a slot less for the second operand, that one's first.
        constexpr int M = XT * YT;
        constexpr bool SKEW = SA > SB;
        auto place = [](int c) { return !SKEW ? c * H * M / CHUNKS : c < CB ? c * M / CB : M + (c - CB) * 2 * M / CA; };
        constexpr int FIRST = SKEW ? CB : (CHUNKS + H - 1) / H;   // items before the stage's end
        now.oa = now.ob = 0;
        const uint32_t mine = scalar_of(lds0 + wave * 1024);
#pragma unroll
        for (int s = 0; s < SA; ++s) {
            stage_a(s);
            if (s < SB) stage_b(s);
#pragma unroll
            for (int i = 0; i < CA; ++i)                           // (the loop goes on with what is left out here)
                if (s < SA - 1 || (!SKEW && i < FIRST)) load_to_lds(now.A, now.va[i], now.oa, mine + s * TILE_A + i * 4096);
#pragma unroll
            for (int i = 0; i < CB; ++i)
                if (s < SB - 1 || (SKEW && s < SB) || (!SKEW && CA + i < FIRST)) load_to_lds(now.B, now.vb[i], now.ob, mine + BASE_B + s * TILE_B + i * 4096);
        }
        wait_loads<SKEW ? (SB - 1) * CHUNKS : (SA - 2) * CHUNKS + FIRST>();
        wait_fragments_and_barrier();
        int at_a = 0, at_b = BASE_B;
#pragma unroll
        for (int i = 0; i < FRAGS; ++i) read(0, i, at_a, at_b, 0);
        uint32_t before_a = scalar_of(mine + (SA - 1) * TILE_A), before_b = scalar_of(mine + BASE_B + (SB - 1) * TILE_B);
        for (int s = 0; s < stages; ++s) {
            // (behind the last stage the loads go nowhere and the fragments that are read are not used)
            const int next_a = at_a + TILE_A < BASE_B ? at_a + TILE_A : 0, next_b = at_b + TILE_B < S::LDS ? at_b + TILE_B : BASE_B;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                constexpr int LAST = H - 1;
                if (h == LAST) {
                    stage_b(s + SB);
                    stage_a(s + SA);
                    before_a = scalar_of(mine + at_a), before_b = scalar_of(mine + at_b);
                    wait_loads<(SB - 2) * CHUNKS + (SA - SB) * CA>();
                    wait_fragments_and_barrier();
                }
                // One wave has a SIMD to itself and issues one instruction in four cycles or more, a few beside each product of
                // 32: the reads and loads are dealt out between the products, in this order and no other.
                const int from = h == LAST ? 0 : (h + 1) * M;   // products since the barrier
#pragma unroll
                for (int m = 0; m < M; ++m) {
#pragma unroll
                    for (int i = m * FRAGS / M; i < (m + 1) * FRAGS / M; ++i)
                        read((h + 1) & 1, i, h == LAST ? next_a : at_a, h == LAST ? next_b : at_b, (h + 1) % H);
                    acc[m / YT][m % YT] = mma32<T>(fb[h & 1][m % YT], fa[h & 1][m / YT], acc[m / YT][m % YT]);
                    unrolled<CHUNKS>([&](auto item) {   // item c: chunk i of the first operand, or of the second
                        constexpr int c = decltype(item)::value;
                        constexpr bool first = SKEW ? c >= CB : c < CA;
                        constexpr int i = SKEW ? (c >= CB ? c - CB : c) : c < CA ? c : c - CA;
                        if (place(c) != from + m) return;
                        if constexpr (first) load_to_lds<i * 4096>(now.A, now.va[i], now.oa, before_a);
                        else load_to_lds<i * 4096>(now.B, now.vb[i], now.ob, before_b);
                    });
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            at_a = next_a, at_b = next_b;
        }
        wait_loads<0>();
    }

    // Results leave through LDS, so that a wave stores whole runs of a row: 16-byte chunks, the chunk index XORed with the
    // row because the 32 rows of a register would meet in one bank otherwise.  (Straight from the registers a store would
    // touch 32 rows with 16 bytes each.)
    const float alpha = !real ? 0.0f : (float)a.alpha * (MODE == ROWS && a.scales ? ((const float*)a.scales)[t.group] : 1.0f), beta = (float)a.beta;
    if constexpr (MODE == PAIR) {
        // B's columns are a pair, hi and lo `pad` apart: their sums are added here, in f32, unless an infinity of A's is in them (finite_only)
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
        // four columns a thread; the direction in which the result is contiguous goes along the lanes
        const int rows = a.M - m0 < TM ? a.M - m0 : TM;
        const bool down = a.c_row == 1, across = a.c_n == 1 && a.c_row % 4 == 0 && a.c_group % 4 == 0 && ((uintptr_t)a.C & 7) == 0;
        for (int id = tid; id < TM * 16; id += 256) {
            const int r = down ? id % TM : id / 16, c = 4 * (down ? id / TM : id % 16);
            if (r >= rows || c >= a.r) continue;
            const char* const row = lds + r * (TN * 4);
            const f32x4 hi = *(const f32x4*)(row + (((c >> 2) ^ (r & 15)) << 4));
            const f32x4 lo = *(const f32x4*)(row + ((((c + a.pad) >> 2) ^ (r & 15)) << 4));
            T* const out = (T*)a.C + t.group * a.c_group + (m0 + r) * a.c_row + c * a.c_n;
            T v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (T)(alpha * (__builtin_isfinite(hi[i]) ? hi[i] + lo[i] : hi[i]));
            if (across && c + 4 <= a.r) {
                __builtin_memcpy(out, v, 8);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < a.r) out[i * a.c_n] = v[i];
            }
        }
        return;
    }
    if constexpr (MODE == ROWS)
        if (a.wide) {
            // f32 results, 32 WM rows at a time through LDS as in the pair's case
            static_assert(32 * S::WM * TN * 4 <= S::LDS, "a pass's results fit the stages");
            constexpr int CHUNKS_W = TN / 4;
#pragma unroll
            for (int x = 0; x < XT; ++x) {
                __syncthreads();
                const int r = wm * 32 + (lane & 31);
#pragma unroll
                for (int y = 0; y < YT; ++y)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int chunk = (wn * YT + y) * 8 + 2 * g + (lane >> 5);
                        const f32x4 v = {alpha * acc[x][y][4 * g], alpha * acc[x][y][4 * g + 1], alpha * acc[x][y][4 * g + 2], alpha * acc[x][y][4 * g + 3]};
                        *(f32x4*)(lds + r * (TN * 4) + ((chunk ^ (r & 15)) << 4)) = v;
                    }
                __syncthreads();
                for (int id = tid; id < 32 * S::WM * CHUNKS_W; id += 256) {
                    const int s = id / CHUNKS_W, chunk = id % CHUNKS_W, row = ((s >> 5) * XT + x) * 32 + (s & 31), n = n0 + 4 * chunk;
                    if (row >= t.rows || n >= a.N) continue;
                    *(f32x4*)((float*)a.C + (t.first + row) * a.c_row + n) = *(const f32x4*)(lds + s * (TN * 4) + ((chunk ^ (s & 15)) << 4));
                }
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
    constexpr int TM = S::TM, TN = S::TN;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    char* const lds = (char*)smem_raw;
    const int tiles_n = (a.N + TN - 1) / TN;
    Tile t;
    if constexpr (MODE == ROWS) {
        if (!find_tile(a, TM, tiles_n, block_of(a), t)) return;
        if constexpr (TM == 256) {
            // a group's last tile is seldom full: half or a quarter of the rows in half or 0.4 of the time
            typedef Shape<1, 4, 2, S::YT / 2, S::KB, S::SA, S::SB> Quarter;
            typedef Shape<2, 2, 2, S::YT, S::KB, S::SA, S::SB> Half;
            static_assert(Quarter::TN == TN && Half::TN == TN && Half::LDS <= S::LDS, "the same columns");
            if (t.rows <= 64) {
                fast_tile<T, MODE, BKFAST, Quarter>(a, t, lds);
                return;
            }
            if (t.rows <= 128) {
                fast_tile<T, MODE, BKFAST, Half>(a, t, lds);
                return;
            }
        }
    } else if constexpr (MODE == OUTER || MODE == PAIR) {
        if (!outer_tile(a, TM, TN, block_of(a), t)) return;
    } else {
        if (!shared_tile(a, TM, tiles_n, block_of(a), t)) return;
    }
    fast_tile<T, MODE, BKFAST, S>(a, t, lds);
}

// Whether the kernel can take a call: rows that start 16-byte aligned and end with a chunk, spans that 32 bits address.
inline bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
inline bool fast_rows(const void* p, int64_t rows, int64_t stride, int64_t inner_stride, int64_t inner) {
    return aligned(p, 16) && inner_stride == 1 && inner % 8 == 0 && stride % 8 == 0 && stride >= inner && (rows - 1) * stride * 2 + inner * 2 < MOST_SPAN;
}
template <int MODE> inline bool fast_takes(const Args& a, bool bkfast) {
    if (MODE == PAIR) return a.pad > 0 && a.pad <= 64 && !a.use_beta && fast_rows(a.A, a.a_rows, a.a_row, a.a_col, a.M) && fast_rows(a.B, a.b_rows, a.b_k, a.b_n, 2 * a.pad);
    if (a.c_n != 1 || a.c_row % 4 || a.N % 4 || !aligned(a.C, a.wide ? 16 : 8)) return false;
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
