// ragged.hpp -- products over rows in groups: the kernel that every type, layout and direction can take, and the
// pieces it shares with the faster ones (k_ragged_*.hip instantiate it, ragged.cpp checks and dispatches).
//
//   rows    C[p, :] = alpha * sum_k A[src(p), k] * B[g(p), k, :] + beta * C[p, :]        for p in group g(p)
//   outer   C[g, i, :] = alpha * sum_{p in g} A[src(p), i] * B[p, :] + beta * C[g, i, :]
//   shared  C[t, :] = sum_k A[t, k] * B[k, :] + sum_j V[p, j] * E[g(p), j, :]            t = order[p], p = 0 .. n_rows
//
// with the groups' offsets, and the order that src() reads, in device memory: the host knows neither how many rows a
// group has nor which, so a launch has as many blocks as the rows could need and each block finds its tile in the
// offsets itself.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gemm_common.hpp"

namespace tfh {
namespace ragged {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));

// E: elements of a 16-byte chunk.  mma() multiplies one chunk of each operand per lane: lane l = 16 q + j holds row j and
// the k's of its chunk; 16-bit types take the whole chunk in one instruction (k = 8 q + e), f32 and f64 in E of them,
// instruction e taking the k's E q + e -- any assignment of k's to lanes is right that both operands share.
// The first operand's row index becomes the accumulator's register index: row() of register r.
template <class T> struct Num;
template <> struct Num<__bf16> {
    static constexpr int E = 8;
    typedef float acc;   // what sums are held in
    typedef f32x4 acc4;
    __device__ static __forceinline__ acc4 mma(u32x4 a, u32x4 b, acc4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ static __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Num<_Float16> {
    static constexpr int E = 8;
    typedef float acc;
    typedef f32x4 acc4;
    __device__ static __forceinline__ acc4 mma(u32x4 a, u32x4 b, acc4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    __device__ static __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Num<float> {
    static constexpr int E = 4;
    typedef float acc;
    typedef f32x4 acc4;
    __device__ static __forceinline__ acc4 mma(u32x4 a, u32x4 b, acc4 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
    __device__ static __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Num<double> {
    static constexpr int E = 2;
    typedef double acc;
    typedef f64x4 acc4;
    __device__ static __forceinline__ acc4 mma(u32x4 a, u32x4 b, acc4 c) {
        const f64x2 x = __builtin_bit_cast(f64x2, a), y = __builtin_bit_cast(f64x2, b);
#pragma unroll
        for (int e = 0; e < 2; ++e) c = __builtin_amdgcn_mfma_f64_16x16x4f64(x[e], y[e], c, 0, 0, 0);
        return c;
    }
    __device__ static __forceinline__ int row(int q, int r) { return q + 4 * r; }
};

// The kernel's view of a call.  Strides in elements.  K, N: extents of the contracted axis and of C's columns (rows and
// shared); outer: M and N are C[g]'s extents.
struct Args {
    const void* A;
    const void* B;
    void* C;
    const int32_t* offsets;   // n_groups + 1
    const int32_t* order;     // null: rows lie group by group
    int64_t a_row, a_col;     // A[row, k] (rows, shared), A[row, i] (outer)
    int64_t b_group, b_k, b_n;   // B[g, k, n]; outer: B[p, n] with b_k the row stride
    int64_t b_rows;           // outer: rows that B has
    int64_t c_group, c_row, c_n;
    int64_t n_rows;           // rows in the order
    int64_t a_rows;           // rows that A has: an index beyond them reads as zeros
    int32_t n_groups, fan;
    int32_t M, N, K;
    int32_t gather;           // A's row of p is order[p] / fan, else p
    int32_t scatter;          // C's row of p is order[p], else p
    int32_t zero_rest;        // rows: the rows behind the last group are written as zeros, else left alone
    int32_t use_beta;
    int32_t wide;             // rows: C is of the sums' type (parts that are added up before they are rounded); no beta, no scatter
    double alpha, beta;
    // shared: the low-rank part, V[p, 0 .. r) against E[g, j, n]; rows of no group are without it.  V is of the sums' type, or
    // (pad > 0) a pair of the operands' type: row p is hi[0 .. pad), lo[0 .. pad), V = up[p] (hi + lo), zeros from r on
    const void* V;
    const void* E;
    int64_t v_row, e_group, e_k, e_n;
    int32_t r, pad;
    float* up;                // f16: the power of two by which row p was scaled down; null: 1 (written with V, read with it)
    const void* scales;       // rows: factors of the groups' results (of the accumulators' type) beside alpha, or null
    uint32_t grid_x;          // the launch's blocks along x; the launcher sets it (a dimension has less than 2^32 threads)
};

enum Mode { ROWS = 0, OUTER = 1, SHARED = 2, PAIR = 3 };   // PAIR: outer with a pair of V's form for B (ragged_fast.hpp)

// E elements of type C from a row of S that starts at any element: `count` of them are there, the others read as zeros.
template <class S, class C>
__device__ __forceinline__ u32x4 load_chunk(const S* p, int64_t stride, int count) {
    constexpr int E = Num<C>::E;
    u32x4 v = {0, 0, 0, 0};
    if (count >= E && stride == 1) {
        if constexpr (sizeof(S) == sizeof(C)) {
            __builtin_memcpy(&v, p, 16);
        } else {
            S s[E];
            C c[E];
            __builtin_memcpy(s, p, E * sizeof(S));
#pragma unroll
            for (int i = 0; i < E; ++i) c[i] = (C)s[i];
            __builtin_memcpy(&v, c, 16);
        }
    } else if (count > 0) {
        C c[E];
#pragma unroll
        for (int i = 0; i < E; ++i) c[i] = i < count ? (C)p[i * stride] : (C)0;
        __builtin_memcpy(&v, c, 16);
    }
    return v;
}

// The same in two parts for rows of elements next to each other, at least E of them: a load of the E elements up to the row's
// end where that lies inside the chunk, which nothing waits for, and, when it is wanted, what of it is put in place.
template <class T> __device__ __forceinline__ u32x4 load_unit(const T* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <class T> __device__ __forceinline__ void settle_unit(u32x4& v, int count) {
    constexpr int E = Num<T>::E;
    struct { uint64_t lo, hi; } w = __builtin_bit_cast(decltype(w), v);
    const int s = count >= E ? 0 : count <= 0 ? 128 : (E - count) * (int)sizeof(T) * 8;   // bits that are not there
    if (s >= 128) w = {0, 0};
    else if (s >= 64) w = {w.hi >> (s - 64), 0};
    else if (s > 0) w = {w.lo >> s | w.hi << (64 - s), w.hi >> s};
    v = __builtin_bit_cast(u32x4, w);
}

// ---- tiles in LDS -------------------------------------------------------------------------------------------------
// An operand's tile is 128 bytes of k by TM rows.  k-fast: [row][8 chunks], the chunk index XORed with the row so that
// the 16 rows of a fragment read spread over the banks.  row-fast: [k][TM elements], whose 16-bit fragments are read by
// the transposing LDS load (four rows of k by 16 columns, 8 bytes a lane); the XOR there moves the 32-byte pieces that
// the rows of one instruction touch to different banks.
template <class T> __device__ __forceinline__ uint32_t kfast_at(uint32_t row, uint32_t chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
template <class T> __device__ __forceinline__ uint32_t rowfast_swizzle(uint32_t k) {
    if constexpr (sizeof(T) == 2) return ((k & 3) | (((k >> 3) & 1) << 2)) << 1;
    else if constexpr (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
    else return 0;
}
template <class T, int TM> __device__ __forceinline__ uint32_t rowfast_at(uint32_t k, uint32_t chunk) {
    constexpr uint32_t chunks = TM * (uint32_t)sizeof(T) / 16;   // of a row; a narrow tile uses fewer bits of the XOR
    return k * (TM * (uint32_t)sizeof(T)) + ((chunk ^ (rowfast_swizzle<T>(k) & (chunks - 1))) << 4);
}
// The chunk (h = 0, 1: which half of the 128 bytes of k) of 16 rows from `row`, as mma() takes it.
template <class T, int TM, bool KFAST>
__device__ __forceinline__ u32x4 fragment(const char* tile, int row, int h, int lane) {
    const int q = lane >> 4, j = lane & 15;
    if constexpr (KFAST) {
        return *(const u32x4*)(tile + kfast_at<T>(row + j, q + 4 * h));
    } else if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
        const int k = (q + 4 * h) * 8 + (j >> 2), col = row + 4 * (j & 3);
        const uint32_t within = (col * 2) & 15, chunk = (col * 2) >> 4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(tile + rowfast_at<T, TM>(k, chunk) + within));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(tile + rowfast_at<T, TM>(k + 4, chunk) + within));
        struct { s16x4 a, b; } both = {lo, hi};
        return __builtin_bit_cast(u32x4, both);
    } else {
        constexpr int E = Num<T>::E;
        T e[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t k = (q + 4 * h) * E + i, at = (row + j) * (uint32_t)sizeof(T);
            e[i] = *(const T*)(tile + rowfast_at<T, TM>(k, at >> 4) + (at & 15));
        }
        u32x4 v;
        __builtin_memcpy(&v, e, 16);
        return v;
    }
}

// ---- which tile a block works on --------------------------------------------------------------------------------------
__device__ __forceinline__ int clamp_row(int32_t o, int64_t n_rows) { return o < 0 ? 0 : o > n_rows ? (int)n_rows : o; }
struct Tile {
    int group;   // n_groups: the rows behind the last group
    int first, rows, tile_m, tile_n;
};
__device__ __forceinline__ uint32_t block_of(const Args& a) { return blockIdx.y * a.grid_x + blockIdx.x; }
// Beyond so many groups no block adds all of their tiles up (which every wave of every block would have to wait for): tiles then end at
// whole multiples of their rows, counted from the first row of all, as well as with their group.  A group's rows are so cut into
// one tile more than need be, and which tile is a block's takes a binary search only (f32,
// 64 x 64: 4096 groups of 16 rows 216 us, and 57 so; 16 384 of them 2875 and 219; 65 536 of 4 rows, 32 x 32: 40 ms and 509 us).
constexpr int MANY_GROUPS = 2048;
__host__ __device__ inline int64_t many_tiles(int64_t n_rows, int64_t groups, int tm) {
    const int64_t cuts = groups + (n_rows + tm - 1) / tm;
    return cuts < n_rows ? cuts : n_rows;
}
__device__ __forceinline__ bool find_tile_of_many(const Args& a, int tm, int tiles_n, uint32_t block, Tile& t) {
    const int groups = a.n_groups + (a.zero_rest ? 1 : 0);
    const int64_t tiles = many_tiles(a.n_rows, groups, tm);
    if (block >= tiles * tiles_n) return false;
    const uint32_t want = (uint32_t)gemm::logical_block(block, (uint64_t)(tiles * tiles_n));
    const int k = (int)(want / (uint32_t)tiles_n);
    auto start_of = [&](int g) { return g > a.n_groups ? (int)a.n_rows : clamp_row(a.offsets[g], a.n_rows); };
    const bool by_row = tiles == a.n_rows;   // fewer rows than cuts: a tile for each row, of which those that start none are left out
    // Cuts in order: groups' starts and the multiples of tm, a group's first where they are equal; group g's is cut g + (multiples before).
    auto cut_of = [&](int g) { return by_row ? (int64_t)start_of(g) : (int64_t)g + (start_of(g) + tm - 1) / tm; };
    int low = 0, high = groups;   // the first group whose cut (row) lies behind the k-th
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (cut_of(mid) > k) high = mid;
        else low = mid + 1;
    }
    if (low == 0) return false;
    t.group = low - 1, t.tile_m = 0, t.tile_n = (int)(want % (uint32_t)tiles_n);
    const int from = start_of(low - 1), end = start_of(low);
    int64_t first;
    bool starts;
    if (by_row) first = k, starts = k == from || k % tm == 0;
    else starts = true, first = cut_of(low - 1) == k ? from : ((int64_t)k - low) * tm;
    int64_t next = by_row || first != from ? (first / tm + 1) * tm : (first + tm - 1) / tm * tm;
    if (!by_row && first == from && cut_of(low - 1) != k) next = first + tm;   // the multiple that a group starts at
    t.first = (int)first;
    t.rows = (int)((next < end ? next : end) - first);
    return starts && first >= from && first < a.n_rows && t.rows > 0;
}
// Tiles are dealt group by group; inside a group as tile_of() walks a matrix.  Every wave does this for itself: the
// lanes take 64 groups at a time.  Returns false when the block has none.
__device__ __forceinline__ bool find_tile(const Args& a, int tm, int tiles_n, uint32_t block, Tile& t) {
    if (a.n_groups > MANY_GROUPS) return find_tile_of_many(a, tm, tiles_n, block, t);
    const int lane = threadIdx.x & 63;
    const int groups = a.n_groups + (a.zero_rest ? 1 : 0);
    auto rows_of = [&](int g) {
        if (g >= groups) return 0;
        const int from = clamp_row(a.offsets[g], a.n_rows);
        const int to = g < a.n_groups ? clamp_row(a.offsets[g + 1], a.n_rows) : (int)a.n_rows;
        return to > from ? to - from : 0;
    };
    // (a launch has fewer blocks than 2^31, and so there are fewer tiles; the scalars tell the compiler that they are)
    uint32_t total = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) total += (uint32_t)((rows_of(g0 + lane) + tm - 1) / tm);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d, 64);
    total = __builtin_amdgcn_readfirstlane(total) * (uint32_t)tiles_n;
    if (block >= total) return false;
    // every XCD walks one contiguous range of the tiles
    uint32_t want = __builtin_amdgcn_readfirstlane((uint32_t)gemm::logical_block(block, total));
    for (int g0 = 0; g0 < groups; g0 += 64) {
        const int rows = rows_of(g0 + lane);
        const uint32_t mine = (uint32_t)((rows + tm - 1) / tm) * (uint32_t)tiles_n;
        uint32_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d, 64);
            if (lane >= d) upto += o;
        }
        const uint32_t here = __builtin_amdgcn_readlane(upto, 63);
        if (want < here) {
            const int at = __builtin_ctzll(__ballot(want < upto));
            const uint32_t rest = want - __builtin_amdgcn_readlane(upto - mine, at);
            const int rows_g = __builtin_amdgcn_readlane(rows, at);
            t.group = g0 + at;
            gemm::tile_of(rest, (rows_g + tm - 1) / tm, tiles_n, t.tile_m, t.tile_n);
            t.first = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[t.group], a.n_rows)) + t.tile_m * tm;
            t.rows = rows_g - t.tile_m * tm < tm ? rows_g - t.tile_m * tm : tm;
            return true;
        }
        want -= here;
    }
    return false;
}
// Shared: the rows' tiles, of whatever groups.
__device__ __forceinline__ bool shared_tile(const Args& a, int tm, int tiles_n, uint32_t block, Tile& t) {
    const int tiles_m = (int)((a.n_rows + tm - 1) / tm);
    const uint32_t total = (uint32_t)tiles_m * (uint32_t)tiles_n;
    if (block >= total) return false;
    gemm::tile_of((uint32_t)gemm::logical_block(block, total), tiles_m, tiles_n, t.tile_m, t.tile_n);
    t.group = 0;
    t.first = t.tile_m * tm;
    t.rows = a.n_rows - t.first < tm ? (int)(a.n_rows - t.first) : tm;
    return true;
}
// Outer products: every group has as many tiles, but each takes as long as the group has rows.  They are dealt to the XCDs in
// patches of up to 4 x 4, which share operands in an XCD's L2, the longest group's first (of up to 64 groups; of more, one
// wave's worth of sorting, the sums even out) and forth and back over the XCDs, so that all of them end at about the same time.
struct Patches {
    int tm, tn, pm, pn, across, each;   // a group's tiles, a patch's, patches along M, patches of a group
    __host__ __device__ Patches(const Args& a, int TM, int TN) {
        tm = (a.M + TM - 1) / TM, tn = (a.N + TN - 1) / TN;
        pm = tm < 4 ? tm : 4, pn = tn < 4 ? tn : 4;
        across = (tm + pm - 1) / pm, each = across * ((tn + pn - 1) / pn);
    }
    __host__ __device__ int64_t blocks(int n_groups) const { return ((int64_t)n_groups * across * ((tn + pn - 1) / pn) + 7) / 8 * 8 * (pm * pn); }
};
__device__ __forceinline__ bool outer_tile(const Args& a, int TM, int TN, uint32_t block, Tile& t) {
    const Patches s(a, TM, TN);
    const uint32_t size = s.pm * s.pn, xcd = block % gemm::XCDS, at = block / gemm::XCDS, turn = at / size, w = at % size;
    const uint32_t patch = turn * gemm::XCDS + (turn & 1 ? gemm::XCDS - 1 - xcd : xcd);
    if (patch >= (uint32_t)a.n_groups * s.each) return false;
    const uint32_t rank = patch / s.each, u = patch % s.each;
    t.tile_m = (u % s.across) * s.pm + w % s.pm, t.tile_n = (u / s.across) * s.pn + w / s.pm;
    if (t.tile_m >= s.tm || t.tile_n >= s.tn) return false;
    t.group = rank;
    if (a.n_groups <= 64) {
        const int lane = threadIdx.x & 63;
        const int from = lane < a.n_groups ? clamp_row(a.offsets[lane], a.n_rows) : 0, to = lane < a.n_groups ? clamp_row(a.offsets[lane + 1], a.n_rows) : 0;
        const int64_t mine = lane < a.n_groups ? (int64_t)(to > from ? to - from : 0) * 64 + 63 - lane : -1;
        uint32_t longer = 0;
        for (int g = 0; g < a.n_groups; ++g) longer += __shfl(mine, g, 64) > mine;
        t.group = __builtin_ctzll(__ballot(longer == rank && lane < a.n_groups));
    }
    t.first = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[t.group], a.n_rows));
    const int to = __builtin_amdgcn_readfirstlane(clamp_row(a.offsets[t.group + 1], a.n_rows));
    t.rows = to > t.first ? to - t.first : 0;
    return true;
}
// The group that holds row p (clamped offsets ascending), n_groups for the rows behind the last one.
__device__ __forceinline__ int group_of(const Args& a, int p) {
    int lo = 0, hi = a.n_groups;   // the first group that ends behind p
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.offsets[mid + 1] > p) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// Calls f(g, from, to) for the groups that rows first .. last belong to, in order; the lanes read 64 groups' offsets at a time.
template <class F> __device__ __forceinline__ void each_group(const Args& a, int first, int last, F f) {
    const int lane = threadIdx.x & 63;
    for (int g0 = a.n_groups > 256 ? __builtin_amdgcn_readfirstlane(group_of(a, first)) & ~63 : 0; g0 < a.n_groups; g0 += 64) {
        int from = 0, to = 0;
        if (g0 + lane < a.n_groups) from = clamp_row(a.offsets[g0 + lane], a.n_rows), to = clamp_row(a.offsets[g0 + lane + 1], a.n_rows);
        uint64_t found = __ballot(to > from && to > first && from <= last);
        while (found) {
            const int b = __builtin_ctzll(found);
            found &= found - 1;
            f(g0 + b, (int)__builtin_amdgcn_readlane(from, b), (int)__builtin_amdgcn_readlane(to, b));
        }
        if (__ballot(to > last)) break;
    }
}
// The row of A that row p of the order reads; -1: none (the order names a row that is not there).
__device__ __forceinline__ int64_t source_row(const Args& a, int p) {
    int64_t s = p;
    if (a.gather && a.order) {
        const int o = a.order[p];
        s = o < 0 ? -1 : o / a.fan;
    }
    return s < a.a_rows ? s : -1;
}

// ---- the kernels for every type, layout and direction -----------------------------------------------------------------
// Tiles of 32 XT x 32 YT, four waves, operands through registers into a double-buffered LDS tile, 128 bytes of k at a time;
// the loads run two such stages ahead (one in large tiles).
//
// Bound by the matrix cores where rows are many, by the wait for loads where blocks are few.  Reached: f32, 32 768 rows of 16 groups,
// 2048 x 1024: 125 TFLOP/s (82 % of a library product's rate); bf16 rows that start at any address, 2047 x 1023: 610, where the
// aligned kernels reach 1000; f64, 8192 x 4096 x 4096: 66 of 76, 24 000 rows of 48 groups, 512 x 384: 46 -- nine tiles a compute
// unit, three at a time, each of which starts and ends with nothing to multiply.
constexpr int GENERAL_THREADS = 256;
// Waits for this wave's LDS accesses only: global loads stay in flight over the barrier.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One stage (128 bytes of k of type C) of a wave's 16 XT x 16 YT results.  Where not all rows take part, those in
// [from, to) of the tile take the products and the others keep what they have: a row that is not a group's must not see
// 0 * infinity from that group's factors.
template <class C, bool AKFAST, bool BKFAST, int XT, int YT, bool ALL>
__device__ __forceinline__ void multiply_stage(typename Num<C>::acc4 (&acc)[XT][YT], const char* stage, int wm, int wn, int lane, int from, int to) {
    constexpr int TM = 32 * XT, TN = 32 * YT;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        u32x4 fa[XT], fb[YT];
#pragma unroll
        for (int x = 0; x < XT; ++x) fa[x] = fragment<C, TM, AKFAST>(stage, (wm * XT + x) * 16, h, lane);
#pragma unroll
        for (int y = 0; y < YT; ++y) fb[y] = fragment<C, TN, BKFAST>(stage + TM * 128, (wn * YT + y) * 16, h, lane);
#pragma unroll
        for (int x = 0; x < XT; ++x) {
            const int r = (wm * XT + x) * 16 + (lane & 15);
            const bool mine = ALL || (r >= from && r < to);
#pragma unroll
            for (int y = 0; y < YT; ++y) {
                const typename Num<C>::acc4 v = Num<C>::mma(fb[y], fa[x], acc[x][y]);
                if constexpr (ALL) acc[x][y] = v;
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[x][y][i] = mine ? v[i] : acc[x][y][i];
            }
        }
    }
}
// A whole k loop: load(k0, ra, rb) fetches a stage's chunks, settle(k0, ra, rb) makes them what the tiles take.  Loads two
// stages ahead are made for those behind the last one too (of anything that is there): were they left out on a condition, the wait
// for one stage's would have to count on that, and would wait for the next one's as well.  With KW teams of four waves, team w takes
// the stages w, w + KW, ...; all of them go through the loop as often, so that they meet at its barriers.
template <class C, bool AKFAST, bool BKFAST, int XT, int YT, int KW, bool ALL, class Load, class Settle>
__device__ __forceinline__ void k_loop(typename Num<C>::acc4 (&acc)[XT][YT], char* lds, int k_end, int wm, int wn, int lane, int team, int from, int to,
                                       Load load_at, Settle settle_at) {
    constexpr int TM = 32 * XT, TN = 32 * YT, BK = 128 / (int)sizeof(C);
    const int kend = KW == 1 ? k_end : (k_end + KW * BK - 1) / (KW * BK) * BK;   // of the team's own stages, which are next to each other here
    auto load = [&](int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) { load_at(k0 * KW + team * BK, ra, rb); };
    auto settle = [&](int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) { settle_at(k0 * KW + team * BK, ra, rb); };
    constexpr int RA = TM * (int)sizeof(C) / 16, RB = TN * (int)sizeof(C) / 16;   // chunks of a row of k in a row-fast tile
    const int tid = threadIdx.x % GENERAL_THREADS, cc = tid & 7, cr = tid >> 3;
    auto store_stage = [&](char* stage, int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) {
        settle(k0, ra, rb);
#pragma unroll
        for (int i = 0; i < XT; ++i) {
            const int id = tid + GENERAL_THREADS * i;
            if constexpr (AKFAST) *(u32x4*)(stage + kfast_at<C>(cr + 32 * i, cc)) = ra[i];
            else *(u32x4*)(stage + rowfast_at<C, TM>(id / RA, id % RA)) = ra[i];
        }
#pragma unroll
        for (int i = 0; i < YT; ++i) {
            const int id = tid + GENERAL_THREADS * i;
            if constexpr (BKFAST) *(u32x4*)(stage + TM * 128 + kfast_at<C>(cr + 32 * i, cc)) = rb[i];
            else *(u32x4*)(stage + TM * 128 + rowfast_at<C, TN>(id / RB, id % RB)) = rb[i];
        }
    };
    if (kend <= 0) return;
    constexpr int STAGE = (TM + TN) * 128;
    if constexpr (XT + YT > 4) {   // a large tile's registers hold one stage beside the one that is multiplied
        u32x4 a0[XT], b0[YT];
        load(0, a0, b0);
        lds_barrier();
        store_stage(lds, 0, a0, b0);
        lds_barrier();
        int at = 0;
        for (int k0 = 0; k0 < kend; k0 += BK) {
            if (k0 + BK < kend) load(k0 + BK, a0, b0);
            multiply_stage<C, AKFAST, BKFAST, XT, YT, ALL>(acc, lds + at, wm, wn, lane, from, to);
            at ^= STAGE;
            if (k0 + BK < kend) store_stage(lds + at, k0 + BK, a0, b0);
            lds_barrier();
        }
    } else {
        u32x4 a0[XT], b0[YT], a1[XT], b1[YT];
        load(0, a0, b0);
        load(BK, a1, b1);
        lds_barrier();   // the last loop's tiles have been read
        store_stage(lds, 0, a0, b0);
        lds_barrier();
        int k0 = 0;
        for (; k0 + BK < kend; k0 += 2 * BK) {
            load(k0 + 2 * BK, a0, b0);
            multiply_stage<C, AKFAST, BKFAST, XT, YT, ALL>(acc, lds, wm, wn, lane, from, to);
            store_stage(lds + STAGE, k0 + BK, a1, b1);
            lds_barrier();
            load(k0 + 3 * BK, a1, b1);
            multiply_stage<C, AKFAST, BKFAST, XT, YT, ALL>(acc, lds + STAGE, wm, wn, lane, from, to);
            if (k0 + 2 * BK < kend) store_stage(lds, k0 + 2 * BK, a0, b0);
            lds_barrier();
        }
        if (k0 < kend) multiply_stage<C, AKFAST, BKFAST, XT, YT, ALL>(acc, lds, wm, wn, lane, from, to);
    }
}

// TA, TB: the operands' types; C: the type multiplied in (theirs, or that of the sums); TO: the result's.  UNIT: both operands
// contiguous in the direction in which they are read (B along k if BKFAST), of type C, and no shorter than a chunk.  KW: teams of
// four waves that share out k, for launches of few blocks, whose time is that of one block's loads after each other.
template <class TA, class TB, class C, class TO, int MODE, bool BKFAST, bool UNIT, int XT, int YT, int KW>
__global__ __launch_bounds__(GENERAL_THREADS * KW, KW == 1 ? 2 : 4) void ragged_general_kernel(const Args a) {
    typedef Num<C> NT;
    typedef typename NT::acc W;
    constexpr int E = NT::E, TM = 32 * XT, TN = 32 * YT, BK = 128 / (int)sizeof(C);
    constexpr bool AKFAST = MODE != OUTER;
    __shared__ __align__(16) char all_lds[KW * 2 * (TM + TN) * 128];
    const int tid = threadIdx.x % GENERAL_THREADS, team = KW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / GENERAL_THREADS);
    char* const lds = all_lds + team * 2 * (TM + TN) * 128;
    const int lane = tid & 63, wave = tid >> 6, wm = wave & 1, wn = wave >> 1, q = lane >> 4, j = lane & 15;
    const int tiles_n = (a.N + TN - 1) / TN;
    Tile t;
    if constexpr (MODE == ROWS) {
        if (!find_tile(a, TM, tiles_n, block_of(a), t)) return;
    } else if constexpr (MODE == OUTER) {
        if (!outer_tile(a, TM, TN, block_of(a), t)) return;
    } else {
        if (!shared_tile(a, TM, tiles_n, block_of(a), t)) return;
    }
    const bool real = MODE != ROWS || t.group < a.n_groups;   // the rows behind the last group have nothing to multiply
    const int n0 = t.tile_n * TN, m0 = t.tile_m * TM;
    typename NT::acc4 acc[XT][YT];
#pragma unroll
    for (int x = 0; x < XT; ++x)
#pragma unroll
        for (int y = 0; y < YT; ++y) acc[x][y] = (typename NT::acc4){0, 0, 0, 0};

    // This thread's chunks of a stage.  k-fast: chunk tid % 8 of rows tid / 8 + 32 i; row-fast: chunks tid + 256 i of [k][row].
    const int cc = tid & 7, cr = tid >> 3;

    if constexpr (MODE == SHARED) {
        constexpr int EW = Num<W>::E, RW = TN * (int)sizeof(W) / 16;
        each_group(a, t.first, t.first + t.rows - 1, [&](int g, int from, int to) {
            const TB* const Eg = (const TB*)a.E + g * a.e_group;
            auto load = [&](int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) {
#pragma unroll
                for (int i = 0; i < XT; ++i) {
                    const int k = k0 + cc * EW, r = cr + 32 * i;
                    ra[i] = load_chunk<W, W>((const W*)a.V + (int64_t)(t.first + r) * a.v_row + k, 1, r < t.rows ? a.r - k : 0);
                }
#pragma unroll
                for (int i = 0; i < YT; ++i) {
                    const int id = tid + GENERAL_THREADS * i;
                    if constexpr (BKFAST) {
                        const int k = k0 + cc * EW, n = n0 + cr + 32 * i;
                        rb[i] = load_chunk<TB, W>(Eg + n * a.e_n + k * a.e_k, a.e_k, n < a.N ? a.r - k : 0);
                    } else {
                        const int k = k0 + id / RW, n = n0 + (id % RW) * EW;
                        rb[i] = load_chunk<TB, W>(Eg + k * a.e_k + n * a.e_n, a.e_n, k < a.r ? a.N - n : 0);
                    }
                }
            };
            k_loop<W, true, BKFAST, XT, YT, KW, false>(acc, lds, a.r, wm, wn, lane, team, from - t.first, to - t.first, load, [](int, u32x4 (&)[XT], u32x4 (&)[YT]) {});
        });
    }

    const TA* const A = (const TA*)a.A;
    int64_t arow[XT];   // k-fast A: the source rows of this thread's chunks (-1: none)
    if constexpr (AKFAST) {
#pragma unroll
        for (int i = 0; i < XT; ++i) arow[i] = cr + 32 * i < t.rows && real ? source_row(a, t.first + cr + 32 * i) : -1;
    }
    const TB* const B = (const TB*)a.B + (MODE == ROWS && real ? t.group * a.b_group : 0);
    const int kend = MODE == OUTER ? t.rows : real ? a.K : 0;
    constexpr int RA = TM * (int)sizeof(C) / 16, RB = TN * (int)sizeof(C) / 16;
    // How many elements of chunk i are there, for the stage at k0.  (A row of A that is none, in outer mode, reads as zeros.)
    auto count_a = [&](int i, int k0) {
        const int id = tid + GENERAL_THREADS * i;
        return AKFAST ? (arow[i] >= 0 ? kend - k0 - cc * E : 0) : k0 + id / RA < kend ? a.M - m0 - (id % RA) * E : 0;
    };
    auto count_b = [&](int i, int k0) {
        const int id = tid + GENERAL_THREADS * i;
        return BKFAST ? (n0 + cr + 32 * i < a.N ? kend - k0 - cc * E : 0) : k0 + id / RB < kend ? a.N - n0 - (id % RB) * E : 0;
    };
    if constexpr (UNIT) {
        // Where this thread's chunks of a stage start, moved back to the row's last E elements where that ends inside one; rows and
        // columns beyond the tile's read the first ones.
        const int64_t step_b = KW * (BKFAST ? BK : BK * a.b_k);
        const TA* pa[XT];
        const TB* pb[YT];
#pragma unroll
        for (int i = 0; i < XT; ++i) {
            const int id = tid + GENERAL_THREADS * i, m = m0 + (id % RA) * E;
            if constexpr (AKFAST) pa[i] = A + (arow[i] > 0 ? arow[i] * a.a_row : 0) + team * BK + cc * E;
            else pa[i] = A + (m + E <= a.M ? m : a.M - E);
        }
#pragma unroll
        for (int i = 0; i < YT; ++i) {
            const int id = tid + GENERAL_THREADS * i, n = n0 + (id % RB) * E;
            if constexpr (BKFAST) pb[i] = B + (n0 + cr + 32 * i < a.N ? (n0 + cr + 32 * i) * a.b_n : 0) + team * BK + cc * E;
            else pb[i] = B + ((MODE == OUTER ? t.first : 0) + team * BK + id / RB) * a.b_k + (n + E <= a.N ? n : a.N - E);
        }
        const bool edge_b = !BKFAST && n0 + TN > a.N;   // both the same for all of a wave
        bool edge;
        if constexpr (AKFAST) {
            bool gone = false;
#pragma unroll
            for (int i = 0; i < XT; ++i) gone |= arow[i] < 0;
            edge = __any(gone);
        } else {
            edge = m0 + TM > a.M || (a.gather && a.order) || t.first + kend > a.a_rows;
        }
        uint32_t none = 0;   // outer: chunks of a stage on their way whose row of A is none, the stages' bits apart
        // whole stages move the pointers on, those behind them leave them there, at k = k_at
        const int kwhole = kend / BK * BK, k_at = KW == 1 ? kwhole : team * BK + (kwhole > team * BK ? (kwhole - team * BK + KW * BK - 1) / (KW * BK) * (KW * BK) : 0);
        auto load = [&](int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) {
            if constexpr (!AKFAST) {
                const bool found = !(a.gather && a.order) && t.first + kend <= a.a_rows;
#pragma unroll
                for (int i = 0; i < XT; ++i) {
                    const int id = tid + GENERAL_THREADS * i, k = k0 + id / RA;
                    const int64_t s = k >= kend ? -1 : found ? t.first + k : source_row(a, t.first + k);
                    const uint32_t bit = 1u << (((k0 / (KW * BK)) & 3) * 8 + i);
                    none = s < 0 ? none | bit : none & ~bit;
                    ra[i] = load_unit<TA>(pa[i] + (s < 0 ? 0 : s) * a.a_row);
                }
            }
            if (k0 < kwhole) {
                if constexpr (AKFAST)
#pragma unroll
                    for (int i = 0; i < XT; ++i) ra[i] = load_unit<TA>(pa[i]), pa[i] += KW * BK;
#pragma unroll
                for (int i = 0; i < YT; ++i) rb[i] = load_unit<TB>(pb[i]), pb[i] += step_b;
            } else {
                const int count = kend - k0 - cc * E;
                if constexpr (AKFAST)
#pragma unroll
                    for (int i = 0; i < XT; ++i) ra[i] = load_unit<TA>(pa[i] - (count >= E ? 0 : count > 0 ? E - count : k_at + cc * E));
#pragma unroll
                for (int i = 0; i < YT; ++i) {
                    const int id = tid + GENERAL_THREADS * i;
                    if constexpr (BKFAST) rb[i] = load_unit<TB>(pb[i] - (count >= E ? 0 : count > 0 ? E - count : k_at + cc * E));
                    else rb[i] = load_unit<TB>(pb[i] - (k0 + id / RB < kend ? 0 : (k_at + id / RB) * a.b_k));
                }
            }
        };
        auto settle = [&](int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) {
            const bool whole = k0 + BK <= kend;
            if (!whole || edge)
#pragma unroll
                for (int i = 0; i < XT; ++i) {
                    int count = count_a(i, k0);
                    if constexpr (!AKFAST)
                        if (none >> (((k0 / (KW * BK)) & 3) * 8 + i) & 1) count = 0;
                    settle_unit<C>(ra[i], count);
                }
            if (!whole || edge_b)
#pragma unroll
                for (int i = 0; i < YT; ++i) settle_unit<C>(rb[i], count_b(i, k0));
        };
        k_loop<C, AKFAST, BKFAST, XT, YT, KW, true>(acc, lds, kend, wm, wn, lane, team, 0, 0, load, settle);
    } else {
        auto load = [&](int k0, u32x4 (&ra)[XT], u32x4 (&rb)[YT]) {
#pragma unroll
            for (int i = 0; i < XT; ++i) {
                const int id = tid + GENERAL_THREADS * i;
                int count = count_a(i, k0);
                const TA* p;
                if constexpr (AKFAST) {
                    p = A + arow[i] * a.a_row + (k0 + cc * E) * a.a_col;
                } else {
                    const int64_t s = count > 0 ? source_row(a, t.first + k0 + id / RA) : -1;
                    if (s < 0) count = 0;
                    p = A + s * a.a_row + (m0 + (id % RA) * E) * a.a_col;
                }
                ra[i] = load_chunk<TA, C>(p, a.a_col, count);
            }
#pragma unroll
            for (int i = 0; i < YT; ++i) {
                const int id = tid + GENERAL_THREADS * i;
                const TB* p;
                if constexpr (BKFAST) {
                    p = B + (n0 + cr + 32 * i) * a.b_n + (k0 + cc * E) * a.b_k;
                } else {
                    const int64_t k = MODE == OUTER ? t.first + k0 + id / RB : k0 + id / RB;
                    p = B + k * a.b_k + (n0 + (id % RB) * E) * a.b_n;
                }
                rb[i] = load_chunk<TB, C>(p, BKFAST ? a.b_k : a.b_n, count_b(i, k0));
            }
        };
        k_loop<C, AKFAST, BKFAST, XT, YT, KW, true>(acc, lds, kend, wm, wn, lane, team, 0, 0, load, [](int, u32x4 (&)[XT], u32x4 (&)[YT]) {});
    }

    if constexpr (KW > 1) {   // the teams' sums, added in their order
        static_assert(sizeof(acc) * GENERAL_THREADS <= 2 * (TM + TN) * 128, "a team's sums fit its tiles");
        __syncthreads();
        if (team > 0) __builtin_memcpy(lds + tid * sizeof(acc), acc, sizeof(acc));
        __syncthreads();
        for (int w = 1; team == 0 && w < KW; ++w) {
            typename NT::acc4 more[XT][YT];
            __builtin_memcpy(more, all_lds + w * 2 * (TM + TN) * 128 + tid * sizeof(acc), sizeof(acc));
#pragma unroll
            for (int x = 0; x < XT; ++x)
#pragma unroll
                for (int y = 0; y < YT; ++y) acc[x][y] += more[x][y];
        }
    }

    W alpha = (W)a.alpha;
    const W beta = (W)a.beta;
    if constexpr (MODE == ROWS)
        if (a.scales && real) alpha *= ((const W*)a.scales)[t.group];
    if (a.c_n == 1 && !a.use_beta) {
        // Through LDS, so that a wave stores whole runs of a row, 16 bytes a lane; the chunk index is XORed with the row because the
        // rows of a register would meet in one bank otherwise.  (Straight from the registers a store has 32 bytes of each of 16 rows,
        // an element a lane: the gradients of 40 matrices of 3776 x 1861 from 50 rows, f16: 620 us so, 320 by LDS.)
        constexpr int PER = 16 / (int)sizeof(TO), ROW = TN / PER;   // elements of a chunk, chunks of a row
        static_assert(TM * TN * sizeof(TO) <= 2 * (TM + TN) * 128, "the results fit a team's tiles");
        auto place = [&](int r, int n) { return all_lds + r * (TN * (int)sizeof(TO)) + (((n / PER) ^ (r & (ROW - 1))) << 4) + n % PER * (int)sizeof(TO); };
        __syncthreads();
        if (KW == 1 || team == 0)
#pragma unroll
            for (int x = 0; x < XT; ++x)
#pragma unroll
                for (int y = 0; y < YT; ++y) {
                    TO out[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = real ? (TO)(alpha * acc[x][y][i]) : (TO)0;
                    const int r = (wm * XT + x) * 16 + j, n = (wn * YT + y) * 16;
                    if constexpr (sizeof(TO) == 8) {   // (every fourth column in a lane)
#pragma unroll
                        for (int i = 0; i < 4; ++i) *(TO*)place(r, n + NT::row(q, i)) = out[i];
                    } else {
                        __builtin_memcpy(place(r, n + NT::row(q, 0)), out, sizeof(out));
                    }
                }
        __syncthreads();
        const int rows = MODE == OUTER ? (a.M - m0 < TM ? a.M - m0 : TM) : t.rows;
        for (int id = threadIdx.x; id < rows * ROW; id += GENERAL_THREADS * KW) {
            const int r = id / ROW, n = id % ROW * PER;
            if (n0 + n >= a.N) continue;
            int64_t row = MODE == OUTER ? m0 + r : t.first + r;
            if constexpr (MODE != OUTER)
                if (a.scatter && a.order) {
                    row = a.order[row];
                    if (row < 0 || row >= a.n_rows) continue;
                }
            TO* const c = (TO*)a.C + (MODE == OUTER ? t.group * a.c_group : 0) + row * a.c_row + n0 + n;
            TO out[PER];
            __builtin_memcpy(out, place(r, n), 16);
            if (n0 + n + PER <= a.N) {
                __builtin_memcpy(c, out, 16);
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (n0 + n + i < a.N) c[i] = out[i];
            }
        }
        return;
    }
    if (team > 0) return;
#pragma unroll
    for (int x = 0; x < XT; ++x) {
        const int r = (wm * XT + x) * 16 + j;
        if (MODE == OUTER ? m0 + r >= a.M : r >= t.rows) continue;
        int64_t row = MODE == OUTER ? m0 + r : t.first + r;
        if constexpr (MODE != OUTER)
            if (a.scatter && a.order) {
                row = a.order[row];
                if (row < 0 || row >= a.n_rows) continue;
            }
        TO* const c = (TO*)a.C + (MODE == OUTER ? t.group * a.c_group : 0) + row * a.c_row;
#pragma unroll
        for (int y = 0; y < YT; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = n0 + (wn * YT + y) * 16 + NT::row(q, i);
                if (n >= a.N) continue;
                W v = real ? alpha * acc[x][y][i] : (W)0;
                if (a.use_beta && real) v += beta * (W)c[n * a.c_n];
                c[n * a.c_n] = (TO)v;
            }
    }
}

}  // namespace ragged
}  // namespace tfh
