// ragged_launch.hpp -- chooses and launches a kernel on rows in groups; one translation unit per operand type includes it.
#pragma once
#include <atomic>
#include <type_traits>

#include "launch.hpp"
#include "ragged.hpp"
#include "ragged_fast.hpp"
#include "ragged_few.hpp"
#include "ragged_thin.hpp"
#include "ragged_api.hpp"

namespace tfh {
namespace ragged {

inline int64_t tiles(int64_t n, int64_t t) { return (n + t - 1) / t; }
// The grid of a launch (launch_grid), and Args that know it.
inline int32_t grid_of(int64_t blocks, int threads, Args& a, dim3& grid) {
    if (int32_t e = launch_grid(blocks, threads, &a.grid_x, &grid.y)) return e;
    grid.x = a.grid_x;
    return TFH_OK;
}
// Blocks of a launch over the groups' rows: no more tiles than the rows fill and one more, partly filled, for each group.
inline int64_t row_tiles(const Args& a, int tm) {
    const int64_t groups = a.n_groups + (a.zero_rest ? 1 : 0);
    if (a.n_groups > MANY_GROUPS) return many_tiles(a.n_rows, groups, tm);
    return a.n_rows / tm + (groups < a.n_rows ? groups : a.n_rows);
}

// A kernel's dynamic LDS beyond the default, once for each device: the attribute is of the device that is current.
inline void allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& allowed) {
    int device = 0;
    (void)hipGetDevice(&device);
    const uint64_t bit = (uint64_t)1 << (device & 63);
    if (allowed.load(std::memory_order_relaxed) & bit) return;
    (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    allowed.fetch_or(bit, std::memory_order_relaxed);
}

// "(kernel<arguments>)" as tfh_last_kernel spells them.
template <class T> constexpr const char* type_name() {
    if constexpr (__is_same(T, __bf16)) return "bf16";
    else if constexpr (__is_same(T, _Float16)) return "f16";
    else if constexpr (__is_same(T, float)) return "float";
    else return "double";
}
constexpr const char* mode_name(int mode) { return mode == ROWS ? "rows" : mode == OUTER ? "outer" : mode == SHARED ? "shared" : "pair"; }

template <class TA, class TB, class C, class TO, int MODE, bool BKFAST, bool UNIT, int XT, int YT, int KW = 1>
int32_t launch_general_tiles(const Args& a, void* stream) {
    const int64_t tn = tiles(a.N, 32 * YT);
    const int64_t blocks = MODE == ROWS ? row_tiles(a, 32 * XT) * tn
                           : MODE == OUTER ? Patches(a, 32 * XT, 32 * YT).blocks(a.n_groups) : tiles(a.n_rows, 32 * XT) * tn;
    if (blocks <= 0) return TFH_OK;
    Args args = a;
    dim3 grid;
    if (int32_t e = grid_of(blocks, GENERAL_THREADS * KW, args, grid)) return e;
    static const std::string label = std::string("(ragged_general_kernel<") + type_name<TA>() + ", " + type_name<TB>() + ", " + type_name<C>() + ", " +
                                     type_name<TO>() + ", " + mode_name(MODE) + (BKFAST ? ", k, " : ", n, ") + (UNIT ? "unit, " : "any, ") +
                                     std::to_string(32 * XT) + "x" + std::to_string(32 * YT) + (KW > 1 ? ", " + std::to_string(KW) : std::string()) + ">)";
    TFH_LAUNCH_NAMED(label.c_str(), (ragged_general_kernel<TA, TB, C, TO, MODE, BKFAST, UNIT, XT, YT, KW>), grid, dim3(GENERAL_THREADS * KW), 0, (hipStream_t)stream, args);
    return hip_check(hipGetLastError(), "product over groups of rows");
}
// Whether both operands are contiguous in the direction in which the kernel reads them, and long enough for a chunk.
template <class C, int MODE, bool BKFAST> bool unit_strides(const Args& a) {
    constexpr int E = Num<C>::E;
    if (a.a_rows < 1) return false;   // not one row to read where there is none to multiply
    if (MODE == OUTER) return a.a_col == 1 && a.M >= E && a.b_n == 1 && a.N >= E;
    return a.a_col == 1 && a.K >= E && (BKFAST ? a.b_k == 1 : a.b_n == 1 && a.N >= E);
}
// Few blocks wait for their loads, stage after stage: tiles of 32 x 32 then, four times the blocks of 64 x 64, and four teams to
// share out k, where that has eight stages at least and the blocks are fewer than one a compute unit, or two where k has 32 stages
// (f64, 236 rows, 1472 x 38: 65 us against 24; 200 bf16 rows of four groups, 4001 x 1001: 63 and 29, of two, 4096 x 512, aligned: 38
// and 13; 248 blocks, f16, 3001 x 500: 42 and 37; 299 blocks, 1001 x 777: 18 and 29; 330, f64, 256 x 640: 27 and 29, 1024 x 640: 81 and
// 67; 702, f32, 1000 x 800: 79 and 87).  Gradients: fewer than two, from more than 512 rows of a group on (8192 of four, 256 x 256:
// 38 and 11; 16 384 of eight, 512 x 256: 38 and 29; of 32 groups, 128 x 128, 512 rows each: 11 and 13).  `bytes`: of an operand's
// element; aligned 16-bit operands leave their own kernels for this one as well.
template <int MODE> bool starved(const Args& a, int bytes) {
    const int64_t blocks = MODE == OUTER ? Patches(a, 64, 64).blocks(a.n_groups) : (MODE == ROWS ? row_tiles(a, 64) : tiles(a.n_rows, 64)) * tiles(a.N, 64);
    const int64_t k = MODE == OUTER ? a.n_rows / a.n_groups : a.K;
    return blocks < (MODE == OUTER || k * bytes >= 4096 ? 512 : 256) && k * bytes >= 1024 + (MODE == OUTER ? bytes : 0);
}
template <class TA, class TB, class C, class TO, int MODE, bool BKFAST>
int32_t launch_general(const Args& a, void* stream) {
    if constexpr (__is_same(TA, C) && __is_same(TB, C))
        if (unit_strides<C, MODE, BKFAST>(a)) {
            // 128 x 128 tiles where the rows fill them and there are enough for the machine: of 16 bits from one a compute unit on
            // (32 768 rows of 16 groups, 2047 x 1023: 241 us against 377; 168 of them, 3000 x 1001 x 777: 31 against 25), of f32, where
            // the matrix units take 16 times as long, from eight (2048 x 1024: 1096 against 1172; 24 000 rows of 48 groups, 512 x 384: 140
            // against 108).  f64's sums take registers that such tiles do not have.
            if constexpr (sizeof(C) < 8) {
                const int64_t rows = MODE == OUTER ? a.M : MODE == ROWS ? a.n_rows / a.n_groups : a.n_rows;
                const int64_t blocks = (MODE == OUTER ? a.n_groups * tiles(a.M, 128) : MODE == ROWS ? a.n_rows / 128 + a.n_groups / 2 : tiles(a.n_rows, 128)) * tiles(a.N, 128);
                if (rows > 96 && a.N > 96 && blocks >= (sizeof(C) == 4 ? 2048 : 256)) return launch_general_tiles<TA, TB, C, TO, MODE, BKFAST, true, 4, 4>(a, stream);
            }
            if (starved<MODE>(a, sizeof(C))) return launch_general_tiles<TA, TB, C, TO, MODE, BKFAST, true, 1, 1, 4>(a, stream);
            return launch_general_tiles<TA, TB, C, TO, MODE, BKFAST, true, 2, 2>(a, stream);
        }
    // (an adapter's factor, bf16 rows by f32 sums, 5448 of two groups, 2543 x 24: 199 us, and 41 so)
    if (starved<MODE>(a, sizeof(C))) return launch_general_tiles<TA, TB, C, TO, MODE, BKFAST, false, 1, 1, 4>(a, stream);
    return launch_general_tiles<TA, TB, C, TO, MODE, BKFAST, false, 2, 2>(a, stream);
}
template <class T, int MODE, bool BKFAST, class S>
int32_t launch_fast(const Args& a, void* stream) {
    const int64_t tn = tiles(a.N, S::TN);
    const int64_t blocks = MODE == ROWS ? row_tiles(a, S::TM) * tn
                           : MODE == OUTER || MODE == PAIR ? Patches(a, S::TM, S::TN).blocks(a.n_groups) : tiles(a.n_rows, S::TM) * tn;
    if (blocks <= 0) return TFH_OK;
    Args args = a;
    dim3 grid;
    if (int32_t e = grid_of(blocks, 256, args, grid)) return e;
    static std::atomic<uint64_t> allowed{0};
    allow_lds(reinterpret_cast<const void*>(&ragged_fast_kernel<T, MODE, BKFAST, S>), S::LDS, allowed);
    static const std::string label = std::string("(ragged_fast_kernel<") + type_name<T>() + ", " + mode_name(MODE) + (BKFAST ? ", k, " : ", n, ") +
                                     std::to_string(S::TM) + "x" + std::to_string(S::TN) + ">)";
    TFH_LAUNCH_NAMED(label.c_str(), (ragged_fast_kernel<T, MODE, BKFAST, S>), grid, dim3(256), S::LDS, (hipStream_t)stream, args);
    return hip_check(hipGetLastError(), "product over groups of rows");
}
typedef Shape<2, 2, 4, 4, 128, 3, 2> Large;     // 256 x 256
typedef Shape<2, 2, 4, 2, 64, 3, 3> Tall;      // 256 x 128, two to a compute unit
typedef Shape<2, 2, 2, 2> Middle;   // 128 x 128
typedef Shape<2, 2, 1, 2, 128, 3, 3> Slim;   // 64 x 128
typedef Shape<1, 4, 1, 1> Small;    // 32 x 128
// Whether tiles of 256 x 256, one to a compute unit, come in rounds of the machine's 256 units that are full enough.  If not,
// tiles of half the columns, two to a unit: those take a tenth longer for the same work where k is 2048, a fifth from 4096 on and
// hardly any where it is short, since one works while the other starts or ends, and leave less of the machine idle.  How full the
// last round is follows from the sizes for one group only; of several, it is half on average, and so are the groups' last tiles.
// (bf16, uneven groups, large and tall tiles: 65 536 rows of 64, 2048 x 2048, nine rounds: 595 and 640 us; 32 768 of 32,
// 1024 x 2048, four and a half: 187 and 168; 49 152 of 48, 1024 x 2048, seven: 265 and 253; 8192 of 16, 2048 x 2048, one and a
// quarter: 104 and 91; 4096 of 8, 0.6: 54 and 56.)
inline bool fills_rounds(const Args& a) {
    const int64_t tn = tiles(a.N, 256), t = a.n_groups > 1 ? (a.n_rows * 2 / 256 + a.n_groups) * tn / 2 : tiles(a.n_rows, 256) * tn;
    const int64_t k = a.K < 4096 ? a.K : 4096;
    if (t < 256) return t > 128;
    return (a.n_groups > 1 ? 2 * t + 256 : tiles(t, 256) * 512) * 20480 <= 2 * t * (20480 + k);
}
template <class T, int MODE, bool BKFAST>
int32_t launch_shape(const Args& a, void* stream) {
    const int64_t rows = MODE == OUTER ? a.M : a.n_rows / a.n_groups;
    if (rows > 192) return MODE == OUTER || !fills_rounds(a) ? launch_fast<T, MODE, BKFAST, Tall>(a, stream) : launch_fast<T, MODE, BKFAST, Large>(a, stream);
    if (rows > 48) return launch_fast<T, MODE, BKFAST, Middle>(a, stream);
    return launch_fast<T, MODE, BKFAST, Small>(a, stream);
}
template <class T, int MODE, int TR>
int32_t launch_few(const Args& a, void* stream) {
    const int64_t blocks = (MODE == ROWS ? row_tiles(a, 16 * TR) : tiles(a.n_rows, 16 * TR)) * tiles(a.N, 16);
    if (blocks <= 0) return TFH_OK;
    Args args = a;
    dim3 grid;
    if (int32_t e = grid_of(blocks, few_threads<MODE>(), args, grid)) return e;
    static std::atomic<uint64_t> allowed{0};
    allow_lds(reinterpret_cast<const void*>(&ragged_few_kernel<T, MODE, TR>), few_lds<TR>(), allowed);
    static const std::string label = std::string("(ragged_few_kernel<") + type_name<T>() + ", " + mode_name(MODE) + ", " + std::to_string(16 * TR) + ">)";
    TFH_LAUNCH_NAMED(label.c_str(), (ragged_few_kernel<T, MODE, TR>), grid, dim3(few_threads<MODE>()), few_lds<TR>(), (hipStream_t)stream, args);
    return hip_check(hipGetLastError(), "product over groups of rows");
}
template <class T, bool BKFAST, int YT, int WAVES>
int32_t launch_thin_waves(const Args& a, void* stream) {
    const int64_t blocks = row_tiles(a, THIN_ROWS);
    if (blocks <= 0) return TFH_OK;
    Args args = a;
    dim3 grid;
    if (int32_t e = grid_of(blocks, 64 * WAVES, args, grid)) return e;
    static std::atomic<uint64_t> allowed{0};
    allow_lds(reinterpret_cast<const void*>(&ragged_thin_kernel<T, BKFAST, YT, WAVES>), (thin_lds<YT, WAVES>()), allowed);
    static const std::string label = std::string("(ragged_thin_kernel<") + type_name<T>() + (BKFAST ? ", k, " : ", n, ") + std::to_string(32 * YT) + ">)";
    TFH_LAUNCH_NAMED(label.c_str(), (ragged_thin_kernel<T, BKFAST, YT, WAVES>), grid, dim3(64 * WAVES), (thin_lds<YT, WAVES>()), (hipStream_t)stream, args);
    return hip_check(hipGetLastError(), "product over groups of rows");
}

template <class T, bool BKFAST, int YT>
int32_t launch_thin(const Args& a, void* stream) {
    // Eight waves to share out k where each block has a compute unit to itself; four, whose tiles leave room for a second block, beyond
    // (8192 rows of 16 groups, 4096 k's, from HBM: 31 and 25 us)
    if constexpr (YT == 1)
        if (row_tiles(a, THIN_ROWS) <= 256) return launch_thin_waves<T, BKFAST, YT, 8>(a, stream);
    return launch_thin_waves<T, BKFAST, YT, 4>(a, stream);
}

template <class T> int32_t launch_product(int kind, const Args& a, void* stream) {
    typedef typename Num<T>::acc W;
    // B's columns contiguous: its tiles keep the direction in which they are read
    const bool columns = a.b_n == 1 && a.b_k != 1;
    if constexpr (sizeof(T) == 2) {
        // Few rows of few groups, likewise: 8 rows of as many 2048 x 1024 matrices take 14 us so and 22 with 32 x 128 tiles, 64
        // rows of 50 of them 72 and 41 (the matrices bound that, and larger blocks read them better).
        if (kind == PRODUCT_ROWS && !columns && few_takes<ROWS>(a)) {
            const int64_t used = a.n_groups < a.n_rows ? a.n_groups : a.n_rows, each = a.n_rows / used, t16 = tiles(a.N, 16);
            if (each <= 16 && (a.n_rows / 16 + used) * t16 <= 1024) return launch_few<T, ROWS, 1>(a, stream);
            if (each <= 32 && (a.n_rows / 32 + used) * t16 <= 1024) return launch_few<T, ROWS, 2>(a, stream);
            if (each <= 64 && (a.n_rows / 64 + used) * t16 <= 1024) return launch_few<T, ROWS, 4>(a, stream);
        }
        if (kind == PRODUCT_ROWS && !starved<ROWS>(a, 2) && fast_takes<ROWS>(a, !columns))
            return columns ? launch_shape<T, ROWS, false>(a, stream) : launch_shape<T, ROWS, true>(a, stream);
        if (kind == PRODUCT_OUTER && !starved<OUTER>(a, 2) && fast_takes<OUTER>(a, false)) return launch_shape<T, OUTER, false>(a, stream);
        // Few rows: sixteen columns a block.  64 rows by 4096 columns and k's take 16 us so and 86 with 128 x 128 tiles, whose 32
        // blocks leave the machine idle; 1024 blocks take as long as those tiles do with 128.
        if (kind == PRODUCT_SHARED && a.pad > 0 && !columns && few_takes<SHARED>(a) && tiles(a.n_rows, 64) * tiles(a.N, 16) <= 1024)
            return a.n_rows <= 16 ? launch_few<T, SHARED, 1>(a, stream) : a.n_rows <= 32 ? launch_few<T, SHARED, 2>(a, stream) : launch_few<T, SHARED, 4>(a, stream);
        // Tiles of 128 x 128 that span the groups: larger ones of one group each leave more of the rows' tiles half empty (8192 rows
        // of 16 groups, 4096 x 4096, on the same inputs again: 285 us against 345, 298 with others each time; 16 384 of 8: 530 and 580; 4096 of
        // 8, 2048 x 4096: 92 and 112).
        if (kind == PRODUCT_SHARED && a.pad > 0) return columns ? launch_fast<T, SHARED, false, Middle>(a, stream) : launch_fast<T, SHARED, true, Middle>(a, stream);
        // (eight groups of 4096 rows, 4096 and 2048 x 64: 26 us in tiles of 64 rows, three stages on their way, 34 in those of 128)
        if (kind == PRODUCT_OUTER_V && a.pad > 0)
            return a.n_groups * tiles(a.M, 128) < 512 ? launch_fast<T, PAIR, false, Slim>(a, stream) : launch_fast<T, PAIR, false, Middle>(a, stream);
        if (kind == PRODUCT_MIDDLE && thin_takes(a, !columns)) {
            if (columns) return a.N <= 32 ? launch_thin<T, false, 1>(a, stream) : a.N <= 64 ? launch_thin<T, false, 2>(a, stream) : launch_thin<T, false, 4>(a, stream);
            return a.N <= 32 ? launch_thin<T, true, 1>(a, stream) : a.N <= 64 ? launch_thin<T, true, 2>(a, stream) : launch_thin<T, true, 4>(a, stream);
        }
    }
    switch (kind) {
        case PRODUCT_ROWS:
            if (a.wide) return columns ? launch_general<T, T, T, W, ROWS, false>(a, stream) : launch_general<T, T, T, W, ROWS, true>(a, stream);
            return columns ? launch_general<T, T, T, T, ROWS, false>(a, stream) : launch_general<T, T, T, T, ROWS, true>(a, stream);
        case PRODUCT_MIDDLE: return columns ? launch_general<T, T, T, W, ROWS, false>(a, stream) : launch_general<T, T, T, W, ROWS, true>(a, stream);
        case PRODUCT_SHARED: return columns ? launch_general<T, T, T, T, SHARED, false>(a, stream) : launch_general<T, T, T, T, SHARED, true>(a, stream);
        case PRODUCT_OUTER: return launch_general<T, T, T, T, OUTER, false>(a, stream);
        default: return launch_general<T, W, W, T, OUTER, false>(a, stream);
    }
}

}  // namespace ragged
}  // namespace tfh
