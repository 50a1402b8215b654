// ragged_launch.hpp -- chooses and launches a kernel on rows in groups; one translation unit per operand type includes it.
#pragma once
#include "launch.hpp"
#include "ragged.hpp"
#include "ragged_fast.hpp"
#include "ragged_api.hpp"

namespace tfh {
namespace ragged {

inline int64_t tiles(int64_t n, int64_t t) { return (n + t - 1) / t; }
// Blocks of a launch over the groups' rows: no more tiles than the rows fill and one more, partly filled, for each group.
inline int64_t row_tiles(const Args& a, int tm) {
    const int64_t groups = a.n_groups + (a.zero_rest ? 1 : 0);
    return a.n_rows / tm + (groups < a.n_rows ? groups : a.n_rows);
}

template <class TA, class TB, class C, class TO, int MODE, bool BKFAST>
int32_t launch_general(const Args& a, void* stream) {
    constexpr int XT = 2, YT = 2;
    const int64_t tn = tiles(a.N, 32 * YT);
    const int64_t blocks = MODE == ROWS ? row_tiles(a, 32 * XT) * tn
                           : MODE == OUTER ? a.n_groups * tiles(a.M, 32 * XT) * tn : tiles(a.n_rows, 32 * XT) * tn;
    if (blocks <= 0) return TFH_OK;
    if (blocks > 0x7fffffff) return set_error(TFH_ERR_INVALID_ARGUMENT, "the product needs %lld blocks, more than one launch has", (long long)blocks);
    TFH_LAUNCH_TIMED((ragged_general_kernel<TA, TB, C, TO, MODE, BKFAST, XT, YT>), dim3((unsigned)blocks), dim3(GENERAL_THREADS), 0, (hipStream_t)stream, a);
    return hip_check(hipGetLastError(), "product over groups of rows");
}

template <class T, int MODE, bool BKFAST, class S>
int32_t launch_fast(const Args& a, void* stream) {
    const int64_t tn = tiles(a.N, S::TN);
    const int64_t blocks = MODE == ROWS ? row_tiles(a, S::TM) * tn
                           : MODE == OUTER ? a.n_groups * tiles(a.M, S::TM) * tn : tiles(a.n_rows, S::TM) * tn;
    if (blocks <= 0) return TFH_OK;
    if (blocks > 0x7fffffff) return set_error(TFH_ERR_INVALID_ARGUMENT, "the product needs %lld blocks, more than one launch has", (long long)blocks);
    static const bool once = [] {
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&ragged_fast_kernel<T, MODE, BKFAST, S>), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS);
        return true;
    }();
    (void)once;
    TFH_LAUNCH_TIMED((ragged_fast_kernel<T, MODE, BKFAST, S>), dim3((unsigned)blocks), dim3(256), S::LDS, (hipStream_t)stream, a);
    return hip_check(hipGetLastError(), "product over groups of rows");
}
typedef Shape<2, 2, 4, 4> Large;    // 256 x 256
typedef Shape<2, 2, 2, 2> Middle;   // 128 x 128
typedef Shape<1, 4, 1, 1> Small;    // 32 x 128
template <class T, int MODE, bool BKFAST>
int32_t launch_shape(const Args& a, void* stream) {
    const int64_t rows = MODE == OUTER ? a.M : a.n_rows / a.n_groups;
    if (rows > 192) return launch_fast<T, MODE, BKFAST, Large>(a, stream);
    if (rows > 48) return launch_fast<T, MODE, BKFAST, Middle>(a, stream);
    return launch_fast<T, MODE, BKFAST, Small>(a, stream);
}

template <class T> int32_t launch_product(int kind, const Args& a, void* stream) {
    typedef typename Num<T>::acc W;
    // B's columns contiguous: its tiles keep the direction in which they are read
    const bool columns = a.b_n == 1 && a.b_k != 1;
    if constexpr (sizeof(T) == 2) {
        if (kind == PRODUCT_ROWS && fast_takes<ROWS>(a, !columns))
            return columns ? launch_shape<T, ROWS, false>(a, stream) : launch_shape<T, ROWS, true>(a, stream);
        if (kind == PRODUCT_OUTER && fast_takes<OUTER>(a, false)) return launch_shape<T, OUTER, false>(a, stream);
    }
    switch (kind) {
        case PRODUCT_ROWS: return columns ? launch_general<T, T, T, T, ROWS, false>(a, stream) : launch_general<T, T, T, T, ROWS, true>(a, stream);
        case PRODUCT_MIDDLE: return columns ? launch_general<T, T, T, W, ROWS, false>(a, stream) : launch_general<T, T, T, W, ROWS, true>(a, stream);
        case PRODUCT_SHARED: return columns ? launch_general<T, T, T, T, SHARED, false>(a, stream) : launch_general<T, T, T, T, SHARED, true>(a, stream);
        case PRODUCT_OUTER: return launch_general<T, T, T, T, OUTER, false>(a, stream);
        case PRODUCT_OUTER_V: return launch_general<T, W, W, T, OUTER, false>(a, stream);
        default: return launch_general<W, T, W, T, OUTER, false>(a, stream);
    }
}

}  // namespace ragged
}  // namespace tfh
