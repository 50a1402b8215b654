// ragged_launch.hpp -- chooses and launches a kernel on rows in groups; one translation unit per operand type includes it.
#pragma once
#include "launch.hpp"
#include "ragged.hpp"
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

template <class T> int32_t launch_product(int kind, const Args& a, void* stream) {
    typedef typename Num<T>::acc W;
    // B's columns contiguous: its tiles keep the direction in which they are read
    const bool columns = a.b_n == 1 && a.b_k != 1;
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
