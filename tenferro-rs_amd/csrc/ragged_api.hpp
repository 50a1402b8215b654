// ragged_api.hpp -- what ragged.cpp (argument checks, dispatch) and the kernels on rows in groups agree on.
#pragma once
#include <cstddef>
#include <cstdint>

#include "internal.hpp"

namespace tfh {
namespace ragged {

// `blocks` blocks as a grid of x times y, each dimension of which has less than 2^32 threads and x a multiple of the XCDs: block
// y * grid x + x, those from `blocks` on with nothing to do.  More than 2^31 are refused.
inline int32_t launch_grid(int64_t blocks, int threads, uint32_t* x, uint32_t* y) {
    if (blocks > 0x7fffffff) return set_error(TFH_ERR_INVALID_ARGUMENT, "the call needs %lld blocks, more than a launch has", (long long)blocks);
    const int64_t most = ((int64_t)1 << 31) / threads / 8 * 8;
    *x = (uint32_t)(blocks < most ? blocks : most);
    *y = (uint32_t)((blocks + *x - 1) / *x);
    return TFH_OK;
}

// Rows by group (k_row_groups.hip).
struct GroupArgs {
    const void* ids;          // element of row i: (i / inner) * s_outer + (i % inner) * s_inner
    int64_t s_outer, s_inner;
    int32_t inner, id64;
    int32_t n_rows, n_groups;
    int32_t* offsets;
    int32_t* order;
    int32_t* positions;       // may be null
    int32_t* counts;          // [blocks + 1][n_groups + 1] in the workspace (more than one block)
    int32_t blocks;
};
size_t group_rows_workspace(int64_t n_rows, int32_t n_groups);
int32_t launch_group_rows(GroupArgs a, void* stream);

// A token's rows joined (k_combine.hip).  Strides in elements.
struct CombineArgs {
    const void* x;            // [n_rows, n] rows in order
    int64_t x_row, x_n;
    int32_t x_wide;           // x is of the sums' type (no gradient)
    const void* w;            // [tokens, fan], of the sums' type, or null (ones)
    int64_t w_token, w_fan;
    void* y;                  // [tokens, n]; the gradient's: dy
    int64_t y_row, y_n;
    void* dx;                 // the gradient's [n_rows, n], may be null
    int64_t dx_row, dx_n;
    void* dw;                 // the gradient's [tokens, fan], may be null
    int64_t dw_token, dw_fan;
    const int32_t* positions;
    const int32_t* offsets;
    const int32_t* order;     // the gradient's, may be null
    int64_t n_rows, tokens;
    int32_t n_groups, fan, n;
};
int32_t launch_combine(int dtype, const CombineArgs& a, void* stream);
int32_t launch_combine_grad(int dtype, const CombineArgs& a, void* stream);

// Products (k_ragged_*.hip): one entry per operand type, which chooses among its kernels.
struct Args;
enum Kind {
    PRODUCT_ROWS,      // rows in, rows out, all of the type
    PRODUCT_OUTER,     // a group's rows summed over, all of the type
    PRODUCT_SHARED,    // one matrix for all rows and a low-rank part by group
    PRODUCT_MIDDLE,    // rows in, rows out in the sums' type or as a pair (Args::pad)
    PRODUCT_OUTER_V    // a group's rows summed over, B what PRODUCT_MIDDLE has written
};
int32_t launch_bf16(int kind, const Args& a, void* stream);
int32_t launch_f16(int kind, const Args& a, void* stream);
int32_t launch_f32(int kind, const Args& a, void* stream);
int32_t launch_f64(int kind, const Args& a, void* stream);

}  // namespace ragged
}  // namespace tfh
