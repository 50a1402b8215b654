// ragged.cpp -- the entry points on rows in groups: argument checks and the calls they are made of.
#include <exception>
#include <initializer_list>

#include <hip/hip_runtime.h>

#include "ragged_api.hpp"
#include "ragged_thin.hpp"

namespace tfh {
namespace ragged {
namespace {

constexpr int64_t MOST = 0x7ff00000;   // rows, extents: 32-bit indices may run past one by the largest step of a loop

bool known(int32_t dtype) { return dtype == TFH_BF16 || dtype == TFH_F16 || dtype == TFH_F32 || dtype == TFH_F64; }
size_t sums_size(int32_t dtype) { return dtype == TFH_F64 ? 8 : 4; }

int32_t check_dtype(int32_t dtype) {
    if (!known(dtype)) return set_error(TFH_ERR_INVALID_ARGUMENT, "operations on rows in groups take bf16, f16, f32 and f64; got dtype %d", dtype);
    return TFH_OK;
}
int32_t check_groups(const tfh_row_groups* g, bool positions) {
    if (!g) return set_error(TFH_ERR_INVALID_ARGUMENT, "null row groups");
    if (g->n_groups < 1 || g->n_groups > MOST) return set_error(TFH_ERR_INVALID_ARGUMENT, "row groups need at least one group and less than 2^31 - 2^20, got %d", g->n_groups);
    if (g->n_rows < 0 || g->n_rows > MOST) return set_error(TFH_ERR_INVALID_ARGUMENT, "row groups: %lld rows are out of range", (long long)g->n_rows);
    if (g->fan < 1) return set_error(TFH_ERR_INVALID_ARGUMENT, "row groups: a fan of %d", g->fan);
    if (g->n_rows % g->fan) return set_error(TFH_ERR_INVALID_ARGUMENT, "row groups: %lld rows are no multiple of the fan %d", (long long)g->n_rows, g->fan);
    if (!g->offsets) return set_error(TFH_ERR_INVALID_ARGUMENT, "row groups without offsets");
    if (positions && g->n_rows && !g->positions) return set_error(TFH_ERR_INVALID_ARGUMENT, "row groups without positions");
    return TFH_OK;
}
int32_t check_view(const char* what, const tfh_view* v, std::initializer_list<int64_t> dims, bool output) {
    if (!v) return set_error(TFH_ERR_INVALID_ARGUMENT, "%s: null view", what);
    if (v->rank != (int32_t)dims.size()) return set_rank_mismatch((int64_t)dims.size(), v->rank);
    bool same = true, empty = false;
    int64_t want[3] = {0, 0, 0};
    int d = 0;
    for (int64_t n : dims) {
        want[d] = n;
        same = same && v->dims[d] == n;
        empty = empty || n == 0;
        ++d;
    }
    if (!same) return set_shape_mismatch(want, (int)dims.size(), v->dims, v->rank);
    if (!v->base && !empty) return set_error(TFH_ERR_INVALID_ARGUMENT, "%s: null base pointer", what);
    if (v->flags & TFH_VIEW_CONJ) return set_error(TFH_ERR_INVALID_ARGUMENT, "%s: TFH_VIEW_CONJ is not taken by operations on rows in groups", what);
    if (output)
        for (d = 0; d < v->rank; ++d)
            if (v->dims[d] > 1 && v->strides[d] == 0 && !empty) return set_error(TFH_ERR_INVALID_ARGUMENT, "%s: an output with a stride of 0", what);
    return TFH_OK;
}
int32_t check_extent(const char* what, int64_t n) {
    if (n < 0 || n > MOST) return set_error(TFH_ERR_INVALID_ARGUMENT, "%s: an extent of %lld is out of range", what, (long long)n);
    return TFH_OK;
}
int32_t check_workspace(const void* workspace, size_t have, size_t need) {
    if (need == 0) return TFH_OK;
    if (!workspace || have < need) return set_error(TFH_ERR_INVALID_ARGUMENT, "the call needs %zu bytes of workspace, got %zu", need, workspace ? have : 0);
    if ((uintptr_t)workspace & 15) return set_error(TFH_ERR_INVALID_ARGUMENT, "the workspace is not 16-byte aligned");
    return TFH_OK;
}
int32_t rank_of(const char* what, const tfh_view* v, int rank) {
    if (!v) return set_error(TFH_ERR_INVALID_ARGUMENT, "%s: null view", what);
    if (v->rank != rank) return set_rank_mismatch(rank, v->rank);
    return TFH_OK;
}

int32_t product(int32_t dtype, int kind, const Args& a, void* stream) {
    const int prof = prof_begin(PROF_CONTRACT, stream);
    int32_t e;
    switch (dtype) {
        case TFH_BF16: e = launch_bf16(kind, a, stream); break;
        case TFH_F16: e = launch_f16(kind, a, stream); break;
        case TFH_F32: e = launch_f32(kind, a, stream); break;
        default: e = launch_f64(kind, a, stream);
    }
    prof_end(prof, stream);
    return e;
}

int64_t wide_row(int64_t n) { return (n + 3) & ~(int64_t)3; }   // of the sums' type in scratch: 16-byte aligned

Args base_args(const tfh_row_groups& g) {
    Args a = {};
    a.offsets = g.offsets;
    a.order = g.order;
    a.n_rows = g.n_rows;
    a.n_groups = g.n_groups;
    a.fan = g.fan;
    a.alpha = 1;
    return a;
}
void set_a(Args& a, int dtype, const tfh_view& v) {
    a.A = view_ptr(v, dtype);
    a.a_rows = v.dims[0];
    a.a_row = v.strides[0];
    a.a_col = v.strides[1];
}

int32_t ragged_gemm(int32_t dtype, const tfh_row_groups* g, int32_t flags, double alpha, const tfh_view* a, const tfh_view* b,
                    double beta, const tfh_view* c, void* stream) {
    if (int32_t e = check_dtype(dtype)) return e;
    if (int32_t e = check_groups(g, false)) return e;
    if (flags & ~(TFH_ROWS_GATHER_A | TFH_ROWS_SCATTER_C | TFH_ROWS_ZERO_REST)) return set_error(TFH_ERR_INVALID_ARGUMENT, "unknown flags %d", flags);
    const bool gather = flags & TFH_ROWS_GATHER_A, scatter = flags & TFH_ROWS_SCATTER_C;
    if ((gather || scatter) && !g->order && g->n_rows) return set_error(TFH_ERR_INVALID_ARGUMENT, "rows are gathered or scattered by an order, and there is none");
    if (int32_t e = rank_of("A", a, 2)) return e;
    if (int32_t e = rank_of("B", b, 3)) return e;
    const int64_t K = a->dims[1], N = b->dims[2];
    if (int32_t e = check_extent("K", K)) return e;
    if (int32_t e = check_extent("N", N)) return e;
    if (int32_t e = check_view("A", a, {gather ? g->n_rows / g->fan : g->n_rows, K}, false)) return e;
    if (int32_t e = check_view("B", b, {g->n_groups, K, N}, false)) return e;
    if (int32_t e = check_view("C", c, {g->n_rows, N}, true)) return e;
    if (g->n_rows == 0 || N == 0) return TFH_OK;
    Args p = base_args(*g);
    set_a(p, dtype, *a);
    p.B = view_ptr(*b, dtype);
    p.b_group = b->strides[0], p.b_k = b->strides[1], p.b_n = b->strides[2];
    p.C = view_ptr(*c, dtype);
    p.c_row = c->strides[0], p.c_n = c->strides[1];
    p.N = (int32_t)N, p.K = (int32_t)K;
    p.gather = gather, p.scatter = scatter;
    p.zero_rest = (flags & TFH_ROWS_ZERO_REST) != 0;
    p.alpha = alpha, p.beta = beta;
    p.use_beta = beta != 0;
    return product(dtype, PRODUCT_ROWS, p, stream);
}

int32_t ragged_gemm_grad(int32_t dtype, const tfh_row_groups* g, int32_t flags, double alpha, const tfh_view* a, const tfh_view* dc,
                         double beta, const tfh_view* db, void* stream) {
    if (int32_t e = check_dtype(dtype)) return e;
    if (int32_t e = check_groups(g, false)) return e;
    if (flags & ~TFH_ROWS_GATHER_A) return set_error(TFH_ERR_INVALID_ARGUMENT, "unknown flags %d", flags);
    const bool gather = flags & TFH_ROWS_GATHER_A;
    if (gather && !g->order && g->n_rows) return set_error(TFH_ERR_INVALID_ARGUMENT, "rows are gathered by an order, and there is none");
    if (int32_t e = rank_of("A", a, 2)) return e;
    if (int32_t e = rank_of("dC", dc, 2)) return e;
    const int64_t K = a->dims[1], N = dc->dims[1];
    if (int32_t e = check_extent("K", K)) return e;
    if (int32_t e = check_extent("N", N)) return e;
    if (int32_t e = check_view("A", a, {gather ? g->n_rows / g->fan : g->n_rows, K}, false)) return e;
    if (int32_t e = check_view("dC", dc, {g->n_rows, N}, false)) return e;
    if (int32_t e = check_view("dB", db, {g->n_groups, K, N}, true)) return e;
    if (K == 0 || N == 0) return TFH_OK;
    Args p = base_args(*g);
    set_a(p, dtype, *a);
    p.B = view_ptr(*dc, dtype);
    p.b_rows = g->n_rows;
    p.b_k = dc->strides[0], p.b_n = dc->strides[1];
    p.C = view_ptr(*db, dtype);
    p.c_group = db->strides[0], p.c_row = db->strides[1], p.c_n = db->strides[2];
    p.M = (int32_t)K, p.N = (int32_t)N;
    p.gather = gather;
    p.alpha = alpha, p.beta = beta;
    p.use_beta = beta != 0;
    return product(dtype, PRODUCT_OUTER, p, stream);
}

// The gradient of the product's A.  Where several places read a row, their parts are kept in the sums' type and rounded once, as
// they are joined: a part may lie beyond the operands' range, or cancel against another, and the row's sum not.
size_t grad_a_bytes(int32_t dtype, int64_t n_rows, int64_t k, int32_t fan, int32_t flags) {
    return (flags & TFH_ROWS_GATHER_A) && fan > 1 ? (size_t)n_rows * wide_row(k) * sums_size(dtype) : 0;
}
int32_t ragged_gemm_grad_a(int32_t dtype, const tfh_row_groups* g, int32_t flags, double alpha, const tfh_view* dc, const tfh_view* b,
                           const tfh_view* da, void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t e = check_dtype(dtype)) return e;
    if (flags & ~TFH_ROWS_GATHER_A) return set_error(TFH_ERR_INVALID_ARGUMENT, "unknown flags %d", flags);
    const bool gather = flags & TFH_ROWS_GATHER_A, joined = gather && g && g->fan > 1;
    if (int32_t e = check_groups(g, joined)) return e;
    if (gather && !g->order && g->n_rows) return set_error(TFH_ERR_INVALID_ARGUMENT, "rows are gathered by an order, and there is none");
    if (int32_t e = rank_of("dC", dc, 2)) return e;
    if (int32_t e = rank_of("B", b, 3)) return e;
    const int64_t K = b->dims[1], N = dc->dims[1], sources = gather ? g->n_rows / g->fan : g->n_rows;
    if (int32_t e = check_extent("K", K)) return e;
    if (int32_t e = check_extent("N", N)) return e;
    if (int32_t e = check_view("dC", dc, {g->n_rows, N}, false)) return e;
    if (int32_t e = check_view("B", b, {g->n_groups, K, N}, false)) return e;
    if (int32_t e = check_view("dA", da, {sources, K}, true)) return e;
    if (int32_t e = check_workspace(workspace, workspace_bytes, grad_a_bytes(dtype, g->n_rows, K, g->fan, flags))) return e;
    if (g->n_rows == 0 || K == 0) return TFH_OK;
    Args p = base_args(*g);
    set_a(p, dtype, *dc);
    p.B = view_ptr(*b, dtype);
    p.b_group = b->strides[0], p.b_k = b->strides[2], p.b_n = b->strides[1];
    p.N = (int32_t)K, p.K = (int32_t)N;
    p.alpha = alpha;
    p.zero_rest = 1;
    if (joined) {
        p.C = workspace, p.c_row = wide_row(K), p.c_n = 1;
        p.wide = 1;
    } else {
        p.C = view_ptr(*da, dtype), p.c_row = da->strides[0], p.c_n = da->strides[1];
        p.scatter = gather;
    }
    if (int32_t e = product(dtype, PRODUCT_ROWS, p, stream)) return e;
    if (!joined) return TFH_OK;
    CombineArgs c = {};
    c.x = workspace, c.x_row = wide_row(K), c.x_n = 1;
    c.x_wide = 1;
    c.y = view_ptr(*da, dtype), c.y_row = da->strides[0], c.y_n = da->strides[1];
    c.positions = g->positions, c.offsets = g->offsets;
    c.n_rows = g->n_rows, c.tokens = sources;
    c.n_groups = g->n_groups, c.fan = g->fan, c.n = (int32_t)K;
    const int prof = prof_begin(PROF_REDUCE, stream);
    const int32_t e = launch_combine(dtype, c, stream);
    prof_end(prof, stream);
    return e;
}

int32_t combine(int32_t dtype, const tfh_row_groups* g, const tfh_view* x, const tfh_view* w, const tfh_view* y, const tfh_view* dx,
                const tfh_view* dw, bool gradient, void* stream) {
    if (int32_t e = check_dtype(dtype)) return e;
    if (int32_t e = check_groups(g, true)) return e;
    const int64_t tokens = g->n_rows / g->fan;
    if (int32_t e = rank_of(gradient ? "dY" : "Y", y, 2)) return e;
    const int64_t N = y->dims[1];
    if (int32_t e = check_extent("N", N)) return e;
    if (!gradient || dw)
        if (int32_t e = check_view("X", x, {g->n_rows, N}, false)) return e;
    if (w)
        if (int32_t e = check_view("weights", w, {tokens, g->fan}, false)) return e;
    if (int32_t e = check_view(gradient ? "dY" : "Y", y, {tokens, N}, !gradient)) return e;
    if (dx)
        if (int32_t e = check_view("dX", dx, {g->n_rows, N}, true)) return e;
    if (dw)
        if (int32_t e = check_view("dweights", dw, {tokens, g->fan}, true)) return e;
    if (tokens == 0 || (gradient ? !dx && !dw : N == 0)) return TFH_OK;
    const int sums = dtype == TFH_F64 ? TFH_F64 : TFH_F32;
    CombineArgs c = {};
    if (!gradient || dw) c.x = view_ptr(*x, dtype), c.x_row = x->strides[0], c.x_n = x->strides[1];
    if (w) c.w = view_ptr(*w, sums), c.w_token = w->strides[0], c.w_fan = w->strides[1];
    c.y = view_ptr(*y, dtype), c.y_row = y->strides[0], c.y_n = y->strides[1];
    if (dx) c.dx = view_ptr(*dx, dtype), c.dx_row = dx->strides[0], c.dx_n = dx->strides[1];
    if (dw) c.dw = view_ptr(*dw, sums), c.dw_token = dw->strides[0], c.dw_fan = dw->strides[1];
    c.positions = g->positions, c.offsets = g->offsets, c.order = g->order;
    c.n_rows = g->n_rows, c.tokens = tokens;
    c.n_groups = g->n_groups, c.fan = g->fan, c.n = (int32_t)N;
    const int prof = prof_begin(PROF_REDUCE, stream);
    const int32_t e = gradient ? launch_combine_grad(dtype, c, stream) : launch_combine(dtype, c, stream);
    prof_end(prof, stream);
    return e;
}

// The middle product X . A of the adapters, in scratch: rows in the sums' type, 16-byte aligned, or a pair of the operands'
// type with a power of two per row (f16).
int64_t pair_pad(int64_t rank) { return (rank + 31) & ~(int64_t)31; }
size_t middle_bytes(int32_t dtype, int64_t n_rows, int64_t rank) {
    if (rank == 0) return 0;
    if (dtype == TFH_F32 || dtype == TFH_F64) return (size_t)n_rows * wide_row(rank) * sums_size(dtype);
    return (size_t)n_rows * pair_pad(rank) * 4 + (((size_t)n_rows * 4 + 15) & ~(size_t)15);
}
int middle_count(int32_t dtype, bool gradient) { return !gradient ? 1 : dtype == TFH_F32 || dtype == TFH_F64 ? 2 : 3; }

struct Adapter {
    int32_t dtype;
    const tfh_row_groups* g;
    const tfh_view *x, *w, *a, *b, *scales;
    int64_t K, N, R;
};
int32_t check_adapter(Adapter& d) {
    if (int32_t e = check_dtype(d.dtype)) return e;
    if (int32_t e = check_groups(d.g, false)) return e;
    if (d.g->fan != 1) return set_error(TFH_ERR_INVALID_ARGUMENT, "adapters take one row a token, got a fan of %d", d.g->fan);
    if (int32_t e = rank_of("W", d.w, 2)) return e;
    if (int32_t e = rank_of("A", d.a, 3)) return e;
    d.K = d.w->dims[0], d.N = d.w->dims[1], d.R = d.a->dims[2];
    if (int32_t e = check_extent("K", d.K)) return e;
    if (int32_t e = check_extent("N", d.N)) return e;
    if (int32_t e = check_extent("R", d.R)) return e;
    if (int32_t e = check_view("X", d.x, {d.g->n_rows, d.K}, false)) return e;
    if (int32_t e = check_view("W", d.w, {d.K, d.N}, false)) return e;
    if (int32_t e = check_view("A", d.a, {d.g->n_groups, d.K, d.R}, false)) return e;
    if (int32_t e = check_view("B", d.b, {d.g->n_groups, d.R, d.N}, false)) return e;
    if (d.scales) {
        if (int32_t e = check_view("scales", d.scales, {d.g->n_groups}, false)) return e;
        if (d.scales->strides[0] != 1 && d.g->n_groups > 1) return set_error(TFH_ERR_STRIDED, "scales have to be contiguous");
    }
    return TFH_OK;
}
// V[p, :] = scales[g] * X[order[p], :] . F[g], F [K, R] by strides.
Args middle_args(const Adapter& d, const tfh_view& x, int64_t K, const tfh_view& f, int k_axis, int r_axis, void* v, bool pair) {
    Args p = base_args(*d.g);
    set_a(p, d.dtype, x);
    p.B = view_ptr(f, d.dtype);
    p.b_group = f.strides[0], p.b_k = f.strides[k_axis], p.b_n = f.strides[r_axis];
    p.C = v;
    p.pad = pair ? (int32_t)pair_pad(d.R) : 0;
    p.c_row = pair ? 2 * p.pad : wide_row(d.R), p.c_n = 1;
    if (pair && d.dtype == TFH_F16) p.up = (float*)((char*)v + (size_t)d.g->n_rows * p.pad * 4);
    p.N = (int32_t)d.R, p.K = (int32_t)K;
    p.gather = d.g->order != nullptr;
    if (d.scales) p.scales = view_ptr(*d.scales, d.dtype == TFH_F64 ? TFH_F64 : TFH_F32);
    return p;
}
// Y = X . W + V . E[g]: X [n_rows, K], W [K, N] by (w_k, w_n), E [R, N] of f by (r_axis, n_axis).
Args shared_args(const Adapter& d, const tfh_view& x, int64_t K, int64_t N, int64_t w_k, int64_t w_n, const tfh_view& f, int r_axis,
                 int n_axis, void* v, const tfh_view& y, bool pair) {
    Args p = base_args(*d.g);
    set_a(p, d.dtype, x);
    p.B = view_ptr(*d.w, d.dtype);
    p.b_k = w_k, p.b_n = w_n;
    p.C = view_ptr(y, d.dtype);
    p.c_row = y.strides[0], p.c_n = y.strides[1];
    p.N = (int32_t)N, p.K = (int32_t)K;
    p.gather = p.scatter = d.g->order != nullptr;
    p.V = v;
    p.pad = pair ? (int32_t)pair_pad(d.R) : 0;
    p.v_row = pair ? 2 * p.pad : wide_row(d.R);
    if (pair && d.dtype == TFH_F16) p.up = (float*)((char*)v + (size_t)d.g->n_rows * p.pad * 4);
    p.E = view_ptr(f, d.dtype);
    p.e_group = f.strides[0], p.e_k = f.strides[r_axis], p.e_n = f.strides[n_axis];
    p.r = (int32_t)d.R;
    return p;
}
// Whether the two are done by the kernels that keep the middle as a pair.
bool by_pair(int32_t dtype, const Args& middle, const Args& shared) {
    if (dtype != TFH_BF16 && dtype != TFH_F16) return false;
    // W's columns contiguous and so few tiles that k has to be shared out, which the kernel for sums does (200 rows, 4096 x 1024, rank
    // 16: 44 us with the pair's tiles, 16 with that; 400 rows, 512 x 512: 14 and 9; 256 tiles of 64 x 64, 1024 x 1024: 29 and 37)
    const bool columns = shared.b_n == 1 && shared.b_k != 1;
    if (columns && shared.K >= 512 && ((shared.n_rows + 63) / 64) * (int64_t)((shared.N + 63) / 64) <= 128) return false;
    return thin_takes(middle, !(middle.b_n == 1 && middle.b_k != 1)) && fast_takes<SHARED>(shared, !columns);
}
// Y = X . W + scales (X . F[g]) . E[g]; `v`: scratch, left as a pair or as sums (`*pair`).
int32_t both(const Adapter& d, const tfh_view& x, int64_t K, int64_t N, int64_t w_k, int64_t w_n, const tfh_view& f, int f_k, int f_r, const tfh_view& e,
             int e_r, int e_n, void* v, const tfh_view& y, bool* pair, void* stream) {
    *pair = false;
    if (d.R > 0) {
        Args m = middle_args(d, x, K, f, f_k, f_r, v, true), s = shared_args(d, x, K, N, w_k, w_n, e, e_r, e_n, v, y, true);
        *pair = by_pair(d.dtype, m, s);
    }
    if (d.R > 0)
        if (int32_t err = product(d.dtype, PRODUCT_MIDDLE, middle_args(d, x, K, f, f_k, f_r, v, *pair), stream)) return err;
    return product(d.dtype, PRODUCT_SHARED, shared_args(d, x, K, N, w_k, w_n, e, e_r, e_n, v, y, *pair), stream);
}

int32_t adapter_gemm(Adapter d, const tfh_view* y, void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t e = check_adapter(d)) return e;
    if (int32_t e = check_view("Y", y, {d.g->n_rows, d.N}, true)) return e;
    if (int32_t e = check_workspace(workspace, workspace_bytes, middle_bytes(d.dtype, d.g->n_rows, d.R))) return e;
    if (d.g->n_rows == 0 || d.N == 0) return TFH_OK;
    bool pair;
    return both(d, *d.x, d.K, d.N, d.w->strides[0], d.w->strides[1], *d.a, 1, 2, *d.b, 1, 2, workspace, *y, &pair, stream);
}

// A factor's gradient: G[g] = sum over the group's rows of X[order[p], :]^T . V[p, :] with V = scales Z[order[p], :] . F[g], in
// the view `grad` by (x_axis, r_axis).  `have`: V from before, as a pair or as sums; null or of the other form: it is made
// again, in `spare`.  A pair in bf16; f16's pairs carry a factor for each row, for which a sum over rows has no place.
int32_t factor_gradient(const Adapter& d, const tfh_view& x, int64_t K, const tfh_view& z, int64_t KZ, const tfh_view& f, int f_k, int f_r,
                        const tfh_view& grad, int x_axis, int r_axis, void* have, bool have_pair, void* spare, void* stream) {
    Args p = base_args(*d.g);
    set_a(p, d.dtype, x);
    p.gather = d.g->order != nullptr;
    p.b_rows = d.g->n_rows;
    p.C = view_ptr(grad, d.dtype), p.c_group = grad.strides[0], p.c_row = grad.strides[x_axis], p.c_n = grad.strides[r_axis];
    p.M = (int32_t)K, p.r = (int32_t)d.R;
    p.b_n = 1;
    Args q = p;
    q.pad = (int32_t)pair_pad(d.R), q.N = 2 * q.pad, q.b_k = 2 * q.pad, q.B = spare;
    p.N = (int32_t)d.R, p.b_k = wide_row(d.R);
    const Args as_pair = middle_args(d, z, KZ, f, f_k, f_r, spare, true);
    const bool pair = d.dtype == TFH_BF16 && fast_takes<PAIR>(q, false) && thin_takes(as_pair, !(as_pair.b_n == 1 && as_pair.b_k != 1));
    void* v = have && have_pair == pair ? have : spare;
    if (v == spare && d.g->n_rows)
        if (int32_t e = product(d.dtype, PRODUCT_MIDDLE, pair ? as_pair : middle_args(d, z, KZ, f, f_k, f_r, spare, false), stream)) return e;
    Args& out = pair ? q : p;
    out.B = v;
    return product(d.dtype, PRODUCT_OUTER_V, out, stream);
}

int32_t adapter_gemm_grad(Adapter d, const tfh_view* dy, const tfh_view* dx, const tfh_view* da, const tfh_view* db, void* workspace,
                          size_t workspace_bytes, void* stream) {
    if (int32_t e = check_adapter(d)) return e;
    const int64_t rows = d.g->n_rows;
    if (int32_t e = check_view("dY", dy, {rows, d.N}, false)) return e;
    if (dx)
        if (int32_t e = check_view("dX", dx, {rows, d.K}, true)) return e;
    if (da)
        if (int32_t e = check_view("dA", da, {d.g->n_groups, d.K, d.R}, true)) return e;
    if (db)
        if (int32_t e = check_view("dB", db, {d.g->n_groups, d.R, d.N}, true)) return e;
    const size_t each = middle_bytes(d.dtype, rows, d.R);
    if (int32_t e = check_workspace(workspace, workspace_bytes, each * middle_count(d.dtype, true))) return e;
    char* const u = (char*)workspace;
    bool pair = false, made = false;
    if (rows && dx && d.K) {
        if (int32_t e = both(d, *dy, d.N, d.K, d.w->strides[1], d.w->strides[0], *d.b, 2, 1, *d.a, 2, 1, u, *dx, &pair, stream)) return e;
        made = true;
    }
    if (d.R == 0) return TFH_OK;
    if (da && d.K)
        if (int32_t e = factor_gradient(d, *d.x, d.K, *dy, d.N, *d.b, 2, 1, *da, 1, 2, made ? u : nullptr, pair, u + each, stream)) return e;
    if (db && d.N)
        if (int32_t e = factor_gradient(d, *dy, d.N, *d.x, d.K, *d.a, 1, 2, *db, 2, 1, nullptr, false, u + (middle_count(d.dtype, true) - 1) * each, stream)) return e;
    return TFH_OK;
}

int32_t group_rows(int32_t id_bits, const tfh_view* ids, int32_t n_groups, int32_t* offsets, int32_t* order, int32_t* positions,
                   void* workspace, size_t workspace_bytes, void* stream) {
    if (id_bits != 32 && id_bits != 64) return set_error(TFH_ERR_INVALID_ARGUMENT, "indices of 32 or 64 bits, got %d", id_bits);
    if (!ids) return set_error(TFH_ERR_INVALID_ARGUMENT, "ids: null view");
    if (ids->rank != 1 && ids->rank != 2) return set_rank_mismatch(1, ids->rank);
    if (n_groups < 1 || n_groups > TFH_MAX_ROW_GROUPS) return set_error(TFH_ERR_INVALID_ARGUMENT, "%d groups: 1 to %d are taken", n_groups, TFH_MAX_ROW_GROUPS);
    const int64_t outer = ids->dims[0], inner = ids->rank == 2 ? ids->dims[1] : 1;
    if (outer < 0 || inner < 0 || outer > MOST || inner > MOST || outer * inner > MOST) return set_error(TFH_ERR_INVALID_ARGUMENT, "too many rows to group");
    const int64_t rows = outer * inner;
    if (ids->flags & TFH_VIEW_CONJ) return set_error(TFH_ERR_INVALID_ARGUMENT, "ids: TFH_VIEW_CONJ is not taken by operations on rows in groups");
    if (rows && !ids->base) return set_error(TFH_ERR_INVALID_ARGUMENT, "ids: null base pointer");
    if (!offsets || (rows && !order)) return set_error(TFH_ERR_INVALID_ARGUMENT, "null output pointer");
    if (int32_t e = check_workspace(workspace, workspace_bytes, group_rows_workspace(rows, n_groups))) return e;
    GroupArgs a = {};
    a.ids = (const char*)ids->base + ids->offset * (id_bits / 8);
    a.s_outer = ids->strides[0], a.s_inner = ids->rank == 2 ? ids->strides[1] : 0;
    a.inner = (int32_t)inner;
    if (ids->rank == 2 && (inner <= 1 || outer <= 1 || a.s_outer == a.s_inner * inner)) {   // one stride throughout: no division per row
        if (inner > 1) a.s_outer = a.s_inner;
        a.inner = 1;
    }
    a.id64 = id_bits == 64;
    a.n_rows = (int32_t)rows, a.n_groups = n_groups;
    a.offsets = offsets, a.order = order, a.positions = positions;
    a.counts = (int32_t*)workspace;
    const int prof = prof_begin(PROF_COPY, stream);
    const int32_t e = launch_group_rows(a, stream);
    prof_end(prof, stream);
    return e;
}

// Nothing leaves an entry point but a status.
template <class F> int32_t guarded(const char* name, F f) {
    try {
        const int32_t e = f();
        if (!e) clear_error();
        return e;
    } catch (const std::exception& ex) {
        return set_error(TFH_ERR_DEVICE, "%s: %s", name, ex.what());
    } catch (...) {
        return set_error(TFH_ERR_DEVICE, "%s: unknown exception", name);
    }
}

}  // namespace
}  // namespace ragged
}  // namespace tfh

using namespace tfh;

extern "C" {

size_t tfh_group_rows_workspace(int64_t n_rows, int32_t n_groups) {
    return n_rows < 0 || n_rows > ragged::MOST || n_groups < 1 || n_groups > TFH_MAX_ROW_GROUPS ? 0 : ragged::group_rows_workspace(n_rows, n_groups);
}
int32_t tfh_group_rows(int32_t id_bits, const tfh_view* ids, int32_t n_groups, int32_t* offsets, int32_t* order, int32_t* positions,
                       void* workspace, size_t workspace_bytes, tfh_stream stream) {
    return ragged::guarded("tfh_group_rows", [&] { return ragged::group_rows(id_bits, ids, n_groups, offsets, order, positions, workspace, workspace_bytes, stream); });
}
int32_t tfh_ragged_gemm(int32_t dtype, const tfh_row_groups* groups, int32_t flags, double alpha, const tfh_view* a, const tfh_view* b,
                        double beta, const tfh_view* c, tfh_stream stream) {
    return ragged::guarded("tfh_ragged_gemm", [&] { return ragged::ragged_gemm(dtype, groups, flags, alpha, a, b, beta, c, stream); });
}
int32_t tfh_ragged_gemm_grad(int32_t dtype, const tfh_row_groups* groups, int32_t flags, double alpha, const tfh_view* a,
                             const tfh_view* dc, double beta, const tfh_view* db, tfh_stream stream) {
    return ragged::guarded("tfh_ragged_gemm_grad", [&] { return ragged::ragged_gemm_grad(dtype, groups, flags, alpha, a, dc, beta, db, stream); });
}
size_t tfh_ragged_gemm_grad_a_workspace(int32_t dtype, int64_t n_rows, int64_t k, int32_t fan, int32_t flags) {
    return !ragged::known(dtype) || n_rows < 0 || k < 0 || n_rows > ragged::MOST || k > ragged::MOST ? 0 : ragged::grad_a_bytes(dtype, n_rows, k, fan, flags);
}
int32_t tfh_ragged_gemm_grad_a(int32_t dtype, const tfh_row_groups* groups, int32_t flags, double alpha, const tfh_view* dc,
                               const tfh_view* b, const tfh_view* da, void* workspace, size_t workspace_bytes, tfh_stream stream) {
    return ragged::guarded("tfh_ragged_gemm_grad_a", [&] {
        return ragged::ragged_gemm_grad_a(dtype, groups, flags, alpha, dc, b, da, workspace, workspace_bytes, stream);
    });
}
int32_t tfh_combine_rows(int32_t dtype, const tfh_row_groups* groups, const tfh_view* x, const tfh_view* weights, const tfh_view* y,
                         tfh_stream stream) {
    return ragged::guarded("tfh_combine_rows", [&] { return ragged::combine(dtype, groups, x, weights, y, nullptr, nullptr, false, stream); });
}
int32_t tfh_combine_rows_grad(int32_t dtype, const tfh_row_groups* groups, const tfh_view* x, const tfh_view* weights,
                              const tfh_view* dy, const tfh_view* dx, const tfh_view* dweights, tfh_stream stream) {
    return ragged::guarded("tfh_combine_rows_grad", [&] { return ragged::combine(dtype, groups, x, weights, dy, dx, dweights, true, stream); });
}
size_t tfh_adapter_workspace(int32_t dtype, int64_t n_rows, int64_t rank, int32_t gradient) {
    return !ragged::known(dtype) || n_rows < 0 || rank < 0 || n_rows > ragged::MOST || rank > ragged::MOST ? 0
           : ragged::middle_bytes(dtype, n_rows, rank) * ragged::middle_count(dtype, gradient != 0);
}
int32_t tfh_adapter_gemm(int32_t dtype, const tfh_row_groups* groups, const tfh_view* x, const tfh_view* w, const tfh_view* a,
                         const tfh_view* b, const tfh_view* scales, const tfh_view* y, void* workspace, size_t workspace_bytes,
                         tfh_stream stream) {
    return ragged::guarded("tfh_adapter_gemm", [&] {
        return ragged::adapter_gemm({dtype, groups, x, w, a, b, scales, 0, 0, 0}, y, workspace, workspace_bytes, stream);
    });
}
int32_t tfh_adapter_gemm_grad(int32_t dtype, const tfh_row_groups* groups, const tfh_view* x, const tfh_view* w, const tfh_view* a,
                              const tfh_view* b, const tfh_view* scales, const tfh_view* dy, const tfh_view* dx, const tfh_view* da,
                              const tfh_view* db, void* workspace, size_t workspace_bytes, tfh_stream stream) {
    return ragged::guarded("tfh_adapter_gemm_grad", [&] {
        return ragged::adapter_gemm_grad({dtype, groups, x, w, a, b, scales, 0, 0, 0}, dy, dx, da, db, workspace, workspace_bytes, stream);
    });
}

}  // extern "C"
