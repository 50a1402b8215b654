// k_combine.hip -- a token's rows joined again, and the gradient.
//
//   y[t, :] = sum_j w[t, j] x[pos[t fan + j], :]        dx[p, :] = w[t, j] dy[t, :]        dw[t, j] = <x[p, :], dy[t, :]>
//
// with p = pos[t fan + j]; a choice without a place (p < 0) adds nothing, whatever its weight holds.  One wave a token:
// its row of y (dy) is made (read) once, in 16-byte pieces, with the places and weights in scalar registers and two pieces of every
// choice in flight.  HBM bound: 16 384 tokens of four choices, 2048 bf16 columns: 74 us, 4.5 TB/s of reads and writes (a copy: 5.1);
// the gradients of 8192: 66 us, 4.6 TB/s; 8192 tokens of f32 parts into bf16: 57 us, 5.3 TB/s, some of it from L2.
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "ragged.hpp"
#include "ragged_api.hpp"

namespace tfh {
namespace ragged {
namespace {

constexpr int CHUNKS = 2;   // 16-byte pieces of a row that a lane has in flight for each of the choices

// E elements, 16 bytes of a T, of a row from its n-th on, of which the row has `total`.  UNIT: next to each other, and E of them at least; a piece
// that the row ends in is its last E elements instead.
template <class T, bool UNIT> __device__ __forceinline__ u32x4 piece(const T* row, int64_t stride, int n, int total) {
    constexpr int E = Num<T>::E;
    if constexpr (UNIT) return load_unit<T>(row + (n + E <= total ? n : total - E));
    else return load_chunk<T, T>(row + n * stride, stride, total - n);
}
template <class T, bool UNIT, int E> __device__ __forceinline__ void put_piece(T* row, int64_t stride, int n, int total, const T (&e)[E]) {
    if constexpr (UNIT) {
        if (n < total) __builtin_memcpy(row + (n + E <= total ? n : total - E), e, sizeof(e));
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (n + i < total) row[(n + i) * stride] = e[i];
    }
}
// The places and weights of choices j0 .. j0 + F of token t, the same for the whole wave.
template <int F, class W> __device__ __forceinline__ void choices_of(const CombineArgs& a, int64_t t, int j0, int (&p)[F], W (&w)[F]) {
#pragma unroll
    for (int j = 0; j < F; ++j) {
        p[j] = -1;
        w[j] = 0;
        if (j0 + j < a.fan) {
            p[j] = a.positions[t * a.fan + j0 + j];
            if (p[j] >= a.n_rows) p[j] = -1;
            if (p[j] >= 0) w[j] = a.w ? ((const W*)a.w)[t * a.w_token + (j0 + j) * a.w_fan] : (W)1;
        }
    }
}

// X: x's type, T or that of the sums (parts of a sum that is rounded here for the first time).
template <class T, class X, int F, bool UNIT>
__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
    typedef typename Num<T>::acc W;
    constexpr int E = Num<X>::E;
    const int lane = threadIdx.x & 63, step = 64 * E * gridDim.y;
    const int64_t t = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.tokens) return;
    int p[F];
    W w[F];
    choices_of(a, t, 0, p, w);
    for (int n0 = (blockIdx.y * 64 + lane) * E; n0 < a.n; n0 += CHUNKS * step) {
        W sum[CHUNKS][E] = {};
        for (int j0 = 0;;) {
            u32x4 v[F][CHUNKS];
#pragma unroll
            for (int j = 0; j < F; ++j)
                if (p[j] >= 0)
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) v[j][c] = piece<X, UNIT>((const X*)a.x + p[j] * a.x_row, a.x_n, n0 + c * step, a.n);
#pragma unroll
            for (int j = 0; j < F; ++j)
                if (p[j] >= 0)
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        X e[E];
                        __builtin_memcpy(e, &v[j][c], 16);
#pragma unroll
                        for (int i = 0; i < E; ++i) sum[c][i] += w[j] * (W)e[i];
                    }
            j0 += F;
            if (j0 >= a.fan) break;
            choices_of(a, t, j0, p, w);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            T out[E];
#pragma unroll
            for (int i = 0; i < E; ++i) out[i] = (T)sum[c][i];
            put_piece<T, UNIT, E>((T*)a.y + t * a.y_row, a.y_n, n0 + c * step, a.n, out);
        }
        if (a.fan > F) choices_of(a, t, 0, p, w);
    }
}

template <class T, int F, bool UNIT>
__global__ __launch_bounds__(256) void combine_grad_kernel(const CombineArgs a, int token_blocks, int rest_blocks) {
    typedef typename Num<T>::acc W;
    constexpr int E = Num<T>::E, STEP = 64 * E;
    const int lane = threadIdx.x & 63, block = (int)(blockIdx.z * gridDim.x + blockIdx.x);
    if (block >= token_blocks) {
        // the rows behind the last group get zeros, and those before whose row's position is not theirs: no token writes them.  A
        // lane looks at a row, its wave clears those found.
        if (!a.dx || block >= token_blocks + rest_blocks) return;
        const T zero[E] = {};
        const int end = clamp_row(a.offsets[a.n_groups], a.n_rows);
        for (int64_t p0 = ((block - token_blocks) * 4 + (threadIdx.x >> 6)) * (int64_t)64; p0 < a.n_rows; p0 += rest_blocks * 256) {
            const int64_t p = p0 + lane;
            bool left = p < a.n_rows;
            if (left && p < end) {
                const int64_t i = a.order ? a.order[p] : p;
                left = i < 0 || i >= a.n_rows || a.positions[i] != p;
            }
            for (uint64_t found = __ballot(left); found; found &= found - 1)
                for (int n = lane * E; n < a.n; n += STEP) put_piece<T, UNIT, E>((T*)a.dx + (p0 + __builtin_ctzll(found)) * a.dx_row, a.dx_n, n, a.n, zero);
        }
        return;
    }
    const int64_t t = (int64_t)block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.tokens) return;
    for (int j0 = 0; j0 < a.fan; j0 += F) {
        W w[F], dot[F] = {};
        int p[F];
        choices_of(a, t, j0, p, w);
        for (int n0 = lane * E; n0 < a.n; n0 += CHUNKS * STEP) {
            u32x4 d[CHUNKS], v[F][CHUNKS];
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) d[c] = piece<T, UNIT>((const T*)a.y + t * a.y_row, a.y_n, n0 + c * STEP, a.n);
            if (a.dw)
#pragma unroll
                for (int j = 0; j < F; ++j)
                    if (p[j] >= 0)
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) v[j][c] = piece<T, UNIT>((const T*)a.x + p[j] * a.x_row, a.x_n, n0 + c * STEP, a.n);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                T de[E];
                __builtin_memcpy(de, &d[c], 16);
                // elements that the piece before has: of a row's last piece, which may start before n, and of none behind the row
                const int n = n0 + c * STEP, seen = !UNIT ? 0 : n >= a.n ? E : n + E > a.n ? n + E - a.n : 0;
#pragma unroll
                for (int j = 0; j < F; ++j) {
                    if (p[j] < 0) continue;
                    if (a.dw) {
                        T e[E];
                        __builtin_memcpy(e, &v[j][c], 16);
#pragma unroll
                        for (int i = 0; i < E; ++i) dot[j] += i >= seen ? (W)e[i] * (W)de[i] : (W)0;
                    }
                    if (a.dx) {
                        T out[E];
#pragma unroll
                        for (int i = 0; i < E; ++i) out[i] = (T)(w[j] * (W)de[i]);
                        put_piece<T, UNIT, E>((T*)a.dx + p[j] * a.dx_row, a.dx_n, n, a.n, out);
                    }
                }
            }
        }
        if (a.dw) {
#pragma unroll
            for (int j = 0; j < F; ++j) {
#pragma unroll
                for (int s = 1; s < 64; s <<= 1) dot[j] += __shfl_xor(dot[j], s, 64);
                if (lane == 0 && j0 + j < a.fan) ((W*)a.dw)[t * a.dw_token + (j0 + j) * a.dw_fan] = dot[j];
            }
        }
    }
}

template <class T> constexpr const char* name_of(const char* bf16, const char* f16, const char* f32, const char* f64) {
    return __is_same(T, __bf16) ? bf16 : __is_same(T, _Float16) ? f16 : __is_same(T, float) ? f32 : f64;
}

template <class T, class X, int F, bool UNIT> int32_t combine_as(const CombineArgs& a, hipStream_t st) {
    const int64_t blocks = (a.tokens + 3) / 4, pieces = (a.n + 64 * Num<X>::E - 1) / (64 * Num<X>::E);
    // few tokens: their columns are dealt to several blocks, so that more waves wait for memory
    const int64_t split = blocks >= 512 ? 1 : pieces < 512 / blocks ? pieces : 512 / blocks;
    uint32_t x, z;
    if (int32_t e = launch_grid(blocks, 256, &x, &z)) return e;
    TFH_LAUNCH_NAMED(name_of<T>("(combine_kernel<bf16>)", "(combine_kernel<f16>)", "(combine_kernel<float>)", "(combine_kernel<double>)"),
                     (combine_kernel<T, X, F, UNIT>), dim3(x, (unsigned)(split < 1 ? 1 : split), z), dim3(256), 0, st, a);
    return hip_check(hipGetLastError(), "combine launch");
}
template <class T, int F, bool UNIT> int32_t combine_grad_as(const CombineArgs& a, hipStream_t st) {
    const int64_t blocks = (a.tokens + 3) / 4, rest = a.n_rows < 64 * 256 ? (a.n_rows + 255) / 256 : 64;
    uint32_t x, z;
    if (int32_t e = launch_grid(blocks + rest, 256, &x, &z)) return e;
    TFH_LAUNCH_NAMED(name_of<T>("(combine_grad_kernel<bf16>)", "(combine_grad_kernel<f16>)", "(combine_grad_kernel<float>)", "(combine_grad_kernel<double>)"),
                     (combine_grad_kernel<T, F, UNIT>), dim3(x, 1, z), dim3(256), 0, st, a, (int)blocks, (int)rest);
    return hip_check(hipGetLastError(), "combine gradient launch");
}
template <class T, class X> int32_t combine_from(const CombineArgs& a, hipStream_t st) {
    const bool unit = a.x_n == 1 && a.y_n == 1 && a.n >= Num<X>::E;
    if (!unit) return combine_as<T, X, 4, false>(a, st);
    return a.fan <= 2 ? combine_as<T, X, 2, true>(a, st) : a.fan <= 4 ? combine_as<T, X, 4, true>(a, st) : combine_as<T, X, 8, true>(a, st);
}
template <class T> int32_t combine_of(const CombineArgs& a, hipStream_t st) {
    if (a.x_wide) return combine_from<T, typename Num<T>::acc>(a, st);
    return combine_from<T, T>(a, st);
}
template <class T> int32_t combine_grad_of(const CombineArgs& a, hipStream_t st) {
    const bool unit = (!a.dw || a.x_n == 1) && a.y_n == 1 && (!a.dx || a.dx_n == 1) && a.n >= Num<T>::E;
    if (!unit) return combine_grad_as<T, 4, false>(a, st);
    return a.fan <= 2 ? combine_grad_as<T, 2, true>(a, st) : a.fan <= 4 ? combine_grad_as<T, 4, true>(a, st) : combine_grad_as<T, 8, true>(a, st);
}

}  // namespace

int32_t launch_combine(int dtype, const CombineArgs& a, void* stream) {
    switch (dtype) {
        case TFH_BF16: return combine_of<__bf16>(a, (hipStream_t)stream);
        case TFH_F16: return combine_of<_Float16>(a, (hipStream_t)stream);
        case TFH_F32: return combine_of<float>(a, (hipStream_t)stream);
        default: return combine_of<double>(a, (hipStream_t)stream);
    }
}
int32_t launch_combine_grad(int dtype, const CombineArgs& a, void* stream) {
    switch (dtype) {
        case TFH_BF16: return combine_grad_of<__bf16>(a, (hipStream_t)stream);
        case TFH_F16: return combine_grad_of<_Float16>(a, (hipStream_t)stream);
        case TFH_F32: return combine_grad_of<float>(a, (hipStream_t)stream);
        default: return combine_grad_of<double>(a, (hipStream_t)stream);
    }
}

}  // namespace ragged
}  // namespace tfh
