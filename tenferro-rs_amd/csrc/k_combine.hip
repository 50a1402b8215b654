// k_combine.hip -- a token's rows joined again, and the gradient.
//
//   y[t, :] = sum_j w[t, j] x[pos[t fan + j], :]        dx[p, :] = w[t, j] dy[t, :]        dw[t, j] = <x[p, :], dy[t, :]>
//
// with p = pos[t fan + j]; a choice without a place (p < 0) adds nothing, whatever its weight holds.  One wave a token:
// its row of y (dy) is made (read) once, in 16-byte pieces.  HBM bound.
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "ragged.hpp"
#include "ragged_api.hpp"

namespace tfh {
namespace ragged {
namespace {

constexpr int AT_ONCE = 8;   // choices of a token whose loads are in flight together

template <class T>
__device__ __forceinline__ void store_chunk(T* p, int64_t stride, int count, const T (&e)[Num<T>::E]) {
    if (count >= Num<T>::E && stride == 1) {
        __builtin_memcpy(p, e, 16);
    } else {
#pragma unroll
        for (int i = 0; i < Num<T>::E; ++i)
            if (i < count) p[i * stride] = e[i];
    }
}

template <class T>
__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
    typedef typename Num<T>::acc W;
    constexpr int E = Num<T>::E;
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    for (int n = (blockIdx.y * 64 + lane) * E; n < a.n; n += 64 * E * gridDim.y) {
        W sum[E] = {};
        for (int j0 = 0; j0 < a.fan; j0 += AT_ONCE) {
            u32x4 v[AT_ONCE];
            W w[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                w[j] = 0;
                int p = -1;
                if (j0 + j < a.fan) {
                    p = a.positions[t * a.fan + j0 + j];
                    if (p >= a.n_rows) p = -1;
                    if (p >= 0) w[j] = a.w ? ((const W*)a.w)[t * a.w_token + (j0 + j) * a.w_fan] : (W)1;
                }
                v[j] = load_chunk<T, T>((const T*)a.x + p * a.x_row + n * a.x_n, a.x_n, p >= 0 ? a.n - n : 0);
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                T e[E];
                __builtin_memcpy(e, &v[j], 16);
#pragma unroll
                for (int i = 0; i < E; ++i) sum[i] += w[j] * (W)e[i];
            }
        }
        T out[E];
#pragma unroll
        for (int i = 0; i < E; ++i) out[i] = (T)sum[i];
        store_chunk<T>((T*)a.y + t * a.y_row + n * a.y_n, a.y_n, a.n - n, out);
    }
}

template <class T>
__global__ __launch_bounds__(256) void combine_grad_kernel(const CombineArgs a, int token_blocks) {
    typedef typename Num<T>::acc W;
    constexpr int E = Num<T>::E;
    const int lane = threadIdx.x & 63;
    if ((int)blockIdx.x >= token_blocks) {
        // the rows behind the last group get zeros
        if (!a.dx) return;
        const T zero[E] = {};
        const int from = clamp_row(a.offsets[a.n_groups], a.n_rows);
        for (int64_t p = from + ((int)blockIdx.x - token_blocks) * 4 + (threadIdx.x >> 6); p < a.n_rows; p += ((int)gridDim.x - token_blocks) * 4)
            for (int n = lane * E; n < a.n; n += 64 * E) store_chunk<T>((T*)a.dx + p * a.dx_row + n * a.dx_n, a.dx_n, a.n - n, zero);
        return;
    }
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    for (int j0 = 0; j0 < a.fan; j0 += AT_ONCE) {
        W w[AT_ONCE], dot[AT_ONCE];
        int p[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            p[j] = -1;
            w[j] = dot[j] = 0;
            if (j0 + j < a.fan) {
                p[j] = a.positions[t * a.fan + j0 + j];
                if (p[j] >= a.n_rows) p[j] = -1;
                if (p[j] >= 0) w[j] = a.w ? ((const W*)a.w)[t * a.w_token + (j0 + j) * a.w_fan] : (W)1;
            }
        }
        for (int n = lane * E; n < a.n; n += 64 * E) {
            const u32x4 d = load_chunk<T, T>((const T*)a.y + t * a.y_row + n * a.y_n, a.y_n, a.n - n);
            u32x4 v[AT_ONCE];
            if (a.dw)
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j)
                    v[j] = load_chunk<T, T>((const T*)a.x + p[j] * a.x_row + n * a.x_n, a.x_n, p[j] >= 0 ? a.n - n : 0);
            T de[E];
            __builtin_memcpy(de, &d, 16);
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                if (p[j] < 0) continue;
                if (a.dw) {
                    T e[E];
                    __builtin_memcpy(e, &v[j], 16);
#pragma unroll
                    for (int i = 0; i < E; ++i) dot[j] += (W)e[i] * (W)de[i];
                }
                if (a.dx) {
                    T out[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) out[i] = (T)(w[j] * (W)de[i]);
                    store_chunk<T>((T*)a.dx + p[j] * a.dx_row + n * a.dx_n, a.dx_n, a.n - n, out);
                }
            }
        }
        if (a.dw) {
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
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

template <class T> int32_t combine_of(const CombineArgs& a, hipStream_t st) {
    const int64_t blocks = (a.tokens + 3) / 4, pieces = (a.n + 64 * Num<T>::E - 1) / (64 * Num<T>::E);
    // few tokens: their columns are dealt to several blocks, so that more waves wait for memory
    const int64_t split = blocks >= 512 ? 1 : pieces < 512 / blocks ? pieces : 512 / blocks;
    TFH_LAUNCH_NAMED(name_of<T>("(combine_kernel<bf16>)", "(combine_kernel<f16>)", "(combine_kernel<float>)", "(combine_kernel<double>)"), combine_kernel<T>, dim3((unsigned)blocks, (unsigned)(split < 1 ? 1 : split)), dim3(256), 0, st, a);
    return hip_check(hipGetLastError(), "combine launch");
}
template <class T> int32_t combine_grad_of(const CombineArgs& a, hipStream_t st) {
    const int64_t blocks = (a.tokens + 3) / 4, rest = a.n_rows < 256 ? (a.n_rows + 3) / 4 : 64;
    TFH_LAUNCH_NAMED(name_of<T>("(combine_grad_kernel<bf16>)", "(combine_grad_kernel<f16>)", "(combine_grad_kernel<float>)", "(combine_grad_kernel<double>)"),
                     combine_grad_kernel<T>, dim3((unsigned)(blocks + rest)), dim3(256), 0, st, a, (int)blocks);
    return hip_check(hipGetLastError(), "combine gradient launch");
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
