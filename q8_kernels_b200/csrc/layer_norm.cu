// Layer norm over the last dim, forward and backward:
//   z = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = z * w + b
//   dx = rstd * (g w - mean(g w) - z mean(g w z)),  dw = sum_rows g z,  db = sum_rows g
//
// Both passes are bound by HBM: the forward reads x and writes y, the backward reads x and g and writes dx.  A row lives in the
// registers of T threads between its reductions and its output, so each element is read once.  The variance is taken from
// the differences to the mean (a second sum over the registers, not E[x^2] - mean^2, which loses all digits of a row whose mean is
// large against its spread).  Sums, statistics and the gradients of w and b are fp32.
//
// Columns of a thread: VEC (dim a multiple of 8, all rows 16-byte aligned): items of 8 consecutive elements, 16- or 32-byte
// accesses.  Otherwise single elements T apart: a warp then reads 32 consecutive elements, and the columns of a thread are the same
// in every row, wherever the rows start, which the sums over rows need.

#include <type_traits>
#include "common.cuh"

namespace q8k {

constexpr int kLnItem = 8;
constexpr int kLnMaxDim = 16384;

// What thread `t` of a row's T threads owns in its item i: column of element j, and whether it exists.
template <int T, bool VEC> __device__ __forceinline__ int ln_col(int t, int i, int j) {
    return VEC ? (t + i * T) * kLnItem + j : t + (i * kLnItem + j) * T;
}

template <typename E, int T, bool VEC>
__device__ __forceinline__ void ln_load(const E* __restrict__ row, int dim, int t, int i, float (&v)[kLnItem]) {
    if constexpr (VEC) {
        if (ln_col<T, VEC>(t, i, 0) < dim) load_vec<E, kLnItem>(row + ln_col<T, VEC>(t, i, 0), v);
        else {
#pragma unroll
            for (int j = 0; j < kLnItem; ++j) v[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kLnItem; ++j) v[j] = ln_col<T, VEC>(t, i, j) < dim ? to_float<E>(row[ln_col<T, VEC>(t, i, j)]) : 0.f;
    }
}

template <typename E, int T, bool VEC>
__device__ __forceinline__ void ln_store(E* __restrict__ row, int dim, int t, int i, const float (&v)[kLnItem]) {
    if constexpr (VEC) {
        if (ln_col<T, VEC>(t, i, 0) < dim) store_vec<E, kLnItem>(row + ln_col<T, VEC>(t, i, 0), v);
    } else {
#pragma unroll
        for (int j = 0; j < kLnItem; ++j)
            if (ln_col<T, VEC>(t, i, j) < dim) row[ln_col<T, VEC>(t, i, j)] = from_float<E>(v[j]);
    }
}

// Sums of N values over the T threads of a row, the same in each of them.  `red` is the row group's own shared memory
// (N * T / 32 floats); a barrier stands before its reuse.
template <int T, int N>
__device__ __forceinline__ void ln_row_sum(float (&v)[N], float* red) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
    if constexpr (T > 32) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) red[warp * N + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = red[k];
#pragma unroll
            for (int w = 1; w < T / 32; ++w) v[k] += red[w * N + k];
        }
        __syncthreads();
    }
}

// G rows per CTA, T threads each (G > 1 only with T = 32, where a row needs no barrier).
template <typename Tx, typename Ty, int ITEMS, int T, int G, bool VEC>
__global__ void __launch_bounds__(T * G)
layer_norm_kernel(const Tx* __restrict__ x, int64_t x_stride, const float* __restrict__ w, const float* __restrict__ b,
                  Ty* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int dim, float eps) {
    static_assert(G == 1 || T == 32, "row groups of more than a warp would need barriers of their own");
    __shared__ float red[T / 32];
    const int t = G > 1 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = (int64_t)blockIdx.x * G + (G > 1 ? threadIdx.x >> 5 : 0);
    pdl_wait();
    pdl_release();
    if (G > 1 && row >= rows) return;
    const Tx* xr = x + row * x_stride;
    float v[ITEMS][kLnItem];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        ln_load<Tx, T, VEC>(xr, dim, t, i, v[i]);
#pragma unroll
        for (int j = 0; j < kLnItem; ++j) s[0] += v[i][j];
    }
    ln_row_sum<T>(s, red);
    const float inv = 1.0f / (float)dim;
    const float mean = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int j = 0; j < kLnItem; ++j) {
            if (ln_col<T, VEC>(t, i, VEC ? 0 : j) < dim) {
                const float d = v[i][j] - mean;
                s[0] = fmaf(d, d, s[0]);
            }
        }
    }
    ln_row_sum<T>(s, red);
    const float rstd = 1.0f / sqrtf(fmaf(s[0], inv, eps));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        float wv[kLnItem], bv[kLnItem], o[kLnItem];
        if (w != nullptr) ln_load<float, T, VEC>(w, dim, t, i, wv);
        if (b != nullptr) ln_load<float, T, VEC>(b, dim, t, i, bv);
#pragma unroll
        for (int j = 0; j < kLnItem; ++j) {
            o[j] = (v[i][j] - mean) * rstd;
            if (w != nullptr) o[j] = b != nullptr ? fmaf(o[j], wv[j], bv[j]) : o[j] * wv[j];
            else if (b != nullptr) o[j] += bv[j];
        }
        ln_store<Ty, T, VEC>(y + row * (int64_t)dim, dim, t, i, o);
    }
    if (t == 0) {
        if (mean_out != nullptr) mean_out[row] = mean;
        if (rstd_out != nullptr) rstd_out[row] = rstd;
    }
}

// A CTA walks over rows and keeps its columns' sums of g z and g in registers; they go to part[group][2][dim] at the end and
// layer_norm_wgrad_kernel adds the groups up in a fixed order: no atomics, the same bits in every run.
template <typename Tx, typename Tg, int ITEMS, int T, int G, bool VEC, bool WGRAD>
__global__ void __launch_bounds__(T * G)
layer_norm_backward_kernel(const Tx* __restrict__ x, int64_t x_stride, const Tg* __restrict__ g, const float* __restrict__ mean,
                           const float* __restrict__ rstd, const float* __restrict__ w, Tx* __restrict__ dx, float* __restrict__ part,
                           int64_t rows, int dim) {
    static_assert(G == 1 || T == 32, "row groups of more than a warp would need barriers of their own");
    __shared__ float red[2 * (T / 32)];
    const int t = G > 1 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t group = (int64_t)blockIdx.x * G + (G > 1 ? threadIdx.x >> 5 : 0);
    pdl_wait();
    pdl_release();
    float dw[WGRAD ? ITEMS : 1][kLnItem], db[WGRAD ? ITEMS : 1][kLnItem];
    if constexpr (WGRAD) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < kLnItem; ++j) dw[i][j] = db[i][j] = 0.f;
    }
    const float inv = 1.0f / (float)dim;
    for (int64_t row = group; row < rows; row += (int64_t)gridDim.x * G) {
        float z[ITEMS][kLnItem], gv[ITEMS][kLnItem];
        const float m = mean[row], r = rstd[row];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            ln_load<Tx, T, VEC>(x + row * x_stride, dim, t, i, z[i]);
            ln_load<Tg, T, VEC>(g + row * (int64_t)dim, dim, t, i, gv[i]);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            float wv[kLnItem];
            if (w != nullptr) ln_load<float, T, VEC>(w, dim, t, i, wv);
#pragma unroll
            for (int j = 0; j < kLnItem; ++j) {                // columns that do not exist have g = 0: they add nothing
                z[i][j] = (z[i][j] - m) * r;
                if constexpr (WGRAD) {
                    dw[i][j] = fmaf(gv[i][j], z[i][j], dw[i][j]);
                    db[i][j] += gv[i][j];
                }
                if (w != nullptr) gv[i][j] *= wv[j];
                s[0] += gv[i][j];
                s[1] = fmaf(gv[i][j], z[i][j], s[1]);
            }
        }
        if (dx == nullptr) continue;                           // only the sums over rows are wanted
        ln_row_sum<T>(s, red);
        const float a = s[0] * inv, c = s[1] * inv;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            float o[kLnItem];
#pragma unroll
            for (int j = 0; j < kLnItem; ++j) o[j] = r * (gv[i][j] - fmaf(z[i][j], c, a));
            ln_store<Tx, T, VEC>(dx + row * (int64_t)dim, dim, t, i, o);
        }
    }
    if constexpr (WGRAD) {
        float* p = part + group * 2 * (int64_t)dim;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            ln_store<float, T, VEC>(p, dim, t, i, dw[i]);
            ln_store<float, T, VEC>(p + dim, dim, t, i, db[i]);
        }
    }
}

// dw[c] = sum over groups of part[group][0][c], db[c] likewise of part[group][1][c]: a CTA takes 32 of the 2 * dim columns, warp k the
// groups k, k + 8, ..., and the eight sums are added in shared memory.
constexpr int kLnSumWarps = 8;
__global__ void __launch_bounds__(32 * kLnSumWarps)
layer_norm_wgrad_kernel(const float* __restrict__ part, int groups, float* __restrict__ dw, float* __restrict__ db, int dim) {
    __shared__ float sums[kLnSumWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    const bool in = c < 2 * (int64_t)dim;
    pdl_wait();
    pdl_release();
    float s = 0.f;
    if (in) {
#pragma unroll 8
        for (int k = warp; k < groups; k += kLnSumWarps) s += part[k * 2 * (int64_t)dim + c];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && in) {
        s = sums[0][lane];
#pragma unroll
        for (int k = 1; k < kLnSumWarps; ++k) s += sums[k][lane];
        float* out = c < dim ? dw : db;
        if (out != nullptr) out[c < dim ? c : c - dim] = s;
    }
}

// ------------------------------------------------------------------ host side
// Calls f(items, threads per row, rows per CTA) with the row's layout as integral constants.
template <typename F> static int ln_layout(int dim, F&& f) {
    const int items = (dim + kLnItem - 1) / kLnItem;
#define Q8K_LN(I, T, G) return f(std::integral_constant<int, I>(), std::integral_constant<int, T>(), std::integral_constant<int, G>())
    if (items <= 32) Q8K_LN(1, 32, 4);
    if (items <= 128) Q8K_LN(1, 128, 1);
    if (items <= 256) Q8K_LN(1, 256, 1);
    if (items <= 512) Q8K_LN(2, 256, 1);
    if (items <= 1024) Q8K_LN(4, 256, 1);
    Q8K_LN(4, 512, 1);
#undef Q8K_LN
}

// Row groups of a backward pass that sums over rows: as many CTAs as the device holds, or one row each.
static int ln_groups(int64_t rows, int dim) {
    int groups = 0;
    ln_layout(dim, [&](auto, auto t, auto g) {
        const int64_t ctas = (int64_t)gemm_num_sms() * (1024 / (t.value * g.value));
        const int64_t need = (rows + g.value - 1) / g.value;
        groups = (int)(need < ctas ? need : ctas) * g.value;
        return 0;
    });
    return groups;
}

static int check_ln(const char* op, int64_t rows, int dim, int64_t x_stride) {
    Q8K_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL, Q8K_ERR_INVALID_ARG, "%s: rows %lld out of range", op, (long long)rows);
    Q8K_REQUIRE(dim > 0, Q8K_ERR_INVALID_ARG, "%s: dim %d must be positive", op, dim);
    Q8K_REQUIRE(dim <= kLnMaxDim, Q8K_ERR_UNSUPPORTED, "%s: dim %d exceeds %d", op, dim, kLnMaxDim);
    Q8K_REQUIRE(x_stride >= 0, Q8K_ERR_INVALID_ARG, "%s: negative row stride", op);
    return Q8K_OK;
}

static bool ln_aligned(const void* p, int dtype) {
    const int size = dtype_size(dtype);
    return size > 0 && reinterpret_cast<uintptr_t>(p) % size == 0;
}

template <typename Tx, typename Ty>
static int launch_ln(const void* x, int64_t x_stride, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t rows,
                     int dim, float eps, bool vec, cudaStream_t st) {
    return ln_layout(dim, [&](auto i, auto t, auto g) {
        constexpr int I = decltype(i)::value, T = decltype(t)::value, G = decltype(g)::value;
        auto kern = vec ? layer_norm_kernel<Tx, Ty, I, T, G, true> : layer_norm_kernel<Tx, Ty, I, T, G, false>;
        Q8K_CUDA_OK(launch_dependent(kern, (unsigned)((rows + G - 1) / G), T * G, 0, st, 1, (const Tx*)x, x_stride, w, b, (Ty*)y, mean,
                                     rstd, rows, dim, eps));
        return Q8K_OK;
    });
}

template <typename Tx, typename Tg>
static int launch_ln_backward(const void* x, int64_t x_stride, const void* g, const float* mean, const float* rstd, const float* w,
                              void* dx, float* part, int64_t rows, int dim, bool vec, cudaStream_t st) {
    return ln_layout(dim, [&](auto i, auto t, auto gr) {
        constexpr int I = decltype(i)::value, T = decltype(t)::value, G = decltype(gr)::value;
        // without sums over rows nothing is gained by a CTA that takes more than its G rows
        const unsigned grid = part != nullptr ? (unsigned)(ln_groups(rows, dim) / G) : (unsigned)((rows + G - 1) / G);
        auto kern = part != nullptr ? (vec ? layer_norm_backward_kernel<Tx, Tg, I, T, G, true, true>
                                           : layer_norm_backward_kernel<Tx, Tg, I, T, G, false, true>)
                                    : (vec ? layer_norm_backward_kernel<Tx, Tg, I, T, G, true, false>
                                           : layer_norm_backward_kernel<Tx, Tg, I, T, G, false, false>);
        Q8K_CUDA_OK(launch_dependent(kern, grid, T * G, 0, st, 1, (const Tx*)x, x_stride, (const Tg*)g, mean, rstd, w, (Tx*)dx, part,
                                     rows, dim));
        return Q8K_OK;
    });
}

}  // namespace q8k

using namespace q8k;

extern "C" int q8k_layer_norm(const void* x, int x_dtype, int64_t x_row_stride, const float* weight, const float* bias, void* y,
                              int y_dtype, float* mean, float* rstd, int64_t rows, int dim, float eps, void* stream) {
    const char* op = "layer_norm";
    if (int rc = check_ln(op, rows, dim, x_row_stride)) return rc;
    if (rows == 0) return Q8K_OK;
    Q8K_REQUIRE(x && y, Q8K_ERR_INVALID_ARG, "%s: null pointer", op);
    Q8K_REQUIRE(ln_aligned(x, x_dtype) && ln_aligned(y, y_dtype) && ln_aligned(weight, Q8K_DT_F32) && ln_aligned(bias, Q8K_DT_F32),
                Q8K_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element, or an unknown type", op);
    const bool vec = dim % kLnItem == 0 && aligned16(x) && (x_row_stride * dtype_size(x_dtype)) % 16 == 0 && aligned16(y) &&
                     aligned16(weight) && aligned16(bias);
    cudaStream_t st = (cudaStream_t)stream;
#define Q8K_LN_FWD(DX, DY)                                                                       \
    if (x_dtype == DX && y_dtype == DY)                                                          \
        return launch_ln<DType<DX>::type, DType<DY>::type>(x, x_row_stride, weight, bias, y, mean, rstd, rows, dim, eps, vec, st)
    Q8K_LN_FWD(Q8K_DT_BF16, Q8K_DT_BF16);
    Q8K_LN_FWD(Q8K_DT_BF16, Q8K_DT_E4M3);
    Q8K_LN_FWD(Q8K_DT_F16, Q8K_DT_F16);
    Q8K_LN_FWD(Q8K_DT_F32, Q8K_DT_F32);
    Q8K_LN_FWD(Q8K_DT_F32, Q8K_DT_BF16);
    Q8K_LN_FWD(Q8K_DT_F32, Q8K_DT_F16);
#undef Q8K_LN_FWD
    set_error_detail("%s: dtype pair (%d -> %d) not supported", op, x_dtype, y_dtype);
    return Q8K_ERR_UNSUPPORTED;
}

extern "C" size_t q8k_layer_norm_backward_workspace_bytes(int64_t rows, int dim) {
    if (rows <= 0 || dim <= 0 || dim > kLnMaxDim) return 0;
    return (size_t)ln_groups(rows, dim) * 2 * (size_t)dim * sizeof(float);
}

extern "C" int q8k_layer_norm_backward(const void* x, int x_dtype, int64_t x_row_stride, const void* grad, int grad_dtype,
                                       const float* mean, const float* rstd, const float* weight, void* dx, float* dweight,
                                       float* dbias, int64_t rows, int dim, void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "layer_norm_backward";
    if (int rc = check_ln(op, rows, dim, x_row_stride)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const bool sums = dweight != nullptr || dbias != nullptr;
    Q8K_REQUIRE(ln_aligned(dweight, Q8K_DT_F32) && ln_aligned(dbias, Q8K_DT_F32), Q8K_ERR_INVALID_ARG, "%s: misaligned gradient", op);
    if (rows == 0) {                                           // sums over no rows
        if (dweight != nullptr) Q8K_CUDA_OK(cudaMemsetAsync(dweight, 0, (size_t)dim * sizeof(float), st));
        if (dbias != nullptr) Q8K_CUDA_OK(cudaMemsetAsync(dbias, 0, (size_t)dim * sizeof(float), st));
        return Q8K_OK;
    }
    if (dx == nullptr && !sums) return Q8K_OK;
    Q8K_REQUIRE(x && grad && mean && rstd, Q8K_ERR_INVALID_ARG, "%s: null pointer", op);
    Q8K_REQUIRE(ln_aligned(x, x_dtype) && ln_aligned(dx, x_dtype) && ln_aligned(grad, grad_dtype) && ln_aligned(weight, Q8K_DT_F32),
                Q8K_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element, or an unknown type", op);
    float* part = nullptr;
    if (sums) {
        Q8K_REQUIRE(workspace != nullptr && aligned16(workspace), Q8K_ERR_INVALID_ARG, "%s: null or misaligned workspace", op);
        Q8K_REQUIRE(workspace_bytes >= q8k_layer_norm_backward_workspace_bytes(rows, dim), Q8K_ERR_WORKSPACE,
                    "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, q8k_layer_norm_backward_workspace_bytes(rows, dim));
        part = (float*)workspace;
    }
    const bool vec = dim % kLnItem == 0 && aligned16(x) && (x_row_stride * dtype_size(x_dtype)) % 16 == 0 && aligned16(grad) &&
                     aligned16(dx) && aligned16(weight);
    int rc = Q8K_ERR_UNSUPPORTED;
#define Q8K_LN_BWD(DX, DG)                                                                       \
    if (x_dtype == DX && grad_dtype == DG)                                                       \
        rc = launch_ln_backward<DType<DX>::type, DType<DG>::type>(x, x_row_stride, grad, mean, rstd, weight, dx, part, rows, dim, vec, st)
    Q8K_LN_BWD(Q8K_DT_BF16, Q8K_DT_BF16);
    else Q8K_LN_BWD(Q8K_DT_F16, Q8K_DT_F16);
    else Q8K_LN_BWD(Q8K_DT_F32, Q8K_DT_F32);
    else Q8K_LN_BWD(Q8K_DT_F32, Q8K_DT_BF16);
    else Q8K_LN_BWD(Q8K_DT_F32, Q8K_DT_F16);
    else set_error_detail("%s: dtype pair (%d, gradient %d) not supported", op, x_dtype, grad_dtype);
#undef Q8K_LN_BWD
    if (rc != Q8K_OK || !sums) return rc;
    Q8K_CUDA_OK(launch_dependent(layer_norm_wgrad_kernel, (unsigned)((2 * (int64_t)dim + 31) / 32), 32 * kLnSumWarps, 0, st, 1, part,
                                 ln_groups(rows, dim), dweight, dbias, dim));
    return Q8K_OK;
}
