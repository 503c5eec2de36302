// igs_layer_norm / igs_layer_norm_grad over rows of D values (one feature vector a row).
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  xhat = (x - mean) rstd
//   y    = xhat w + b
//   g    = dy w,  dx = rstd (g - sum g / D - xhat sum(g xhat) / D)
//   dw   = sum over rows of dy xhat,  db = sum over rows of dy
//
// All of it in 32 bits, one rounding per result.  The mean is kept as its distance `shift` from
// the row's first value, mean = x[0] + shift: sums and differences of a row far from zero then
// have the size of its spread, not of its distance from zero, and a constant row has variance 0
// exactly.
//
// No atomics: the column sums go through partial sums of fixed blocks of rows, which are added
// in a fixed order.
#include "feature.cuh"

namespace igs {

constexpr int LN_THREADS = 256;

struct NormArgs {
    const void* x;
    const void* w;  // NULL: ones
    const void* b;  // NULL: zeros
    void* y;
    float* shift;   // NULL, or [rows]
    float* rstd;    // NULL, or [rows]
    long long rows, D, row_stride;
    float eps;
};

struct NormGradArgs {
    const void* dy;
    const void* x;
    const void* w;
    const float* shift;
    const float* rstd;
    void* dx;         // NULL: not wanted
    void* dw;
    void* db;
    float* part;      // [splits][2][D] partial column sums
    long long rows, D, row_stride;
    int splits;
};

// Sum over the block, the same bits in every thread; s_red holds two floats per warp, used in
// turn so that one barrier a call suffices: `turn` alternates between calls.
__device__ __forceinline__ float block_sum_all(float v, float* s_red, int turn) {
    v = warp_sum(v);
    float* red = s_red + turn * 32;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    float t = 0.f;
    for (int i = 0; i < warps; ++i) t += red[i];
    return t;
}

// Rows of any width: one CTA per row, the row read three times (from L2 after the first).
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_any_kernel(NormArgs a) {
    __shared__ float s_red[64];
    const W* w = static_cast<const W*>(a.w);
    const W* b = static_cast<const W*>(a.b);
    const float inv_d = 1.f / (float)a.D;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.row_stride;
        T* y = static_cast<T*>(a.y) + r * a.D;
        const float x0 = to_f(x[0]);
        float sum = 0.f;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) sum += to_f(x[c]) - x0;
        const float shift = block_sum_all(sum, s_red, 0) * inv_d;
        float sq = 0.f;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float d = (to_f(x[c]) - x0) - shift;
            sq = fmaf(d, d, sq);
        }
        const float rstd = 1.f / sqrtf(block_sum_all(sq, s_red, 1) * inv_d + a.eps);
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float xhat = ((to_f(x[c]) - x0) - shift) * rstd;
            y[c] = from_f<T>(fmaf(xhat, w ? to_f(w[c]) : 1.f, b ? to_f(b[c]) : 0.f));
        }
        if (threadIdx.x == 0 && a.shift) {
            a.shift[r] = shift;
            a.rstd[r] = rstd;
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_dx_any_kernel(NormGradArgs a) {
    __shared__ float s_red[64];
    const W* w = static_cast<const W*>(a.w);
    const float inv_d = 1.f / (float)a.D;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.row_stride;
        const T* dy = static_cast<const T*>(a.dy) + r * a.D;
        T* dx = static_cast<T*>(a.dx) + r * a.D;
        const float x0 = to_f(x[0]), shift = a.shift[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.f);
            s1 += g;
            s2 = fmaf(g, ((to_f(x[c]) - x0) - shift) * rstd, s2);
        }
        const float m1 = block_sum_all(s1, s_red, 0) * inv_d;
        const float m2 = block_sum_all(s2, s_red, 1) * inv_d;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.f);
            dx[c] = from_f<T>(rstd * (g - m1 - ((to_f(x[c]) - x0) - shift) * rstd * m2));
        }
    }
}

// grid (columns / 32, row splits), block 32 x 8: the column sums over one block of rows
constexpr int LN_COL_ROWS = 8;
template <typename T>
__global__ void __launch_bounds__(32 * LN_COL_ROWS) layer_norm_columns_kernel(NormGradArgs a) {
    __shared__ float s_w[LN_COL_ROWS][32], s_b[LN_COL_ROWS][32];
    const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
    const long long per = (a.rows + a.splits - 1) / a.splits;
    const long long lo = blockIdx.y * per, hi = lo + per < a.rows ? lo + per : a.rows;
    float sw = 0.f, sb = 0.f;
    if (c < a.D) {
        for (long long r = lo + threadIdx.y; r < hi; r += LN_COL_ROWS) {
            const float dy = to_f(static_cast<const T*>(a.dy)[r * a.D + c]);
            const T* x = static_cast<const T*>(a.x) + r * a.row_stride;
            sw = fmaf(dy, ((to_f(x[c]) - to_f(x[0])) - a.shift[r]) * a.rstd[r], sw);
            sb += dy;
        }
    }
    s_w[threadIdx.y][threadIdx.x] = sw;
    s_b[threadIdx.y][threadIdx.x] = sb;
    __syncthreads();
    if (threadIdx.y == 0 && c < a.D) {
        for (int i = 1; i < LN_COL_ROWS; ++i) {
            sw += s_w[i][threadIdx.x];
            sb += s_b[i][threadIdx.x];
        }
        float* part = a.part + (long long)blockIdx.y * 2 * a.D;
        part[c] = sw;
        part[a.D + c] = sb;
    }
}

// the partial sums of all splits, in split order
template <typename W>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_finish_kernel(NormGradArgs a) {
    const long long i = (long long)blockIdx.x * LN_THREADS + threadIdx.x;
    if (i >= 2 * a.D) return;
    float s = 0.f;
    for (int p = 0; p < a.splits; ++p) s += a.part[(long long)p * 2 * a.D + i];
    if (i < a.D) {
        if (a.dw) static_cast<W*>(a.dw)[i] = from_f<W>(s);
    } else if (a.db) {
        static_cast<W*>(a.db)[i - a.D] = from_f<W>(s);
    }
}

// Row splits of the column sums: a pure function of the sizes.
static int norm_splits(long long rows, long long D) {
    const long long slabs = (D + 31) / 32;
    long long want = 148 * 8 / slabs;
    if (want < 1) want = 1;
    if (want > (rows + 31) / 32) want = (rows + 31) / 32;
    return (int)(want < 1 ? 1 : want);
}

static int norm_args_ok(long long rows, long long D, long long row_stride, int dtype, int wdtype) {
    if (rows < 0 || D < 1 || row_stride < 0) return IGS_ERR_ARG;
    if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != IGS_F32)) return IGS_ERR_ARG;
    if (D > (1ll << 30)) return IGS_ERR_LIMIT;
    return IGS_OK;
}

static unsigned row_grid(long long rows) { return (unsigned)(rows < (1ll << 30) ? rows : (1ll << 30)); }

}  // namespace igs

using namespace igs;

extern "C" int igs_layer_norm(const void* x, int dtype, long long rows, long long D, long long row_stride,
                              const void* weight, const void* bias, int wdtype, float eps, void* y, float* shift,
                              float* rstd, int device, void* stream) {
    const int rc = norm_args_ok(rows, D, row_stride, dtype, wdtype);
    if (rc) return rc;
    if (!(eps >= 0.f) || (!shift != !rstd)) return IGS_ERR_ARG;
    if (rows == 0) return IGS_OK;
    if (!x || !y) return IGS_ERR_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    NormArgs a{x, weight, bias, y, shift, rstd, rows, D, row_stride, eps};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (wdtype == dtype)
            layer_norm_any_kernel<T, T><<<row_grid(rows), LN_THREADS, 0, s>>>(a);
        else
            layer_norm_any_kernel<T, float><<<row_grid(rows), LN_THREADS, 0, s>>>(a);
        return 0;
    });
    count_launch();
    return (int)cudaGetLastError();
}

extern "C" size_t igs_layer_norm_grad_workspace_bytes(long long rows, long long D) {
    if (rows <= 0 || D <= 0) return 256;
    return align_up((size_t)norm_splits(rows, D) * 2 * (size_t)D * sizeof(float), 256);
}

extern "C" int igs_layer_norm_grad(const void* dy, const void* x, int dtype, long long rows, long long D,
                                   long long row_stride, const void* weight, int wdtype, const float* shift,
                                   const float* rstd, void* dx, void* dweight, void* dbias, void* workspace,
                                   size_t workspace_bytes, int device, void* stream) {
    const int rc = norm_args_ok(rows, D, row_stride, dtype, wdtype);
    if (rc) return rc;
    const size_t wsize = dtype_size(wdtype);
    if (rows > 0 && (!dy || !x || !shift || !rstd)) return IGS_ERR_ARG;
    const bool columns = dweight || dbias;
    if (rows > 0 && columns && (!workspace || workspace_bytes < igs_layer_norm_grad_workspace_bytes(rows, D)))
        return IGS_ERR_WORKSPACE;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {  // sums over no rows
        cudaError_t e = cudaSuccess;
        if (dweight) e = cudaMemsetAsync(dweight, 0, (size_t)D * wsize, s);
        if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, (size_t)D * wsize, s);
        return (int)e;
    }
    NormGradArgs a{dy, x, weight, shift, rstd, dx, dweight, dbias, static_cast<float*>(workspace), rows, D, row_stride,
                   norm_splits(rows, D)};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (dx) {
            if (wdtype == dtype)
                layer_norm_dx_any_kernel<T, T><<<row_grid(rows), LN_THREADS, 0, s>>>(a);
            else
                layer_norm_dx_any_kernel<T, float><<<row_grid(rows), LN_THREADS, 0, s>>>(a);
            count_launch();
        }
        if (columns) {
            const dim3 grid((unsigned)((D + 31) / 32), (unsigned)a.splits);
            layer_norm_columns_kernel<T><<<grid, dim3(32, LN_COL_ROWS), 0, s>>>(a);
            count_launch();
            const unsigned fin = (unsigned)((2 * D + LN_THREADS - 1) / LN_THREADS);
            if (wdtype == dtype)
                layer_norm_finish_kernel<T><<<fin, LN_THREADS, 0, s>>>(a);
            else
                layer_norm_finish_kernel<float><<<fin, LN_THREADS, 0, s>>>(a);
            count_launch();
        }
        return 0;
    });
    return (int)cudaGetLastError();
}
