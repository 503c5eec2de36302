// igs_layer_norm, and in layer_norm_grad.cu its gradient, over rows of D values (one feature vector a row).
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
#include "layer_norm.cuh"

namespace igs {

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

// Rows that fit the registers of a group of G threads, ITEMS packs of V values a thread: one read
// of x, one write of y.  A group takes R rows at a time, so that their sums overlap and a weight
// is loaded once for all of them.
template <typename T, typename W, int V, int G, int ITEMS, int R>
__global__ void __launch_bounds__(norm_block(G)) layer_norm_kernel(NormArgs a) {
    constexpr int GROUPS = norm_block(G) / G;
    __shared__ float s_red[G > 32 ? 2 * (G / 32) * R : 1];
    const int lane = threadIdx.x % G;
    const float inv_d = 1.f / (float)a.D;
    const int packs = (int)(a.D / V);
    const long long row0 = ((long long)blockIdx.x * GROUPS + threadIdx.x / G) * R;
    // (a group past the last row stays to take part in its warp's or block's sums)

    Pack<T, V> x[R][ITEMS];
    float x0[R], sum[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* src = static_cast<const T*>(a.x) + (row0 + r) * a.row_stride;
        const bool ok = row0 + r < a.rows;
        x0[r] = ok ? to_f(src[0]) : 0.f;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int p = k * G + lane;
            if (ok && p < packs) x[r][k] = reinterpret_cast<const Pack<T, V>*>(src)[p];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        sum[r] = 0.f;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (k * G + lane < packs && row0 + r < a.rows) {
#pragma unroll
                for (int j = 0; j < V; ++j) sum[r] += to_f(x[r][k].v[j]) - x0[r];
            }
    }
    group_sum<G, R>(sum, s_red, 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        sum[r] *= inv_d;  // the shift
        rstd[r] = 0.f;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (k * G + lane < packs && row0 + r < a.rows) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = (to_f(x[r][k].v[j]) - x0[r]) - sum[r];
                    rstd[r] = fmaf(d, d, rstd[r]);
                }
            }
    }
    group_sum<G, R>(rstd, s_red, 1);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        rstd[r] = 1.f / sqrtf(rstd[r] * inv_d + a.eps);
        if (lane == 0 && a.shift && row0 + r < a.rows) {
            a.shift[row0 + r] = sum[r];
            a.rstd[row0 + r] = rstd[r];
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int p = k * G + lane;
        if (p >= packs) continue;
        float w[V], b[V];
        load_weights<W, V>(a.w, (long long)p * V, 1.f, w);
        load_weights<W, V>(a.b, (long long)p * V, 0.f, b);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (row0 + r >= a.rows) continue;
            Pack<T, V> y;
#pragma unroll
            for (int j = 0; j < V; ++j)
                y.v[j] = from_f<T>(fmaf(((to_f(x[r][k].v[j]) - x0[r]) - sum[r]) * rstd[r], w[j], b[j]));
            reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.y) + (row0 + r) * a.D)[p] = y;
        }
    }
}

// Rows of any width: one CTA per row, the row read three times (from L2 after the first).
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_any_kernel(NormArgs a) {
    __shared__ float s_red[LN_RED];
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

// Calls f(G, ITEMS, R) with the narrowest group of threads that holds `packs` packs of V values: a warp
// where 32 values a thread do (sums without a barrier), else up to 1024 threads; false when none does.
template <int V, typename F>
static bool with_norm_group(long long packs, F&& f) {
    constexpr int I = V == 1 ? 16 : 32 / V;  // packs a thread of a wide group
    if (packs <= 8) f(Int<8>{}, Int<1>{}, Int<2>{});
    else if (packs <= 32) f(Int<32>{}, Int<1>{}, Int<4>{});
    else if (packs <= 32 * (8 / (V < 8 ? V : 8)) && V < 8) f(Int<32>{}, Int<8 / (V < 8 ? V : 8)>{}, Int<2>{});
    else if (packs <= 32 * (16 / V)) f(Int<32>{}, Int<16 / V>{}, Int<2>{});
    else if (packs <= 32 * (32 / V)) f(Int<32>{}, Int<32 / V>{}, Int<1>{});
    else if (packs <= 128 * I) f(Int<128>{}, Int<I>{}, Int<1>{});
    else if (packs <= 256 * I) f(Int<256>{}, Int<I>{}, Int<1>{});
    else if (packs <= 512 * I) f(Int<512>{}, Int<I>{}, Int<1>{});
    else if (packs <= 1024 * I) f(Int<1024>{}, Int<I>{}, Int<1>{});
    else return false;
    return true;
}

template <typename T, typename W, int V>
static bool launch_norm_packs(const NormArgs& a, cudaStream_t s) {
    return with_norm_group<V>(a.D / V, [&](auto g, auto items, auto r) {
        constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value, R = decltype(r)::value;
        constexpr int PER = norm_block(G) / G * R;
        layer_norm_kernel<T, W, V, G, ITEMS, R><<<row_grid((a.rows + PER - 1) / PER), norm_block(G), 0, s>>>(a);
    });
}

template <typename T, typename W>
static void launch_norm(const NormArgs& a, cudaStream_t s) {
    const int bytes = norm_pack_bytes(a.x, a.y, nullptr, a.w, a.b, a.D, a.row_stride, sizeof(T), sizeof(W));
    bool done = false;
    if (bytes == 16) done = launch_norm_packs<T, W, 16 / sizeof(T)>(a, s);
    else if (bytes == 4) done = launch_norm_packs<T, W, 4 / sizeof(T)>(a, s);
    else done = launch_norm_packs<T, W, 1>(a, s);
    if (!done) layer_norm_any_kernel<T, W><<<row_grid(a.rows), LN_THREADS, 0, s>>>(a);
}

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
        if (wdtype == dtype) launch_norm<T, T>(a, s);
        else launch_norm<T, float>(a, s);
        return 0;
    });
    count_launch();
    return (int)cudaGetLastError();
}
