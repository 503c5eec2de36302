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

// V weights as floats; without any, the value they stand for
template <typename W, int V>
__device__ __forceinline__ void load_weights(const void* w, long long c, float none, float (&out)[V]) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = none;
        return;
    }
    const Pack<W, V> p = *reinterpret_cast<const Pack<W, V>*>(static_cast<const W*>(w) + c);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = to_f(p.v[j]);
}

// N sums over the G threads of a row's group at once, the same bits in every one of them.  Groups
// of up to a warp are lanes of one warp; a wider group is the whole block, and s_red (two halves
// used in turn, so that one barrier a call suffices) holds N floats per warp.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* s_red, int turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int d = (G < 32 ? G : 32) / 2; d > 0; d >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
    }
    if constexpr (G > 32) {
        constexpr int WARPS = G / 32;
        float* red = s_red + turn * (WARPS * N);
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) red[(threadIdx.x >> 5) * N + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) t += red[w * N + i];
            v[i] = t;
        }
    }
}

__host__ __device__ constexpr int norm_block(int G) { return G < 128 ? 128 : G; }

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

// The gradient of the same rows: one read of x and dy, one write of dx, and the column sums kept
// in registers over all rows that a block takes (a thread's columns are the same in every row).
// Block b takes the batches b, b + gridDim.x, ... of GROUPS * R rows; its groups' sums are added in
// order at the end and written as partial b.
template <typename T, typename W, int V, int G, int ITEMS, int R>
__global__ void __launch_bounds__(norm_block(G)) layer_norm_grad_kernel(NormGradArgs a) {
    constexpr int GROUPS = norm_block(G) / G;
    constexpr int COLS = G * ITEMS * V;  // columns a group covers
    __shared__ float s_red[G > 32 ? 2 * (G / 32) * 2 * R : 1];
    __shared__ float s_cols[GROUPS > 1 ? GROUPS * 2 * COLS : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_d = 1.f / (float)a.D;
    const int packs = (int)(a.D / V);

    float w[ITEMS][V], dw[ITEMS][V], db[ITEMS][V];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[k][j] = dw[k][j] = db[k][j] = 0.f;
        if (k * G + lane < packs) load_weights<W, V>(a.w, (long long)(k * G + lane) * V, 1.f, w[k]);
    }

    int turn = 0;
    for (long long base = (long long)blockIdx.x * (GROUPS * R); base < a.rows; base += (long long)gridDim.x * (GROUPS * R)) {
        const long long row0 = base + group * R;
        Pack<T, V> x[R][ITEMS], dy[R][ITEMS];
        float x0[R], shift[R], rstd[R], s[2 * R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool ok = row0 + r < a.rows;
            const T* xs = static_cast<const T*>(a.x) + (row0 + r) * a.row_stride;
            const T* ds = static_cast<const T*>(a.dy) + (row0 + r) * a.D;
            x0[r] = ok ? to_f(xs[0]) : 0.f;
            shift[r] = ok ? a.shift[row0 + r] : 0.f;
            rstd[r] = ok ? a.rstd[row0 + r] : 0.f;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                const int p = k * G + lane;
                if (ok && p < packs) {
                    x[r][k] = reinterpret_cast<const Pack<T, V>*>(xs)[p];
                    dy[r][k] = reinterpret_cast<const Pack<T, V>*>(ds)[p];
                } else {  // (a row past the last adds nothing to any sum: rstd is zero too)
#pragma unroll
                    for (int j = 0; j < V; ++j) x[r][k].v[j] = dy[r][k].v[j] = from_f<T>(0.f);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k * G + lane >= packs) continue;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = to_f(dy[r][k].v[j]), xhat = ((to_f(x[r][k].v[j]) - x0[r]) - shift[r]) * rstd[r];
                    const float g = d * w[k][j];
                    s[2 * r] += g;
                    s[2 * r + 1] = fmaf(g, xhat, s[2 * r + 1]);
                    dw[k][j] = fmaf(d, xhat, dw[k][j]);
                    db[k][j] += d;
                }
            }
        }
        if (a.dx) {  // (the same for every thread)
            group_sum<G, 2 * R>(s, s_red, turn);
            turn ^= 1;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (row0 + r >= a.rows) continue;
                const float m1 = s[2 * r] * inv_d, m2 = s[2 * r + 1] * inv_d;
                T* out = static_cast<T*>(a.dx) + (row0 + r) * a.D;
#pragma unroll
                for (int k = 0; k < ITEMS; ++k) {
                    const int p = k * G + lane;
                    if (p >= packs) continue;
                    Pack<T, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float xhat = ((to_f(x[r][k].v[j]) - x0[r]) - shift[r]) * rstd[r];
                        o.v[j] = from_f<T>(rstd[r] * (to_f(dy[r][k].v[j]) * w[k][j] - m1 - xhat * m2));
                    }
                    reinterpret_cast<Pack<T, V>*>(out)[p] = o;
                }
            }
        }
    }

    if (!a.dw && !a.db) return;
    float* part = a.part + (long long)blockIdx.x * 2 * a.D;
    if constexpr (GROUPS > 1) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s_cols[(group * 2) * COLS + (k * G + lane) * V + j] = dw[k][j];
                s_cols[(group * 2 + 1) * COLS + (k * G + lane) * V + j] = db[k][j];
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * COLS; i += norm_block(G)) {
            const int which = i / COLS, c = i % COLS;
            float t = 0.f;
            for (int g = 0; g < GROUPS; ++g) t += s_cols[(g * 2 + which) * COLS + c];
            if (c < a.D) part[which * a.D + c] = t;
        }
    } else {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int p = k * G + lane;
            if (p >= packs) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                part[(long long)p * V + j] = dw[k][j];
                part[a.D + (long long)p * V + j] = db[k][j];
            }
        }
    }
}

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

// The partial sums of all splits: every 16th by one thread, then the 16 in order.  Block 32 x 16:
// 32 of the 2 D sums.
constexpr int LN_FINISH_ROWS = 16;
template <typename W>
__global__ void __launch_bounds__(32 * LN_FINISH_ROWS) layer_norm_finish_kernel(NormGradArgs a) {
    __shared__ float s_sum[LN_FINISH_ROWS][32];
    const long long i = (long long)blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (i < 2 * a.D) {
#pragma unroll 8
        for (int p = threadIdx.y; p < a.splits; p += LN_FINISH_ROWS) s += a.part[(long long)p * 2 * a.D + i];
    }
    s_sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y || i >= 2 * a.D) return;
#pragma unroll
    for (int k = 1; k < LN_FINISH_ROWS; ++k) s += s_sum[k][threadIdx.x];
    if (i < a.D) {
        if (a.dw) static_cast<W*>(a.dw)[i] = from_f<W>(s);
    } else if (a.db) {
        static_cast<W*>(a.db)[i - a.D] = from_f<W>(s);
    }
}

// The most partial sums a call writes, a pure function of the sizes and the device (which path
// runs also depends on alignment): about 8192 columns' worth of blocks on an SM.
static int norm_splits(long long rows, long long D, int sms) {
    long long per_sm = 8192 / D;
    per_sm = per_sm < 2 ? 2 : per_sm > 8 ? 8 : per_sm;
    const long long most = per_sm * sms;
    return (int)(rows < most ? rows : most);
}

// Calls f(G, ITEMS) with the narrowest group of up to MOST_G threads that holds `packs` packs of V
// values, up to MOST values a thread; false when none does.
template <int N>
struct Int {
    static constexpr int value = N;
};
template <int V, int MOST, int MOST_G, typename F>
static bool with_group(long long packs, F&& f) {
    constexpr int I = MOST / V, H = (I + 1) / 2;  // packs a thread, half of them
    if (packs <= 8) f(Int<8>{}, Int<1>{});
    else if (packs <= 32) f(Int<32>{}, Int<1>{});
    else if (packs <= 128 * H) f(Int<128>{}, Int<H>{});
    else if (packs <= 128 * I) f(Int<128>{}, Int<I>{});
    else if (packs <= 256 * I) f(Int<256>{}, Int<I>{});
    else if (packs <= 512 * I) f(Int<512>{}, Int<I>{});
    else if constexpr (MOST_G > 512) {
        if (packs > 1024 * I) return false;
        f(Int<1024>{}, Int<I>{});
    } else return false;
    return true;
}

static int norm_args_ok(long long rows, long long D, long long row_stride, int dtype, int wdtype) {
    if (rows < 0 || D < 1 || row_stride < 0) return IGS_ERR_ARG;
    if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != IGS_F32)) return IGS_ERR_ARG;
    if (D > (1ll << 30)) return IGS_ERR_LIMIT;
    return IGS_OK;
}

// Whether packs of `bytes` can be moved: every row of x, y (dy, dx) and the weights start on one.
static bool packs_fit(const void* x, const void* y, const void* w, const void* b, long long D, long long row_stride,
                      size_t tsize, size_t wsize, size_t bytes) {
    const size_t wbytes = bytes / tsize * wsize < 16 ? bytes / tsize * wsize : 16;
    return aligned_to(x, bytes) && aligned_to(y, bytes) && aligned_to(w, wbytes) && aligned_to(b, wbytes) &&
           (size_t)D * tsize % bytes == 0 && (size_t)row_stride * tsize % bytes == 0;
}

static unsigned row_grid(long long rows) { return (unsigned)(rows < (1ll << 30) ? rows : (1ll << 30)); }

template <typename T, typename W, int V>
static bool launch_norm_packs(const NormArgs& a, cudaStream_t s) {
    return with_group<V, V == 1 ? 8 : 32, 1024>(a.D / V, [&](auto g, auto items) {
        constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value, R = ITEMS * V <= 16 ? 2 : 1;
        constexpr int PER = norm_block(G) / G * R;
        layer_norm_kernel<T, W, V, G, ITEMS, R><<<row_grid((a.rows + PER - 1) / PER), norm_block(G), 0, s>>>(a);
    });
}

template <typename T, typename W>
static void launch_norm(const NormArgs& a, cudaStream_t s) {
    bool done = false;
    if (packs_fit(a.x, a.y, a.w, a.b, a.D, a.row_stride, sizeof(T), sizeof(W), 16))
        done = launch_norm_packs<T, W, 16 / sizeof(T)>(a, s);
    else
        done = launch_norm_packs<T, W, 1>(a, s);
    if (!done) layer_norm_any_kernel<T, W><<<row_grid(a.rows), LN_THREADS, 0, s>>>(a);
}

// `a.splits` comes in as the most blocks and goes out as the blocks that wrote partial sums
template <typename T, typename W, int V>
static bool launch_norm_grad_packs(NormGradArgs& a, cudaStream_t s) {
    return with_group<V, V == 1 ? 8 : 16, 512>(a.D / V, [&](auto g, auto items) {
        constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value;
        constexpr int R = (G <= 128 ? 2 : 1) * (ITEMS * V <= 8 && G > 32 && G < 512 ? 2 : 1);  // rows that fit the registers
        constexpr int PER = norm_block(G) / G * R;
        const long long batches = (a.rows + PER - 1) / PER;
        if (batches < a.splits) a.splits = (int)batches;
        layer_norm_grad_kernel<T, W, V, G, ITEMS, R><<<a.splits, norm_block(G), 0, s>>>(a);
    });
}

template <typename T, typename W>
static void launch_norm_grad(NormGradArgs& a, cudaStream_t s) {
    bool done = false;
    // (a gradient that is not wanted has no address: nothing is stored, any alignment fits)
    if (packs_fit(a.x, a.dy, a.w, nullptr, a.D, a.row_stride, sizeof(T), sizeof(W), 16) && aligned_to(a.dx, 16))
        done = launch_norm_grad_packs<T, W, 16 / sizeof(T)>(a, s);
    else
        done = launch_norm_grad_packs<T, W, 1>(a, s);
    if (done) {
        count_launch();
    } else {
        if (a.dx) {
            layer_norm_dx_any_kernel<T, W><<<row_grid(a.rows), LN_THREADS, 0, s>>>(a);
            count_launch();
        }
        if (a.dw || a.db) {
            const dim3 grid((unsigned)((a.D + 31) / 32), (unsigned)a.splits);
            layer_norm_columns_kernel<T><<<grid, dim3(32, LN_COL_ROWS), 0, s>>>(a);
            count_launch();
        }
    }
    if (a.dw || a.db) {
        layer_norm_finish_kernel<W><<<(unsigned)((2 * a.D + 31) / 32), dim3(32, LN_FINISH_ROWS), 0, s>>>(a);
        count_launch();
    }
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

extern "C" size_t igs_layer_norm_grad_workspace_bytes(long long rows, long long D, int device) {
    if (rows <= 0 || D <= 0) return 256;
    return align_up((size_t)norm_splits(rows, D, sm_count(device)) * 2 * (size_t)D * sizeof(float), 256);
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
    if (rows > 0 && columns && (!workspace || workspace_bytes < igs_layer_norm_grad_workspace_bytes(rows, D, device)))
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
    if (!dx && !columns) return IGS_OK;
    NormGradArgs a{dy, x, weight, shift, rstd, dx, dweight, dbias, static_cast<float*>(workspace), rows, D, row_stride,
                   norm_splits(rows, D, sm_count(device))};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (wdtype == dtype) launch_norm_grad<T, T>(a, s);
        else launch_norm_grad<T, float>(a, s);
        return 0;
    });
    return (int)cudaGetLastError();
}
