// igs_layer_norm_grad; the formulas are in layer_norm.cu.
//
// One pass over x and dy: a block keeps the sums of its columns in registers while rows stream by,
// so that dx, dw and db cost one read of each input.  What bounds it is memory: three passes over
// [rows, D] (x, dy, dx), about 13 instructions a value.  A row's two sums need every thread of its
// group between its loads and its stores; so that memory does not wait for them, each thread copies
// its packs of the next rows to shared memory of its own ahead of time (cp.async; no thread reads
// another's, no barrier is needed for it).  65536 rows of 1024 bf16: 72 us with the column sums'
// second step; the sum of two such tensors, the same traffic, takes 59.
#include "layer_norm.cuh"

namespace igs {

struct NormGradArgs {
    const void* dy;
    const void* x;
    const void* w;
    const RowStats* stats;
    void* dx;         // NULL: not wanted
    void* dw;
    void* db;
    float* part;      // [splits][2][D] partial column sums
    long long rows, D, row_stride;
    int splits;
};


// Block b takes the batches b, b + gridDim.x, ... of GROUPS * R rows; ITEMS packs of V values a thread,
// the same columns in every row.  Its groups' column sums are added in order at the end and written
// as partial b.
template <typename T, typename W, int V, int G, int ITEMS, int FULL, int R>
__global__ void __launch_bounds__(norm_block(G), norm_blocks(G)) layer_norm_grad_kernel(NormGradArgs a) {
    constexpr int BLOCK = norm_block(G), GROUPS = BLOCK / G;
    constexpr int COLS = G * ITEMS * V;  // columns a group covers
    constexpr bool ASYNC = norm_async<T, V>;
    constexpr int STAGES = norm_stages<T, V>(2 * ITEMS * R, BLOCK);
    extern __shared__ __align__(16) unsigned char s_mem[];
    __shared__ __align__(16) float s_red[G > 32 ? 2 * (G / 32) * 2 * R : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_d = 1.f / (float)a.D;
    const int packs = (int)(a.D / V), mine = packs - lane;  // (item k is there when k G < mine)
    const long long step = (long long)gridDim.x * (GROUPS * R);

    Vals<V> dw[ITEMS], db[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) dw[k] = db[k] = splat<V>(0.f);

    // shared memory: the ring, slot [stage][row][x or dy][item][thread]; then the weights
    constexpr int PACK = sizeof(Pack<T, V>);
    float* s_w = reinterpret_cast<float*>(s_mem + (ASYNC ? STAGES * R * 2 * ITEMS * BLOCK * PACK : 0));
    Pack<T, V>* ring = reinterpret_cast<Pack<T, V>*>(s_mem) + threadIdx.x;
    const auto slot = [&](int stage, int r, int which, int k) {
        return ring + ((stage * R + r) * 2 + which) * ITEMS * BLOCK + k * BLOCK;
    };
    // (addresses advance by a fixed number of bytes: this thread's first pack of a batch's first row)
    const long long first = (long long)blockIdx.x * (GROUPS * R) + group * R;
    const long long x_row = a.row_stride * (long long)sizeof(T), y_row = a.D * (long long)sizeof(T);
    const char* x_ahead = static_cast<const char*>(a.x) + first * x_row + lane * PACK;
    const char* dy_ahead = static_cast<const char*>(a.dy) + first * y_row + lane * PACK;
    const char *x_now = x_ahead, *dy_now = dy_ahead;  // (used where nothing is copied ahead)
    char* out = static_cast<char*>(a.dx) + first * y_row + lane * PACK;
    // A group makes `steps` steps, the last with `tail` rows (none or fewer, where narrow groups share a
    // warp).  A warp goes on while it has a row; narrower groups share one and go on together, a wider
    // group is the block: barriers and exchanges are met by all of their threads.
    const long long ours = a.rows - (G == 32 ? first : first - group * R);
    const int steps = ours > 0 ? (int)((ours + step - 1) / step) : 0;
    const int tail = (int)(a.rows - first - (steps - 1) * step < R ? a.rows - first - (steps - 1) * step : R);
    int fetched = 0;
    const auto fetch = [&](int stage) {
        const int n = fetched < steps - 1 ? R : fetched == steps - 1 ? tail : 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= n) break;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k >= FULL && k * G >= mine) continue;
                copy_async<PACK>(slot(stage, r, 0, k), x_ahead + r * x_row + k * (G * PACK));
                copy_async<PACK>(slot(stage, r, 1, k), dy_ahead + r * y_row + k * (G * PACK));
            }
        }
        x_ahead += step * x_row;
        dy_ahead += step * y_row;
        ++fetched;
    };
    if constexpr (ASYNC) {
#pragma unroll
        for (int q = 0; q < STAGES - 1; ++q) {
            fetch(q);
            copy_commit();
        }
    }
    // (a row's statistics are loaded one batch ahead; a row past the last has a factor of zero)
    RowStats next[R];
    const RowStats* stats = a.stats + first;
    const auto fetch_stats = [&](int i) {
        const int n = i < steps - 1 ? R : i == steps - 1 ? tail : 0;
#pragma unroll
        for (int r = 0; r < R; ++r) next[r] = r < n ? stats[r] : RowStats{0.f, 0.f, 0.f, 0.f};
        stats += step;
    };
    fetch_stats(0);
    stage_weights<W, V>(s_w, a.w, 1.f, (int)a.D, packs, BLOCK);
    __syncthreads();

    int turn = 0, stage = 0;
    for (int i = 0; i < steps; ++i) {
        const int left = i < steps - 1 ? R : tail;
        Vals<V> xh[R][ITEMS], g[R][ITEMS];  // xhat and dy w
        float rstd[R], s[2 * R];
        if constexpr (ASYNC) {
            fetch(stage == 0 ? STAGES - 1 : stage - 1);
            copy_commit();
            copy_wait<STAGES - 1>();
        }
        Vals<V> s1[R], s2[R], pivot[R], f[R], t[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            rstd[r] = next[r].rstd;
            s1[r] = s2[r] = splat<V>(0.f);
            pivot[r] = splat<V>(next[r].pivot);  // xhat = (x - pivot) rstd - shift rstd
            f[r] = splat<V>(rstd[r]);
            t[r] = splat<V>(-next[r].shift * rstd[r]);
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if (k >= FULL && k * G >= mine) continue;
            const Vals<V> w = staged_weights<V>(s_w, k * G + lane, packs);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if ((R > 1 || G < 32) && r >= left) continue;
                Pack<T, V> px, pd;
                if constexpr (ASYNC) {
                    px = *slot(stage, r, 0, k);
                    pd = *slot(stage, r, 1, k);
                } else {
                    px = *reinterpret_cast<const Pack<T, V>*>(x_now + r * x_row + k * (G * PACK));
                    pd = *reinterpret_cast<const Pack<T, V>*>(dy_now + r * y_row + k * (G * PACK));
                }
                const Vals<V> d = to_vals<T, V>(pd);
                xh[r][k] = fma(sub(to_vals<T, V>(px), pivot[r]), f[r], t[r]);
                g[r][k] = mul(d, w);
                s1[r] = add(s1[r], g[r][k]);
                s2[r] = fma(g[r][k], xh[r][k], s2[r]);
                dw[k] = fma(d, xh[r][k], dw[k]);
                db[k] = add(db[k], d);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[2 * r] = total(s1[r]);
            s[2 * r + 1] = total(s2[r]);
        }
        x_now += step * x_row;
        dy_now += step * y_row;
        fetch_stats(i + 1);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (a.dx) {  // (the same for every thread)
            group_sum<G, 2 * R>(s, s_red, turn);
            turn ^= 1;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r >= left) continue;
                // rstd (g - m1 - xhat m2)
                const Vals<V> c1 = splat<V>(-(s[2 * r] * inv_d) * rstd[r]), c2 = splat<V>(-(s[2 * r + 1] * inv_d) * rstd[r]);
#pragma unroll
                for (int k = 0; k < ITEMS; ++k) {
                    if (k >= FULL && k * G >= mine) continue;
                    *reinterpret_cast<Pack<T, V>*>(out + r * y_row + k * (G * PACK)) =
                        to_pack<T, V>(fma(xh[r][k], c2, fma(g[r][k], f[r], c1)));
                }
            }
            out += step * y_row;
        }
    }

    if constexpr (ASYNC) copy_wait<0>();
    let_next_start();
    if (!a.dw && !a.db) return;
    float* part = a.part + (long long)blockIdx.x * 2 * a.D;
    if constexpr (GROUPS > 1) {
        float* s_cols = reinterpret_cast<float*>(s_mem);  // [group][dw, db][columns], over the ring
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const Pack<float, V> pw = to_pack<float, V>(dw[k]), pb = to_pack<float, V>(db[k]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s_cols[(group * 2) * COLS + (k * G + lane) * V + j] = pw.v[j];
                s_cols[(group * 2 + 1) * COLS + (k * G + lane) * V + j] = pb.v[j];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * COLS; i += BLOCK) {
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
            // (D is a multiple of V: whole packs of up to 16 bytes)
            reinterpret_cast<Pack<float, V>*>(part)[p] = to_pack<float, V>(dw[k]);
            reinterpret_cast<Pack<float, V>*>(part + a.D)[p] = to_pack<float, V>(db[k]);
        }
    }
}

// Rows of any width, first part: one CTA per row, the row read twice (from L2 the second time).
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_dx_any_kernel(NormGradArgs a) {
    __shared__ __align__(16) float s_red[LN_RED];
    const W* w = static_cast<const W*>(a.w);
    const float inv_d = 1.f / (float)a.D;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.row_stride;
        const T* dy = static_cast<const T*>(a.dy) + r * a.D;
        T* dx = static_cast<T*>(a.dx) + r * a.D;
        const RowStats st = a.stats[r];
        float s1 = 0.f, s2 = 0.f;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.f);
            s1 += g;
            s2 = fmaf(g, ((to_f(x[c]) - st.pivot) - st.shift) * st.rstd, s2);
        }
        const float m1 = block_sum_all(s1, s_red, 0) * inv_d;
        const float m2 = block_sum_all(s2, s_red, 1) * inv_d;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.f);
            dx[c] = from_f<T>(st.rstd * (g - m1 - ((to_f(x[c]) - st.pivot) - st.shift) * st.rstd * m2));
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
            const RowStats st = a.stats[r];
            sw = fmaf(dy, ((to_f(static_cast<const T*>(a.x)[r * a.row_stride + c]) - st.pivot) - st.shift) * st.rstd, sw);
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

// The partial sums of all splits: every 32nd by one thread, then the 32 in order.  Block 32 x 32:
// 32 of the 2 D sums.
constexpr int LN_FINISH_ROWS = 32;
template <typename W>
__global__ void __launch_bounds__(32 * LN_FINISH_ROWS) layer_norm_finish_kernel(NormGradArgs a) {
    __shared__ float s_sum[LN_FINISH_ROWS][32];
    const long long i = (long long)blockIdx.x * 32 + threadIdx.x;
    wait_for_previous();
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

// `a.splits` comes in as the most blocks and goes out as the blocks that wrote partial sums
template <typename T, typename W, int V>
static bool launch_norm_grad_packs(NormGradArgs& a, int device, cudaStream_t s) {
    return with_stream_group<T, V>(a.D / V, [&](auto g, auto items, auto full) {
        constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value, FULL = decltype(full)::value;
        constexpr int R = G >= 512 ? 1 : ITEMS * V <= 8 ? 4 : ITEMS * V <= 16 ? 2 : 1;
        // (64 values a thread, xhat and dy w; a fifth of the instances, all of 16-bit types, spill up to
        // 152 bytes of them)
        constexpr int BLOCK = norm_block(G), PER = BLOCK / G * R;
        constexpr size_t ring = norm_async<T, V> ? sizeof(Pack<T, V>) * norm_stages<T, V>(2 * ITEMS * R, BLOCK) * R * 2 * ITEMS * BLOCK : 0;
        constexpr size_t cols = BLOCK > G ? (size_t)BLOCK * ITEMS * V * 2 * sizeof(float) : 0;
        constexpr size_t widest = ring + (size_t)G * ITEMS * V * sizeof(float), most = widest > cols ? widest : cols;
        const size_t used = ring + (size_t)a.D * sizeof(float), smem = used > cols ? used : cols;
        static int cached[64];
        const auto kernel = layer_norm_grad_kernel<T, W, V, G, ITEMS, FULL, R>;
        const long long resident = (long long)blocks_per_sm(kernel, BLOCK, most, device, cached) * sm_count(device);
        const long long batches = (a.rows + PER - 1) / PER;
        if (resident < a.splits) a.splits = (int)resident;
        if (batches < a.splits) a.splits = (int)batches;
        kernel<<<a.splits, BLOCK, smem, s>>>(a);
    });
}

template <typename T, typename W>
static void launch_norm_grad(NormGradArgs& a, int device, cudaStream_t s) {
    const int bytes = norm_pack_bytes(a.x, a.dy, a.dx, a.w, nullptr, a.D, a.row_stride, sizeof(T), sizeof(W));
    bool done = false;
    if (bytes == 16) done = launch_norm_grad_packs<T, W, 16 / sizeof(T)>(a, device, s);
    else if (bytes == 4) done = launch_norm_grad_packs<T, W, 4 / sizeof(T)>(a, device, s);
    else done = launch_norm_grad_packs<T, W, 1>(a, device, s);
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
        launch_chained(layer_norm_finish_kernel<W>, (unsigned)((2 * a.D + 31) / 32), dim3(32, LN_FINISH_ROWS), 0, s, a);
        count_launch();
    }
}

}  // namespace igs

using namespace igs;

extern "C" size_t igs_layer_norm_grad_workspace_bytes(long long rows, long long D, int device) {
    if (rows <= 0 || D <= 0) return 256;
    return align_up((size_t)norm_splits(rows, D, sm_count(device)) * 2 * (size_t)D * sizeof(float), 256);
}

extern "C" int igs_layer_norm_grad(const void* dy, const void* x, int dtype, long long rows, long long D,
                                   long long row_stride, const void* weight, int wdtype, const float* stats,
                                   void* dx, void* dweight, void* dbias, void* workspace,
                                   size_t workspace_bytes, int device, void* stream) {
    const int rc = norm_args_ok(rows, D, row_stride, dtype, wdtype);
    if (rc) return rc;
    const size_t wsize = dtype_size(wdtype);
    if (rows > 0 && (!dy || !x || !stats || !aligned_to(stats, 16))) return IGS_ERR_ARG;
    const bool columns = dweight || dbias;
    if (rows > 0 && columns &&
        (!workspace || !aligned_to(workspace, 16) || workspace_bytes < igs_layer_norm_grad_workspace_bytes(rows, D, device)))
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
    NormGradArgs a{dy, x, weight, reinterpret_cast<const RowStats*>(stats), dx, dweight, dbias, static_cast<float*>(workspace), rows, D, row_stride,
                   norm_splits(rows, D, sm_count(device))};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (wdtype == dtype) launch_norm_grad<T, T>(a, device, s);
        else launch_norm_grad<T, float>(a, device, s);
        return 0;
    });
    return (int)cudaGetLastError();
}
