// igs_layer_norm_grad; the formulas are in layer_norm.cu.
//
// One pass over x and dy: a block keeps the sums of its columns in registers while rows stream by,
// so that dx, dw and db cost one read of each input.  What bounds it is memory: three passes over
// [rows, D] (x, dy, dx), about 13 instructions a value.  A row's two sums need every thread of its
// group between its loads and its stores; so that memory does not wait for them, each thread copies
// its packs of the next rows to shared memory of its own ahead of time (cp.async; no thread reads
// another's, no barrier is needed for it).
#include "layer_norm.cuh"

namespace igs {

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


// What a thread copies ahead: PACK bytes of 4 or 16.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// 16-bit values one by one cannot be copied that way.
template <typename T, int V>
constexpr bool norm_async = sizeof(Pack<T, V>) >= 4;
// Batches of R rows in the ring, the one being worked on included: as many as fit 384 bytes a thread,
// two to four.
template <typename T, int V>
__host__ __device__ constexpr int norm_stages(int items, int r) {
    const int n = 384 / (int)(sizeof(Pack<T, V>) * 2 * items * r);
    return n < 2 ? 2 : n > 4 ? 4 : n;
}

// Block b takes the batches b, b + gridDim.x, ... of GROUPS * R rows; ITEMS packs of V values a thread,
// the same columns in every row.  Its groups' column sums are added in order at the end and written
// as partial b.
template <typename T, typename W, int V, int G, int ITEMS, int R>
__global__ void __launch_bounds__(norm_block(G)) layer_norm_grad_kernel(NormGradArgs a) {
    constexpr int BLOCK = norm_block(G), GROUPS = BLOCK / G;
    constexpr int COLS = G * ITEMS * V;  // columns a group covers
    constexpr bool ASYNC = norm_async<T, V>;
    constexpr int STAGES = norm_stages<T, V>(ITEMS, R);
    extern __shared__ __align__(16) unsigned char s_mem[];
    __shared__ float s_red[G > 32 ? 2 * (G / 32) * 2 * R : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_d = 1.f / (float)a.D;
    const int packs = (int)(a.D / V);
    const long long step = (long long)gridDim.x * (GROUPS * R);

    float w[ITEMS][V], dw[ITEMS][V], db[ITEMS][V];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[k][j] = dw[k][j] = db[k][j] = 0.f;
        if (k * G + lane < packs) load_weights<W, V>(a.w, (long long)(k * G + lane) * V, 1.f, w[k]);
    }

    // slot [stage][row][x or dy][item][thread]
    Pack<T, V>* ring = reinterpret_cast<Pack<T, V>*>(s_mem) + threadIdx.x;
    const auto slot = [&](int stage, int r, int which, int k) {
        return ring + ((stage * R + r) * 2 + which) * ITEMS * BLOCK + k * BLOCK;
    };
    const auto fetch = [&](long long row0, int stage) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (row0 + r >= a.rows) continue;
            const Pack<T, V>* xs = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.x) + (row0 + r) * a.row_stride);
            const Pack<T, V>* ds = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.dy) + (row0 + r) * a.D);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k * G + lane >= packs) continue;
                copy_async<sizeof(Pack<T, V>)>(slot(stage, r, 0, k), xs + k * G + lane);
                copy_async<sizeof(Pack<T, V>)>(slot(stage, r, 1, k), ds + k * G + lane);
            }
        }
    };

    const long long first = (long long)blockIdx.x * (GROUPS * R) + group * R;
    if constexpr (ASYNC) {
#pragma unroll
        for (int q = 0; q < STAGES - 1; ++q) {
            fetch(first + q * step, q);
            copy_commit();
        }
    }
    // (the three numbers of a row are loaded one batch ahead)
    float next_x0[R], next_shift[R], next_rstd[R];
    const auto fetch_row = [&](long long row0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool ok = row0 + r < a.rows;
            next_x0[r] = ok ? to_f(static_cast<const T*>(a.x)[(row0 + r) * a.row_stride]) : 0.f;
            next_shift[r] = ok ? a.shift[row0 + r] : 0.f;
            next_rstd[r] = ok ? a.rstd[row0 + r] : 0.f;
        }
    };
    fetch_row(first);

    int turn = 0, stage = 0;
    // (every group of a block makes the same number of steps: a barrier is met by all of its threads)
    for (long long row0 = first, base = first - group * R; base < a.rows; row0 += step, base += step) {
        Pack<T, V> x[R][ITEMS], dy[R][ITEMS];
        float x0[R], shift[R], rstd[R], s[2 * R];
        if constexpr (ASYNC) {
            fetch(row0 + (STAGES - 1) * step, (stage + STAGES - 1) % STAGES);
            copy_commit();
            copy_wait<STAGES - 1>();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            x0[r] = next_x0[r];
            shift[r] = next_shift[r];
            rstd[r] = next_rstd[r];
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                const int p = k * G + lane;
                if (row0 + r < a.rows && p < packs) {
                    if constexpr (ASYNC) {
                        x[r][k] = *slot(stage, r, 0, k);
                        dy[r][k] = *slot(stage, r, 1, k);
                    } else {
                        x[r][k] = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.x) + (row0 + r) * a.row_stride)[p];
                        dy[r][k] = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.dy) + (row0 + r) * a.D)[p];
                    }
                } else {  // (a row past the last adds nothing to any sum: rstd is zero too)
#pragma unroll
                    for (int j = 0; j < V; ++j) x[r][k].v[j] = dy[r][k].v[j] = from_f<T>(0.f);
                }
            }
        }
        fetch_row(row0 + step);
        stage = (stage + 1) % STAGES;
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

    if constexpr (ASYNC) copy_wait<0>();
    if (!a.dw && !a.db) return;
    float* part = a.part + (long long)blockIdx.x * 2 * a.D;
    if constexpr (GROUPS > 1) {
        float* s_cols = reinterpret_cast<float*>(s_mem);  // [group][dw, db][columns], over the ring
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s_cols[(group * 2) * COLS + (k * G + lane) * V + j] = dw[k][j];
                s_cols[(group * 2 + 1) * COLS + (k * G + lane) * V + j] = db[k][j];
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
#pragma unroll
            for (int j = 0; j < V; ++j) {
                part[(long long)p * V + j] = dw[k][j];
                part[a.D + (long long)p * V + j] = db[k][j];
            }
        }
    }
}

// Rows of any width, first part: one CTA per row, the row read twice (from L2 the second time).
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS) layer_norm_dx_any_kernel(NormGradArgs a) {
    __shared__ float s_red[LN_RED];
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

// The partial sums of all splits: every 32nd by one thread, then the 32 in order.  Block 32 x 32:
// 32 of the 2 D sums.
constexpr int LN_FINISH_ROWS = 32;
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

// Calls f(G, ITEMS, R) with the narrowest group of threads that holds `packs` packs of V values, at most
// 16 values a thread (their weights and column sums take 48 registers); false when none does.
template <int V, typename F>
static bool with_norm_grad_group(long long packs, F&& f) {
    constexpr int I = 16 / V, H = (I + 1) / 2;  // packs a thread, half of them
    if (packs <= 8) f(Int<8>{}, Int<1>{}, Int<2>{});
    else if (packs <= 32) f(Int<32>{}, Int<1>{}, Int<2>{});
    else if (packs <= 128 * H) f(Int<128>{}, Int<H>{}, Int<2>{});
    else if (packs <= 128 * I) f(Int<128>{}, Int<I>{}, Int<2>{});
    else if (packs <= 256 * I) f(Int<256>{}, Int<I>{}, Int<1>{});
    else if (packs <= 512 * I) f(Int<512>{}, Int<I>{}, Int<1>{});
    else return false;
    return true;
}

// Blocks of a kernel that an SM holds, found once per device; the first call also allows the kernel
// its shared memory.
template <typename K>
static int blocks_per_sm(K kernel, int block, size_t smem, int device, int (&cached)[64]) {
    if (device >= 0 && device < 64 && cached[device]) return cached[device];
    int n = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, block, smem) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = 1;
    }
    if (device >= 0 && device < 64) cached[device] = n;
    return n;
}

// `a.splits` comes in as the most blocks and goes out as the blocks that wrote partial sums
template <typename T, typename W, int V>
static bool launch_norm_grad_packs(NormGradArgs& a, int device, cudaStream_t s) {
    return with_norm_grad_group<V>(a.D / V, [&](auto g, auto items, auto rr) {
        constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value, R = decltype(rr)::value;
        constexpr int BLOCK = norm_block(G), PER = BLOCK / G * R;
        constexpr size_t ring = norm_async<T, V> ? sizeof(Pack<T, V>) * norm_stages<T, V>(ITEMS, R) * R * 2 * ITEMS * BLOCK : 0;
        constexpr size_t cols = BLOCK > G ? (size_t)BLOCK * ITEMS * V * 2 * sizeof(float) : 0;
        constexpr size_t smem = ring > cols ? ring : cols;
        static int cached[64];
        const auto kernel = layer_norm_grad_kernel<T, W, V, G, ITEMS, R>;
        const long long resident = (long long)blocks_per_sm(kernel, BLOCK, smem, device, cached) * sm_count(device);
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
        layer_norm_finish_kernel<W><<<(unsigned)((2 * a.D + 31) / 32), dim3(32, LN_FINISH_ROWS), 0, s>>>(a);
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
        if (wdtype == dtype) launch_norm_grad<T, T>(a, device, s);
        else launch_norm_grad<T, float>(a, device, s);
        return 0;
    });
    return (int)cudaGetLastError();
}
