// igs_layer_norm, and in layer_norm_grad.cu its gradient, over rows of D values (one feature vector a row).
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  xhat = (x - mean) rstd
//   y    = xhat w + b
//   g    = dy w,  dx = rstd (g - sum g / D - xhat sum(g xhat) / D)
//   dw   = sum over rows of dy xhat,  db = sum over rows of dy
//
// All of it in 32 bits, one rounding per result, in two passes over a row's registers.  The first finds
// a pivot, the mean up to rounding: x[0] plus the mean of x - x[0], which is x[0] itself in a constant
// row.  The second sums c = x - pivot and c^2 together: mean = pivot + shift with shift = sum c / D, and
// var = sum c^2 / D - shift^2.  Whatever the pivot's rounding was is in c and so in shift: rows far from
// zero, and rows whose first value lies far from the others, keep what 32 bits can hold of their values'
// distances from the mean, and a constant row has variance 0 exactly.  (With x - x[0] in place of x - pivot
// in the second pass, the first pass's differences kept, N(0,1) rows whose first value is 1000 had a
// relative error of 2e-5 in the others; now 1e-7.)
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
    RowStats* stats;  // NULL, or [rows]
    long long rows, D, row_stride;
    float eps;
};

// Few rows, where latency counts: every row has its own group of G threads, ITEMS packs of V values a
// thread, held in registers between its one read and its one write.
template <typename T, typename W, int V, int G, int ITEMS>
__global__ void __launch_bounds__(norm_block(G)) layer_norm_kernel(NormArgs a) {
    __shared__ __align__(16) float s_red[G > 32 ? 2 * (G / 32) * 2 : 1];
    const int lane = threadIdx.x % G;
    const float inv_d = 1.f / (float)a.D;
    const int packs = (int)(a.D / V);
    const long long row = (long long)blockIdx.x * (norm_block(G) / G) + threadIdx.x / G;
    // (a group past the last row stays to take part in its warp's sums)
    const int mine = row < a.rows ? packs - lane : 0;  // item k is there when k G < mine

    const T* src = static_cast<const T*>(a.x) + row * a.row_stride;
    const float x0 = row < a.rows ? to_f(src[0]) : 0.f;
    Pack<T, V> x[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k * G < mine) x[k] = reinterpret_cast<const Pack<T, V>*>(src)[k * G + lane];

    Vals<V> d[ITEMS], sum = splat<V>(0.f);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        if (k * G >= mine) continue;
        d[k] = to_vals<T, V>(x[k]);
        sum = add(sum, sub(d[k], splat<V>(x0)));
    }
    float first[1] = {total(sum)};
    group_sum<G, 1>(first, s_red, 0);
    const float pivot = fmaf(first[0], inv_d, x0);
    Vals<V> sq = splat<V>(0.f);
    sum = splat<V>(0.f);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        if (k * G >= mine) continue;
        d[k] = sub(d[k], splat<V>(pivot));
        sum = add(sum, d[k]);
        sq = fma(d[k], d[k], sq);
    }
    float both[2] = {total(sum), total(sq)};
    group_sum<G, 2>(both, s_red, 1);
    const float shift = both[0] * inv_d, rstd = inverse_deviation(both[1] * inv_d, shift, a.eps);
    if (mine <= 0) return;
    if (lane == 0 && a.stats) a.stats[row] = RowStats{pivot, shift, rstd, 0.f};
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        if (k * G >= mine) continue;
        const int p = k * G + lane;
        const Vals<V> w = load_weights<W, V>(a.w, p, 1.f), b = load_weights<W, V>(a.b, p, 0.f);
        reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.y) + row * a.D)[p] =
            to_pack<T, V>(fma(fma(d[k], splat<V>(rstd), splat<V>(-shift * rstd)), w, b));
    }
}

// Many rows: blocks stay and rows stream by, R at a time a group, so that the weights are read from
// memory once a block, and each thread copies its packs of the next batches to shared memory of its own
// ahead of time (cp.async), so that memory does not wait for a row's sums.  Bound by memory: 65536
// rows of 1024 bf16 take 46 us, a copy of them 43 (one group of registers a row, its weights read from L1
// each time: 57, that pipe 96 % busy).
template <typename T, typename W, int V, int G, int ITEMS, int FULL, int R>
__global__ void __launch_bounds__(norm_block(G), norm_blocks(G)) layer_norm_stream_kernel(NormArgs a) {
    constexpr int BLOCK = norm_block(G), GROUPS = BLOCK / G, PACK = sizeof(Pack<T, V>);
    constexpr bool ASYNC = norm_async<T, V>;
    constexpr int STAGES = norm_stages<T, V>(ITEMS * R, BLOCK);
    extern __shared__ __align__(16) unsigned char s_mem[];
    __shared__ __align__(16) float s_red[G > 32 ? 2 * (G / 32) * 2 * R : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_d = 1.f / (float)a.D;
    const int packs = (int)(a.D / V), mine = packs - lane;  // (item k is there when k G < mine)
    const long long step = (long long)gridDim.x * (GROUPS * R);

    // shared memory: the ring, slot [stage][row][item][thread]; then weights and biases
    Pack<T, V>* ring = reinterpret_cast<Pack<T, V>*>(s_mem) + threadIdx.x;
    const auto slot = [&](int stage, int r, int k) { return ring + ((stage * R + r) * ITEMS + k) * BLOCK; };
    float* s_w = reinterpret_cast<float*>(s_mem + (ASYNC ? STAGES * R * ITEMS * BLOCK * PACK : 0));
    float* s_b = s_w + a.D;

    // (addresses advance by a fixed number of bytes: this thread's first pack of a batch's first row)
    const long long first = (long long)blockIdx.x * (GROUPS * R) + group * R;
    const long long x_row = a.row_stride * (long long)sizeof(T), y_row = a.D * (long long)sizeof(T);
    const char* ahead = static_cast<const char*>(a.x) + first * x_row + lane * PACK;
    const char* firsts = static_cast<const char*>(a.x) + first * x_row;
    char* out = static_cast<char*>(a.y) + first * y_row + lane * PACK;
    const char* now = ahead;  // (used where nothing is copied ahead)
    // A group makes `steps` steps, the last with `tail` rows (none or fewer, where narrow groups share a
    // warp).  A warp goes on while it has a row; narrower groups share one and go on together, a wider
    // group is the block: barriers and exchanges are met by all of their threads.
    const long long ours = a.rows - (G == 32 ? first : first - group * R);
    const int steps = ours > 0 ? (int)((ours + step - 1) / step) : 0;
    const int tail = (int)(a.rows - first - (steps - 1) * step < R ? a.rows - first - (steps - 1) * step : R);
    RowStats* stats = a.stats ? a.stats + first : nullptr;
    int fetched = 0;
    const auto fetch = [&](int stage) {
        const int n = fetched < steps - 1 ? R : fetched == steps - 1 ? tail : 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= n) break;
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
                if (k < FULL || k * G < mine) copy_async<PACK>(slot(stage, r, k), ahead + r * x_row + k * (G * PACK));
        }
        ahead += step * x_row;
        ++fetched;
    };
    if constexpr (ASYNC) {
#pragma unroll
        for (int q = 0; q < STAGES - 1; ++q) {
            fetch(q);
            copy_commit();
        }
    }
    stage_weights<W, V>(s_w, a.w, 1.f, (int)a.D, packs, BLOCK);
    stage_weights<W, V>(s_b, a.b, 0.f, (int)a.D, packs, BLOCK);
    // A row's first value: lane 0 holds it; in groups wider than a warp it is loaded one batch ahead.
    float next[R];
    const auto fetch_first = [&](int i) {
        if constexpr (G > 32) {
            const int n = i < steps - 1 ? R : i == steps - 1 ? tail : 0;
#pragma unroll
            for (int r = 0; r < R; ++r) next[r] = r < n ? to_f(*reinterpret_cast<const T*>(firsts + r * x_row)) : 0.f;
            firsts += step * x_row;
        }
    };
    fetch_first(0);
    __syncthreads();

    int stage = 0;
    for (int i = 0; i < steps; ++i) {
        const int left = i < steps - 1 ? R : tail;
        Vals<V> d[R][ITEMS];
        float x0[R], pivot[R], both[2 * R];
        if constexpr (ASYNC) {
            fetch(stage == 0 ? STAGES - 1 : stage - 1);
            copy_commit();
            copy_wait<STAGES - 1>();
        }
        // (rows past the last are computed on whatever the ring holds, and not stored)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Pack<T, V> x[ITEMS];
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k >= FULL && k * G >= mine) continue;
                if constexpr (ASYNC) x[k] = *slot(stage, r, k);
                else if (r < left) x[k] = *reinterpret_cast<const Pack<T, V>*>(now + r * x_row + k * (G * PACK));
            }
            if constexpr (G > 32) x0[r] = next[r];
            else x0[r] = __shfl_sync(0xffffffffu, to_f(x[0].v[0]), 0, G);
            Vals<V> sum = splat<V>(0.f);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k >= FULL && k * G >= mine) continue;
                d[r][k] = to_vals<T, V>(x[k]);
                sum = add(sum, sub(d[r][k], splat<V>(x0[r])));
            }
            pivot[r] = total(sum);
        }
        now += step * x_row;
        fetch_first(i + 1);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        group_sum<G, R>(pivot, s_red, 0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            pivot[r] = fmaf(pivot[r], inv_d, x0[r]);
            Vals<V> sum = splat<V>(0.f), sq = splat<V>(0.f);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (k >= FULL && k * G >= mine) continue;
                d[r][k] = sub(d[r][k], splat<V>(pivot[r]));
                sum = add(sum, d[r][k]);
                sq = fma(d[r][k], d[r][k], sq);
            }
            both[2 * r] = total(sum);
            both[2 * r + 1] = total(sq);
        }
        group_sum<G, 2 * R>(both, s_red, 1);
        float rstd[R], offset[R];  // xhat = d rstd + offset
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float shift = both[2 * r] * inv_d;
            rstd[r] = inverse_deviation(both[2 * r + 1] * inv_d, shift, a.eps);
            offset[r] = -shift * rstd[r];
            if (lane == 0 && stats && r < left) stats[r] = RowStats{pivot[r], shift, rstd[r], 0.f};
        }
        if (stats) stats += step;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if (k >= FULL && k * G >= mine) continue;
            const Vals<V> w = staged_weights<V>(s_w, k * G + lane, packs), b = staged_weights<V>(s_b, k * G + lane, packs);
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < left)
                    *reinterpret_cast<Pack<T, V>*>(out + r * y_row + k * (G * PACK)) =
                        to_pack<T, V>(fma(fma(d[r][k], splat<V>(rstd[r]), splat<V>(offset[r])), w, b));
        }
        out += step * y_row;
    }
    if constexpr (ASYNC) copy_wait<0>();
}

// Rows of any width: one CTA per row, the row read three times (from L2 after the first), eight CTAs an
// SM to have enough of them on their way (1024 rows of 20000 fp32: 68 us, with six 92).
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS, 8) layer_norm_any_kernel(NormArgs a) {
    __shared__ __align__(16) float s_red[LN_RED];
    const W* w = static_cast<const W*>(a.w);
    const W* b = static_cast<const W*>(a.b);
    const float inv_d = 1.f / (float)a.D;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.row_stride;
        T* y = static_cast<T*>(a.y) + r * a.D;
        const float x0 = to_f(x[0]);
        float sum = 0.f;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) sum += to_f(x[c]) - x0;
        const float pivot = fmaf(block_sum_all(sum, s_red, 0), inv_d, x0);
        float sum_d = 0.f, sum_sq = 0.f;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float d = to_f(x[c]) - pivot;
            sum_d += d;
            sum_sq = fmaf(d, d, sum_sq);
        }
        float both[2] = {sum_d, sum_sq};
        group_sum<LN_THREADS, 2>(both, s_red, 1);
        const float shift = both[0] * inv_d, rstd = inverse_deviation(both[1] * inv_d, shift, a.eps), offset = -shift * rstd;
        for (long long c = threadIdx.x; c < a.D; c += LN_THREADS) {
            const float xhat = fmaf(to_f(x[c]) - pivot, rstd, offset);
            y[c] = from_f<T>(fmaf(xhat, w ? to_f(w[c]) : 1.f, b ? to_f(b[c]) : 0.f));
        }
        if (threadIdx.x == 0 && a.stats) a.stats[r] = RowStats{pivot, shift, rstd, 0.f};
    }
}

// Calls f(G, ITEMS) with the narrowest group of threads that holds `packs` packs of V values, false when
// none does: at most 16 values a thread, up to 1024 threads.
template <int V, typename F>
static bool with_norm_group(long long packs, F&& f) {
    constexpr int I = 16 / V, H = (I + 1) / 2;  // packs a thread, half of them
    if (packs <= 8) f(Int<8>{}, Int<1>{});
    else if (packs <= 32) f(Int<32>{}, Int<1>{});
    else if (packs <= 128 * H) f(Int<128>{}, Int<H>{});
    else if (packs <= 256 * H) f(Int<256>{}, Int<H>{});
    else if (packs <= 512 * H) f(Int<512>{}, Int<H>{});
    else if (packs <= 512 * I) f(Int<512>{}, Int<I>{});
    else if (packs <= 1024 * I) f(Int<1024>{}, Int<I>{});
    else return false;
    return true;
}

template <typename T, typename W, int V>
static bool launch_norm_packs(const NormArgs& a, int device, cudaStream_t s) {
    // Rows stream once every SM has several to keep its blocks busy; below, one group a row answers sooner
    // (128 x 1024 fp32: 2.5 us, half of what streaming took).
    if (a.rows >= 8ll * sm_count(device)) {
        const bool done = with_stream_group<T, V>(a.D / V, [&](auto g, auto items, auto full) {
            constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value, FULL = decltype(full)::value;
            constexpr int R = G >= 256 ? 2 : ITEMS * V <= 16 ? 4 : 2;  // 64 values a thread (few spill)
            constexpr int BLOCK = norm_block(G), PER = BLOCK / G * R;
            constexpr size_t ring = norm_async<T, V> ? sizeof(Pack<T, V>) * norm_stages<T, V>(ITEMS * R, BLOCK) * R * ITEMS * BLOCK : 0;
            constexpr size_t most = ring + (size_t)BLOCK / (BLOCK / G) * ITEMS * V * 2 * sizeof(float);  // (of the widest row)
            static int cached[64];
            const auto kernel = layer_norm_stream_kernel<T, W, V, G, ITEMS, FULL, R>;
            const long long resident = (long long)blocks_per_sm(kernel, BLOCK, most, device, cached) * sm_count(device);
            const long long batches = (a.rows + PER - 1) / PER;
            kernel<<<(unsigned)(batches < resident ? batches : resident), BLOCK, ring + (size_t)a.D * 2 * sizeof(float), s>>>(a);
        });
        if (done) return true;
    }
    return with_norm_group<V>(a.D / V, [&](auto g, auto items) {
        constexpr int G = decltype(g)::value, ITEMS = decltype(items)::value, PER = norm_block(G) / G;
        layer_norm_kernel<T, W, V, G, ITEMS><<<row_grid((a.rows + PER - 1) / PER), norm_block(G), 0, s>>>(a);
    });
}

template <typename T, typename W>
static void launch_norm(const NormArgs& a, int device, cudaStream_t s) {
    const int bytes = norm_pack_bytes(a.x, a.y, nullptr, a.w, a.b, a.D, a.row_stride, sizeof(T), sizeof(W));
    bool done = false;
    if (bytes == 16) done = launch_norm_packs<T, W, 16 / sizeof(T)>(a, device, s);
    else if (bytes == 4) done = launch_norm_packs<T, W, 4 / sizeof(T)>(a, device, s);
    else done = launch_norm_packs<T, W, 1>(a, device, s);
    if (!done) layer_norm_any_kernel<T, W><<<row_grid(a.rows), LN_THREADS, 0, s>>>(a);
}

}  // namespace igs

using namespace igs;

extern "C" int igs_layer_norm(const void* x, int dtype, long long rows, long long D, long long row_stride,
                              const void* weight, const void* bias, int wdtype, float eps, void* y, float* stats,
                              int device, void* stream) {
    const int rc = norm_args_ok(rows, D, row_stride, dtype, wdtype);
    if (rc) return rc;
    if (!(eps >= 0.f) || !aligned_to(stats, 16)) return IGS_ERR_ARG;
    if (rows == 0) return IGS_OK;
    if (!x || !y) return IGS_ERR_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    NormArgs a{x, weight, bias, y, reinterpret_cast<RowStats*>(stats), rows, D, row_stride, eps};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (wdtype == dtype) launch_norm<T, T>(a, device, s);
        else launch_norm<T, float>(a, device, s);
        return 0;
    });
    count_launch();
    return (int)cudaGetLastError();
}
