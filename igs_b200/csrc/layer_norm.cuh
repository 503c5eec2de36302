// Shared by layer_norm.cu and layer_norm_grad.cu: how a row is given to threads, and sums over them.
#pragma once

#include "feature.cuh"

namespace igs {

// What the gradient needs of a row, one 16-byte load: its pivot, mean - pivot, rstd.
struct alignas(16) RowStats {
    float pivot, shift, rstd, unused;
};

// 1 / sqrt(var + eps) from the mean of the squared distances from the pivot and the mean's own distance
// `shift` from it.  The subtraction takes off at most half in rows that the type can tell from constant
// ones; it is a fused one, so that an infinite mean square stays what it is.  (NaN passes the comparison.)
__device__ __forceinline__ float inverse_deviation(float mean_square, float shift, float eps) {
    const float var = fmaf(-shift, shift, mean_square);
    return rsqrtf((var < 0.f ? 0.f : var) + eps);
}

// V weights; without any, the value they stand for
template <typename W, int V>
__device__ __forceinline__ Vals<V> load_weights(const void* w, int pack, float none) {
    if (!w) return splat<V>(none);
    // (a pack may be longer than the 16 bytes that one load moves)
    return to_vals<W, V>(static_cast<const Pack<W, V>*>(w)[pack]);
}

__host__ __device__ constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// N sums (a power of two, at most 32) over the G threads of a row's group at once, the same bits in
// every one of them.  Groups of up to a warp are lanes of one warp; a wider group is the whole
// block, and s_red (on a 16-byte boundary; two halves used in turn, so that one barrier a call suffices)
// holds N floats per warp.  Within a warp the first log2 N steps halve the number of sums a lane carries: N - 1
// exchanges and 5 - log2 N more, instead of 5 N.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* s_red, int turn) {
    if constexpr (G < 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int d = G / 2; d > 0; d >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
        }
    } else {
        const int lane = threadIdx.x & 31;
        int d = 16;
#pragma unroll
        for (int n = N; n > 1; n >>= 1, d >>= 1) {
            const bool upper = lane & d;
#pragma unroll
            for (int i = 0; i < n / 2; ++i) {
                const float keep = upper ? v[i + n / 2] : v[i], send = upper ? v[i] : v[i + n / 2];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
            }
        }
#pragma unroll
        for (; d > 0; d >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
        constexpr int SHIFT = 5 - log2_of(N);  // lane l now holds sum l >> SHIFT
        if constexpr (G == 32) {
            const float mine = v[0];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, mine, i << SHIFT);
        } else {
            constexpr int WARPS = G / 32;
            float* red = s_red + turn * (WARPS * N);
            if ((lane & ((1 << SHIFT) - 1)) == 0) red[(threadIdx.x >> 5) * N + (lane >> SHIFT)] = v[0];
            __syncthreads();
            constexpr int Q = N < 4 ? N : 4;  // sums that one load reads
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
#pragma unroll
                for (int q = 0; q < N / Q; ++q) {
                    const Pack<float, Q> t = reinterpret_cast<const Pack<float, Q>*>(red + w * N)[q];
#pragma unroll
                    for (int i = 0; i < Q; ++i) v[q * Q + i] += t.v[i];
                }
            }
        }
    }
}

// Threads of a block whose groups have G threads: four warps, or one wider group
__host__ __device__ constexpr int norm_block(int G) { return G <= 32 ? 128 : G; }
// Blocks that an SM is to hold: 384 threads with 168 registers each
__host__ __device__ constexpr int norm_blocks(int G) { return norm_block(G) >= 256 ? 1 : 384 / norm_block(G); }

// Weights in shared memory in 32 bits, as a thread reads its packs of V: the 16-byte quarters of all
// packs in planes of their own, so that the lanes of a warp read neighbouring 16 bytes.
template <int V>
__device__ __forceinline__ int weight_place(int column, int packs) {
    if constexpr (V <= 4) return column;
    const int p = column / V, j = column % V;
    return (j / 4) * packs * 4 + p * 4 + j % 4;
}
template <typename W, int V>
__device__ __forceinline__ void stage_weights(float* s_w, const void* w, float none, int D, int packs, int block) {
    for (int c = threadIdx.x; c < D; c += block)
        s_w[weight_place<V>(c, packs)] = w ? to_f(static_cast<const W*>(w)[c]) : none;
}
template <int V>
__device__ __forceinline__ Vals<V> staged_weights(const float* s_w, int pack, int packs) {
    if constexpr (V <= 4) return to_vals<float, V>(reinterpret_cast<const Pack<float, V>*>(s_w)[pack]);
    else {
        Vals<V> r;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const Vals<4> t = to_vals<float, 4>(reinterpret_cast<const Pack<float, 4>*>(s_w)[q * packs + pack]);
            r.v[2 * q] = t.v[0];
            r.v[2 * q + 1] = t.v[1];
        }
        return r;
    }
}

// Calls f(G, ITEMS, FULL) with the narrowest group of threads that holds `packs` packs of V values of T,
// false when none does: up to 32 values a thread of 16-bit types, 16 of 32-bit ones (the same bytes in
// flight a thread).  As few threads a row as possible, since what a row costs beside its values (sums
// across its threads, addresses, its statistics) is paid per thread.  The first FULL items are
// there in every thread: a check per item costs registers and moves (in the gradient of 65536 x 1024 bf16
// 7 % of the time with the last of four items checked, 15 % with all).
template <int N>
struct Int {
    static constexpr int value = N;
};
template <typename T, int V, typename F>
inline bool with_stream_group(long long packs, F&& f) {
    constexpr int J = 16 / V, I = sizeof(T) == 2 && V > 1 ? 2 * J : J;  // the most packs a thread
    constexpr int Q = I / 4, H = I / 2;
    // (widths that fill their group to the last thread, as round ones do, have no check at all)
    const auto go = [&](auto g, auto items, auto full) {
        if constexpr (V * sizeof(T) == 16) {
            if (packs == (long long)decltype(g)::value * decltype(items)::value) return f(g, items, items);
        }
        f(g, items, full);
    };
    if (packs <= 8) go(Int<8>{}, Int<1>{}, Int<0>{});
    else if (packs <= 32) go(Int<32>{}, Int<1>{}, Int<0>{});
    else if (Q > 1 && packs <= 32 * Q) go(Int<32>{}, Int<Q>{}, Int<1>{});
    else if (packs <= 32 * H) go(Int<32>{}, Int<H>{}, Int<Q>{});
    else if (packs <= 32 * (H + Q)) go(Int<32>{}, Int<H + Q>{}, Int<H>{});
    else if (packs <= 32 * I) go(Int<32>{}, Int<I>{}, Int<H + Q>{});
    else if (packs <= 64 * (H + Q)) go(Int<64>{}, Int<H + Q>{}, Int<H>{});
    else if (packs <= 64 * I) go(Int<64>{}, Int<I>{}, Int<H + Q>{});
    else if (packs <= 128 * (H + Q)) go(Int<128>{}, Int<H + Q>{}, Int<H>{});
    else if (packs <= 128 * I) go(Int<128>{}, Int<I>{}, Int<H + Q>{});
    else if (I == J && packs <= 256 * J) go(Int<256>{}, Int<J>{}, Int<J / 2>{});
    else if (packs <= 512 * J) go(Int<512>{}, Int<J>{}, Int<J / 2>{});
    else return false;
    return true;
}

// The pack sizes in bytes that the kernels move, the widest that fits: every row of x, y (dy, dx)
// and the weights start on one.
inline int norm_pack_bytes(const void* x, const void* y, const void* z, const void* w, const void* b, long long D,
                           long long row_stride, size_t tsize, size_t wsize) {
    for (size_t bytes : {size_t(16), size_t(4)}) {
        const size_t wbytes = bytes / tsize * wsize < 16 ? bytes / tsize * wsize : 16;
        if (bytes > tsize && aligned_to(x, bytes) && aligned_to(y, bytes) && aligned_to(z, bytes) && aligned_to(w, wbytes) &&
            aligned_to(b, wbytes) && (size_t)D * tsize % bytes == 0 && (size_t)row_stride * tsize % bytes == 0)
            return (int)bytes;
    }
    return (int)tsize;
}

// 16-bit values one by one cannot be copied that way.
template <typename T, int V>
constexpr bool norm_async = sizeof(Pack<T, V>) >= 4;
// Batches in a thread's ring of copies, the one being worked on included, when a batch is `packs` packs
// a thread: as many as fit 384 bytes a thread (256 in blocks of 512, whose weights take up to 64 KB of
// shared memory), two to four.
template <typename T, int V>
__host__ __device__ constexpr int norm_stages(int packs, int block) {
    const int n = (block < 512 ? 384 : 256) / (int)(sizeof(Pack<T, V>) * packs);
    return n < 2 ? 2 : n > 4 ? 4 : n;
}

// Blocks of a kernel that an SM holds, found once per device; the first call also allows the kernel
// its shared memory.
template <typename K>
inline int blocks_per_sm(K kernel, int block, size_t smem, int device, int (&cached)[64]) {
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

inline int norm_args_ok(long long rows, long long D, long long row_stride, int dtype, int wdtype) {
    if (rows < 0 || D < 1 || row_stride < 0) return IGS_ERR_ARG;
    if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != IGS_F32)) return IGS_ERR_ARG;
    if (D > (1ll << 30)) return IGS_ERR_LIMIT;
    return IGS_OK;
}

inline unsigned row_grid(long long rows) { return (unsigned)(rows < (1ll << 30) ? rows : (1ll << 30)); }

constexpr int LN_THREADS = 256;  // of the kernels for rows of any width

// Sum over a block of LN_THREADS, the same bits in every thread; `turn` alternates between calls.
__device__ __forceinline__ float block_sum_all(float v, float* s_red, int turn) {
    float t[1] = {v};
    group_sum<LN_THREADS, 1>(t, s_red, turn);
    return t[0];
}
constexpr int LN_RED = 2 * 2 * (LN_THREADS / 32);  // (for two sums at once)

}  // namespace igs
