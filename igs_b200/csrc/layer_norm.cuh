// Shared by layer_norm.cu and layer_norm_grad.cu: how a row is given to threads, and sums over them.
#pragma once

#include "feature.cuh"

namespace igs {

// V weights as floats; without any, the value they stand for
template <typename W, int V>
__device__ __forceinline__ void load_weights(const void* w, long long c, float none, float (&out)[V]) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = none;
        return;
    }
    // (a pack may be longer than the 16 bytes that one load moves)
    const Pack<W, V> p = *reinterpret_cast<const Pack<W, V>*>(static_cast<const W*>(w) + c);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = to_f(p.v[j]);
}

__host__ __device__ constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// N sums (a power of two, at most 32) over the G threads of a row's group at once, the same bits in
// every one of them.  Groups of up to a warp are lanes of one warp; a wider group is the whole
// block, and s_red (two halves used in turn, so that one barrier a call suffices) holds N floats
// per warp.  Within a warp the first log2 N steps halve the number of sums a lane carries: N - 1
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
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) t += red[w * N + i];
                v[i] = t;
            }
        }
    }
}

// Threads of a block whose groups have G threads
__host__ __device__ constexpr int norm_block(int G) { return G < 128 ? 128 : G; }

template <int N>
struct Int {
    static constexpr int value = N;
};

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
constexpr int LN_RED = 2 * (LN_THREADS / 32);

}  // namespace igs
