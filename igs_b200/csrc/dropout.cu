// igs_dropout: y = x / (1 - p) where the generator keeps the value, 0 where it does not.
//
// The mask is a function of (seed, offset, place) and is never stored: Philox4x32 with 7 rounds
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011; 7 is the
// fewest rounds that the paper finds to pass every test of BigCrush).  Value i takes word i % 4
// of the block with counter (i / 4, offset), both 64 bits, under the key `seed`, and is kept when
// the word is at least p * 2^32.  The gradient is the same call on the upstream gradient.
// A dropped value is zero whatever was there, NaN and infinities included.
#include "feature.cuh"

namespace igs {

constexpr int PHILOX_ROUNDS = 7;
constexpr int DROPOUT_THREADS = 256;
constexpr long long DROPOUT_MAX = 1ll << 42;  // values a call takes: the grid stays within 2^31 - 1 blocks

struct PhiloxKeys {
    uint32_t k0[PHILOX_ROUNDS], k1[PHILOX_ROUNDS];
    uint32_t off_lo, off_hi;
};

__device__ __forceinline__ PhiloxKeys philox_keys(unsigned long long seed, unsigned long long offset) {
    PhiloxKeys k;
    uint32_t a = (uint32_t)seed, b = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < PHILOX_ROUNDS; ++r) {
        k.k0[r] = a;
        k.k1[r] = b;
        a += 0x9E3779B9u;
        b += 0xBB67AE85u;
    }
    k.off_lo = (uint32_t)offset;
    k.off_hi = (uint32_t)(offset >> 32);
    return k;
}

__device__ __forceinline__ uint4 philox(const PhiloxKeys& k, unsigned long long block) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = k.off_lo, c3 = k.off_hi;
#pragma unroll
    for (int r = 0; r < PHILOX_ROUNDS; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k.k0[r];
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k.k1[r];
        c3 = (uint32_t)a;
    }
    return make_uint4(c0, c1, c2, c3);
}

struct DropoutArgs {
    const void* x;
    void* y;
    long long n;
    unsigned long long seed, offset;
    const long long* state;  // NULL, or (seed, offset) on the device; `offset` above is added to its offset
    uint32_t threshold;      // floor(p * 2^32)
    float scale;             // 1 / (1 - p)
};

template <typename T>
__device__ __forceinline__ T dropped(T x, uint32_t word, const DropoutArgs& a) {
    return word >= a.threshold ? from_f<T>(to_f(x) * a.scale) : from_f<T>(0.f);
}

// A thread takes DROPOUT_UNROLL groups of V neighbouring values, all loads first; V is 16 bytes'
// worth (one or two generator blocks) or, where x or y is off the 16-byte boundary, four values
// moved one by one.  The last n % V values go to the last block's first threads.
constexpr int DROPOUT_UNROLL = 4;
template <typename T, int V, bool ALIGNED>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_kernel(DropoutArgs a) {
    unsigned long long seed = a.seed, offset = a.offset;
    if (a.state) {
        seed = (unsigned long long)a.state[0];
        offset += (unsigned long long)a.state[1];
    }
    const PhiloxKeys keys = philox_keys(seed, offset);
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const long long groups = a.n / V;
    const long long g0 = (long long)blockIdx.x * (DROPOUT_THREADS * DROPOUT_UNROLL) + threadIdx.x;
    Pack<T, V> in[DROPOUT_UNROLL];
#pragma unroll
    for (int u = 0; u < DROPOUT_UNROLL; ++u) {
        const long long g = g0 + u * DROPOUT_THREADS;
        if (g >= groups) continue;
        if constexpr (ALIGNED) {
            in[u] = reinterpret_cast<const Pack<T, V>*>(x)[g];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) in[u].v[j] = x[g * V + j];
        }
    }
#pragma unroll
    for (int u = 0; u < DROPOUT_UNROLL; ++u) {
        const long long g = g0 + u * DROPOUT_THREADS;
        if (g >= groups) continue;
        Pack<T, V> out;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const uint4 r = philox(keys, (unsigned long long)(g * (V / 4) + q));
            out.v[4 * q] = dropped(in[u].v[4 * q], r.x, a);
            out.v[4 * q + 1] = dropped(in[u].v[4 * q + 1], r.y, a);
            out.v[4 * q + 2] = dropped(in[u].v[4 * q + 2], r.z, a);
            out.v[4 * q + 3] = dropped(in[u].v[4 * q + 3], r.w, a);
        }
        if constexpr (ALIGNED) {
            reinterpret_cast<Pack<T, V>*>(y)[g] = out;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) y[g * V + j] = out.v[j];
        }
    }
    const long long i = groups * V + threadIdx.x;
    if (blockIdx.x == gridDim.x - 1 && i < a.n) {
        const uint4 r = philox(keys, (unsigned long long)(i / 4));
        const uint32_t w = i % 4 == 0 ? r.x : i % 4 == 1 ? r.y : i % 4 == 2 ? r.z : r.w;
        y[i] = dropped(x[i], w, a);
    }
}

}  // namespace igs

using namespace igs;

extern "C" int igs_dropout(const void* x, int dtype, long long n, double p, unsigned long long seed,
                           unsigned long long offset, const long long* state, void* y, int device, void* stream) {
    if (n < 0 || !dtype_ok(dtype) || !(p >= 0.0 && p <= 1.0)) return IGS_ERR_ARG;
    if (n > DROPOUT_MAX) return IGS_ERR_LIMIT;
    if (n == 0) return IGS_OK;
    if (!x || !y) return IGS_ERR_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    if (p * 4294967296.0 >= 4294967296.0)  // nothing is kept: no word reaches 2^32, and 1 / (1 - p) has no value
        return (int)cudaMemsetAsync(y, 0, (size_t)n * dtype_size(dtype), s);

    DropoutArgs a{x, y, n, seed, offset, state, (uint32_t)(p * 4294967296.0), (float)(1.0 / (1.0 - p))};
    const bool aligned = aligned_to(x, 16) && aligned_to(y, 16);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T);
        const long long per = (long long)(aligned ? V : 4) * DROPOUT_THREADS * DROPOUT_UNROLL;
        const unsigned grid = (unsigned)((n + per - 1) / per);
        if (aligned)
            dropout_kernel<T, V, true><<<grid, DROPOUT_THREADS, 0, s>>>(a);
        else
            dropout_kernel<T, 4, false><<<grid, DROPOUT_THREADS, 0, s>>>(a);
        return 0;
    });
    count_launch();
    return (int)cudaGetLastError();
}
