// igs_dropout: y = x / (1 - p) where the generator keeps the value, 0 where it does not.
//
// The mask is a function of (seed, offset, place) and is never stored: Philox4x32 with 7 rounds
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011; 7 is the
// fewest rounds that the paper finds to pass every test of BigCrush).  Value i takes word i % 4
// of the block with counter (i / 4, offset), both 64 bits, under the key `seed`, and is kept when
// the word is at least p * 2^32.  The gradient is the same call on the upstream gradient.
// A dropped value is zero whatever was there, NaN and infinities included.
//
// What bounds it: memory for fp32 (128 MB in 42 us where a copy takes 43), the integer pipes for 16-bit
// types, where a byte carries twice the words (bf16 48, fp16 45 us).
#include "feature.cuh"

namespace igs {

constexpr int PHILOX_ROUNDS = 7;
constexpr int DROPOUT_THREADS = 256;
constexpr long long DROPOUT_MAX = 1ll << 42;  // values a call takes: the grid stays within 2^31 - 1 blocks

// What a block of threads shares of the generator: the keys of all rounds, and the words that depend on
// the counter's upper three quarters alone.  With c = (lo, hi, o0, o1) the first round is
//   (hi32(o0 M1) ^ hi ^ k0, lo32(o0 M1), hi32(lo M0) ^ o1 ^ k1, lo32(lo M0)),
// whose first two words do not depend on lo, so that the second round's product of the first is shared
// as well: two of the fourteen products of a block of four words are paid once a thread.
struct Philox {
    uint32_t k0[PHILOX_ROUNDS], k1[PHILOX_ROUNDS];
    uint32_t x2;    // o1 ^ k1 of the first round
    uint32_t y2;    // hi32(c0 M0) ^ k1 of the second round, c0 its first word
    uint32_t y3;    // lo32(c0 M0)
    uint32_t x1;    // the first round's second word ^ k0 of the second round
};

__device__ __forceinline__ Philox philox_setup(unsigned long long seed, unsigned long long offset, uint32_t hi) {
    Philox p;
    uint32_t a = (uint32_t)seed, b = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < PHILOX_ROUNDS; ++r) {
        p.k0[r] = a;
        p.k1[r] = b;
        a += 0x9E3779B9u;
        b += 0xBB67AE85u;
    }
    const unsigned long long o = (unsigned long long)(uint32_t)offset * 0xCD9E8D57u;
    const uint32_t c0 = (uint32_t)(o >> 32) ^ hi ^ p.k0[0];
    p.x2 = (uint32_t)(offset >> 32) ^ p.k1[0];
    p.x1 = (uint32_t)o ^ p.k0[1];
    const unsigned long long t = (unsigned long long)c0 * 0xD2511F53u;
    p.y2 = (uint32_t)(t >> 32) ^ p.k1[1];
    p.y3 = (uint32_t)t;
    return p;
}

// the four words of the block whose counter's lowest quarter is lo
__device__ __forceinline__ uint4 philox(const Philox& p, uint32_t lo) {
    const unsigned long long first = (unsigned long long)lo * 0xD2511F53u;
    const unsigned long long second = (unsigned long long)((uint32_t)(first >> 32) ^ p.x2) * 0xCD9E8D57u;
    uint32_t c0 = (uint32_t)(second >> 32) ^ p.x1, c1 = (uint32_t)second;
    uint32_t c2 = p.y2 ^ (uint32_t)first, c3 = p.y3;
#pragma unroll
    for (int r = 2; r < PHILOX_ROUNDS; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ p.k0[r];
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ p.k1[r];
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

// two scaled values, each kept or zero
__device__ __forceinline__ void put_kept(float* out, float a, float b, bool keep_a, bool keep_b) {
    out[0] = keep_a ? a : 0.f;
    out[1] = keep_b ? b : 0.f;
}
template <typename T>
__device__ __forceinline__ void put_kept(T* out, float a, float b, bool keep_a, bool keep_b) {
    Pack<T, 2> p;
    put_pair(p.v, a, b);
    uint32_t u = *reinterpret_cast<const uint32_t*>(&p);
    if (!keep_a) u &= 0xffff0000u;
    if (!keep_b) u &= 0x0000ffffu;
    *reinterpret_cast<uint32_t*>(out) = u;
}

// Four neighbouring values and their block's words.
template <typename T>
__device__ __forceinline__ void drop4(T* v, const uint4& r, const DropoutArgs& a) {
    const f2 scale = pk(a.scale, a.scale);
    float f[4];
    upk(mul2(pair_f(v), scale), f[0], f[1]);
    upk(mul2(pair_f(v + 2), scale), f[2], f[3]);
    put_kept(v, f[0], f[1], r.x >= a.threshold, r.y >= a.threshold);
    put_kept(v + 2, f[2], f[3], r.z >= a.threshold, r.w >= a.threshold);
}

// A thread takes DROPOUT_UNROLL groups of V neighbouring values, all loads first; V is 16 bytes'
// worth (one or two generator blocks) or, where x or y is off the 16-byte boundary, four values
// moved one by one.  The last n % V values go to the last block's first threads.
constexpr int DROPOUT_UNROLL = 4;
template <typename T, int V, bool ALIGNED>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_kernel(DropoutArgs a) {
    unsigned long long seed = a.seed, offset = a.offset;
    constexpr int TILE = DROPOUT_THREADS * DROPOUT_UNROLL;  // groups a block
    const long long groups = a.n / V, g0 = (long long)blockIdx.x * TILE + threadIdx.x;
    const int left = (int)(groups - g0 < TILE ? groups - g0 : TILE);  // group u is there when u DROPOUT_THREADS < left
    const T* x = static_cast<const T*>(a.x) + g0 * V;
    T* y = static_cast<T*>(a.y) + g0 * V;
    Pack<T, V> v[DROPOUT_UNROLL];
#pragma unroll
    for (int u = 0; u < DROPOUT_UNROLL; ++u) {
        if (u * DROPOUT_THREADS >= left) continue;
        if constexpr (ALIGNED) {
            v[u] = reinterpret_cast<const Pack<T, V>*>(x)[u * DROPOUT_THREADS];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[u].v[j] = x[u * DROPOUT_THREADS * V + j];
        }
    }
    if (a.state) {
        seed = (unsigned long long)a.state[0];
        offset += (unsigned long long)a.state[1];
    }
    // (a block's generator counters share their upper half: it takes a power of two of them)
    const unsigned long long q0 = (unsigned long long)g0 * (V / 4);
    const Philox gen = philox_setup(seed, offset, (uint32_t)(q0 >> 32));
#pragma unroll
    for (int u = 0; u < DROPOUT_UNROLL; ++u) {
        if (u * DROPOUT_THREADS >= left) continue;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) drop4(v[u].v + 4 * q, philox(gen, (uint32_t)q0 + u * (DROPOUT_THREADS * (V / 4)) + q), a);
        if constexpr (ALIGNED) {
            reinterpret_cast<Pack<T, V>*>(y)[u * DROPOUT_THREADS] = v[u];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) y[u * DROPOUT_THREADS * V + j] = v[u].v[j];
        }
    }
    const long long i = groups * V + threadIdx.x;
    if (blockIdx.x == gridDim.x - 1 && i < a.n) {
        const uint4 r = philox(philox_setup(seed, offset, (uint32_t)((i / 4) >> 32)), (uint32_t)(i / 4));
        const uint32_t w = i % 4 == 0 ? r.x : i % 4 == 1 ? r.y : i % 4 == 2 ? r.z : r.w;
        const float f = to_f(static_cast<const T*>(a.x)[i]) * a.scale;
        static_cast<T*>(a.y)[i] = from_f<T>(w >= a.threshold ? f : 0.f);
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
