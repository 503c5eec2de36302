// Shared by the feature operators (embed.cu, layer_norm.cu, dropout.cu): the element types they
// take and how a value goes to and from the 32 bits everything is computed in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace igs {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// The one rounding of every result: to nearest, ties to even.
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

inline size_t dtype_size(int dtype) { return dtype == IGS_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == IGS_F32 || dtype == IGS_BF16 || dtype == IGS_F16; }

// Calls f(T{}) with the element type of a dtype code that dtype_ok accepts.
template <typename F>
inline auto with_dtype(int dtype, F&& f) {
    if (dtype == IGS_BF16) return f(__nv_bfloat16{});
    if (dtype == IGS_F16) return f(__half{});
    return f(float{});
}

// V neighbouring values as they lie in memory, moved by one load or store of up to 16 bytes
// (aligned to its size).
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
    T v[V];
};

// V values in 32 bits.  Pairs of neighbours share a packed f32x2 operand: half the instructions to
// issue for the same arithmetic.
template <int V>
struct Vals {
    static_assert(V % 2 == 0, "pairs");
    f2 v[V / 2];
};
template <>
struct Vals<1> {
    float v;
};

template <int V>
__device__ __forceinline__ Vals<V> splat(float x) {
    Vals<V> r;
    if constexpr (V == 1) r.v = x;
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) r.v[i] = pk(x, x);
    }
    return r;
}

__device__ __forceinline__ f2 pair_f(const float* p) { return pk(p[0], p[1]); }
__device__ __forceinline__ f2 pair_f(const __nv_bfloat16* p) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);  // a bfloat16 is the upper half of a float
    return pk(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ f2 pair_f(const __half* p) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
    return pk(f.x, f.y);
}
template <typename T, int V>
__device__ __forceinline__ Vals<V> to_vals(const Pack<T, V>& p) {
    Vals<V> r;
    if constexpr (V == 1) r.v = to_f(p.v[0]);
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) r.v[i] = pair_f(p.v + 2 * i);
    }
    return r;
}

__device__ __forceinline__ void put_pair(float* p, float a, float b) {
    p[0] = a;
    p[1] = b;
}
__device__ __forceinline__ void put_pair(__nv_bfloat16* p, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void put_pair(__half* p, float a, float b) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> to_pack(const Vals<V>& x) {
    Pack<T, V> r;
    if constexpr (V == 1) r.v[0] = from_f<T>(x.v);
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            float a, b;
            upk(x.v[i], a, b);
            put_pair(r.v + 2 * i, a, b);
        }
    }
    return r;
}

template <int V>
__device__ __forceinline__ Vals<V> add(Vals<V> a, const Vals<V>& b) {
    if constexpr (V == 1) a.v += b.v;
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) a.v[i] = add2(a.v[i], b.v[i]);
    }
    return a;
}
template <int V>
__device__ __forceinline__ Vals<V> sub(Vals<V> a, const Vals<V>& b) {
    if constexpr (V == 1) a.v -= b.v;
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) a.v[i] = sub2(a.v[i], b.v[i]);
    }
    return a;
}
template <int V>
__device__ __forceinline__ Vals<V> mul(Vals<V> a, const Vals<V>& b) {
    if constexpr (V == 1) a.v *= b.v;
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) a.v[i] = mul2(a.v[i], b.v[i]);
    }
    return a;
}
// a b + c
template <int V>
__device__ __forceinline__ Vals<V> fma(const Vals<V>& a, const Vals<V>& b, Vals<V> c) {
    if constexpr (V == 1) c.v = fmaf(a.v, b.v, c.v);
    else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) c.v[i] = fma2(a.v[i], b.v[i], c.v[i]);
    }
    return c;
}
template <int V>
__device__ __forceinline__ float total(const Vals<V>& a) {
    if constexpr (V == 1) return a.v;
    else {
        f2 t = a.v[0];
#pragma unroll
        for (int i = 1; i < V / 2; ++i) t = add2(t, a.v[i]);
        float lo, hi;
        upk(t, lo, hi);
        return lo + hi;
    }
}

__host__ __device__ inline bool aligned_to(const void* p, size_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

// Asynchronous copies to shared memory, by which a thread reads ahead of itself: BYTES of 4 or 16, groups in
// order of their commits.
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


// Chains of short kernels: each is launched so that its blocks may start once all blocks of the one
// before have started, and waits for that one's results (its completion, which for the same reason
// includes everything before it) where it first reads them.  Launching and draining then overlap.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
inline void launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;  // the same bits in every lane
}

}  // namespace igs
