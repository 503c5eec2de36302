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

__host__ __device__ inline bool aligned_to(const void* p, size_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;  // the same bits in every lane
}

}  // namespace igs
