// experts.cuh -- device helpers shared by the routed-experts kernels (route.cu, group.cu, combine.cu, expert_*.cu).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace kmc {

// One element type of the routed-experts operators: conversions to and from float32 (to 16 bits: round to nearest
// even, once, where a result is stored), and 16-byte vectors of it.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// V elements read or written as one access (V sizeof(T) = 2, 4, 8 or 16 bytes, aligned to that)
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

}  // namespace kmc
