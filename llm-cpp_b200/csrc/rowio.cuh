// Rows of bf16 or f32 matrices, eight neighbouring elements at a time.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.cuh"

namespace llmgpu {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<bf16>(bf16 v) {
    return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) {
    return __float2bfloat16_rn(v);
}

// Eight neighbouring elements as they lie in memory: loads stay in flight until raw_f32.
template <typename T>
struct Raw8 {
    uint4 q[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void load_raw(const T* p, Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.q[i] = reinterpret_cast<const uint4*>(p)[i];
}
// n < 8 of them, the others 0
template <typename T>
__device__ __forceinline__ void load_raw_n(const T* p, int n, Raw8<T>& r) {
    alignas(16) T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = j < n ? p[j] : from_f32<T>(0.0f);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.q[i] = reinterpret_cast<const uint4*>(t)[i];
}
__device__ __forceinline__ void raw_f32(const Raw8<bf16>& r, float (&v)[8]) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(w[i]);
        v[2 * i + 1] = bf16_hi(w[i]);
    }
}
__device__ __forceinline__ void raw_f32(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[4 * i] = __uint_as_float(r.q[i].x);
        v[4 * i + 1] = __uint_as_float(r.q[i].y);
        v[4 * i + 2] = __uint_as_float(r.q[i].z);
        v[4 * i + 3] = __uint_as_float(r.q[i].w);
    }
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                   pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

template <typename T>
inline bool rows_on_16(const T* p, long long ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
}

}  // namespace llmgpu
