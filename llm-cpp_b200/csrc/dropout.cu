// Dropout from a counter-based generator (philox.cuh): y = resid + (kept ? x * scale : 0), the mask
// formed where it is used and never stored. The backward is the same map of the gradient.
#include "common.cuh"
#include "dropout.cuh"
#include "philox.cuh"

namespace llmgpu {

namespace {

constexpr int kDropThreads = 256;

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

// Any strides and alignment: a warp takes 256 columns of a row, lane i forms the bits of columns
// 8 i .. 8 i + 7, and the elements are visited 32 neighbouring columns at a time.
template <typename TI, typename TO>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const TI* x, long long ldx,
                                                               const TO* resid, long long ldr,
                                                               TO* out, long long ldo, int rows,
                                                               int cols, uint32_t thr, float scale,
                                                               const uint64_t* rng, uint64_t site) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int segs = (cols + 255) / 256;
    const long long total = (long long)rows * segs;
    const DropKey key = drop_key(rng, site);
    for (long long i = ((long long)blockIdx.x * kDropThreads + threadIdx.x) >> 5; i < total;
         i += ((long long)gridDim.x * kDropThreads) >> 5) {
        const int row = (int)(i / segs);
        const int c0 = (int)(i - (long long)row * segs) * 256;
        const uint32_t m = drop_keep8(key, (uint32_t)(c0 >> 3) + lane, (uint32_t)row, thr);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t mj = __shfl_sync(0xffffffffu, m, 4 * j + (lane >> 3));
            const int c = c0 + 32 * j + lane;
            if (c >= cols) continue;
            float v = 0.0f;
            if ((mj >> (lane & 7)) & 1u) v = to_f32(x[row * ldx + c]) * scale;
            if (resid) v += to_f32(resid[row * ldr + c]);
            out[row * ldo + c] = from_f32<TO>(v);
        }
    }
}

template <typename TI, typename TO>
int launch_dropout(const void* x, long long ldx, const void* resid, long long ldr, void* out,
                   long long ldo, int rows, int cols, uint32_t thr, float scale,
                   const uint64_t* rng, uint64_t site, cudaStream_t s) {
    const long long warps = (long long)rows * ((cols + 255) / 256);
    long long blocks = (warps + kDropThreads / 32 - 1) / (kDropThreads / 32);
    if (blocks > 148 * 8) blocks = 148 * 8;
    return launch_kernel(dropout_kernel<TI, TO>, (int)blocks, kDropThreads, 0, s, (const TI*)x, ldx,
                         (const TO*)resid, ldr, (TO*)out, ldo, rows, cols, thr, scale, rng, site);
}

}  // namespace

int dropout_apply(const void* x, int x_f32, long long ldx, const void* resid, long long ldr,
                  void* out, int out_f32, long long ldo, int rows, int cols, float p,
                  const uint64_t* rng, uint64_t site, cudaStream_t s) {
    uint32_t thr;
    float scale;
    if (rows < 0 || cols < 0 || cols > (1 << 30) || !drop_params(p, &thr, &scale)) return -1;
    if (rows == 0 || cols == 0) return 0;
    if (!x || !out || !rng || (rows > 1 && (ldx < cols || ldo < cols || (resid && ldr < cols))))
        return -1;
    if (x_f32)
        return out_f32 ? launch_dropout<float, float>(x, ldx, resid, ldr, out, ldo, rows, cols, thr,
                                                      scale, rng, site, s)
                       : launch_dropout<float, bf16>(x, ldx, resid, ldr, out, ldo, rows, cols, thr,
                                                     scale, rng, site, s);
    return out_f32 ? launch_dropout<bf16, float>(x, ldx, resid, ldr, out, ldo, rows, cols, thr,
                                                 scale, rng, site, s)
                   : launch_dropout<bf16, bf16>(x, ldx, resid, ldr, out, ldo, rows, cols, thr,
                                                scale, rng, site, s);
}

}  // namespace llmgpu
