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

// Eight neighbouring elements, 16 bytes at a time.
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(w[i]);
        v[2 * i + 1] = bf16_hi(w[i]);
    }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0];
    const float4 b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
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

// Rows on 16 bytes: a thread takes 8 columns (one call of the generator) at a time, kDropUnroll of
// them with all loads in flight before the generator's arithmetic. The positions of a thread lie
// gridDim * 256 groups of 8 apart; (dr, dc) is that distance in rows and groups, so the loop
// divides nothing.
constexpr int kDropUnroll = 4;
template <typename TI, typename TO, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_vec_kernel(
    const TI* x, long long ldx, const TO* resid, long long ldr, TO* out, long long ldo,
    uint32_t rows, int cols, uint32_t n8, uint32_t dr, uint32_t dc, uint32_t thr, float scale,
    const uint64_t* rng, uint64_t site) {
    pdl_enter();
    const DropKey key = drop_key(rng, site);
    const uint32_t first = blockIdx.x * kDropThreads + threadIdx.x;
    uint32_t row = first / n8, c8 = first - row * n8;
    while (row < rows) {
        float v[kDropUnroll][8], r[kDropUnroll][8];
        uint32_t ur[kDropUnroll], uc[kDropUnroll];
#pragma unroll
        for (int u = 0; u < kDropUnroll; ++u) {
            ur[u] = row;
            uc[u] = c8;
            const int c = (int)(c8 * 8);
            if (row < rows) {
                if (c + 8 <= cols) {
                    load8(x + row * ldx + c, v[u]);
                    if (RES) load8(resid + row * ldr + c, r[u]);
                } else {
                    for (int j = 0; j < 8; ++j) {
                        v[u][j] = c + j < cols ? to_f32(x[row * ldx + c + j]) : 0.0f;
                        if (RES) r[u][j] = c + j < cols ? to_f32(resid[row * ldr + c + j]) : 0.0f;
                    }
                }
            }
            row += dr;
            c8 += dc;
            if (c8 >= n8) {
                c8 -= n8;
                ++row;
            }
        }
#pragma unroll
        for (int u = 0; u < kDropUnroll; ++u) {
            if (ur[u] >= rows) break;
            if (thr) drop_apply8(key, uc[u], ur[u], thr, scale, v[u]);
            if (RES) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] += r[u][j];
            }
            const int c = (int)(uc[u] * 8);
            if (c + 8 <= cols) {
                store8(out + ur[u] * ldo + c, v[u]);
            } else {
                for (int j = 0; j < 8; ++j)
                    if (c + j < cols) out[ur[u] * ldo + c + j] = from_f32<TO>(v[u][j]);
            }
        }
    }
}

template <typename T>
bool rows_on_16(const T* p, long long ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
}

template <typename TI, typename TO>
int launch_dropout(const void* x, long long ldx, const void* resid, long long ldr, void* out,
                   long long ldo, int rows, int cols, uint32_t thr, float scale,
                   const uint64_t* rng, uint64_t site, cudaStream_t s) {
    if (rows_on_16((const TI*)x, ldx) && rows_on_16((const TO*)out, ldo) &&
        (!resid || rows_on_16((const TO*)resid, ldr))) {
        const uint32_t n8 = (uint32_t)(cols + 7) / 8;
        const long long items = (long long)rows * n8;
        long long blocks = (items + kDropThreads - 1) / kDropThreads;
        if (blocks > 148 * 8) blocks = 148 * 8;
        const uint32_t step = (uint32_t)blocks * kDropThreads;
        return resid ? launch_kernel(dropout_vec_kernel<TI, TO, true>, (int)blocks, kDropThreads, 0, s,
                                     (const TI*)x, ldx, (const TO*)resid, ldr, (TO*)out, ldo,
                                     (uint32_t)rows, cols, n8, step / n8, step % n8, thr, scale, rng,
                                     site)
                     : launch_kernel(dropout_vec_kernel<TI, TO, false>, (int)blocks, kDropThreads, 0, s,
                                     (const TI*)x, ldx, (const TO*)resid, ldr, (TO*)out, ldo,
                                     (uint32_t)rows, cols, n8, step / n8, step % n8, thr, scale, rng,
                                     site);
    }
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
