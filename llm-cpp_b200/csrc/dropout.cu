// Dropout from a counter-based generator (philox.cuh): y = resid + (kept ? x * scale : 0), the mask
// formed where it is used and never stored. The backward is the same map of the gradient.
#include "common.cuh"
#include "dropout.cuh"
#include "philox.cuh"
#include "rowio.cuh"

namespace llmgpu {

namespace {

constexpr int kDropThreads = 256;

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
    const DropKeys key = drop_keys(rng, site);
    for (long long i = ((long long)blockIdx.x * kDropThreads + threadIdx.x) >> 5; i < total;
         i += ((long long)gridDim.x * kDropThreads) >> 5) {
        const int row = (int)(i / segs);
        const int c0 = (int)(i - (long long)row * segs) * 256;
        TI xv[8];
        TO rv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // all loads in flight before the generator's arithmetic
            const int c = c0 + 32 * j + lane;
            if (c < cols) {
                xv[j] = x[row * ldx + c];
                if (resid) rv[j] = resid[row * ldr + c];
            }
        }
        const uint32_t m = drop_keep8(key, (uint32_t)(c0 >> 3) + lane, (uint32_t)row, thr);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t mj = __shfl_sync(0xffffffffu, m, 4 * j + (lane >> 3));
            const int c = c0 + 32 * j + lane;
            if (c >= cols) continue;
            float v = ((mj >> (lane & 7)) & 1u) ? to_f32(xv[j]) * scale : 0.0f;
            if (resid) v += to_f32(rv[j]);
            out[row * ldo + c] = from_f32<TO>(v);
        }
    }
}

// Rows on 16 bytes: a thread takes 8 columns (one call of the generator) at a time, U of them with
// all loads in flight, as raw words, before the generator's arithmetic. The positions of a thread lie
// gridDim * 256 groups of 8 apart; (dr, dc) is that distance in rows and groups, so the loop
// divides nothing.
//
// Bound by memory for f32 (16384 x 4096: bf16 + f32 residual -> f32 106 us, 6.3 TB/s; f32 -> f32 86
// us) and by the generator's integer arithmetic for bf16 -> bf16 (54 us, 5.0 TB/s). U = 3 keeps
// the most blocks resident but for f32 -> f32, where 4 moves more at once (86 against 97 us).
template <typename TI, typename TO, bool RES>
constexpr int kDropUnroll = (!RES && sizeof(TI) == 4 && sizeof(TO) == 4) ? 4 : 3;
template <typename TI, typename TO, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_vec_kernel(
    const TI* x, long long ldx, const TO* resid, long long ldr, TO* out, long long ldo,
    uint32_t rows, int cols, uint32_t n8, uint32_t dr, uint32_t dc, uint32_t thr, float scale,
    const uint64_t* rng, uint64_t site) {
    pdl_enter();
    constexpr int U = kDropUnroll<TI, TO, RES>;
    const DropKeys key = drop_keys(rng, site);
    const uint32_t first = blockIdx.x * kDropThreads + threadIdx.x;
    uint32_t row = first / n8, c8 = first - row * n8;
    while (row < rows) {
        Raw8<TI> xr[U];
        Raw8<TO> rr[U];
        uint32_t ur[U], uc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ur[u] = row;
            uc[u] = c8;
            const int c = (int)(c8 * 8);
            if (row < rows) {
                if (c + 8 <= cols) {
                    load_raw(x + row * ldx + c, xr[u]);
                    if (RES) load_raw(resid + row * ldr + c, rr[u]);
                } else {
                    load_raw_n(x + row * ldx + c, cols - c, xr[u]);
                    if (RES) load_raw_n(resid + row * ldr + c, cols - c, rr[u]);
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
        for (int u = 0; u < U; ++u) {
            if (ur[u] >= rows) break;
            float v[8];
            raw_f32(xr[u], v);
            if (thr) drop_apply8(key, uc[u], ur[u], thr, scale, v);
            if (RES) {
                float r[8];
                raw_f32(rr[u], r);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += r[j];
            }
            const int c = (int)(uc[u] * 8);
            if (c + 8 <= cols) {
                store8(out + ur[u] * ldo + c, v);
            } else {
                for (int j = 0; j < 8; ++j)
                    if (c + j < cols) out[ur[u] * ldo + c + j] = from_f32<TO>(v[j]);
            }
        }
    }
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
    // in place, every element keeps its place
    if ((out == x && ((x_f32 != 0) != (out_f32 != 0) || (rows > 1 && ldo != ldx))) ||
        (out == resid && rows > 1 && ldo != ldr))
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
