// Linear layer with bias, activation, dropout and residual applied where the product's tiles leave
// tensor memory (gemm.cu, kEpiLinear), and its backward: one elementwise pass forms dz in bf16
// and the bias gradient's partial sums, then two products give dx and dw.
#include "linear.cuh"

#include "common.cuh"
#include "philox.cuh"
#include "rowio.cuh"

namespace llmgpu {

namespace {

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
long long ceil8(long long n) { return (n + 7) & ~7ll; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kDzCols = 256;  // columns of a block: 32 lanes of 8
constexpr int kDzRows = 8;    // rows in flight, one per warp

// Row groups of the elementwise backward: enough blocks to fill the device a few times over.
int dz_groups(int M, int N) {
    const int gx = (N + kDzCols - 1) / kDzCols;
    int gy = (148 * 8 + gx - 1) / gx;
    const int most = (M + kDzRows - 1) / kDzRows;
    if (gy > most) gy = most;
    return gy < 1 ? 1 : gy;
}

// Derivatives of a pair of activations, from the same sigmoid as the forward's: gelu(z) = z h with
// h = sigmoid(2u): h + z h (1 - h) 2u'; silu: h (1 + z (1 - h)).
template <int ACT>
__device__ __forceinline__ float2 act_grad_pair(float2 z) {
    constexpr float kLog2 = 1.4426950408889634f;
    if constexpr (ACT == kActRelu) {
        return make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
    } else if constexpr (ACT == kActGelu || ACT == kActSilu) {
        const float2 one = make_float2(1.0f, 1.0f);
        const float2 z2 = fmul2(z, z);
        float2 t;
        if constexpr (ACT == kActGelu) {
            constexpr float c = -1.5957691216f * kLog2;
            t = fmul2(ffma2(z2, make_float2(c * 0.044715f, c * 0.044715f), make_float2(c, c)), z);
        } else {
            t = fmul2(z, make_float2(-kLog2, -kLog2));
        }
        const float2 d = fadd2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), one);
        const float2 h = make_float2(rcp_approx(d.x), rcp_approx(d.y));
        const float2 g = ffma2(h, make_float2(-1.0f, -1.0f), one);  // 1 - h
        if constexpr (ACT == kActGelu) {
            constexpr float k = 1.5957691216f;
            const float2 q =
                fmul2(ffma2(z2, make_float2(k * 0.134145f, k * 0.134145f), make_float2(k, k)), z);
            return ffma2(fmul2(h, g), q, h);
        } else {
            return fmul2(h, ffma2(z, g, one));
        }
    } else {
        return make_float2(1.0f, 1.0f);
    }
}

// dz [M][ldz] (nullable) and the column sums of a block's rows, part[gy][N] (nullable; with one row of
// blocks it is dbias itself, added to when `accumulate`). `vec`: rows of dy and pre start on 16 bytes. A thread takes 8 columns of kDzInFlight rows at a time, their
// loads in flight together as raw words: bound by memory at 8192 x 4096 bf16 (201 MB).
constexpr int kDzInFlight = 2;
template <typename T, int ACT, bool DROP>
__global__ void __launch_bounds__(256) linear_dz_kernel(const T* __restrict__ dy, long long lddy,
                                                        const bf16* __restrict__ pre,
                                                        long long ld_pre, DropArgs drop,
                                                        bf16* __restrict__ dz, long long ldz,
                                                        float* __restrict__ part, int accumulate,
                                                        int M, int N, int vec) {
    pdl_enter();
    const int lane = threadIdx.x & 31, wr = threadIdx.x >> 5;
    const int col = blockIdx.x * kDzCols + lane * 8;
    const int n = min(8, N - col);
    float2 sum[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = make_float2(0.0f, 0.0f);
    if (n > 0) {
        const bool v8 = vec && n == 8;
        DropKeys key;
        if constexpr (DROP) key = drop_keys(drop.rng, drop.site);
        const int step = gridDim.y * kDzRows;
        for (long long row0 = blockIdx.y * kDzRows + wr; row0 < M; row0 += kDzInFlight * step) {
            Raw8<T> dr[kDzInFlight];
            Raw8<bf16> pr[kDzInFlight];
#pragma unroll
            for (int u = 0; u < kDzInFlight; ++u) {
                const long long row = row0 + u * step;
                if (row >= M) break;
                if (v8) {
                    load_raw(dy + row * lddy + col, dr[u]);
                    if (ACT != kActNone) load_raw(pre + row * ld_pre + col, pr[u]);
                } else {
                    load_raw_n(dy + row * lddy + col, n, dr[u]);
                    if (ACT != kActNone) load_raw_n(pre + row * ld_pre + col, n, pr[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kDzInFlight; ++u) {
                const long long row = row0 + u * step;
                if (row >= M) break;
                float v[8];
                raw_f32(dr[u], v);
                if constexpr (DROP)
                    drop_apply8(key, (uint32_t)col >> 3, (uint32_t)row, drop.thr, drop.scale, v);
                if constexpr (ACT != kActNone) {
                    float z[8];
                    raw_f32(pr[u], z);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 y = fmul2(make_float2(v[2 * i], v[2 * i + 1]),
                                               act_grad_pair<ACT>(make_float2(z[2 * i], z[2 * i + 1])));
                        v[2 * i] = y.x;
                        v[2 * i + 1] = y.y;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fadd2(sum[i], make_float2(v[2 * i], v[2 * i + 1]));
                // columns past N, up to the padded stride, are written as zeros
                if (dz) store8(dz + row * ldz + col, v);
            }
        }
    }
    if (!part) return;
    __shared__ float red[kDzRows][kDzCols];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        red[wr][lane * 8 + 2 * i] = sum[i].x;
        red[wr][lane * 8 + 2 * i + 1] = sum[i].y;
    }
    __syncthreads();
    const int c = blockIdx.x * kDzCols + threadIdx.x;
    if (c < N) {
        float t = 0.0f;
#pragma unroll
        for (int r = 0; r < kDzRows; ++r) t += red[r][threadIdx.x];
        float* to = part + (long long)blockIdx.y * N + c;
        *to = accumulate ? *to + t : t;
    }
}

template <typename T, int ACT>
int launch_dz_act(const LinearBwd& a, const DropArgs& drop, dim3 grid, bf16* to, float* sums, int vec,
                  cudaStream_t s) {
    const int accumulate = grid.y == 1 && a.accumulate;
    return launch_kernel(drop.rng ? linear_dz_kernel<T, ACT, true> : linear_dz_kernel<T, ACT, false>,
                         grid, 256, 0, s, (const T*)a.dy, a.lddy, a.pre, a.ld_pre, drop, to,
                         ceil8(a.N), sums, accumulate, a.M, a.N, vec);
}
template <typename T>
int launch_dz(const LinearBwd& a, const DropArgs& drop, dim3 grid, bf16* to, float* sums, int vec,
              cudaStream_t s) {
    switch (a.act) {
        case kActRelu:
            return launch_dz_act<T, kActRelu>(a, drop, grid, to, sums, vec, s);
        case kActGelu:
            return launch_dz_act<T, kActGelu>(a, drop, grid, to, sums, vec, s);
        case kActSilu:
            return launch_dz_act<T, kActSilu>(a, drop, grid, to, sums, vec, s);
        default:
            return launch_dz_act<T, kActNone>(a, drop, grid, to, sums, vec, s);
    }
}

// dbias[c] (+)= sum over the row groups, in a fixed order.
__global__ void __launch_bounds__(1024) linear_db_kernel(const float* __restrict__ part, int groups,
                                                         int N, float* __restrict__ dbias,
                                                         int accumulate) {
    pdl_enter();
    __shared__ float red[32][33];
    const int cc = threadIdx.x & 31, g0 = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cc;
    float t = 0.0f;
    if (c < N)
        for (int g = g0; g < groups; g += 32) t += part[(long long)g * N + c];
    red[g0][cc] = t;
    __syncthreads();
    if (g0 == 0 && c < N) {
        float u = 0.0f;
#pragma unroll
        for (int g = 0; g < 32; ++g) u += red[g][cc];
        dbias[c] = accumulate ? dbias[c] + u : u;
    }
}

}  // namespace

int product(const bf16* A, long long lda, int a_mn, const bf16* B, long long ldb, int b_mn, int M,
            int N, int K, void* out, int out_f32, long long ldo, int accumulate, int num_sms,
            int* err, cudaStream_t s, const float* alpha) {
    if (accumulate && !out_f32) return -1;
    if (M <= kFewRows && !a_mn) {
        RowsArgs r{A, lda, B, ldb, alpha, nullptr, kActNone, {}, accumulate ? out : nullptr, ldo, nullptr, 0,
                   out, out_f32, ldo, M, N, K};
        return rows_product(r, b_mn, s);
    }
    if (K <= kOuterRows && a_mn && b_mn)
        return outer_product(A, lda, B, ldb, M, N, K, out, out_f32, ldo, accumulate, alpha, s);
    GemmArgs g{};
    g.out = out;
    g.ldo = ldo;
    g.splits = 1;
    g.err = err;
    GemmPlan plan;
    int rc;
    const int per16 = out_f32 ? 4 : 8;
    if (!alpha && aligned16(out) && (ldo % per16) == 0 && (N % per16) == 0) {
        g.epi = out_f32 ? kEpiStoreF32 : kEpiStoreBF16;
        g.accumulate = accumulate;
        rc = gemm_make_plan(&plan, A, lda, a_mn, B, ldb, b_mn, M, N, K, g, 0, num_sms);
    } else {  // scaled, or rows that no 16-byte store reaches or that end inside one
        GemmExt x{};
        x.alpha = alpha;
        g.epi = kEpiLinear;
        x.out_f32 = out_f32;
        x.resid = accumulate ? out : nullptr;
        x.ldr = ldo;
        rc = gemm_make_plan(&plan, A, lda, a_mn, B, ldb, b_mn, M, N, K, g, 0, num_sms, &x);
    }
    return rc ? rc : gemm_run(plan, s);
}

int linear_forward(const LinearFwd& a, int num_sms, cudaStream_t s) {
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.act < kActNone || a.act > kActSilu) return -1;
    if (a.M == 0) return 0;
    if (!a.x || !a.w || !a.out) return -1;
    if (!operand_ok(a.x, a.ldx) || !operand_ok(a.w, a.ldw)) return kBadOperand;
    if (a.M <= kFewRows) {
        RowsArgs r{a.x, a.ldx, a.w, a.ldw, nullptr, a.bias, a.act, a.drop, a.resid, a.ldr, a.pre, a.ld_pre,
                   a.out, a.out_f32, a.ldo, a.M, a.N, a.K};
        if (r.drop.thr == 0) r.drop.rng = nullptr;
        return rows_product(r, a.w_mn_major, s);
    }
    GemmArgs g{};
    g.epi = kEpiLinear;
    g.out = a.out;
    g.ldo = a.ldo;
    g.aux = a.pre;
    g.ld_aux = a.ld_pre;
    g.splits = 1;
    g.err = a.err;
    GemmExt x{};
    x.bias = a.bias;
    x.act = a.act;
    x.out_f32 = a.out_f32;
    x.resid = a.resid;
    x.ldr = a.ldr;
    if (a.drop.thr > 0) {
        x.rng = a.drop.rng;
        x.site = a.drop.site;
        x.drop_thr = a.drop.thr;
        x.drop_scale = a.drop.scale;
    }
    GemmPlan plan;
    const int rc = gemm_make_plan(&plan, a.x, a.ldx, 0, a.w, a.ldw, a.w_mn_major, a.M, a.N, a.K, g,
                                  0, num_sms, &x);
    return rc ? rc : gemm_run(plan, s);
}

size_t linear_backward_work(int M, int N, int K) {
    (void)K;
    if (M <= 0 || N <= 0) return 0;
    return align256((size_t)M * ceil8(N) * 2) + align256((size_t)dz_groups(M, N) * N * 4);
}

int linear_backward(const LinearBwd& a, int num_sms, cudaStream_t s) {
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.act < kActNone || a.act > kActSilu) return -1;
    if (a.accumulate && a.dw && !a.dw_f32) return -1;
    if (a.M == 0) {  // no rows: zero gradients, or nothing to add
        if (a.accumulate) return 0;
        const size_t es = a.dw_f32 ? 4 : 2;
        const int rows = a.w_mn_major ? a.K : a.N, cols = a.w_mn_major ? a.N : a.K;
        if (a.dw && cudaMemset2DAsync(a.dw, a.lddw * es, 0, cols * es, rows, s) != cudaSuccess)
            return launch_status();
        if (a.dbias && cudaMemsetAsync(a.dbias, 0, (size_t)a.N * 4, s) != cudaSuccess)
            return launch_status();
        return 0;
    }
    if (!a.dy || (a.act != kActNone && !a.pre)) return -1;
    if ((a.dx && !a.w) || (a.dw && !a.x)) return -1;
    if ((a.dx && !operand_ok(a.w, a.ldw)) || (a.dw && !operand_ok(a.x, a.ldx))) return kBadOperand;
    const bool drops = a.drop.rng && a.drop.thr > 0;
    const bool as_is = !a.dy_f32 && a.act == kActNone && !drops && aligned16(a.dy) &&
                       (a.lddy & 7) == 0;  // dy is the products' operand itself
    const bool need_dz = !as_is && (a.dx || a.dw);
    const bf16* dz = reinterpret_cast<const bf16*>(a.dy);
    long long ldz = a.lddy;
    if (need_dz || a.dbias) {
        if (!a.work || !aligned16(a.work)) return -1;
        bf16* buf = reinterpret_cast<bf16*>(a.work);
        float* part = reinterpret_cast<float*>(reinterpret_cast<char*>(a.work) +
                                               align256((size_t)a.M * ceil8(a.N) * 2));
        const int groups = dz_groups(a.M, a.N);
        DropArgs drop = a.drop;
        if (!drops) drop.rng = nullptr;
        const int per16 = a.dy_f32 ? 4 : 8;
        const int vec = aligned16(a.dy) && (a.lddy % per16) == 0 &&
                        (a.act == kActNone || (aligned16(a.pre) && (a.ld_pre & 7) == 0));
        const dim3 grid((a.N + kDzCols - 1) / kDzCols, groups);
        bf16* to = need_dz ? buf : nullptr;
        float* sums = !a.dbias ? nullptr : groups == 1 ? a.dbias : part;
        int rc = a.dy_f32 ? launch_dz<float>(a, drop, grid, to, sums, vec, s)
                          : launch_dz<bf16>(a, drop, grid, to, sums, vec, s);
        if (rc) return rc;
        if (a.dbias && groups > 1) {
            rc = launch_kernel(linear_db_kernel, (a.N + 31) / 32, 1024, 0, s, part, groups, a.N,
                               a.dbias, a.accumulate);
            if (rc) return rc;
        }
        if (need_dz) {
            dz = buf;
            ldz = ceil8(a.N);
        }
    }
    if (a.dx) {  // dz [M,N] times w
        const int rc = product(dz, ldz, 0, a.w, a.ldw, a.w_mn_major ? 0 : 1, a.M, a.K, a.N, a.dx,
                               a.dx_f32, a.lddx, 0, num_sms, a.err, s);
        if (rc) return rc;
    }
    if (a.dw) {
        const int rc =
            a.w_mn_major
                ? product(a.x, a.ldx, 1, dz, ldz, 1, a.K, a.N, a.M, a.dw, a.dw_f32, a.lddw,
                          a.accumulate, num_sms, a.err, s)
                : product(dz, ldz, 1, a.x, a.ldx, 1, a.N, a.K, a.M, a.dw, a.dw_f32, a.lddw,
                          a.accumulate, num_sms, a.err, s);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace llmgpu
