// Linear layer with bias, activation, dropout and residual applied where the product's tiles leave
// tensor memory (gemm.cu, kEpiLinear), and its backward: one elementwise pass forms dz in bf16
// and the bias gradient's partial sums, then two products give dx and dw. dz is rounded to bf16
// because it is a tensor-core operand; the bias gradient is summed before that rounding, and dw of up
// to 8 rows, whose outer products run on the CUDA cores, takes it in f32. (dx of few rows goes
// through the tensor cores too: dz in three bf16 terms cost it 1 to 5 us of 4 to 11.)
// 8192 x 1024 x 4096: forward gelu 64 us (cuBLAS's bare product 57), backward 133 us (34 dz, 4
// dbias, 95 the products); 8192 x 4096 x 1024 with dropout and f32 residual 68 us.
#include "linear.cuh"

#include "act.cuh"
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
    const int most = (M + 2 * kDzRows - 1) / (2 * kDzRows);  // two rows a warp at least
    if (gy > most) gy = most;
    return gy < 1 ? 1 : gy;
}

// dz [M][ldz] in bf16 and in f32 (each nullable) and the column sums of a block's rows,
// part[gy][N] (nullable; with one row of blocks it is dbias itself, added to when `accumulate`).
// `vec`: rows of dy and pre start on 16 bytes. A thread takes 8 columns of kDzInFlight rows at a
// time, their loads in flight together as raw words. Bound by memory: 8192 x 4096 bf16 gelu, 201 MB,
// 34 us (5.9 TB/s). With an activation alone, the compiler's own choice of registers left a block
// less on an SM than fits with a few spilled bytes: 4 of bf16 rather than 3 (gelu with its dx product
// over K = 64 57 -> 53 us, relu 52 -> 48, silu 56 -> 54), 3 of f32 rather than 2 (gelu 68 -> 63, the
// others as before). With dropout or no activation its choice is as fast or faster.
constexpr int kDzInFlight = 2;
template <typename T, int ACT, bool DROP>
constexpr int kDzBlocks = DROP || ACT == kActNone ? 0 : sizeof(T) == 2 ? 4 : 3;  // 0: its choice
template <typename T, int ACT, bool DROP>
__global__ void __launch_bounds__(256, kDzBlocks<T, ACT, DROP>) linear_dz_kernel(
    const T* __restrict__ dy, long long lddy, const bf16* __restrict__ pre, long long ld_pre,
    DropArgs drop, bf16* __restrict__ dz, float* __restrict__ dz32, long long ldz,
    float* __restrict__ part, int accumulate, int M, int N, int vec) {
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
                // behind act', so that a dropped place is 0 whatever dy and pre hold there
                if constexpr (DROP)
                    drop_apply8(key, (uint32_t)col >> 3, (uint32_t)row, drop.thr, drop.scale, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fadd2(sum[i], make_float2(v[2 * i], v[2 * i + 1]));
                // columns past N, up to the padded stride, are written as zeros
                if (dz) store8(dz + row * ldz + col, v);
                if (dz32) store8(dz32 + row * ldz + col, v);
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
int launch_dz_act(const LinearBwd& a, const DropArgs& drop, dim3 grid, bf16* to, float* to32,
                  float* sums, int vec, cudaStream_t s) {
    const int accumulate = grid.y == 1 && a.accumulate;
    return launch_kernel(drop.rng ? linear_dz_kernel<T, ACT, true> : linear_dz_kernel<T, ACT, false>,
                         grid, 256, 0, s, (const T*)a.dy, a.lddy, a.pre, a.ld_pre, drop, to, to32,
                         ceil8(a.N), sums, accumulate, a.M, a.N, vec);
}
template <typename T>
int launch_dz(const LinearBwd& a, const DropArgs& drop, dim3 grid, bf16* to, float* to32, float* sums,
              int vec, cudaStream_t s) {
    switch (a.act) {
        case kActRelu:
            return launch_dz_act<T, kActRelu>(a, drop, grid, to, to32, sums, vec, s);
        case kActGelu:
            return launch_dz_act<T, kActGelu>(a, drop, grid, to, to32, sums, vec, s);
        case kActSilu:
            return launch_dz_act<T, kActSilu>(a, drop, grid, to, to32, sums, vec, s);
        default:
            return launch_dz_act<T, kActNone>(a, drop, grid, to, to32, sums, vec, s);
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

// out = resid + drop(act(alpha sum_p planes[p] + bias)) over planes [n][M][ldp] of a product split
// along K: a thread takes 8 columns, two planes' loads in flight. Bound by memory.
template <typename TO>
__global__ void __launch_bounds__(256) linear_finish_kernel(const RowsArgs a,
                                                            const float* __restrict__ planes, int n,
                                                            int ldp, uint32_t n8, uint32_t dr,
                                                            uint32_t dc, int vec) {
    pdl_enter();
    const long long plane = (long long)a.M * ldp;
    const float f = a.alpha ? *a.alpha : 1.0f;
    DropKey key{};
    if (a.drop.rng) key = drop_key(a.drop.rng, a.drop.site);
    const uint32_t first = blockIdx.x * 256u + threadIdx.x;
    uint32_t row = first / n8, c8 = first - row * n8;
    const uint32_t rows = (uint32_t)a.M;
    while (row < rows) {
        const int col = (int)(c8 * 8), left = min(8, a.N - col);
        const float* p = planes + (long long)row * ldp + col;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        for (int k0 = 0; k0 < n; k0 += 2) {
            Raw8<float> q[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (k0 + k < n) load_raw(p + (k0 + k) * plane, q[k]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (k0 + k < n) {
                    float w[8];
                    raw_f32(q[k], w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += w[j];
                }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= f;
        if (a.bias)
            for (int j = 0; j < left; ++j) v[j] += a.bias[col + j];
        if (a.pre)
            for (int j = 0; j < left; ++j) a.pre[row * a.ld_pre + col + j] = __float2bfloat16_rn(v[j]);
        with_act(a.act, [&](auto tag) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float2 y = act_pair<decltype(tag)::value>(make_float2(v[j], v[j + 1]));
                v[j] = y.x;
                v[j + 1] = y.y;
            }
        });
        if (a.drop.rng) drop_apply8(key, c8, row, a.drop.thr, a.drop.scale, v);
        TO* o = reinterpret_cast<TO*>(a.out) + row * a.ldo + col;
        const TO* r = reinterpret_cast<const TO*>(a.resid) + row * a.ldr + col;
        if (vec && left == 8) {
            if (a.resid) {
                Raw8<TO> q;
                float w[8];
                load_raw(r, q);
                raw_f32(q, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += w[j];
            }
            store8(o, v);
        } else {
            for (int j = 0; j < left; ++j) o[j] = from_f32<TO>(a.resid ? v[j] + to_f32(r[j]) : v[j]);
        }
        row += dr;
        c8 += dc;
        if (c8 >= n8) {
            c8 -= n8;
            ++row;
        }
    }
}

template <typename TO>
int launch_finish(const RowsArgs& a, const float* planes, int n, int ldp, cudaStream_t s) {
    const uint32_t n8 = (uint32_t)(a.N + 7) / 8;
    const long long items = (long long)a.M * n8, most = 148 * 8;
    const uint32_t blocks = (uint32_t)((items + 255) / 256 < most ? (items + 255) / 256 : most);
    const uint32_t step = blocks * 256;
    const int vec = rows_on_16((const TO*)a.out, a.ldo) &&
                    (!a.resid || rows_on_16((const TO*)a.resid, a.ldr));
    return launch_kernel(linear_finish_kernel<TO>, (int)blocks, 256, 0, s, a, planes, n, ldp, n8,
                         step / n8, step % n8, vec);
}

}  // namespace

// A product whose 128 x 64 tiles fill less than half of the SMs walks its K on few of them, at about
// 0.27 us a k-block; split along K it fills them, for a second kernel of about 4 us. 256 x 4096 x 512:
// 18 us in one piece.
int product_splits(int M, int N, int K) {
    const long long tiles = (long long)((M + 127) / 128) * ((N + 63) / 64);
    const int kb = (K + 63) / 64;
    if (M <= kFewRows || tiles > 74 || kb < 32) return 1;
    long long n = 148 / tiles;
    if (n > kb / 8) n = kb / 8;
    return n > 16 ? 16 : (int)n;
}
size_t product_work(int M, int N, int K) {
    const int n = product_splits(M, N, K);
    return n > 1 ? align256((size_t)n * M * ceil8(N) * 4) : 0;
}

int finish_planes(const RowsArgs& a, const float* planes, int n, int ldp, cudaStream_t s) {
    return a.out_f32 ? launch_finish<float>(a, planes, n, ldp, s)
                     : launch_finish<bf16>(a, planes, n, ldp, s);
}

namespace {

// The k-split product of A and B into planes, then the epilogue `a`.
int split_product(const bf16* A, long long lda, int a_mn, const bf16* B, long long ldb, int b_mn, int K,
                  int n, void* work, const RowsArgs& a, int num_sms, int* err, int early,
                  cudaStream_t s) {
    GemmArgs g{};
    g.epi = kEpiPlaneAdd;
    g.out = work;
    g.ldo = ceil8(a.N);
    g.splits = n;
    g.err = err;
    g.early = early;
    GemmExt x{};
    x.out_f32 = a.out_f32;
    GemmPlan plan;
    int rc = gemm_make_plan(&plan, A, lda, a_mn, B, ldb, b_mn, a.M, a.N, K, g, 0, num_sms, &x);
    if (rc) return rc;
    if ((rc = gemm_run(plan, s)) != 0) return rc;
    return finish_planes(a, reinterpret_cast<const float*>(work), n, (int)ceil8(a.N), s);
}

}  // namespace

int product(const bf16* A, long long lda, int a_mn, const bf16* B, long long ldb, int b_mn, int M,
            int N, int K, void* out, int out_f32, long long ldo, int accumulate, int num_sms,
            int* err, cudaStream_t s, const float* alpha, void* work, int early) {
    if (accumulate && !out_f32) return -1;
    if (M <= kFewRows && !a_mn) {
        RowsArgs r{A, lda, B, ldb, alpha, nullptr, kActNone, {}, accumulate ? out : nullptr, ldo, nullptr, 0,
                   out, out_f32, ldo, M, N, K};
        return rows_product(r, b_mn, s);
    }
    if (K <= kOuterRows && a_mn && b_mn)
        return outer_product(A, lda, B, ldb, 0, M, N, K, out, out_f32, ldo, accumulate, alpha, s);
    if (const int n = work ? product_splits(M, N, K) : 1; n > 1) {
        RowsArgs r{nullptr, 0, nullptr, 0, alpha, nullptr, kActNone, {}, accumulate ? out : nullptr, ldo,
                   nullptr, 0, out, out_f32, ldo, M, N, K};
        return split_product(A, lda, a_mn, B, ldb, b_mn, K, n, work, r, num_sms, err,
                             early, s);
    }
    GemmArgs g{};
    g.out = out;
    g.ldo = ldo;
    g.splits = 1;
    g.err = err;
    g.early = early;
    GemmPlan plan;
    int rc;
    if (!alpha && !out_f32 && aligned16(out) && (ldo & 7) == 0 && (N & 7) == 0) {
        g.epi = kEpiStoreBF16;
        rc = gemm_make_plan(&plan, A, lda, a_mn, B, ldb, b_mn, M, N, K, g,
                            gemm_pick_tile(M, N, K, 1, 1.0, false, true, num_sms), num_sms);
    } else {  // scaled, f32 (whose long sums go by chains), or rows not on or not ending on 16 bytes
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
    if (a.M > kMaxDim || a.N > kMaxDim || a.K > kMaxDim) return -1;
    if (a.M == 0) return 0;
    if (!a.x || !a.w || !a.out) return -1;
    if (a.out == a.resid && a.M > 1 && a.ldo != a.ldr) return -1;  // in place, every element keeps its place
    if (!operand_ok(a.x, a.ldx) || !operand_ok(a.w, a.ldw) || !operand_ok(a.work, 0))
        return kBadOperand;
    const int n = a.work ? product_splits(a.M, a.N, a.K) : 1;
    if (a.M <= kFewRows || n > 1) {
        RowsArgs r{a.x, a.ldx, a.w, a.ldw, nullptr, a.bias, a.act, a.drop, a.resid, a.ldr, a.pre, a.ld_pre,
                   a.out, a.out_f32, a.ldo, a.M, a.N, a.K};
        if (r.drop.thr == 0) r.drop.rng = nullptr;
        return n > 1 ? split_product(a.x, a.ldx, 0, a.w, a.ldw, a.w_mn_major, a.K, n, a.work, r,
                                     num_sms, a.err, 0, s)
                     : rows_product(r, a.w_mn_major, s);
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

namespace {

// The backward's workspace: dz in bf16, the row groups' column sums, the planes of the products (dw's
// follow dx's in the same place), dz in f32 where rows are few. Byte offsets and the whole.
struct BackwardLayout {
    size_t part, planes, dz32, total;
};
BackwardLayout backward_layout(int M, int N, int K) {
    // dw is [N, K] or [K, N]: the larger of the two
    size_t planes = product_work(M, K, N);
    const size_t dw = product_work(N, K, M), dw_mn = product_work(K, N, M);
    if (dw > planes) planes = dw;
    if (dw_mn > planes) planes = dw_mn;
    BackwardLayout l;
    l.part = align256((size_t)M * ceil8(N) * 2);
    l.planes = l.part + align256((size_t)dz_groups(M, N) * N * 4);
    l.dz32 = l.planes + planes;
    l.total = l.dz32 + (M <= kOuterRows ? align256((size_t)M * ceil8(N) * 4) : 0);
    return l;
}

}  // namespace

size_t linear_backward_work(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > kMaxDim || N > kMaxDim || K > kMaxDim) return 0;
    return backward_layout(M, N, K).total;
}

int linear_backward(const LinearBwd& a, int num_sms, cudaStream_t s) {
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.act < kActNone || a.act > kActSilu) return -1;
    if (a.M > kMaxDim || a.N > kMaxDim || a.K > kMaxDim) return -1;
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
    if ((a.dx && !operand_ok(a.w, a.ldw)) || (a.dw && !operand_ok(a.x, a.ldx)) ||
        !operand_ok(a.work, 0))
        return kBadOperand;
    const bool drops = a.drop.rng && a.drop.thr > 0;
    const bool as_is = !a.dy_f32 && a.act == kActNone && !drops && aligned16(a.dy) &&
                       (a.lddy & 7) == 0;  // dy is the products' operand itself
    const bool need_dz = !as_is && (a.dx || a.dw);
    const bf16* dz = reinterpret_cast<const bf16*>(a.dy);
    long long ldz = a.lddy;
    const BackwardLayout l = backward_layout(a.M, a.N, a.K);
    char* const work = reinterpret_cast<char*>(a.work);
    void* planes = work ? work + l.planes : nullptr;
    float* dz32 = nullptr;  // of few rows, for dw
    // the products need not wait for what runs in front of them once dz's own kernel has ended: dx
    // for the second stage of dbias, dw for it and for dx (unless dx's planes lie where dw's go)
    int early = 0;
    if (need_dz || a.dbias) {
        if (!a.work) return -1;
        bf16* buf = reinterpret_cast<bf16*>(work);
        float* part = reinterpret_cast<float*>(work + l.part);
        if (need_dz && a.dw && a.M <= kOuterRows) dz32 = reinterpret_cast<float*>(work + l.dz32);
        const int groups = dz_groups(a.M, a.N);
        DropArgs drop = a.drop;
        if (!drops) drop.rng = nullptr;
        const int per16 = a.dy_f32 ? 4 : 8;
        const int vec = aligned16(a.dy) && (a.lddy % per16) == 0 &&
                        (a.act == kActNone || (aligned16(a.pre) && (a.ld_pre & 7) == 0));
        const dim3 grid((a.N + kDzCols - 1) / kDzCols, groups);
        bf16* to = need_dz && (a.dx || !dz32) ? buf : nullptr;
        float* sums = !a.dbias ? nullptr : groups == 1 ? a.dbias : part;
        int rc = a.dy_f32 ? launch_dz<float>(a, drop, grid, to, dz32, sums, vec, s)
                          : launch_dz<bf16>(a, drop, grid, to, dz32, sums, vec, s);
        if (rc) return rc;
        if (a.dbias && groups > 1) {
            rc = launch_kernel_pdl(linear_db_kernel, (a.N + 31) / 32, 1024, 0, s, part, groups, a.N,
                               a.dbias, a.accumulate);
            if (rc) return rc;
            early = 1;
        }
        if (need_dz) {
            dz = buf;
            ldz = ceil8(a.N);
        }
    }
    if (a.dx) {  // dz [M,N] times w
        const int rc = product(dz, ldz, 0, a.w, a.ldw, a.w_mn_major ? 0 : 1, a.M, a.K, a.N, a.dx,
                               a.dx_f32, a.lddx, 0, num_sms, a.err, s, nullptr, planes, early);
        if (rc) return rc;
        early = (!planes || product_splits(a.M, a.K, a.N) == 1) && leaves_room(a.M, a.K, 1);
    }
    if (a.dw && dz32)
        return a.w_mn_major ? outer_product(a.x, a.ldx, dz32, ldz, 2, a.K, a.N, a.M, a.dw, a.dw_f32,
                                            a.lddw, a.accumulate, nullptr, s)
                            : outer_product(dz32, ldz, a.x, a.ldx, 1, a.N, a.K, a.M, a.dw, a.dw_f32,
                                            a.lddw, a.accumulate, nullptr, s);
    if (a.dw) {
        const int rc =
            a.w_mn_major
                ? product(a.x, a.ldx, 1, dz, ldz, 1, a.K, a.N, a.M, a.dw, a.dw_f32, a.lddw,
                          a.accumulate, num_sms, a.err, s, nullptr, planes, early)
                : product(dz, ldz, 1, a.x, a.ldx, 1, a.N, a.K, a.M, a.dw, a.dw_f32, a.lddw,
                          a.accumulate, num_sms, a.err, s, nullptr, planes, early);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace llmgpu
