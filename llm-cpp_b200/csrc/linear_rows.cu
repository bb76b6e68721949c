// Linear-layer products of a few rows (decoding, single sequences): the weights are streamed once,
// 16 bytes a lane straight into mma.sync fragments, with no tile, tensor map or staging between.
// The legacy matrix instructions carry them because a tcgen05 tile is 128 rows high: 64-wide tcgen05
// tiles took 18 us for 4096 x 4096.
// With bias and gelu, in graph replays, weights in L2 and (other weights of 320 MB in between) in HBM:
//   rows x K x N          w [N, K] L2 / HBM us     w [K, N]          floor (bytes at 6.48 TB/s)
//    1 x 1024 x 4096          3.4 /  4.1            3.5 /  4.0        1.3
//    1 x 4096 x 1024          5.5 /  6.9            9.0 / 10.2        1.3
//    1 x 4096 x 4096          7.2 / 10.4            9.1 / 11.1        5.2
//   16 x 4096 x 4096          8.4 / 11.4           10.7 / 12.9        5.2
// From HBM 3.2 TB/s at best: a launch, the wait for the kernel in front and one DRAM latency stand in a
// row, and w [K, N] has a block to 32 columns only, whatever K is.
#include "common.cuh"
#include "linear.cuh"
#include "philox.cuh"
#include "rowio.cuh"

namespace llmgpu {

namespace {

// D (16 x 8, f32) += A (16 x 16) B (16 x 8), bf16. Lane (g, t) = (lane / 4, lane % 4) holds of A rows g
// and g + 8, k 2t, 2t+1 and 2t+8, 2t+9 (a0..a3: row g, row g + 8, row g upper k, row g + 8 upper k), of
// B the same k in column g, of D columns 2t, 2t + 1 of rows g (d0, d1) and g + 8 (d2, d3).
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The epilogue of one element.
__device__ __forceinline__ void rows_store(const RowsArgs& a, int m, int n, float z) {
    if (a.alpha) z *= *a.alpha;
    if (a.bias) z += a.bias[n];
    if (a.pre) a.pre[m * a.ld_pre + n] = __float2bfloat16_rn(z);
    float y = z;
    if (a.act == kActRelu) {
        y = z <= 0.0f ? 0.0f : z;
    } else if (a.act == kActGelu) {
        const float t = -1.5957691216f * 1.4426950408889634f * z * fmaf(0.044715f * z, z, 1.0f);
        y = z * rcp_approx(1.0f + ex2_approx(t));
    } else if (a.act == kActSilu) {
        y = z * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z));
    }
    if (a.drop.rng) {
        const DropKey key = drop_key(a.drop.rng, a.drop.site);
        const uint32_t keep = drop_keep8(key, (uint32_t)n >> 3, (uint32_t)m, a.drop.thr);
        y = ((keep >> (n & 7)) & 1u) ? y * a.drop.scale : 0.0f;
    }
    if (a.out_f32) {
        if (a.resid) y += reinterpret_cast<const float*>(a.resid)[m * a.ldr + n];
        reinterpret_cast<float*>(a.out)[m * a.ldo + n] = y;
    } else {
        if (a.resid) y += __bfloat162float(reinterpret_cast<const bf16*>(a.resid)[m * a.ldr + n]);
        reinterpret_cast<bf16*>(a.out)[m * a.ldo + n] = __float2bfloat16_rn(y);
    }
}

// E bf16 of a row from k on, zeros past K; whole chunks are aligned to their size.
template <int E>
__device__ __forceinline__ void row_chunk(const bf16* p, int k, int K, uint32_t (&u)[E / 2]) {
    if (k + E <= K) {
        if constexpr (E == 8) {
            const uint4 q = *reinterpret_cast<const uint4*>(p + k);
            u[0] = q.x, u[1] = q.y, u[2] = q.z, u[3] = q.w;
        } else {
            const uint2 q = *reinterpret_cast<const uint2*>(p + k);
            u[0] = q.x, u[1] = q.y;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        const int j = k + 2 * i;
        const uint32_t lo = j < K ? __bfloat16_as_ushort(p[j]) : 0u;
        const uint32_t hi = j + 1 < K ? __bfloat16_as_ushort(p[j + 1]) : 0u;
        u[i] = lo | hi << 16;
    }
}

// ------------------------------------------------------------------------------- w [N, K]
// A warp forms 16 output columns (rows of w: the A operand) by up to 16 rows of x (B, MT tiles of 8)
// over its share of K. A lane's 16 bytes of a row are k 8t .. 8t + 7 of 32: two MMAs whose k are
// permuted alike on both sides. 128 of K are in flight; their sums leave the MMA accumulators
// after each 128, so the tensor cores' truncation does not grow with K. KS warps of a block share
// 16 columns and meet in shared memory.
constexpr int kRowsWarps = 8;
template <int MT>
__global__ void __launch_bounds__(32 * kRowsWarps) linear_rows_kernel(const RowsArgs a, int KS) {
    pdl_enter();
    __shared__ float part[kRowsWarps][16][8 * MT + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int groups = kRowsWarps / KS;  // of 16 columns, in this block
    const int n0 = (blockIdx.x * groups + warp / KS) * 16;
    float sum[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
    const bf16* w0 = a.w + (n0 + g) * a.ldw;
    const bf16* w1 = w0 + 8 * a.ldw;
    const bool in0 = n0 + g < a.N, in1 = n0 + g + 8 < a.N;
    for (int k0 = 128 * (warp % KS) + 8 * t; k0 < a.K + 8 * t; k0 += 128 * KS) {
        uint32_t u0[4][4], u1[4][4], v[MT][4][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int k = k0 + 32 * c;
#pragma unroll
            for (int i = 0; i < 4; ++i) u0[c][i] = u1[c][i] = 0u;
            if (in0 && k < a.K) row_chunk<8>(w0, k, a.K, u0[c]);
            if (in1 && k < a.K) row_chunk<8>(w1, k, a.K, u1[c]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[m][c][i] = 0u;
                if (8 * m + g < a.M && k < a.K)
                    row_chunk<8>(a.x + (8 * m + g) * a.ldx, k, a.K, v[m][c]);
            }
        }
        __syncwarp();
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                mma_16x8x16(d, u0[c][0], u1[c][0], u0[c][1], u1[c][1], v[m][c][0], v[m][c][1]);
                mma_16x8x16(d, u0[c][2], u1[c][2], u0[c][3], u1[c][3], v[m][c][2], v[m][c][3]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[m][j] += d[j];
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        part[warp][g][8 * m + 2 * t] = sum[m][0];
        part[warp][g][8 * m + 2 * t + 1] = sum[m][1];
        part[warp][g + 8][8 * m + 2 * t] = sum[m][2];
        part[warp][g + 8][8 * m + 2 * t + 1] = sum[m][3];
    }
    __syncthreads();
    const int cols = groups * 16;
    for (int i = threadIdx.x; i < cols * a.M; i += 32 * kRowsWarps) {
        const int m = i / cols, c = i - m * cols;
        const int n = blockIdx.x * cols + c;
        if (n >= a.N) continue;
        float z = 0.0f;
        for (int q = 0; q < KS; ++q) z += part[(c >> 4) * KS + q][c & 15][m];
        rows_store(a, m, n, z);
    }
}

// ------------------------------------------------------------------------------- w [K, N]
// A warp forms up to 16 rows (x: A) by 32 columns over its share of K. A lane reads 4 columns of the
// rows k 4t .. 4t + 3 of 16 (8 bytes each); column 4g + j of the 32 is column g of B tile j, its
// pairs of k put together by byte permutes. 64 of K are in flight and leave the accumulators
// together; the block's 16 warps share the columns.
constexpr int kRowsMnWarps = 16;
__global__ void __launch_bounds__(32 * kRowsMnWarps) linear_rows_mn_kernel(const RowsArgs a) {
    pdl_enter();
    __shared__ float part[kRowsMnWarps][16][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 32, n = n0 + 4 * g;
    float sum[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[j][i] = 0.0f;
    const bf16* x0 = a.x + g * a.ldx;
    const bf16* x1 = x0 + 8 * a.ldx;
    const bool in0 = g < a.M, in1 = g + 8 < a.M;
    for (int k0 = 64 * warp; k0 < a.K; k0 += 64 * kRowsMnWarps) {
        uint32_t w[4][4][2], p[4][2], q[4][2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int k = k0 + 16 * c + 4 * t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[c][i][0] = w[c][i][1] = 0u;
                if (k + i < a.K && n < a.N) row_chunk<4>(a.w + (k + i) * a.ldw, n, a.N, w[c][i]);
            }
            p[c][0] = p[c][1] = q[c][0] = q[c][1] = 0u;
            if (in0 && k < a.K) row_chunk<4>(x0, k, a.K, p[c]);
            if (in1 && k < a.K) row_chunk<4>(x1, k, a.K, q[c]);
        }
        __syncwarp();
        float d[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[j][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // element j of the rows k, k + 1 and of k + 2, k + 3
                const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                const uint32_t b0 = __byte_perm(w[c][0][j >> 1], w[c][1][j >> 1], sel);
                const uint32_t b1 = __byte_perm(w[c][2][j >> 1], w[c][3][j >> 1], sel);
                mma_16x8x16(d[j], p[c][0], q[c][0], p[c][1], q[c][1], b0, b1);
            }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[j][i] += d[j][i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // D column 2t (2t + 1) of tile j is column 8t + j (8t + 4 + j)
        part[warp][g][8 * t + j] = sum[j][0];
        part[warp][g][8 * t + 4 + j] = sum[j][1];
        part[warp][g + 8][8 * t + j] = sum[j][2];
        part[warp][g + 8][8 * t + 4 + j] = sum[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * a.M; i += 32 * kRowsMnWarps) {
        const int m = i >> 5, c = i & 31;
        if (n0 + c >= a.N) continue;
        float z = 0.0f;
#pragma unroll
        for (int q = 0; q < kRowsMnWarps; ++q) z += part[q][m][c];
        rows_store(a, m, n0 + c, z);
    }
}

// --------------------------------------------------------------------------------- outer product
// A warp writes 256 columns (8 a lane) of 8 rows; the lane keeps its columns of B in registers, the
// block's 64 rows of A lie in shared memory as f32. KK: K rounded up to a power of two.
// Everything is f32 but what memory holds in bf16.
constexpr int kOuterTile = 64;
__device__ __forceinline__ void outer_chunk(const bf16* p, int col, int N, float2 (&b)[4]) {
    uint32_t u[4];
    row_chunk<8>(p, col, N, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = make_float2(bf16_lo(u[j]), bf16_hi(u[j]));
}
__device__ __forceinline__ void outer_chunk(const float* p, int col, int, float2 (&b)[4]) {
    Raw8<float> q;
    float v[8];
    load_raw(p + col, q);
    raw_f32(q, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = make_float2(v[2 * j], v[2 * j + 1]);
}
template <typename T, int KK, typename TA, typename TB>
__global__ void __launch_bounds__(256) outer_product_kernel(const TA* __restrict__ A, long long lda,
                                                            const TB* __restrict__ B, long long ldb,
                                                            int M, int N, int K, int tiles_n,
                                                            T* out, long long ldo, int accumulate,
                                                            int vec,
                                                            const float* __restrict__ alpha) {
    pdl_enter();
    __shared__ float sa[KK][kOuterTile];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int bm = blockIdx.x / tiles_n, bn = blockIdx.x - bm * tiles_n;
    const int r0 = bm * kOuterTile, col = bn * 256 + 8 * lane;
    const float f = alpha ? *alpha : 1.0f;
    for (int i = threadIdx.x; i < KK * kOuterTile; i += 256) {
        const int k = i / kOuterTile, r = i - k * kOuterTile;
        sa[k][r] = k < K && r0 + r < M ? to_f32(A[k * lda + r0 + r]) : 0.0f;
    }
    float2 b[KK][4];
#pragma unroll
    for (int k = 0; k < KK; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) b[k][j] = make_float2(0.0f, 0.0f);
        if (k < K && col < N) outer_chunk(B + k * ldb, col, N, b[k]);
    }
    __syncthreads();
    if (col >= N) return;
    const int n = min(8, N - col);
#pragma unroll 4
    for (int i = 0; i < kOuterTile / 8; ++i) {
        const int r = warp * (kOuterTile / 8) + i;
        if (r0 + r >= M) return;
        float2 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < KK; ++k) {
            const float av = sa[k][r];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = ffma2(make_float2(av, av), b[k][j], s[j]);
        }
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = s[j].x * f;
            v[2 * j + 1] = s[j].y * f;
        }
        T* o = out + (r0 + r) * ldo + col;
        if (vec && n == 8) {
            if (accumulate) {
                Raw8<T> q;
                float w[8];
                load_raw(o, q);
                raw_f32(q, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += w[j];
            }
            store8(o, v);
        } else {
            for (int j = 0; j < n; ++j)
                o[j] = from_f32<T>(accumulate ? v[j] + to_f32(o[j]) : v[j]);
        }
    }
}

}  // namespace

int rows_product(const RowsArgs& a, int w_mn, cudaStream_t s) {
    if (w_mn)
        return launch_kernel_pdl(linear_rows_mn_kernel, (a.N + 31) / 32, 32 * kRowsMnWarps, 0, s, a);
    // warps to a group of 16 columns: all eight of a block where K has work for them
    const int KS = a.K > 512 ? 8 : a.K > 256 ? 4 : a.K > 128 ? 2 : 1;
    const int cols = 16 * (kRowsWarps / KS);
    const int grid = (a.N + cols - 1) / cols;
    return a.M <= 8 ? launch_kernel_pdl(linear_rows_kernel<1>, grid, 32 * kRowsWarps, 0, s, a, KS)
                    : launch_kernel_pdl(linear_rows_kernel<2>, grid, 32 * kRowsWarps, 0, s, a, KS);
}

namespace {
template <typename T, int KK, typename TA, typename TB>
int launch_outer(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K, void* out,
                 long long ldo, int accumulate, const float* alpha, cudaStream_t s) {
    const int tiles_n = (N + 255) / 256;
    const int grid = tiles_n * ((M + kOuterTile - 1) / kOuterTile);
    const int vec = rows_on_16((const T*)out, ldo);
    return launch_kernel(outer_product_kernel<T, KK, TA, TB>, grid, 256, 0, s, (const TA*)A, lda,
                         (const TB*)B, ldb, M, N, K, tiles_n, (T*)out, ldo, accumulate, vec, alpha);
}
template <typename T, typename TA, typename TB>
int launch_outer_k(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K,
                   void* out, long long ldo, int accumulate, const float* alpha, cudaStream_t s) {
    auto* f = K == 1   ? launch_outer<T, 1, TA, TB>
              : K == 2 ? launch_outer<T, 2, TA, TB>
              : K <= 4 ? launch_outer<T, 4, TA, TB>
                       : launch_outer<T, kOuterRows, TA, TB>;
    return f(A, lda, B, ldb, M, N, K, out, ldo, accumulate, alpha, s);
}
}  // namespace

int outer_product(const void* A, long long lda, const void* B, long long ldb, int f32, int M, int N,
                  int K, void* out, int out_f32, long long ldo, int accumulate, const float* alpha,
                  cudaStream_t s) {
    auto* f = f32 == 1   ? (out_f32 ? launch_outer_k<float, float, bf16> : launch_outer_k<bf16, float, bf16>)
              : f32 == 2 ? (out_f32 ? launch_outer_k<float, bf16, float> : launch_outer_k<bf16, bf16, float>)
                         : (out_f32 ? launch_outer_k<float, bf16, bf16> : launch_outer_k<bf16, bf16, bf16>);
    return f(A, lda, B, ldb, M, N, K, out, ldo, accumulate, alpha, s);
}

}  // namespace llmgpu
