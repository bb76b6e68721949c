// The linear layer with its epilogue (bias, activation, dropout, residual), its backward, and the
// loss head that keeps no logits. All launchers are asynchronous on `s` and return 0 or a
// negative status.
#pragma once
#include "gemm.cuh"
#include "kernels.cuh"

namespace llmgpu {

// Status of an operand whose rows do not start on 16 bytes (the tensor maps need it).
constexpr int kBadOperand = -3;
inline bool operand_ok(const void* p, long long ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0;
}

// Sizes at most: the index arithmetic of tiles stays in 32 bits.
constexpr int kMaxDim = 1 << 30;

// Dropout of a linear layer's output; thr 0 keeps everything.
struct DropArgs {
    const uint64_t* rng;  // device {seed, offset}; null: no dropout
    uint64_t site;
    uint32_t thr;
    float scale;
};

// out[M,N] = resid + drop(act(x[M,K] w^T + bias)); w is [N,K], or [K,N] with w_mn_major. pre
// (nullable, bf16) receives x w^T + bias. out and resid: f32 or bf16.
struct LinearFwd {
    const bf16* x;
    long long ldx;
    const bf16* w;
    long long ldw;
    int w_mn_major;
    const float* bias;
    int act;
    DropArgs drop;
    const void* resid;
    long long ldr;
    bf16* pre;
    long long ld_pre;
    void* out;
    int out_f32;
    long long ldo;
    int M, N, K;
    void* work;  // product_work(M, N, K) bytes, 16-byte aligned; null: K is not split
    int* err;
};
int linear_forward(const LinearFwd& a, int num_sms, cudaStream_t s);

// dz = drop(dy act'(pre)), dbias (+)= column sums of dz, dx = dz w, dw (+)= dz^T x (laid out as w). The
// tensor cores take dz in bf16; dw of up to kOuterRows rows, which they do not form, takes it in f32.
// dx, dw, dbias nullable.
struct LinearBwd {
    const void* dy;
    int dy_f32;
    long long lddy;
    const bf16* x;
    long long ldx;
    const bf16* w;
    long long ldw;
    int w_mn_major;
    const bf16* pre;
    long long ld_pre;
    int act;
    DropArgs drop;
    void* dx;
    int dx_f32;
    long long lddx;
    void* dw;
    int dw_f32;
    long long lddw;
    float* dbias;
    int accumulate;  // into dw (f32 only) and dbias
    int M, N, K;
    void* work;  // linear_backward_work bytes, 16-byte aligned
    int* err;
};
size_t linear_backward_work(int M, int N, int K);
int linear_backward(const LinearBwd& a, int num_sms, cudaStream_t s);

// Loss head on x [rows, C] and w [V, C] (or [C, V] with w_mn_major): row_loss = on (lse - z_t) +
// off sum_{v != t} (lse - z_v), on = 1 - smoothing, off = smoothing / (V - 1) (the gradient of
// cross_entropy_fwd_bwd, whose loss leaves the smoothing out); a row whose target is outside [0, V) is left out: loss 0.
struct HeadArgs {
    const bf16* x;
    long long ldx;
    const bf16* w;
    long long ldw;
    int w_mn_major;
    const int32_t* targets;
    int rows, C, V;
    float smoothing;
    void* work;
    int* err;
};
size_t head_forward_work(int rows, int V);
int head_forward(const HeadArgs& a, float* row_loss, float* lse, int num_sms, cudaStream_t s);
// Gradients of sum_r scale * dloss[r] * row_loss[r] (dloss nullable: ones), in pieces of `piece`
// columns of the vocabulary (0: chosen here). Rows left out contribute nothing, whatever x
// holds there. dx, dw nullable; dw is laid out as w, and added to when `accumulate` (f32 only).
int head_piece(int rows, int C, int V, int piece);
size_t head_backward_work(int rows, int C, int V, int piece);
int head_backward(const HeadArgs& a, const float* lse, const float* dloss, float scale, void* dx,
                  int dx_f32, long long lddx, void* dw, int dw_f32, long long lddw, int accumulate,
                  int piece, int num_sms, cudaStream_t s);

// Products of a few rows (linear_rows.cu): decoding, where every weight is read once and a 128-row
// tile would be empty. out [M <= kFewRows, N] = resid + drop(act(alpha x w^T + bias)), w [N, K] or
// (w_mn) [K, N].
constexpr int kFewRows = 16;
struct RowsArgs {
    const bf16* x;
    long long ldx;
    const bf16* w;
    long long ldw;
    const float* alpha;
    const float* bias;
    int act;
    DropArgs drop;
    const void* resid;
    long long ldr;
    bf16* pre;
    long long ld_pre;
    void* out;
    int out_f32;
    long long ldo;
    int M, N, K;
};
int rows_product(const RowsArgs& a, int w_mn, cudaStream_t s);
// out[M,N] (+)= alpha sum_k A[k,M] B[k,N] over K <= kOuterRows rows: bound by the result's writes.
// A and B are bf16, or one of them (f32: 1 A, 2 B) f32 with rows padded to 8 elements, on 16 bytes.
constexpr int kOuterRows = 8;
int outer_product(const void* A, long long lda, const void* B, long long ldb, int f32, int M, int N,
                  int K, void* out, int out_f32, long long ldo, int accumulate, const float* alpha,
                  cudaStream_t s);

// Splits along K of a product with too few tiles for the device, and the bytes of their planes.
int product_splits(int M, int N, int K);
size_t product_work(int M, int N, int K);
// Whether a product leaves SMs idle for the one behind it to start on: fewer 256 x 256 tiles than the 74
// pairs. Where it fills them, two products at once only compete (8192 x 768 x 50257 backward: 0.8%
// slower).
inline bool leaves_room(int M, int N, int splits) {
    return (long long)((M + 255) / 256) * ((N + 255) / 256) * splits < 74;
}
// out = resid + drop(act(alpha sum of planes [n][M][ldp] + bias)) (x, w of `a` unused); ldp: a
// multiple of 8.
int finish_planes(const RowsArgs& a, const float* planes, int n, int ldp, cudaStream_t s);

// D[M,N] (+)= alpha A B^T on the tcgen05 kernels into bf16 or f32 `out`, any row stride (accumulate:
// f32 only; alpha: device scalar, nullable; work: product_work(M, N, K) bytes, or null; early: see
// GemmArgs, of use where the tcgen05 kernels run).
int product(const bf16* A, long long lda, int a_mn, const bf16* B, long long ldb, int b_mn, int M,
            int N, int K, void* out, int out_f32, long long ldo, int accumulate, int num_sms,
            int* err, cudaStream_t s, const float* alpha = nullptr, void* work = nullptr,
            int early = 0);

}  // namespace llmgpu
