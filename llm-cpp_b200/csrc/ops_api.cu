// Kernel-level C ABI (include/llmgpu_ops.h): thin wrappers that run one kernel
// on caller-owned device buffers, used by the per-kernel parity tests.
#include <cuda_runtime.h>
#include <string.h>

#include "common.cuh"
#include "dropout.cuh"
#include "gemm.cuh"
#include "kernels.cuh"
#include "linear.cuh"
#include "llmgpu_ops.h"
#include "moe.cuh"
#include "philox.cuh"

using namespace llmgpu;

static int device_num_sms() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return n > 0 ? n : 148;
}

extern "C" int llmgpu_op_num_sms(void) { return device_num_sms(); }

extern "C" int llmgpu_op_gemm_pair_slots(void) { return gemm_pair_slots(device_num_sms()); }

extern "C" int llmgpu_op_gemm(const void* A, long long lda, int a_mn_major, const void* B,
                              long long ldb, int b_mn_major, int M, int N, int K, int epi,
                              void* out, long long ldo, int accumulate, const float* resid,
                              long long ldr, void* aux, long long ld_aux, int splits,
                              float* workspace, int col_group, long long group_stride, int bn,
                              int* err, void* stream) {
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    GemmArgs g{};
    g.epi = epi;
    g.accumulate = accumulate;
    g.out = out;
    g.ldo = ldo;
    g.col_group = col_group;
    g.group_stride = group_stride;
    g.resid = resid;
    g.ldr = ldr;
    g.aux = aux;
    g.ld_aux = ld_aux;
    g.splits = splits < 1 ? 1 : splits;
    g.err = err;
    if (g.splits > 1) {
        if (epi != kEpiStoreF32 || workspace == nullptr) return -100;
        g.epi = kEpiSplitPartial;
        g.out = workspace;
        g.ldo = N;
    }
    GemmPlan plan;
    int rc = gemm_make_plan(&plan, A, lda, a_mn_major, B, ldb, b_mn_major, M, N, K, g, bn,
                            device_num_sms());
    if (rc) return rc;
    rc = gemm_run(plan, st);
    if (rc) return rc;
    if (g.splits > 1)
        rc = gemm_splitk_reduce(workspace, g.splits, M, N, reinterpret_cast<float*>(out), ldo,
                                col_group <= 0 ? N : col_group, group_stride, accumulate, st);
    return rc;
}

extern "C" int llmgpu_op_embed(const int32_t* tokens, const float* wte, const float* wpe, float* x,
                               int B, int T, int C, int V, void* stream) {
    return embed_forward(tokens, wte, wpe, x, B, T, C, V, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" long long llmgpu_op_embed_bwd_work(int B, int T, int C) {
    const long long n = (long long)B * T;
    return ((n * 8 + 255) / 256) * 256 + n * C * 4;
}

extern "C" int llmgpu_op_embed_bwd(const int32_t* tokens, const float* dx, float* wte_grad,
                                   float* wpe_grad, int B, int T, int C, int V,
                                   int accumulate_wpe, void* work, void* stream) {
    const long long n = (long long)B * T;
    if (B <= 0 || T <= 0 || C <= 0 || V <= 0 || n > 16384 || !work) return -1;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint64_t* keys = reinterpret_cast<uint64_t*>(work);
    float* scratch = reinterpret_cast<float*>(reinterpret_cast<char*>(work) +
                                              ((n * 8 + 255) / 256) * 256);
    const int rc = embed_sort_keys(tokens, (int)n, V, keys, s);
    if (rc) return rc;
    return embed_backward(keys, dx, wte_grad, wpe_grad, B, T, C, accumulate_wpe, scratch, s);
}

extern "C" int llmgpu_op_norm_fwd(const float* x, const float* gamma, const float* beta,
                                  void* y_bf16, float* mean, float* rstd, int rows, int C, int rms,
                                  void* stream) {
    return norm_forward(x, gamma, beta, reinterpret_cast<bf16*>(y_bf16), mean, rstd, rows, C, rms,
                        reinterpret_cast<cudaStream_t>(stream));
}

extern "C" long long llmgpu_op_norm_bwd_work(int rows, int C) {
    return (long long)norm_backward_grid(rows) * 3 * C;
}

extern "C" int llmgpu_op_norm_bwd(const float* dy, const float* x, const float* gamma,
                                  const float* mean, const float* rstd, const float* resid,
                                  float* dx, void* dx_bf16, float* dgamma, float* dbeta,
                                  float* dxsum, float* work, int rows, int C, int rms,
                                  void* stream) {
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    int nparts = 0;
    int rc = norm_backward(dy, x, gamma, mean, rstd, resid, dx, reinterpret_cast<bf16*>(dx_bf16),
                           work, rows, C, rms, &nparts, st);
    if (rc) return rc;
    return reduce_partials(work, nparts, C, dgamma, dbeta, dxsum, 0, st);
}

extern "C" int llmgpu_op_cross_entropy(void* logits_bf16, int rows, int V, int Vp,
                                       const int32_t* tokens, float* row_loss, float scale,
                                       float smoothing, void* stream) {
    return cross_entropy_fwd_bwd(reinterpret_cast<bf16*>(logits_bf16), rows, V, Vp, tokens,
                                 row_loss, scale, smoothing, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_attention_fwd(const void* qkv, void* out, float* lse, int B, int T,
                                       int H, int hd, const float* rope_cs, void* stream) {
    return attention_forward(reinterpret_cast<const bf16*>(qkv), reinterpret_cast<bf16*>(out), lse,
                             B, T, H, hd, reinterpret_cast<const float2*>(rope_cs),
                             reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_attention_fwd_ws(const void* qkv, void* out, float* lse, int B, int T,
                                          int H, int hd, const float* rope_cs, void* work,
                                          void* stream) {
    return attention_forward(reinterpret_cast<const bf16*>(qkv), reinterpret_cast<bf16*>(out), lse,
                             B, T, H, hd, reinterpret_cast<const float2*>(rope_cs),
                             reinterpret_cast<cudaStream_t>(stream), nullptr, work);
}

extern "C" int llmgpu_op_attention_bwd(const void* qkv, const void* out, const void* dout,
                                       const float* lse, float* dvec, void* dqkv, int B, int T,
                                       int H, int hd, const float* rope_cs, void* work,
                                       void* stream) {
    return attention_backward(reinterpret_cast<const bf16*>(qkv), reinterpret_cast<const bf16*>(out),
                              reinterpret_cast<const bf16*>(dout), lse, dvec,
                              reinterpret_cast<bf16*>(dqkv), B, T, H, hd,
                              reinterpret_cast<const float2*>(rope_cs),
                              reinterpret_cast<cudaStream_t>(stream), nullptr, work);
}

extern "C" long long llmgpu_op_attention_bwd_work(int B, int T, int H, int hd) {
    if (B <= 0 || T <= 0 || H <= 0 || hd > 64 || hd < 8 || hd % 8 != 0) return 0;
    return (long long)attention_work_bytes(B, T, H, hd);
}

extern "C" int llmgpu_op_swiglu_fwd(const void* h13, void* gated, int rows, int F, void* stream) {
    return swiglu_forward(reinterpret_cast<const bf16*>(h13), reinterpret_cast<bf16*>(gated), rows,
                          F, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_swiglu_bwd(const void* dgated, const void* h13, void* dh13, int rows,
                                    int F, void* stream) {
    return swiglu_backward(reinterpret_cast<const bf16*>(dgated), reinterpret_cast<const bf16*>(h13),
                           reinterpret_cast<bf16*>(dh13), rows, F,
                           reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_gemm_grouped(const void* A, long long lda, int a_mn_major, const void* B,
                                      long long ldb, int b_mn_major, int M, int N, int K, int epi,
                                      void* out, long long ldo, int accumulate, void* aux,
                                      long long ld_aux, const int* grp, int groups, int mode,
                                      long long b_grp_rows, long long out_grp_stride, int* err,
                                      void* stream) {
    if (mode != kGroupRows && mode != kGroupK) return -100;
    GemmArgs g{};
    g.epi = epi;
    g.accumulate = accumulate;
    g.out = out;
    g.ldo = ldo;
    g.aux = aux;
    g.ld_aux = ld_aux;
    g.splits = 1;
    g.err = err;
    g.grp = grp;
    g.groups = groups;
    g.grp_mode = mode;
    g.b_grp_rows = b_grp_rows;
    g.out_grp_stride = out_grp_stride;
    GemmPlan plan;
    int rc = gemm_make_plan(&plan, A, lda, a_mn_major, B, ldb, b_mn_major, M, N, K, g, 0,
                            device_num_sms());
    if (rc) return rc;
    return gemm_run(plan, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_moe_route(const float* y, const float* mean, const float* rstd,
                                   const float* gamma, const float* beta, int rms,
                                   const float* gate, int B, int T, int C, int E, int k,
                                   float* probs, int* idx, float* wts, float* ssum,
                                   void* stream) {
    MoeDims m{B, T, C, E, k, moe_capacity(B * T, E, k)};
    return moe_router_forward(m, y, mean, rstd, gamma, beta, rms, gate, probs, idx, wts, ssum,
                              reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_moe_dispatch(const int* idx, int B, int T, int E, int k, int* grp,
                                      int* row_of, int* tok_of, void* stream) {
    MoeDims m{B, T, 8 /* C: unused by the dispatch */, E, k, moe_capacity(B * T, E, k)};
    return moe_dispatch(m, idx, grp, row_of, tok_of, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int llmgpu_op_dropout(const void* x, int x_f32, long long ldx, const void* resid,
                                 long long ldr, void* out, int out_f32, long long ldo, int rows,
                                 int cols, float p, const uint64_t* rng, uint64_t site,
                                 void* stream) {
    return dropout_apply(x, x_f32, ldx, resid, ldr, out, out_f32, ldo, rows, cols, p, rng, site,
                         reinterpret_cast<cudaStream_t>(stream));
}

// Dropout arguments of a linear layer: p = 0 or no generator keeps everything.
static bool linear_drop(float p, const uint64_t* rng, uint64_t site, DropArgs* d) {
    *d = DropArgs{nullptr, site, 0u, 1.0f};
    if (!drop_params(p, &d->thr, &d->scale) || (d->thr > 0 && !rng)) return false;
    if (d->thr > 0) d->rng = rng;
    return true;
}

extern "C" long long llmgpu_op_linear_fwd_work(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > kMaxDim || N > kMaxDim || K > kMaxDim) return 0;
    return (long long)product_work(M, N, K);
}

extern "C" int llmgpu_op_linear_fwd(const void* x, long long ldx, const void* w, long long ldw,
                                    int w_mn_major, const float* bias, int act, float p,
                                    const uint64_t* rng, uint64_t site, const void* resid,
                                    long long ldr, void* pre, long long ld_pre, void* out,
                                    int out_f32, long long ldo, int M, int N, int K, void* work,
                                    int* err, void* stream) {
    LinearFwd a{reinterpret_cast<const bf16*>(x), ldx, reinterpret_cast<const bf16*>(w), ldw,
                w_mn_major != 0, bias, act, {}, resid, ldr, reinterpret_cast<bf16*>(pre), ld_pre,
                out, out_f32 != 0, ldo, M, N, K, work, err};
    if (!linear_drop(p, rng, site, &a.drop)) return -1;
    if (M > 1 && (ldx < K || ldo < N || (resid && ldr < N) || (pre && ld_pre < N))) return -1;
    if (ldw < (w_mn_major ? N : K) && (w_mn_major ? K : N) > 1) return -1;
    return linear_forward(a, device_num_sms(), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" long long llmgpu_op_linear_bwd_work(int M, int N, int K) {
    return (long long)linear_backward_work(M, N, K);
}

extern "C" int llmgpu_op_linear_bwd(const void* dy, int dy_f32, long long lddy, const void* x,
                                    long long ldx, const void* w, long long ldw, int w_mn_major,
                                    const void* pre, long long ld_pre, int act, float p,
                                    const uint64_t* rng, uint64_t site, void* dx, int dx_f32,
                                    long long lddx, void* dw, int dw_f32, long long lddw,
                                    float* dbias, int accumulate, int M, int N, int K, void* work,
                                    int* err, void* stream) {
    LinearBwd a{dy, dy_f32 != 0, lddy, reinterpret_cast<const bf16*>(x), ldx,
                reinterpret_cast<const bf16*>(w), ldw, w_mn_major != 0,
                reinterpret_cast<const bf16*>(pre), ld_pre, act, {}, dx, dx_f32 != 0, lddx, dw,
                dw_f32 != 0, lddw, dbias, accumulate != 0, M, N, K, work, err};
    if (!linear_drop(p, rng, site, &a.drop)) return -1;
    const int wc = w_mn_major ? N : K, wr = w_mn_major ? K : N;  // columns and rows of w
    if (M > 1 && (lddy < N || (dw && ldx < K) || (dx && lddx < K) ||
                  (act != kActNone && ld_pre < N)))
        return -1;
    if (wr > 1 && ((dx && ldw < wc) || (dw && lddw < wc))) return -1;
    return linear_backward(a, device_num_sms(), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" long long llmgpu_op_linear_ce_fwd_work(int rows, int V) {
    return (long long)head_forward_work(rows, V);
}

extern "C" int llmgpu_op_linear_ce_fwd(const void* x, long long ldx, const void* w, long long ldw,
                                       int w_mn_major, const int32_t* targets, int rows, int C,
                                       int V, float smoothing, float* row_loss, float* lse,
                                       void* work, int* err, void* stream) {
    if ((rows > 1 && ldx < C) || (ldw < (w_mn_major ? V : C) && (w_mn_major ? C : V) > 1)) return -1;
    const HeadArgs a{reinterpret_cast<const bf16*>(x), ldx, reinterpret_cast<const bf16*>(w), ldw,
                     w_mn_major != 0, targets, rows, C, V, smoothing, work, err};
    return head_forward(a, row_loss, lse, device_num_sms(), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" long long llmgpu_op_linear_ce_bwd_work(int rows, int C, int V, int piece) {
    if (piece < 0 || piece % 256 != 0) return -1;
    return (long long)head_backward_work(rows, C, V, piece);
}

extern "C" int llmgpu_op_linear_ce_bwd(const void* x, long long ldx, const void* w, long long ldw,
                                       int w_mn_major, const int32_t* targets, const float* lse,
                                       const float* dloss, float scale, int rows, int C, int V,
                                       float smoothing, void* dx, int dx_f32, long long lddx,
                                       void* dw, int dw_f32, long long lddw, int accumulate,
                                       int piece, void* work, int* err, void* stream) {
    const int wc = w_mn_major ? V : C, wr = w_mn_major ? C : V;
    if (rows > 1 && (ldx < C || (dx && lddx < C))) return -1;
    if (wr > 1 && (ldw < wc || (dw && lddw < wc))) return -1;
    const HeadArgs a{reinterpret_cast<const bf16*>(x), ldx, reinterpret_cast<const bf16*>(w), ldw,
                     w_mn_major != 0, targets, rows, C, V, smoothing, work, err};
    return head_backward(a, lse, dloss, scale, dx, dx_f32 != 0, lddx, dw, dw_f32 != 0, lddw,
                         accumulate != 0, piece, device_num_sms(),
                         reinterpret_cast<cudaStream_t>(stream));
}

// Static device memory, so that no call has to allocate it: a first call may be under capture.
__device__ int g_op_error;

extern "C" int llmgpu_op_error_word(int** word) {
    if (!word) return -1;
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_op_error) != cudaSuccess) return launch_status();
    *word = reinterpret_cast<int*>(p);
    return 0;
}

extern "C" int llmgpu_op_take_error(int* code) {
    if (!code) return -1;
    if (cudaDeviceSynchronize() != cudaSuccess ||
        cudaMemcpyFromSymbol(code, g_op_error, sizeof(int)) != cudaSuccess)
        return launch_status();
    const int zero = 0;
    if (*code && cudaMemcpyToSymbol(g_op_error, &zero, sizeof(int)) != cudaSuccess)
        return launch_status();
    return 0;
}

namespace {

// Reads a block of llmgpu_op_call: 8-byte integers and pointers, then doubles.
struct Block {
    const char* at;
    bool fits = true;
    int64_t word() {
        int64_t v;
        memcpy(&v, at, 8);
        at += 8;
        return v;
    }
    void* ptr() { return reinterpret_cast<void*>((uintptr_t)word()); }
    template <typename T>
    T* of() {
        return reinterpret_cast<T*>((uintptr_t)word());
    }
    int i() {
        const int64_t v = word();
        if (v != (int64_t)(int)v) fits = false;
        return (int)v;
    }
    float f() {
        double v;
        memcpy(&v, at, 8);
        at += 8;
        return (float)v;
    }
};

}  // namespace

extern "C" int llmgpu_op_call(int op, const void* args) {
    if (!args) return -1;
    Block b{reinterpret_cast<const char*>(args)};
    // the arguments are read one statement each: a call's own argument list has no order
    switch (op) {
        case LLMGPU_CALL_DROPOUT: {
            const void* x = b.ptr();
            const int x_f32 = b.i();
            const long long ldx = b.word();
            const void* resid = b.ptr();
            const long long ldr = b.word();
            void* out = b.ptr();
            const int out_f32 = b.i();
            const long long ldo = b.word();
            const int rows = b.i(), cols = b.i();
            const uint64_t* rng = b.of<const uint64_t>();
            const uint64_t site = (uint64_t)b.word();
            void* stream = b.ptr();
            const float p = b.f();
            if (!b.fits) return -1;
            return llmgpu_op_dropout(x, x_f32, ldx, resid, ldr, out, out_f32, ldo, rows, cols, p, rng,
                                     site, stream);
        }
        case LLMGPU_CALL_LINEAR_FWD: {
            const void* x = b.ptr();
            const long long ldx = b.word();
            const void* w = b.ptr();
            const long long ldw = b.word();
            const int w_mn = b.i();
            const float* bias = b.of<const float>();
            const int act = b.i();
            const uint64_t* rng = b.of<const uint64_t>();
            const uint64_t site = (uint64_t)b.word();
            const void* resid = b.ptr();
            const long long ldr = b.word();
            void* pre = b.ptr();
            const long long ld_pre = b.word();
            void* out = b.ptr();
            const int out_f32 = b.i();
            const long long ldo = b.word();
            const int M = b.i(), N = b.i(), K = b.i();
            void* work = b.ptr();
            int* err = b.of<int>();
            void* stream = b.ptr();
            const float p = b.f();
            if (!b.fits) return -1;
            return llmgpu_op_linear_fwd(x, ldx, w, ldw, w_mn, bias, act, p, rng, site, resid, ldr, pre,
                                        ld_pre, out, out_f32, ldo, M, N, K, work, err, stream);
        }
        case LLMGPU_CALL_LINEAR_BWD: {
            const void* dy = b.ptr();
            const int dy_f32 = b.i();
            const long long lddy = b.word();
            const void* x = b.ptr();
            const long long ldx = b.word();
            const void* w = b.ptr();
            const long long ldw = b.word();
            const int w_mn = b.i();
            const void* pre = b.ptr();
            const long long ld_pre = b.word();
            const int act = b.i();
            const uint64_t* rng = b.of<const uint64_t>();
            const uint64_t site = (uint64_t)b.word();
            void* dx = b.ptr();
            const int dx_f32 = b.i();
            const long long lddx = b.word();
            void* dw = b.ptr();
            const int dw_f32 = b.i();
            const long long lddw = b.word();
            float* dbias = b.of<float>();
            const int accumulate = b.i(), M = b.i(), N = b.i(), K = b.i();
            void* work = b.ptr();
            int* err = b.of<int>();
            void* stream = b.ptr();
            const float p = b.f();
            if (!b.fits) return -1;
            return llmgpu_op_linear_bwd(dy, dy_f32, lddy, x, ldx, w, ldw, w_mn, pre, ld_pre, act, p, rng,
                                        site, dx, dx_f32, lddx, dw, dw_f32, lddw, dbias, accumulate, M,
                                        N, K, work, err, stream);
        }
        case LLMGPU_CALL_LINEAR_CE_FWD: {
            const void* x = b.ptr();
            const long long ldx = b.word();
            const void* w = b.ptr();
            const long long ldw = b.word();
            const int w_mn = b.i();
            const int32_t* targets = b.of<const int32_t>();
            const int rows = b.i(), C = b.i(), V = b.i();
            float* row_loss = b.of<float>();
            float* lse = b.of<float>();
            void* work = b.ptr();
            int* err = b.of<int>();
            void* stream = b.ptr();
            const float smoothing = b.f();
            if (!b.fits) return -1;
            return llmgpu_op_linear_ce_fwd(x, ldx, w, ldw, w_mn, targets, rows, C, V, smoothing,
                                           row_loss, lse, work, err, stream);
        }
        case LLMGPU_CALL_LINEAR_CE_BWD: {
            const void* x = b.ptr();
            const long long ldx = b.word();
            const void* w = b.ptr();
            const long long ldw = b.word();
            const int w_mn = b.i();
            const int32_t* targets = b.of<const int32_t>();
            const float* lse = b.of<const float>();
            const float* dloss = b.of<const float>();
            const int rows = b.i(), C = b.i(), V = b.i();
            void* dx = b.ptr();
            const int dx_f32 = b.i();
            const long long lddx = b.word();
            void* dw = b.ptr();
            const int dw_f32 = b.i();
            const long long lddw = b.word();
            const int accumulate = b.i(), piece = b.i();
            void* work = b.ptr();
            int* err = b.of<int>();
            void* stream = b.ptr();
            const float scale = b.f(), smoothing = b.f();
            if (!b.fits) return -1;
            return llmgpu_op_linear_ce_bwd(x, ldx, w, ldw, w_mn, targets, lse, dloss, scale, rows, C, V,
                                           smoothing, dx, dx_f32, lddx, dw, dw_f32, lddw, accumulate,
                                           piece, work, err, stream);
        }
        default:
            return -1;
    }
}
