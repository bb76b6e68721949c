// Loss head without logits. Forward: loss = on (lse - z_t) + off sum_{v != t} (lse - z_v) of z = x w^T;
// the product keeps, of each 128 columns of logits, the maximum and the sum of exponentials of
// every row (gemm.cu, kEpiHeadStats), merged by head_merge_kernel. Backward: the logits are formed
// again a piece of the vocabulary at a time, the gradient by them, c (softmax - y), leaves tensor
// memory in bf16 (kEpiHeadGrad), and that piece goes into the products for dx (summed over the
// pieces in f32 planes) and for dw (each of its rows written once).
//
// Bound by the tensor cores (and, over many launches, by the power cap): one product forward,
// three backward, one more than with [rows, V] logits kept, and none of their memory (824 MB at
// 8192 x 50257 in bf16, which would also round the loss). 8192 x 768 x 50257: forward 418 us
// (1.51 PFLOP/s), backward 1430 us (1.33 PFLOP/s counting the recomputed product). Pieces of the
// vocabulary rather than blocks of rows: dw, the largest matrix, is then written once instead of
// summed over row blocks.
#include <cfloat>

#include "common.cuh"
#include "linear.cuh"

namespace llmgpu {

namespace {

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
long long ceil8(long long n) { return (n + 7) & ~7ll; }

constexpr int kSlot = 128;       // vocabulary columns of one (max, sum) slot
constexpr int kMaxSplits = 32;   // planes of the dx product
constexpr int kPairSlots = 74;   // CTA pairs of a B200, for the choice of piece and splits only
// Gradient piece at most, where chosen here. 8192 x 768 x 50257, backward by piece: 1024 columns 3509
// us, 4096 1745, 8192 1684, 18944 1537, the choice below 1430.
constexpr size_t kPieceBytes = (size_t)320 << 20;

int slots_of(int V) { return (V + kSlot - 1) / kSlot; }

// Merges the slots of 32 rows: lanes are rows, the block's warps stride over the slots.
__global__ void __launch_bounds__(1024) head_merge_kernel(const float2* __restrict__ part,
                                                          const float* __restrict__ zsum,
                                                          const float* __restrict__ zt,
                                                          const int32_t* __restrict__ targets,
                                                          int slots, int rows, int V, float on,
                                                          float off, float* __restrict__ row_loss,
                                                          float* __restrict__ lse) {
    pdl_enter();
    constexpr float kLog2 = 1.4426950408889634f;
    __shared__ float sm[32][33], ss[32][33], sz[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int row = blockIdx.x * 32 + lane;
    const float ninf = __int_as_float(0xff800000);
    float m = ninf, s = 0.0f, z = 0.0f;
    if (row < rows) {
        constexpr int U = 8;  // slots in flight
        for (int p0 = w; p0 < slots; p0 += 32 * U) {
            float2 q[U];
            float mn = m;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = p0 + 32 * u;
                q[u] = p < slots ? part[(long long)p * rows + row] : make_float2(ninf, 0.0f);
            }
            if (zsum)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (p0 + 32 * u < slots) z += zsum[(long long)(p0 + 32 * u) * rows + row];
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, q[u].x);
            // a side that holds nothing (sum 0) adds 0; an unordered one passes NaN on
            s = s == 0.0f ? 0.0f : s * ex2_approx((m - mn) * kLog2);
#pragma unroll
            for (int u = 0; u < U; ++u)
                s += q[u].y == 0.0f ? 0.0f : q[u].y * ex2_approx((q[u].x - mn) * kLog2);
            m = mn;
        }
    }
    sm[w][lane] = m;
    ss[w][lane] = s;
    sz[w][lane] = z;
    __syncthreads();
    if (w != 0 || row >= rows) return;
    for (int i = 1; i < 32; ++i) {
        const float mi = sm[i][lane], si = ss[i][lane];
        const float mn = fmaxf(m, mi);
        const float a = s == 0.0f ? 0.0f : s * ex2_approx((m - mn) * kLog2);
        const float b = si == 0.0f ? 0.0f : si * ex2_approx((mi - mn) * kLog2);
        m = mn;
        s = a + b;
        z += sz[i][lane];
    }
    const float l = m + logf(s);
    lse[row] = l;
    const int t = targets[row];
    float loss = 0.0f;
    if (t >= 0 && t < V) {
        const float d = l - zt[row];
        loss = on * d;
        if (zsum) loss += off * (((float)V * l - z) - d);
    }
    row_loss[row] = loss;
}

// Copy of x with zeros in the rows left out (0 times what they hold could be NaN in dw), its row
// stride a multiple of 8 elements. The last block finds the largest finite |dloss| of the rows
// that count: top = {that (1 if it is 0 or there is no dloss), factor times it}, what the gradient by
// the logits is divided by and what the products multiply back.
__global__ void __launch_bounds__(256) head_rows_kernel(const bf16* __restrict__ x, long long ldx,
                                                        const int32_t* __restrict__ targets,
                                                        const float* __restrict__ dloss,
                                                        float factor, int rows, int C, int V,
                                                        bf16* __restrict__ out, int ldo,
                                                        float* __restrict__ top) {
    pdl_enter();
    if (blockIdx.x == gridDim.x - 1) {
        float m = 0.0f;
        if (dloss) {
#pragma unroll 8
            for (int r = threadIdx.x; r < rows; r += 256) {
                const int t = targets[r];
                const float d = fabsf(dloss[r]);
                if (t >= 0 && t < V && d <= FLT_MAX) m = fmaxf(m, d);
            }
        }
        __shared__ float red[8];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
            if (m == 0.0f) m = 1.0f;
            top[0] = m;
            top[1] = factor * m;
        }
        return;
    }
    const int n8 = ldo >> 3;
    const long long total = (long long)rows * n8;
    const long long step = (gridDim.x - 1) * 256ll;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += step) {
        const int row = (int)(i / n8), c = (int)(i - (long long)row * n8) * 8;
        const int t = targets[row];
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (t >= 0 && t < V) {
            const bf16* p = x + row * ldx + c;
            if (c + 8 <= C) {
                u = *reinterpret_cast<const uint4*>(p);
            } else {
                unsigned short h[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    h[j] = c + j < C ? __bfloat16_as_ushort(p[j]) : (unsigned short)0;
                u = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16,
                               h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
            }
        }
        *reinterpret_cast<uint4*>(out + (long long)row * ldo + c) = u;
    }
}

long long waves(long long tiles) { return (tiles + kPairSlots - 1) / kPairSlots; }

// k-splits of the dx product (each into a plane of its own): the count whose last wave of
// 256 x 256 tiles wastes least, a tile costing its k-blocks and about 4 more. Where one piece is
// the whole vocabulary (`all`) and one split would do, the planes' summing kernel is not needed:
// about 12 k-blocks of a pair (4 us).
int dx_splits(int rows, int C, int piece, bool all) {
    const long long tiles = (long long)((rows + 255) / 256) * ((C + 255) / 256);
    const int kb = (piece + 63) / 64;
    // a plane is written (added to) once a piece and read once: 8 bytes an element at about
    // 6 TB/s, against 0.3 us a k-block
    const double plane = (double)rows * C * 8.0 / 6e6 / 0.3;
    int best = 1;
    double cost = 1e30;
    for (int n = 1; n <= kMaxSplits && n <= kb; n += n < 4 ? 1 : n < 16 ? 2 : 8) {
        const double c = (double)waves(tiles * n) * ((double)kb / n + 4.0) + n * plane +
                         (all && n > 1 ? 12.0 : 0.0);
        if (c < cost * 0.97) {
            cost = c;
            best = n;
        }
    }
    return best;
}

struct HeadLayout {
    int piece, splits, ldx, ldg, ldp;
    size_t x, g, planes, top, total;  // byte offsets and the whole
};

HeadLayout head_layout(int rows, int C, int V, int piece) {
    HeadLayout l;
    l.piece = head_piece(rows, C, V, piece);
    l.splits = dx_splits(rows, C, l.piece, l.piece >= V);
    l.ldx = (int)ceil8(C);
    l.ldg = (int)ceil8(l.piece);
    l.ldp = (int)ceil8(C);
    l.x = 0;
    l.g = align256((size_t)rows * l.ldx * 2);
    l.planes = l.g + align256((size_t)rows * l.ldg * 2);
    l.top = l.planes + align256((size_t)l.splits * rows * l.ldp * 4);
    l.total = l.top + 8;
    return l;
}

}  // namespace

int head_piece(int rows, int C, int V, int piece) {
    if (piece > 0) return piece < V ? piece : V;
    const int tc = (C + 255) / 256, tr = (rows + 255) / 256;
    const int all = (V + 255) / 256;
    long long most = (long long)(kPieceBytes / 2 / 256 / (size_t)rows);
    if (most < 1) most = 1;
    if (most >= all) return V;
    // the largest pieces within the bound lose least to launches; among those down to half of
    // it, the one whose products' waves of tiles are fullest
    int best = (int)most;
    double cost = 1e30;
    for (int p = (int)most; p >= 1 && 2 * p >= most; --p) {
        double c = 0.0;
        for (int v = 0; v < all; v += p) {
            const int w = all - v < p ? all - v : p;
            const int n = dx_splits(rows, C, w * 256, false);
            c += (double)waves((long long)tr * w) * ((C + 63) / 64 + 4) +
                 (double)waves((long long)w * tc) * ((rows + 63) / 64 + 4) +
                 (double)waves((long long)tr * tc * n) * (4.0 * w / n + 4);
        }
        if (c < cost) {
            cost = c;
            best = p;
        }
    }
    return best * 256;
}

size_t head_forward_work(int rows, int V) {
    if (rows <= 0 || V <= 0 || rows > kMaxDim || V > kMaxDim) return 0;
    const size_t n = (size_t)slots_of(V) * rows;
    return align256(n * 8) + align256(n * 4) + (size_t)rows * 4;
}

int head_forward(const HeadArgs& a, float* row_loss, float* lse, int num_sms, cudaStream_t s) {
    if (a.rows < 0 || a.C <= 0 || a.V <= 0 || !(a.smoothing >= 0.0f && a.smoothing < 1.0f)) return -1;
    if (a.rows > kMaxDim || a.C > kMaxDim || a.V > kMaxDim) return -1;
    if (a.rows == 0) return 0;
    if (!a.x || !a.w || !a.targets || !row_loss || !lse || !a.work) return -1;
    if (!operand_ok(a.x, a.ldx) || !operand_ok(a.w, a.ldw) || !operand_ok(a.work, 0))
        return kBadOperand;
    const size_t n = (size_t)slots_of(a.V) * a.rows;
    char* w = reinterpret_cast<char*>(a.work);
    GemmArgs g{};
    g.epi = kEpiHeadStats;
    g.splits = 1;
    g.err = a.err;
    GemmExt x{};
    x.targets = a.targets;
    x.v0 = 0;
    x.V = a.V;
    x.part = reinterpret_cast<float2*>(w);
    x.zsum = a.smoothing > 0.0f ? reinterpret_cast<float*>(w + align256(n * 8)) : nullptr;
    x.zt = reinterpret_cast<float*>(w + align256(n * 8) + align256(n * 4));
    GemmPlan plan;
    int rc = gemm_make_plan(&plan, a.x, a.ldx, 0, a.w, a.ldw, a.w_mn_major, a.rows, a.V, a.C, g, 0,
                            num_sms, &x);
    if (rc) return rc;
    rc = gemm_run(plan, s);
    if (rc) return rc;
    return launch_kernel(head_merge_kernel, (a.rows + 31) / 32, 1024, 0, s, x.part, x.zsum, x.zt,
                         a.targets, slots_of(a.V), a.rows, a.V, 1.0f - a.smoothing,
                         a.V > 1 ? a.smoothing / (float)(a.V - 1) : 0.0f, row_loss, lse);
}

size_t head_backward_work(int rows, int C, int V, int piece) {
    if (rows <= 0 || C <= 0 || V <= 0 || rows > kMaxDim || C > kMaxDim || V > kMaxDim) return 0;
    return head_layout(rows, C, V, piece).total;
}

int head_backward(const HeadArgs& a, const float* lse, const float* dloss, float scale, void* dx,
                  int dx_f32, long long lddx, void* dw, int dw_f32, long long lddw, int accumulate,
                  int piece, int num_sms, cudaStream_t s) {
    if (a.rows < 0 || a.C <= 0 || a.V <= 0 || !(a.smoothing >= 0.0f && a.smoothing < 1.0f)) return -1;
    if (a.rows > kMaxDim || a.C > kMaxDim || a.V > kMaxDim) return -1;
    if (piece < 0 || (piece % 256) != 0 || (accumulate && dw && !dw_f32)) return -1;
    const size_t es = dw_f32 ? 4 : 2;
    if (a.rows == 0) {
        if (!dw || accumulate) return 0;
        const size_t r = a.w_mn_major ? a.C : a.V, c = a.w_mn_major ? a.V : a.C;
        return cudaMemset2DAsync(dw, lddw * es, 0, c * es, r, s) == cudaSuccess ? 0
                                                                               : launch_status();
    }
    if (!a.x || !a.w || !a.targets || !lse || !a.work) return -1;
    if (!dx && !dw) return 0;
    if (!operand_ok(a.x, a.ldx) || !operand_ok(a.w, a.ldw) || !operand_ok(a.work, 0))
        return kBadOperand;
    const HeadLayout l = head_layout(a.rows, a.C, a.V, piece);
    char* wk = reinterpret_cast<char*>(a.work);
    bf16* xr = reinterpret_cast<bf16*>(wk + l.x);
    bf16* gp = reinterpret_cast<bf16*>(wk + l.g);
    float* planes = reinterpret_cast<float*>(wk + l.planes);
    float* top = reinterpret_cast<float*>(wk + l.top);
    // a vocabulary of one has nothing to smooth into: the loss is 0, and softmax / on - 1 as well
    const float on = a.V > 1 ? 1.0f - a.smoothing : 1.0f;
    const long long n8 = (long long)a.rows * (l.ldx / 8);
    const int rb = 1 + (int)(n8 < 148ll * 8 * 256 ? (n8 + 255) / 256 : 148 * 8);
    int rc = launch_kernel(head_rows_kernel, rb, 256, 0, s, a.x, a.ldx, a.targets, dloss, scale * on,
                           a.rows, a.C, a.V, xr, l.ldx, top);
    if (rc) return rc;
    const bool one = l.piece >= a.V && l.splits == 1;  // dx straight from one product
    for (int v0 = 0; v0 < a.V; v0 += l.piece) {
        const int pw = a.V - v0 < l.piece ? a.V - v0 : l.piece;
        const bf16* w = a.w + (a.w_mn_major ? (long long)v0 : v0 * a.ldw);
        GemmArgs g{};
        g.epi = kEpiHeadGrad;
        g.out = gp;
        g.ldo = l.ldg;
        g.splits = 1;
        g.err = a.err;
        GemmExt x{};
        x.targets = a.targets;
        x.v0 = v0;
        x.V = a.V;
        x.lse = lse;
        x.dloss = dloss;
        x.top = top;
        x.on = on;
        x.off_on = a.V > 1 ? a.smoothing / (float)(a.V - 1) / on : 0.0f;
        GemmPlan plan;
        rc = gemm_make_plan(&plan, xr, l.ldx, 0, w, a.ldw, a.w_mn_major, a.rows, pw, a.C, g, 0,
                            num_sms, &x);
        if (rc) return rc;
        if ((rc = gemm_run(plan, s)) != 0) return rc;
        if (dx && one) {
            rc = product(gp, l.ldg, 0, w, a.ldw, a.w_mn_major ? 0 : 1, a.rows, a.C, pw, dx, dx_f32,
                         lddx, 0, num_sms, a.err, s, top + 1);
            if (rc) return rc;
        } else if (dx) {
            GemmArgs h{};
            h.epi = kEpiPlaneAdd;
            h.out = planes;
            h.ldo = l.ldp;
            h.accumulate = v0 > 0;
            h.splits = l.splits;
            h.err = a.err;
            // a short last piece may have fewer k-blocks than planes: the planes it does not
            // reach keep their sums
            const int kb = (pw + 63) / 64;
            if (h.splits > kb) h.splits = kb;
            GemmExt none{};
            rc = gemm_make_plan(&plan, gp, l.ldg, 0, w, a.ldw, a.w_mn_major ? 0 : 1, a.rows, a.C,
                                pw, h, 0, num_sms, &none);
            if (rc) return rc;
            if ((rc = gemm_run(plan, s)) != 0) return rc;
        }
        if (dw) {
            // dw need not wait for dx's product
            const int early = dx && leaves_room(a.rows, a.C, one ? 1 : l.splits);
            char* to = reinterpret_cast<char*>(dw) + (a.w_mn_major ? (long long)v0 : v0 * lddw) * es;
            rc = a.w_mn_major ? product(xr, l.ldx, 1, gp, l.ldg, 1, a.C, pw, a.rows, to, dw_f32,
                                        lddw, accumulate, num_sms, a.err, s, top + 1, nullptr, early)
                              : product(gp, l.ldg, 1, xr, l.ldx, 1, pw, a.C, a.rows, to, dw_f32,
                                        lddw, accumulate, num_sms, a.err, s, top + 1, nullptr, early);
            if (rc) return rc;
        }
    }
    if (dx && !one) {
        RowsArgs r{nullptr, 0, nullptr, 0, top + 1, nullptr, kActNone, {}, nullptr, 0, nullptr, 0, dx,
                   dx_f32, lddx, a.rows, a.C, 0};
        rc = finish_planes(r, planes, l.splits, l.ldp, s);
    }
    return rc;
}

}  // namespace llmgpu
