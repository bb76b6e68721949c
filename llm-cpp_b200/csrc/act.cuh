// Activations of the linear layer and their derivatives, on packed pairs in f32.
#pragma once
#include "common.cuh"
#include "gemm.cuh"

namespace llmgpu {

constexpr float kLog2e = 1.4426950408889634f;

// Activations of a pair of pre-activations, z / (1 + exp(-t)) with t = z (silu) or 2 k (z + 0.044715
// z^3) (gelu: 0.5 z (1 + tanh u) = z sigmoid(2u)), from the special-function unit's 2^x and
// reciprocal, a few units in the last place, which an f32 output keeps. Far left, 2^x overflows
// to inf and the result is -0. Packed pairs: 7 issue slots for two gelus besides the 4
// special-function ones, since the epilogue's warps (four a scheduler in the pair kernel, one in the
// others) are what bounds a product of K near 1024.
__device__ __forceinline__ float2 sigmoid_of_log2(float2 t) {  // 1 / (1 + 2^t)
    const float2 d = fadd2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), make_float2(1.f, 1.f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}
template <int ACT>
__device__ __forceinline__ float2 act_pair(float2 z) {
    if constexpr (ACT == kActRelu) {  // NaN stays NaN
        return make_float2(z.x <= 0.0f ? 0.0f : z.x, z.y <= 0.0f ? 0.0f : z.y);
    } else if constexpr (ACT == kActGelu) {
        constexpr float c = -1.5957691216f * kLog2e;
        const float2 w = ffma2(fmul2(z, z), make_float2(c * 0.044715f, c * 0.044715f),
                               make_float2(c, c));
        return fmul2(z, sigmoid_of_log2(fmul2(w, z)));
    } else if constexpr (ACT == kActSilu) {
        return fmul2(z, sigmoid_of_log2(fmul2(z, make_float2(-kLog2e, -kLog2e))));
    } else {
        return z;
    }
}
// Derivatives of a pair of activations, from the same sigmoid as the forward's: gelu(z) = z h with
// h = sigmoid(2u): h + z h (1 - h) 2u'; silu: h (1 + z (1 - h)). Past |z| = 12, h is 0 or 1 in f32 and
// gelu's second term 0: z stops growing there in it, since 0 times an overflowed product would be NaN
// (from 1e13 on for z^3, from 1e37 on for z alone). The sigmoid takes z itself, which keeps a NaN.
template <int ACT>
__device__ __forceinline__ float2 act_grad_pair(float2 z) {
    if constexpr (ACT == kActRelu) {
        return make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
    } else if constexpr (ACT == kActGelu || ACT == kActSilu) {
        const float2 one = make_float2(1.0f, 1.0f);
        float2 zc, z2, t;  // gelu's z within +-12 and its square
        if constexpr (ACT == kActGelu) {
            zc = make_float2(fminf(fmaxf(z.x, -12.0f), 12.0f), fminf(fmaxf(z.y, -12.0f), 12.0f));
            z2 = fmul2(zc, zc);
            constexpr float c = -1.5957691216f * kLog2e;
            t = fmul2(ffma2(z2, make_float2(c * 0.044715f, c * 0.044715f), make_float2(c, c)), z);
        } else {
            t = fmul2(z, make_float2(-kLog2e, -kLog2e));
        }
        const float2 d = fadd2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), one);
        const float2 h = make_float2(rcp_approx(d.x), rcp_approx(d.y));
        const float2 g = ffma2(h, make_float2(-1.0f, -1.0f), one);  // 1 - h
        if constexpr (ACT == kActGelu) {
            constexpr float k = 1.5957691216f;
            const float2 q =
                fmul2(ffma2(z2, make_float2(k * 0.134145f, k * 0.134145f), make_float2(k, k)), zc);
            return ffma2(fmul2(h, g), q, h);
        } else {
            return fmul2(h, ffma2(z, g, one));
        }
    } else {
        return make_float2(1.0f, 1.0f);
    }
}

// f(integral constant) for the activation chosen at run time, so that the choice stands outside loops.
template <int ACT>
struct ActTag {
    static constexpr int value = ACT;
};
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
        case kActRelu:
            f(ActTag<kActRelu>{});
            break;
        case kActGelu:
            f(ActTag<kActGelu>{});
            break;
        case kActSilu:
            f(ActTag<kActSilu>{});
            break;
        default:
            f(ActTag<kActNone>{});
            break;
    }
}

}  // namespace llmgpu
