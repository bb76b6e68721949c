// Launchers of dropout and of the linear layer's elementwise backward.
#pragma once
#include "kernels.cuh"

namespace llmgpu {

// out = resid + (kept ? x * scale : 0) over [rows, cols]; x, resid and out are bf16 or f32 (resid
// of out's type, or null) with row strides in elements. out may be x or resid itself.
int dropout_apply(const void* x, int x_f32, long long ldx, const void* resid, long long ldr,
                  void* out, int out_f32, long long ldo, int rows, int cols, float p,
                  const uint64_t* rng, uint64_t site, cudaStream_t s);

}  // namespace llmgpu
