// Counter-based random bits for dropout: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011), written from the paper's definition.
//
// One call gives 128 bits for 8 neighbouring columns of a row: key = the 64-bit seed, counter =
// (column / 8, row, offset). Column 8 i + j takes 16-bit lane j (low half of word 0 first) and is
// kept when the lane is at least the threshold round(p * 65536): sixteen bits per element halve
// the generator's cost against 32, and the scale of the kept elements uses the quantised
// probability, so the expectation stays exact. An element's fate depends on (seed, offset, row,
// column) alone, not on strides, tiles or the grid, so every kernel that drops the same matrix
// (elementwise, in a product's epilogue, in the backward) forms the same mask and none stores it.
#pragma once
#include <stdint.h>

namespace llmgpu {

struct DropKey {
    uint32_t k0, k1;  // seed
    uint32_t c2, c3;  // offset + site
};
// The same with the ten rounds' keys formed once: twenty registers for twenty additions a call,
// which the elementwise kernels can spare (bf16 16384 x 4096: 62 -> 55 us) and the products'
// epilogue cannot.
struct DropKeys {
    uint32_t k0[10], k1[10];
    uint32_t c2, c3;
};

// Host side: threshold and scale of a drop probability p in [0, 1]; false for any other p.
inline bool drop_params(float p, uint32_t* thr, float* scale) {
    if (!(p >= 0.0f && p <= 1.0f)) return false;
    // p * 65536 is exact (a power of two); round half to even, as numpy and Python do
    const double v = (double)p * 65536.0;
    uint32_t t = (uint32_t)v;
    const double f = v - t;
    if (f > 0.5 || (f == 0.5 && (t & 1u))) ++t;
    *thr = t;
    *scale = t < 65536u ? 65536.0f / (float)(65536u - t) : 0.0f;
    return true;
}

#ifdef __CUDACC__
// rng: {seed, offset} in device memory, read when the kernel runs (a captured launch sees the
// values of its replay).
__device__ __forceinline__ DropKey drop_key(const uint64_t* rng, uint64_t site) {
    const uint64_t seed = rng[0], off = rng[1] + site;
    return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}
__device__ __forceinline__ DropKeys drop_keys(const uint64_t* rng, uint64_t site) {
    const DropKey d = drop_key(rng, site);
    DropKeys k;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        k.k0[r] = d.k0 + r * 0x9E3779B9u;
        k.k1[r] = d.k1 + r * 0xBB67AE85u;
    }
    k.c2 = d.c2;
    k.c3 = d.c3;
    return k;
}
__device__ __forceinline__ uint32_t round_key0(const DropKey& k, int r) { return k.k0 + r * 0x9E3779B9u; }
__device__ __forceinline__ uint32_t round_key1(const DropKey& k, int r) { return k.k1 + r * 0xBB67AE85u; }
__device__ __forceinline__ uint32_t round_key0(const DropKeys& k, int r) { return k.k0[r]; }
__device__ __forceinline__ uint32_t round_key1(const DropKeys& k, int r) { return k.k1[r]; }

template <typename Key>
__device__ __forceinline__ uint4 philox_10(uint4 c, const Key& k) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c.x * 0xD2511F53u;
        const uint64_t b = (uint64_t)c.z * 0xCD9E8D57u;
        c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ round_key0(k, r), (uint32_t)b,
                       (uint32_t)(a >> 32) ^ c.w ^ round_key1(k, r), (uint32_t)a);
    }
    return c;
}

// Columns 8 col8 .. 8 col8 + 7 of `row`: v = kept ? v * scale : 0. thr in [1, 65536]; a lane is at
// least thr when, moved to a word's upper half, it is above (thr << 16) - 1.
template <typename Key>
__device__ __forceinline__ void drop_apply8(const Key& k, uint32_t col8, uint32_t row,
                                            uint32_t thr, float scale, float* v) {
    const uint4 r = philox_10(make_uint4(col8, row, k.c2, k.c3), k);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    const uint32_t below = (thr << 16) - 1u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = (w[i] << 16) > below ? v[2 * i] * scale : 0.0f;
        v[2 * i + 1] = w[i] > below ? v[2 * i + 1] * scale : 0.0f;
    }
}

// Bit j: column 8 * col8 + j of `row` is kept. thr in [0, 65536].
template <typename Key>
__device__ __forceinline__ uint32_t drop_keep8(const Key& k, uint32_t col8, uint32_t row,
                                               uint32_t thr) {
    const uint4 r = philox_10(make_uint4(col8, row, k.c2, k.c3), k);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m |= ((w[i] & 0xFFFFu) >= thr ? 1u : 0u) << (2 * i);
        m |= ((w[i] >> 16) >= thr ? 1u : 0u) << (2 * i + 1);
    }
    return m;
}
#endif

}  // namespace llmgpu
