// What the operators over the top-K lists (balance.cu, gate_dropout.cu) share: one pixel's slots read from pixel_topk [H, W, 10], the
// weight of a slot, and the counter-based generator of the gate dropout.
//
// A slot is filled when its ID lies in [0, N) (and the pixel's mask is set, where there is one). Its weight is w = exp(-sigma) where sigma
// is finite and not negative, and 0 otherwise (the rasterizer's selection skips such a Gaussian, so its lists hold none; lists kept while
// the parameters move on may). The gate is n = w / (sum_j w_j + eps), eps = 1e-4 as in the render.
#pragma once

#include "igs_common.cuh"

namespace igs {

// exp(-sigma), or 0 for a sigma that is negative, NaN or infinite. __expf (2 ulp plus 2^-24 |sigma|) adds no more than the rounding of
// sigma itself, which is 2^-24 relative at best and multiplies the weight's relative error by sigma.
__device__ __forceinline__ float slot_weight(float sigma) { return sigma >= 0.f && sigma < __int_as_float(0x7f800000) ? __expf(-sigma) : 0.f; }

// Philox4x32-10: J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011 (table 2 and section 3.3:
// the multipliers, the Weyl constants of the key and the round). A counter of four words and a key of two give four random words.
__device__ __forceinline__ uint4 philox4x32(uint4 c, uint2 key) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c.x, b = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ key.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ key.y, (uint32_t)a);
        key.x += 0x9E3779B9u, key.y += 0xBB67AE85u;
    }
    return c;
}

// The ten 24-bit draws of a pixel, compared with the threshold: bit k is set where slot k is kept. Two calls give eight words: slot k < 8
// takes the upper 24 bits of word k, slots 8 and 9 the low bytes of words 0, 1, 2 and 3, 4, 5 (the first most significant), which no other
// slot uses; a third call for two slots would cost half as much again.
__device__ __forceinline__ unsigned keep_bits(uint32_t pixel, uint64_t seed, uint64_t offset, uint32_t threshold) {
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const uint32_t o0 = (uint32_t)offset, o1 = (uint32_t)(offset >> 32);
    const uint4 a = philox4x32(make_uint4(pixel, 0u, o0, o1), key), b = philox4x32(make_uint4(pixel, 1u, o0, o1), key);
    const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    unsigned keep = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) keep |= (words[k] >> 8) >= threshold ? 1u << k : 0u;
    const uint32_t d8 = (words[0] & 255u) << 16 | (words[1] & 255u) << 8 | (words[2] & 255u);
    const uint32_t d9 = (words[3] & 255u) << 16 | (words[4] & 255u) << 8 | (words[5] & 255u);
    keep |= d8 >= threshold ? 1u << 8 : 0u;
    keep |= d9 >= threshold ? 1u << 9 : 0u;
    return keep;
}

// Host checks of the lists' geometry, shared by the entry points: ten slots per pixel indexed with 32 bits, coordinates exact in float
inline bool lists_addressable(int img_height, int img_width) {
    return (int64_t)img_height * img_width <= INT32_MAX / kTopK && img_height <= 1 << 24 && img_width <= 1 << 24;
}

}  // namespace igs
