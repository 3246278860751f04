// lq_u4.h -- the 4-bit groups of a paged cache: how a group's scale and bias are chosen, and its codes.
#pragma once

#include "lq_internal.h"

namespace lq {

constexpr int U4_GROUP = 32;  // dims of a key that share a scale and a bias: the depth of one matrix instruction

// The bfloat16 at or above (below) a float32 value, as float32.
__device__ __forceinline__ float bf16_at_or_above(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float((x < 0.0f ? u : u + 0xffffu) & 0xffff0000u);
}
__device__ __forceinline__ float bf16_at_or_below(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float((x < 0.0f ? u + 0xffffu : u) & 0xffff0000u);
}

// A group whose least and largest values are lo and hi; hi = +inf marks one that holds what is not finite.
// The bias is at or below lo and 15 scales reach hi (to 2^-26 of the width: the product with float32's 1 / 15, which lies
// 2^-24.2 of it above it, is rounded by 2^-24 at most), so no value is cut; both are rounded to bfloat16 outward, which
// costs at most 2^-7 of a step and 2^-8 of the bias in resolution.  The product is the rule of the pages (a quotient would
// give the next bfloat16 for widths at the border of two).
struct Group4 {
    float scale, bias, inv;
    __device__ __forceinline__ Group4(float lo, float hi) {
        bias = bf16_at_or_below(lo);
        scale = bf16_at_or_above((hi - bias) * (1.0f / 15.0f));
        inv = 1.0f / scale;
        if (!(inv < INFINITY)) scale = inv = 0.0f;  // every value is the bias
        if (!(hi - bias < INFINITY)) {
            scale = bias = __builtin_nanf("");
            inv = 0.0f;
        }
    }
    __device__ __forceinline__ uint32_t code(float x) const {
        return (uint32_t)fminf(fmaxf(rne((x - bias) * inv), 0.0f), 15.0f);  // NaN: 0
    }
};

}  // namespace lq
