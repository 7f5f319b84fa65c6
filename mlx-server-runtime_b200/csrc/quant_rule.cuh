// The group-wise affine quantization rule, shared by quantize_kernel and the kernel that
// writes a quantized KV cache.
#pragma once

#include "common.cuh"

namespace mlxq {

// The code of one element, clamp(rint(RN(d / s)), 0, n_bins) with RN the IEEE
// quotient, from r = RN(1 / s): q = RN(d * r) is within (2^-23 + 2^-48) |d / s| of
// d / s, and RN(d / s) within 2^-24 |d / s|, so for |q| <= 1024 the two differ by
// less than 2e-4. When q is more than 1e-3 from every half-integer, both round to
// the same integer; otherwise (or when q is outside [-1024, 1024], not a number, or
// r is not a normal float: `fast` false) the IEEE quotient is taken.
// Rounding to an integer adds and subtracts 1.5 * 2^23 (a float in [2^23, 2^24) has
// unit spacing, and the add rounds to nearest even like rintf for |q| < 2^22), and the
// clamped integer is read from the low mantissa bits of the same sum: no conversion
// instructions on the common path.
constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23
constexpr uint32_t kRoundMagicBits = 0x4B400000u;

__device__ __forceinline__ uint32_t quant_code(float d, float s, float r, float n_bins, bool fast) {
    const float q = __fmul_rn(d, r);
    float k = __fsub_rn(__fadd_rn(q, kRoundMagic), kRoundMagic);
    if (!fast || !(fabsf(q) <= 1024.0f) || fabsf(__fsub_rn(q, k)) > 0.499f)
        k = rintf(__fdiv_rn(d, s));
    k = fminf(fmaxf(k, 0.0f), n_bins);
    return __float_as_uint(__fadd_rn(k, kRoundMagic)) - kRoundMagicBits;
}

// Scale and bias of a group from its least and largest value and a first step, its range
// over the number of steps: the end of larger magnitude is kept exactly (bias = that end,
// scale = end / code of zero). There are two rules, which differ in the step alone:
// quantize_kernel divides the range, the cache multiplies it by the steps' reciprocal. The scale
// is made anew from the code of zero, so groups come out the same, bit for bit, unless that code
// differs: where the larger end lies half way between two codes from zero (to 2^-22 of it), as
// with ends of one magnitude. The lower neighbour then spans the range and misses a value by
// 0.54 steps of 15 at most, the upper one clips the far end by up to a step, and what the two
// stand for differs by a step and a half, before scales are rounded to 16 bits. Of normal data,
// 0.37 to 0.63 % of 4-bit and 0.07 to 0.25 % of 8-bit bf16 groups differ (0.05 to 0.09 % in
// f16). In 4 bits the cache's rule took the lower one each time, and so misses values by 0.58
// steps at most where quantize()'s misses them by 0.94 (scales rounded).
__device__ __forceinline__ void quant_group(float lmin, float lmax, float step, float& scale,
                                            float& bias) {
    const bool mask = fabsf(lmin) > fabsf(lmax);
    scale = fmaxf(step, 1e-7f);
    scale = mask ? scale : -scale;
    const float edge = mask ? lmin : lmax;
    const float q0 = rintf(__fdiv_rn(edge, scale));
    bias = 0.0f;
    if (q0 != 0.0f) {
        scale = __fdiv_rn(edge, q0);
        bias = edge;
    }
}

}  // namespace mlxq
