// Per-element arithmetic of the AdamW kernels (adamw.hip) as plain inline functions, so that tests/native/adamw_emulate.cpp runs the
// SAME code on the host (see depthwise_math.h for the pattern).
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      p = p - lr wd p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// States in 8 bits: m and r = sqrt(v) are e4m3 codes (4 exponent bits, 3 mantissa bits, largest value 448) of blocks of 256 elements
// with one f32 scale each, scale = absmax / 448.  r and not v: v spans the square of r's range, which 8 bits do not.
// Rounding is stochastic: from one step to the next r falls by at most (1 - b2) / 2 = 0.05 % of itself (it rises without such a limit, under
// a gradient much larger than r), a nearest rounding of 3 mantissa bits moves only at 6 %, so r would never come down again; a rounding that
// goes up with the probability of the cut-off fraction is right on average.  Its random bits are a counter hash of (seed, step, tensor, element): the same call gives
// the same bits on every machine.  A positive r never rounds to zero (it divides).
#pragma once
#include <stdint.h>
#include <string.h>
#include <math.h>

#ifndef SEMSEG_HD
#ifdef __HIPCC__
#define SEMSEG_HD __host__ __device__ __forceinline__
#else
#define SEMSEG_HD static inline
#endif
#endif

constexpr int ADAM8_BLOCK = 256;                 // elements that share one scale
constexpr float ADAM8_MAX = 448.0f;              // largest e4m3 value
constexpr float ADAM8_TINY = 7.888609052210118e-31f;      // 2^-100: a block below it is stored as zeros (its scale would lose bits)

// what one step needs per tensor, computed once per call on the device (adamw_begin_kernel): the step count lives there
struct AdamCoef {
    float size;        // lr / (1 - b1^t)
    float root;        // 1 / sqrt(1 - b2^t); 0: leave the tensor alone (the gradients are not finite)
    float factor;      // what the gradient is multiplied with
    float decay;       // lr * weight decay
    uint32_t base;     // counter base of the random bits
};
struct AdamHyper {
    float b1, c1, b2, c2, eps;      // c = 1 - b, formed in double
};

SEMSEG_HD uint32_t adam_bits(float x) { uint32_t u; memcpy(&u, &x, 4); return u; }
SEMSEG_HD float adam_float(uint32_t u) { float x; memcpy(&x, &u, 4); return x; }

// 32 bits scrambled: xor-shifts and odd multipliers (the fractional bits of sqrt 2 and sqrt 3); a bijection
SEMSEG_HD uint32_t adam_mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// the coefficients of step t (t >= 1) of one tensor; double: 1 - b^t cancels for small t
SEMSEG_HD AdamCoef adam_coef(double lr, double log_b1, double log_b2, double wd, int t, float factor, uint32_t seed, uint32_t ordinal) {
    AdamCoef c;
    c.size = (float)(lr / -expm1((double)t * log_b1));
    c.root = (float)(1.0 / sqrt(-expm1((double)t * log_b2)));
    c.factor = factor;
    c.decay = (float)(lr * wd);
    c.base = adam_mix(seed ^ adam_mix((uint32_t)t ^ adam_mix(ordinal)));
    return c;
}

// p, one rounding of the difference: the two small terms are added first
SEMSEG_HD float adam_moved(float p, float m, float r, const AdamCoef& c, float eps) {
    const float u = m / fmaf(r, c.root, eps);
    return p - fmaf(c.size, u, c.decay * p);
}

// states in 32 bits
SEMSEG_HD void adam_update32(float& p, float g, float& m, float& v, const AdamCoef& c, const AdamHyper& h) {
    g *= c.factor;
    m = fmaf(h.b1, m, h.c1 * g);
    v = fmaf(h.b2, v, (h.c2 * g) * g);
    p = adam_moved(p, m, sqrtf(v), c, h.eps);
}

// Root and reciprocal of the 8-bit step, which has so few bytes an element that instructions bound it.
// The root decides codes and is rounded to nearest: the hardware's is within one unit of the last place, and of it and its two neighbours
// the one is taken whose half-unit interval holds x -- (s - u/2)^2 = s (s - u) up to u^2/4, so the sign of x - s (s - u), one rounding,
// tells.  Below 2^-96 that difference would leave the range (and the hardware takes a denormal for zero), so x is scaled by 2^64 there and
// the root by 2^-32, both exact.  The reciprocal only moves the parameter: the hardware's, one unit off at most, of a sum that is never
// denormal (the smallest root is 3.7e-23, and semseg_adamw8_step refuses an eps that is).
#if defined(__HIP_DEVICE_COMPILE__)
SEMSEG_HD float adam_root(float value) {
    const bool low = value < 0x1p-96f;
    const float x = low ? value * 0x1p64f : value;
    const float s = __builtin_amdgcn_sqrtf(x);
    const float down = adam_float(adam_bits(s) - 1u), up = adam_float(adam_bits(s) + 1u);
    float r = fmaf(-down, s, x) <= 0.0f ? down : s;
    r = fmaf(-up, s, x) > 0.0f ? up : r;
    r = x > 0.0f && x < INFINITY ? r : s;
    return low ? r * 0x1p-32f : r;
}
SEMSEG_HD float adam_reciprocal(float x) { return __builtin_amdgcn_rcpf(x); }
#else
SEMSEG_HD float adam_root(float x) { return sqrtf(x); }
SEMSEG_HD float adam_reciprocal(float x) { return 1.0f / x; }
#endif

// states in 8 bits, before they are coded again: m and r in 32 bits.  Every product and sum of the states is rounded by itself (no
// contraction): next to a border of the rounding the last bit decides the code, so the definition fixes it.
SEMSEG_HD void adam_update8(float& p, float g, float& m, float& r, const AdamCoef& c, const AdamHyper& h) {
#ifdef __clang__
#pragma clang fp contract(off)
#endif
    g = g * c.factor;
    const float m0 = h.b1 * m, m1 = h.c1 * g;
    m = m0 + m1;
    const float v0 = h.b2 * (r * r), v1 = (h.c2 * g) * g;
    r = adam_root(v0 + v1);
    const float u = m * adam_reciprocal(fmaf(r, c.root, h.eps));
    p = p - fmaf(c.size, u, c.decay * p);
}

// scale of a block from the bit pattern of its largest |value| (patterns order as the values do, NaN above infinity)
SEMSEG_HD float adam8_scale(uint32_t top) {
    if (top >= 0x7f800000u) return adam_float(0x7fc00000u);      // a block that is not finite decodes to NaN
    const float a = adam_float(top);
    return a < ADAM8_TINY ? 0.0f : a * (1.0f / 448.0f);
}
SEMSEG_HD float adam8_inverse(float scale) { return scale > 0.0f ? 1.0f / scale : 0.0f; }

// what is coded: value / scale, limited to the range (the largest may come out a bit above); a positive r is at least the smallest code
SEMSEG_HD float adam8_limited(float a, float low) { return fminf(fmaxf(a, low), ADAM8_MAX); }
SEMSEG_HD float adam8_scaled_m(float m, float inv) { return adam8_limited(m * inv, -ADAM8_MAX); }
SEMSEG_HD float adam8_scaled_r(float r, float inv) { return adam8_limited(r * inv, r > 0.0f ? 0.001953125f : 0.0f); }

// stochastic rounding of |a| <= 448 to the e4m3 grid: 16 random bits are added below the last kept bit of the mantissa, then all below is
// cut off.  Below 2^-6 the grid is even (2^-9): adding 2^-6 puts the value where a float's own bits line up with it.  The hardware's
// conversion (v_cvt_sr_fp8_f32 with the bits on top of its seed) gives the same codes; this form is the host's.
SEMSEG_HD float adam8_round(float x, uint32_t random16) {
    float a = fabsf(x);
    const float low = a < 0.015625f ? 0.015625f : 0.0f;
    a = adam_float((adam_bits(a + low) + (random16 << 4)) & ~0xFFFFFu) - low;
    return copysignf(a, x);
}
