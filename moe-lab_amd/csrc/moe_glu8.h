// The 8-bit form of activations, and the GLUs with their derivatives: shared by the elementwise passes (moe_act8.hip) and the
// products' epilogue (moe_mm.h).
#pragma once
#include "moe_common.h"

namespace moe {

// Blocks of 32 neighbours share one exponent byte s: value = q 2^(s - 133), q in [-127, 127]. s is the biased exponent of
// the block's largest magnitude (so that one keeps 7 bits, 64 <= |q| <= 127), one more where it would round to 128; 0 for a
// block below 2^-126 (whose 16-bit values stay exact), 255 marks a block that holds an infinity or NaN and reads as NaN.
// With a power of two the scaling is exact, so an element is off by its rounding alone, at most half a step 2^(s - 134). The
// block's largest is 63.75 (s one more) to 127.5 steps, so that is at most 1/127.5 of it.
__device__ __forceinline__ uint32_t exponent8(uint32_t top) {   // of the bits of a block's largest magnitude (fp32)
    const uint32_t s = top >> 23;
    return s > 0 && s < 254 && (top & 0x7fffffu) >= 0x7f0000u ? s + 1 : s;   // 127.5 and up
}
__device__ __forceinline__ uint32_t code8(float v, uint32_t s) {   // s < 255
    return (uint32_t)(int)fminf(fmaxf(rintf(ldexpf(v, 133 - (int)s)), -127.f), 127.f) & 255u;
}
__device__ __forceinline__ float value8(uint32_t byte, uint32_t s) {
    return s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf((float)(int8_t)byte, (int)s - 133);
}

// h = f(g) * m(u), with df/dg and dm/du. act 2 clamps g <= 7, |u| <= 7: no gradient where the clamp holds.
__device__ __forceinline__ void glu_parts(int act, float g, float u, float& f, float& m, float& df, float& dm) {
    m = u;
    dm = 1.f;
    if (act == MOE_ACT_GEGLU) {
        const float z = 1.5957691216057308f * (g + 0.044715f * g * g * g), s = sigmoid_fast(z);
        f = g * s;
        // far out sigmoid' is 0 and the polynomial overflows: their product is 0
        const float ds = s * (1.f - s);
        df = s + (ds == 0.f ? 0.f : g * ds * 1.5957691216057308f * (1.f + 0.134145f * g * g));
        return;
    }
    float a = 1.f, on = 1.f;
    if (act == MOE_ACT_GPTOSS) {
        a = 1.702f;
        // comparisons that a NaN fails leave it in place
        on = g > 7.f ? 0.f : 1.f;
        dm = u > 7.f || u < -7.f ? 0.f : 1.f;
        g = g > 7.f ? 7.f : g;
        m = (u > 7.f ? 7.f : u < -7.f ? -7.f : u) + 1.f;
    }
    const float s = sigmoid_fast(a * g), ds = s * (1.f - s);
    f = g * s;
    df = on * (s + (ds == 0.f ? 0.f : a * g * ds));
}

}  // namespace moe
