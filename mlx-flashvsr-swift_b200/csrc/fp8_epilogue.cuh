// fp8_epilogue.cuh — the epilogues of the linear layers on 8-bit operands, in fp32 on pairs of values; the caller rounds
// the result once.
#pragma once

#include "../../include/fvsr_lcsa.h"
#include "sm100.cuh"

namespace fvsr {

namespace sm100 {

// GELU with the tanh approximation, 0.5·x·(1 + tanh(√(2/π)·(x + 0.044715·x³))) = x / (1 + 2^z), z = x·(c0 + c1·x²),
// c0 = −2·√(2/π)·log2(e), c1 = 0.044715·c0, of two values at a time with one reciprocal, of the product of their
// denominators (the special-function unit is what bounds this). x is kept to −7.45, where z is 59.7 and the result −8e-18,
// so that the product stays finite and a value of any size below is off by no more than that (z alone kept to 60 left 2^-60
// of it, which was 87 for −1e20). A NaN stays with its own value: max.NaN keeps it, fminf makes its z 60, so the shared
// reciprocal is finite.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t gelu_tanh2(uint64_t x) {
    constexpr float c0 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, c1 = 0.044715f * c0;
    float x0, x1, z0, z1, d0, d1;
    uf2(x, x0, x1);
    x = f2(max_nan(x0, -7.45f), max_nan(x1, -7.45f));
    uf2(fmul2(x, ffma2(fmul2(x, x), f2(c1, c1), f2(c0, c0))), z0, z1);
    uf2(fadd2(f2(ex2_approx(fminf(z0, 60.0f)), ex2_approx(fminf(z1, 60.0f))), f2(1.0f, 1.0f)), d0, d1);
    const float r = rcp_approx(d0 * d1);
    return fmul2(x, fmul2(f2(d1, d0), f2(r, r)));
}

// What becomes of two neighbouring accumulators: first / last chain of their sum; kAdd: plus the values `add` (the
// residual, or what the chains before left).
template <int kMode, bool kAdd>
__device__ __forceinline__ uint64_t finish2(uint64_t acc, uint64_t bias, uint64_t gate, uint64_t add, bool first, bool last) {
    uint64_t y = first ? fadd2(acc, bias) : acc;
    if (kMode == FVSR_LINEAR_GATED_RESIDUAL)
        y = ffma2(gate, y, add);
    else if (kAdd)
        y = fadd2(y, add);
    if (kMode == FVSR_LINEAR_GELU && last) y = gelu_tanh2(y);
    return y;
}

}  // namespace sm100
}  // namespace fvsr
