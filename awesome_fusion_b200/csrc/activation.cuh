// The activation of the pair form's fused epilogue (pair.cu).
#pragma once

namespace afb {

// 1 / (1 + 2^t), t = -v log2(e), without a branch.  The rounding error of the product t comes back as a first-order factor (TwoProduct by
// fused multiply-add, Ogita, Rump and Oishi 2005): without it, as in exp(), it grows with |v|.  Beyond the clamp the result is 0 or 1 in fp32;
// NaN and infinities come back with the v that the caller multiplies by.
__device__ __forceinline__ float sigmoid(float v) {
    const float x = fminf(fmaxf(v, -128.f), 128.f);
    constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f, kLog2eLow = 1.92596299e-8f;   // log2(e) = kLog2e + kLog2eLow
    const float t = x * -kLog2e, low = fmaf(x, -kLog2eLow, fmaf(x, -kLog2e, -t));
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    const float better = fmaf(e, low * kLn2, e);
    e = t < 128.f ? better : e;   // infinite from there on
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}

}  // namespace afb
