// Activations of the dense products' epilogues.
#pragma once
#include "linear.h"
#include "wkv7_common.cuh"

namespace wkv7 {
namespace lin {

// ---- activations -----------------------------------------------------------------------------------------
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_f(float x) { return rcp_mufu(1.f + ex2_approx(-LOG2E * x)); }
__device__ __forceinline__ float tanh_f(float x) {
    // (1 - e) / (1 + e), e = exp(-2 |x|): relative error 2e-6 from |x| = 0.1 on; the series' first four terms below (next one: 2e-10)
    const float t = fabsf(x), e = ex2_approx(-2.f * LOG2E * t), x2 = x * x;
    const float big = copysignf((1.f - e) * rcp_mufu(1.f + e), x);
    const float small = x * (1.f + x2 * (-1.f / 3.f + x2 * (2.f / 15.f - x2 * (17.f / 315.f))));
    return t < 0.1f ? small : big;
}
constexpr float GELU_C = 1.5957691216057308f;  // 2 sqrt(2 / pi): gelu(x) = x sigmoid(GELU_C (x + 0.044715 x^3))
__device__ __forceinline__ float gelu_s(float x) { return sigmoid_f(GELU_C * x * (1.f + 0.044715f * x * x)); }
__device__ __forceinline__ float sqrt_f(float x) {  // relative error 2^-23
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float relu_f(float x) { return x < 0.f ? 0.f : x; }  // (a NaN stays one)

template <int ACT> __device__ __forceinline__ float act(float x) {
    switch (ACT) {
        case kActRelu: return relu_f(x);
        case kActRelu2: { const float r = relu_f(x); return r * r; }
        case kActTanh: return tanh_f(x);
        case kActSigmoid: return sigmoid_f(x);
        case kActSilu: return x * sigmoid_f(x);
        case kActGelu: return x * gelu_s(x);
        default: return x;
    }
}

}  // namespace lin
}  // namespace wkv7
