// What the kernels of 8-bit linear layers share: the scale of a block, the rounding to e4m3, the gated activation.
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace ph_fp8 {

constexpr int BLOCK = 128;                                     // values that share a scale
constexpr float TOP = 448.0f;                                  // the largest e4m3 value
constexpr float LEAST = 448.0f * 1.17549435e-38f;              // 448 * 2^-126

// max and min that keep what is no number
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Two values to e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// The gated activation of a (gate, up) pair.  kind 0: silu(g) * u; 1 clamped swish: g' = min(g, limit), u' = clamp(u, -limit,
// limit), g' * sigmoid(alpha g') * (u' + shift); 2: gelu(g) * u in the tanh form, 0.5 g (1 + tanh(y)) = g sigmoid(2 y),
// y = sqrt(2/pi) (g + 0.044715 g^3).
struct Gate {
    int kind;
    float alpha, limit, shift;
};
__device__ __forceinline__ float gated_value(const Gate& gate, float g, float u) {
    if (gate.kind == 0) return __fdividef(g, 1.0f + __expf(-g)) * u;
    if (gate.kind == 2) return __fdividef(g, 1.0f + __expf(-1.5957691216057308f * (g + 0.044715f * g * g * g))) * u;
    g = min_nan(g, gate.limit);
    u = min_nan(max_nan(u, -gate.limit), gate.limit);
    return __fdividef(g, 1.0f + __expf(-gate.alpha * g)) * (u + gate.shift);
}

}  // namespace ph_fp8
