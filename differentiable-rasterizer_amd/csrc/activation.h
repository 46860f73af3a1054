// Activations of the layers with products, and their slopes.
#pragma once

#include "layers.h"

namespace drh_nn {

constexpr float LOG2_E = 1.44269504088896341f, SQRT_HALF = 0.70710678118654752f, INV_SQRT_2PI = 0.39894228040143268f;
constexpr float TANH_C = 0.79788456080286536f, TANH_A = 0.044715f;

// EXACT: for results in 32 bits, with the library's functions; else for values that are
// rounded to 16 bits afterwards, by single instructions.

// 1 / (1 + exp(-v))
template <bool EXACT>
__device__ inline float logistic(float v) {
    return EXACT ? 1.0f / (1.0f + expf(-v)) : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2_E * v));
}

// One instruction each, which passes NaN.
__device__ inline float not_below(float z, float lo) { return __builtin_elementwise_maximum(z, lo); }
__device__ inline float not_above(float z, float hi) { return __builtin_elementwise_minimum(z, hi); }

// act(z), and act'(z) in `slope`. Below -128 every value and slope is 0 in 32 bits, above 64
// every value z and slope 1; the bounds keep infinity times zero out of the products there.
template <bool EXACT, int ACT>
__device__ inline float act(float z, float& slope) {
    if constexpr (ACT == DRH_ACT_NONE) {
        slope = 1.0f;
        return z;
    } else if constexpr (ACT == DRH_ACT_RELU) {
        slope = z > 0.0f ? 1.0f : 0.0f;
        return z < 0.0f ? 0.0f : z;
    } else {
        z = not_below(z, -128.0f);
        const float c = not_above(z, 64.0f);
        if constexpr (ACT == DRH_ACT_SILU) {
            const float s = logistic<EXACT>(c);
            slope = s * fmaf(c, 1.0f - s, 1.0f);
            return z * s;
        } else if constexpr (ACT == DRH_ACT_GELU_TANH) {
            const float u = TANH_A * c * c, s = logistic<EXACT>(2.0f * TANH_C * fmaf(u, c, c));  // (1 + tanh) / 2
            slope = fmaf(2.0f * TANH_C * c * s * (1.0f - s), fmaf(3.0f, u, 1.0f), s);
            return z * s;
        } else {
            // Phi(c) and exp(-c^2 / 2). Phi is made from its own tail and not as (1 + erf) / 2, which
            // cancels below zero: at -5 that leaves two bits.
            float phi, e;
            if constexpr (EXACT) {
                phi = 0.5f * erfcf(-SQRT_HALF * c);
                e = expf(-0.5f * c * c);
            } else {
                // Phi(-|c|) = e t P(t), t = 1 / (1 + 0.292 |c|), in the manner of Abramowitz and Stegun
                // 7.1.26, with P fitted to stay within 1e-7 of Phi and 6e-5 of its value down to -13
                e = __builtin_amdgcn_exp2f(c * c * (-0.5f * LOG2_E));
                const float t = __builtin_amdgcn_rcpf(fmaf(0.292f, fabsf(c), 1.0f));
                float q = fmaf(t, -0.0867610723f, 0.27079457f);
                q = fmaf(t, q, -0.0762883946f);
                q = fmaf(t, q, 0.170907423f);
                q = fmaf(t, q, 0.103905939f);
                q = fmaf(t, q, 0.117441483f);
                q *= t * e;
                phi = c < 0.0f ? q : 1.0f - q;
            }
            slope = fmaf(c * INV_SQRT_2PI, e, phi);
            return z * phi;
        }
    }
}

// The type that slopes are kept in.
template <class T>
using Kept = std::conditional_t<sizeof(T) == 4, float, f16>;
template <class T>
constexpr float KEPT_SCALE = sizeof(T) == 4 ? 1.0f : 32768.0f;

// act(z) and its slope for the activation `kind`, the same for all lanes.
template <bool EXACT>
__device__ inline float act_of(int kind, float z, float& slope) {
    switch (kind) {
        case DRH_ACT_RELU: return act<EXACT, DRH_ACT_RELU>(z, slope);
        case DRH_ACT_GELU: return act<EXACT, DRH_ACT_GELU>(z, slope);
        case DRH_ACT_GELU_TANH: return act<EXACT, DRH_ACT_GELU_TANH>(z, slope);
        case DRH_ACT_SILU: return act<EXACT, DRH_ACT_SILU>(z, slope);
        default: return act<EXACT, DRH_ACT_NONE>(z, slope);
    }
}

// f(activation) as a constant.
template <class F>
int with_act(int act, F&& f) {
    using std::integral_constant;
    switch (act) {
        case DRH_ACT_RELU: return f(integral_constant<int, DRH_ACT_RELU>());
        case DRH_ACT_GELU: return f(integral_constant<int, DRH_ACT_GELU>());
        case DRH_ACT_GELU_TANH: return f(integral_constant<int, DRH_ACT_GELU_TANH>());
        case DRH_ACT_SILU: return f(integral_constant<int, DRH_ACT_SILU>());
        default: return f(integral_constant<int, DRH_ACT_NONE>());
    }
}

}  // namespace drh_nn
