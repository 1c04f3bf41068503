// The activations of gated experts and of products in 8 bits, and their slopes (device code).
#pragma once
#include "gelu_terms.hpp"

#include "../../include/fmoe_hip.h"

namespace fmoe {

__host__ __device__ inline bool is_gate_activation(int a) {
    return a == FMOE_ACT_NONE || a == FMOE_ACT_RELU || a == FMOE_ACT_GELU || a == FMOE_ACT_SILU;
}

// kNarrow: the result is rounded to a 16-bit type.  Then sigma(x) = 1 / (1 + e^-x) takes the hardware's exponential and reciprocal, off by
// up to (2 + |x|) 2^-23 of itself, and GELU the rational form of erf (1.5e-7); float32 takes the library's functions.
template <bool kNarrow> __device__ __forceinline__ float logistic(float x) {
    if (kNarrow) return __builtin_amdgcn_rcpf(1.f + __expf(-x));
    return 1.f / (1.f + expf(-x));
}
struct ActTerms { float value, slope; };
// act(x) and act'(x).  A NaN stays one.
template <bool kNarrow> __device__ __forceinline__ ActTerms gate_terms(float x, int act) {
    if (act == FMOE_ACT_SILU) {
        const float s = logistic<kNarrow>(x);
        return ActTerms{x * s, s * fmaf(x, 1.f - s, 1.f)};
    }
    if (act == FMOE_ACT_GELU) {
        if (kNarrow) {
            const gemm::GeluTerms g = gemm::gelu_terms(x);
            return ActTerms{x * g.cdf, fmaf(x, g.pdf, g.cdf)};
        }
        const float cdf = 0.5f + 0.5f * erff(x * 0.70710678118654752440f);
        return ActTerms{x * cdf, fmaf(x, 0.39894228040143267794f * expf(-0.5f * x * x), cdf)};
    }
    if (act == FMOE_ACT_RELU) return ActTerms{x < 0.f ? 0.f : x, x > 0.f ? 1.f : x == x ? 0.f : x};
    return ActTerms{x, 1.f};
}
template <bool kNarrow> __device__ __forceinline__ float gate_act(float x, int act) { return gate_terms<kNarrow>(x, act).value; }
// ReLU (floor 0) or none (minus infinity), which of them known when the kernel runs
struct ReluOrNone { float floor; };
template <bool kNarrow> __device__ __forceinline__ float gate_act(float x, ReluOrNone act) { return x < act.floor ? act.floor : x; }

}  // namespace fmoe
