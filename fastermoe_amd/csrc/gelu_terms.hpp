// GELU's two functions of its argument (device code).
#pragma once
#include <hip/hip_runtime.h>

namespace fmoe {
namespace gemm {

// erf by Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7): a reciprocal, an exponential and
// five multiply-adds instead of the library routine's branches.  The same exponential,
// exp(-x^2/2), is the Gaussian of GELU's derivative.
struct GeluTerms {
    float cdf;  // Phi(x) = 0.5 (1 + erf(x / sqrt 2))
    float pdf;  // phi(x) = exp(-x^2 / 2) / sqrt(2 pi)
};
__device__ __forceinline__ GeluTerms gelu_terms(float x) {
    const float z = fabsf(x) * 0.70710678118654752440f;
    const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * z);
    const float e = __expf(-z * z);
    const float poly = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float erf_abs = 1.f - poly * e;
    const float half_erf = 0.5f * (x < 0.f ? -erf_abs : erf_abs);
    return GeluTerms{0.5f + half_erf, 0.39894228040143267794f * e};
}

}  // namespace gemm
}  // namespace fmoe
