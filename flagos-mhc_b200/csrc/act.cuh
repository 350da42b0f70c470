// act.cuh -- activations of the linear layer and the gated feed-forward block, in fp32.
#pragma once

#include "common.cuh"

namespace mhc {

// expf / division are the fast intrinsics (a few ulp of fp32, against outputs that keep 8 or
// 11 bits).  The sigmoid forms keep their relative accuracy in the negative tail, where
// 1 + tanh or 1 + erf would cancel.
__device__ __forceinline__ float sigmoid_fast(float z) {
  return __fdividef(1.f, 1.f + __expf(-z));
}

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluK = 0.044715f;

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == MHC_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN passes
  if constexpr (ACT == MHC_ACT_GELU) return 0.5f * z * erfcf(-0.7071067811865476f * z);
  // 0.5 z (1 + tanh(u)) = z sigmoid(2u)
  if constexpr (ACT == MHC_ACT_GELU_TANH)
    return z * sigmoid_fast(2.f * kGeluC * z * fmaf(kGeluK * z, z, 1.f));
  if constexpr (ACT == MHC_ACT_SILU) return z * sigmoid_fast(z);
  return z;
}

// value and derivative
template <int ACT>
__device__ __forceinline__ void act_both(float z, float& a, float& da) {
  if constexpr (ACT == MHC_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    da = z > 0.f ? 1.f : (z == z ? 0.f : z);
  } else if constexpr (ACT == MHC_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.7071067811865476f * z);
    a = z * cdf;
    da = fmaf(z * 0.3989422804014327f, __expf(-0.5f * z * z), cdf);
  } else if constexpr (ACT == MHC_ACT_GELU_TANH) {
    const float s = sigmoid_fast(2.f * kGeluC * z * fmaf(kGeluK * z, z, 1.f));
    a = z * s;
    // beyond |z| = 12 the sigmoid is 0 or 1 in fp32; the clamp keeps 0 * inf out
    const float zc = fminf(fmaxf(z, -12.f), 12.f);
    da = fmaf(zc * s * (1.f - s), 2.f * kGeluC * fmaf(3.f * kGeluK * zc, zc, 1.f), s);
  } else if constexpr (ACT == MHC_ACT_SILU) {
    const float s = sigmoid_fast(z);
    a = z * s;
    da = s * fmaf(z, 1.f - s, 1.f);
  } else {
    a = z;
    da = 1.f;
  }
}

#define MHC_DISPATCH_ACT(A_, FN)                          \
  switch (A_) {                                           \
    case MHC_ACT_NONE: return FN(MHC_ACT_NONE);           \
    case MHC_ACT_RELU: return FN(MHC_ACT_RELU);           \
    case MHC_ACT_GELU: return FN(MHC_ACT_GELU);           \
    case MHC_ACT_GELU_TANH: return FN(MHC_ACT_GELU_TANH); \
    case MHC_ACT_SILU: return FN(MHC_ACT_SILU);           \
    default: return MHC_ERR_INVALID_ARGUMENT;             \
  }

}  // namespace mhc
