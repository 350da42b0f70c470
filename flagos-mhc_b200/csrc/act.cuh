// act.cuh -- activations of the linear layer and the gated feed-forward block, in fp32.
#pragma once

#include "common.cuh"

namespace mhc {

// exp and division are the fast intrinsics, against outputs that keep 8 or 11 bits: exp(x) is off
// by 2 + 1.2 |x| units in the last place, so a few where the functions are of any size and about 1e-5
// relative at the far negative end.  The sigmoid forms keep their relative accuracy in the negative
// tail, where 1 + tanh or 1 + erf would cancel; below -87.3 the sigmoid (1e-38 and less) is 0.
__device__ __forceinline__ float sigmoid_fast(float z) {
  return __fdividef(1.f, 1.f + __expf(-z));
}

// The functions that vanish for z -> -inf are 0 there, and their derivatives 0 or 1 beyond either
// end: a z kept in fp16 may have become infinite.  The factors z are clamped where the other
// factor is exactly 0 already, so that no 0 * inf arises (NaN still passes, by the other factor).
__device__ __forceinline__ float floor_z(float z) { return fmaxf(z, -128.f); }
__device__ __forceinline__ float clamp_z(float z) { return fminf(fmaxf(z, -128.f), 128.f); }

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluK = 0.044715f;

// The normal distribution function, and e = exp(-z^2 / 2).  With x = |z| / sqrt(2),
// erfc(x) = e t P(t), t = 1 / (1 + 0.38 x): P is a fit of erfcx(x) / t of degree 6, weighted for
// the relative error over x = 0 .. 9.5 (1.1e-6; 1.4e-6 with fp32 arithmetic), so the negative tail
// keeps its accuracy.  The backward needs e anyway; with erfcf it was bound by its instructions
// (65536 x 4096 elements: 606 us, 312 us for silu).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  e = __expf(-0.5f * z * z);
  const float t = __fdividef(1.f, fmaf(0.38f * 0.7071067811865476f, fabsf(z), 1.f));
  float p = -0.1250499039888382f;
  p = fmaf(p, t, 0.3346192240715027f);
  p = fmaf(p, t, -0.06771065294742584f);
  p = fmaf(p, t, 0.2460743486881256f);
  p = fmaf(p, t, 0.18135355412960052f);
  p = fmaf(p, t, 0.2164105623960495f);
  p = fmaf(p, t, 0.21430183947086334f);
  const float q = 0.5f * t * p * e;
  return z < 0.f ? q : 1.f - q;
}

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == MHC_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN passes
  if constexpr (ACT == MHC_ACT_GELU) {
    float e;
    return floor_z(z) * normal_cdf(z, e);
  }
  // 0.5 z (1 + tanh(u)) = z sigmoid(2u)
  if constexpr (ACT == MHC_ACT_GELU_TANH)
    return floor_z(z) * sigmoid_fast(2.f * kGeluC * z * fmaf(kGeluK * z, z, 1.f));
  if constexpr (ACT == MHC_ACT_SILU) return floor_z(z) * sigmoid_fast(z);
  return z;
}

// value and derivative
template <int ACT>
__device__ __forceinline__ void act_both(float z, float& a, float& da) {
  if constexpr (ACT == MHC_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    da = z > 0.f ? 1.f : (z == z ? 0.f : z);
  } else if constexpr (ACT == MHC_ACT_GELU) {
    float e;
    const float cdf = normal_cdf(z, e);
    a = floor_z(z) * cdf;
    da = fmaf(clamp_z(z) * 0.3989422804014327f, e, cdf);
  } else if constexpr (ACT == MHC_ACT_GELU_TANH) {
    const float s = sigmoid_fast(2.f * kGeluC * z * fmaf(kGeluK * z, z, 1.f));
    a = floor_z(z) * s;
    // beyond |z| = 12 the sigmoid is 0 or 1 in fp32
    const float zc = fminf(fmaxf(z, -12.f), 12.f);
    da = fmaf(zc * s * (1.f - s), 2.f * kGeluC * fmaf(3.f * kGeluK * zc, zc, 1.f), s);
  } else if constexpr (ACT == MHC_ACT_SILU) {
    const float s = sigmoid_fast(z);
    a = floor_z(z) * s;
    da = s * fmaf(clamp_z(z), 1.f - s, 1.f);
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
