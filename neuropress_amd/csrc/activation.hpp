// Activations of the epilogues, in f32: to 2^-20 of their argument.  None is infinite or NaN at a finite argument whose activation is not; those of minus infinity but
// ReLU's are NaN, as a product of it and zero.
#pragma once

#include "common.hpp"

namespace npamd {

__device__ __forceinline__ float silu_f32(float v) { return v * __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// v Phi(v), Phi by erfc: exp(z^2) erfc(z) / 2, z = |v| / sqrt(2), is a polynomial in t = 1 / (1 + 0.51 z) without a constant term, to 9e-7 relative (fitted up to z = 10,
// past which exp(-z^2) is zero).  GELU itself is off by up to 7e-6 relative where it is small, far below zero (5e-6 from
// -9 on, 2e-6 from -6): the exponent is rounded, 2^-24 of some v^2.
__device__ __forceinline__ float gelu_cdf_f32(float v) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.51f * 0.70710678f, fabsf(v), 1.f));
  float q = 0.047250088304281235f;
  q = __builtin_fmaf(q, t, -0.17956776916980743f);
  q = __builtin_fmaf(q, t, 0.17922323942184448f);
  q = __builtin_fmaf(q, t, 0.02752617374062538f);
  q = __builtin_fmaf(q, t, 0.1395331472158432f);
  q = __builtin_fmaf(q, t, 0.14207614958286285f);
  q = __builtin_fmaf(q, t, 0.14395874738693237f);
  const float half = q * t * __builtin_amdgcn_exp2f(v * v * -0.72134752f);  // exp(-v^2 / 2)
  return v < 0.f ? half : 1.f - half;
}
__device__ __forceinline__ float gelu_f32(float v) { return v * gelu_cdf_f32(v); }

// (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u))
__device__ __forceinline__ float gelu_tanh_f32(float v) {
  const float u = v * __builtin_fmaf(0.044715f * v, v, 1.f);
  return v * __builtin_amdgcn_rcpf(1.f + __expf(-1.5957691f * u));
}

// f(value) becomes every value's activation; `act` is the same for every thread of a launch, and looked at once.
template <class Each>
__device__ __forceinline__ void activate_all(int act, Each&& each) {
  switch (act) {
    case NPAMD_ACT_RELU: each([](float v) { return v < 0.f ? 0.f : v; }); break;  // a NaN stays one
    case NPAMD_ACT_GELU: each([](float v) { return gelu_f32(v); }); break;
    case NPAMD_ACT_GELU_TANH: each([](float v) { return gelu_tanh_f32(v); }); break;
    case NPAMD_ACT_SILU: each([](float v) { return silu_f32(v); }); break;
    default: break;
  }
}

__device__ __forceinline__ float activate(int act, float v) {
  activate_all(act, [&](auto f) { v = f(v); });
  return v;
}

}  // namespace npamd
