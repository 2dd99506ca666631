// Activations of the epilogues, in f32.
#pragma once

#include "common.hpp"

namespace npamd {

__device__ __forceinline__ float silu_f32(float v) { return v / (1.f + __expf(-v)); }

// `act` is the same for every thread of a launch.
__device__ __forceinline__ float activate(int act, float v) {
  switch (act) {
    case NPAMD_ACT_RELU: return v < 0.f ? 0.f : v;  // a NaN stays one
    case NPAMD_ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678f);
    case NPAMD_ACT_GELU_TANH: return v / (1.f + __expf(-1.5957691f * (v + 0.044715f * v * v * v)));  // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u))
    case NPAMD_ACT_SILU: return silu_f32(v);
    default: return v;
  }
}

}  // namespace npamd
