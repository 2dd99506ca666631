// Reductions over a wave in registers, dot products of eight values, and 16-byte loads at any address.
#pragma once

#include "common.hpp"

namespace npamd {

// Over a wave without LDS: each step takes a lane's value from another lane's register.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_move(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, lane_move<0x111, 0xF>(v));  // from 1, 2, 4, 8 lanes before, within 16 lanes
  v = max(v, lane_move<0x112, 0xF>(v));
  v = max(v, lane_move<0x114, 0xF>(v));
  v = max(v, lane_move<0x118, 0xF>(v));
  v = max(v, lane_move<0x142, 0xA>(v));  // lane 15 to the next 16, lane 31 to the upper half
  v = max(v, lane_move<0x143, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// The sum, in lane 63.
__device__ __forceinline__ float wave_sum_last(float v) {
  auto add = [&](uint32_t from) { v += __builtin_bit_cast(float, from); };
  auto bits = [&] { return __builtin_bit_cast(uint32_t, v); };
  add(lane_move<0x111, 0xF>(bits()));
  add(lane_move<0x112, 0xF>(bits()));
  add(lane_move<0x114, 0xF>(bits()));
  add(lane_move<0x118, 0xF>(bits()));
  add(lane_move<0x142, 0xA>(bits()));
  add(lane_move<0x143, 0xC>(bits()));
  return v;
}

// The sum, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum_last(v)), 63));
}

// sum + the dot product of eight values each, in f32.
template <int ACT>
__device__ __forceinline__ float add_dot8(const u32x4& a, const u32x4& b, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum = __builtin_fmaf(act_bits_to_f32<ACT>(a[i] & 0xFFFFu), act_bits_to_f32<ACT>(b[i] & 0xFFFFu), sum);
    sum = __builtin_fmaf(act_bits_to_f32<ACT>(a[i] >> 16), act_bits_to_f32<ACT>(b[i] >> 16), sum);
  }
  return sum;
}

// Four dwords at any even address: the card's memory takes them as they lie.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

}  // namespace npamd
