// What the norms share: rows in registers in pieces of 16 bytes, sums over a block.
#pragma once

#include "common.hpp"
#include "wave_ops.hpp"

namespace npamd {

// Rows of a launch that gives each a block of 256 threads: a launch has fewer than 2^32 threads.
constexpr int64_t kRowsAtOnce = 1 << 23;
constexpr int kMaxWidth = 1 << 27;

// The sum over a block of 256 threads, in every one of them.  `part`: four floats of the block's own for this sum.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = wave_reduce_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

// A row in registers goes in pieces of 16 bytes, V values, at whatever address; a row that does not end with a piece has its last one end with the row, and the values
// that the piece before has too count once (and are stored twice, the same).
template <int DT>
struct Pieces {
  static constexpr int V = DT == NPAMD_F32 ? 4 : 8, kBytes = DT == NPAMD_F32 ? 4 : 2;
  // Value `at` of a row, which is the same for all lanes.
  static __device__ __forceinline__ u32x4 load(const uint8_t* row, int at) { return *reinterpret_cast<const u32x4_any*>(row + (uint32_t)at * kBytes); }
  static __device__ __forceinline__ void store(uint8_t* row, int at, const u32x4& v) { *reinterpret_cast<u32x4_any*>(row + (uint32_t)at * kBytes) = v; }
  static __host__ __device__ __forceinline__ const uint8_t* row_of(const void* p, int64_t row, int64_t ld) { return (const uint8_t*)p + row * ld * kBytes; }
  // What is made of a piece from here on is made anew: kept since it was made before, it would take two to four times the registers.
  static __device__ __forceinline__ void forget(u32x4& v) {
    if constexpr (DT != NPAMD_F32) asm volatile("" : "+v"(v));
  }
  static __device__ __forceinline__ void unpack(const u32x4& v, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == NPAMD_F32) {
        f[i] = __builtin_bit_cast(float, (uint32_t)v[i]);
      } else {
        f[2 * i] = act_bits_to_f32<DT>(v[i] & 0xFFFFu);
        f[2 * i + 1] = act_bits_to_f32<DT>(v[i] >> 16);
      }
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&f)[V]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == NPAMD_F32) v[i] = __builtin_bit_cast(uint32_t, f[i]);
      else if constexpr (DT == NPAMD_BF16) v[i] = f32_to_bf16_bits(f[2 * i]) | (f32_to_bf16_bits(f[2 * i + 1]) << 16);
      else v[i] = f32_to_f16_bits(f[2 * i]) | (f32_to_f16_bits(f[2 * i + 1]) << 16);
    }
    return v;
  }
};

}  // namespace npamd
