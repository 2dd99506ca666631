// Sums over strips of rows, added up in their order.
#pragma once

#include "dense_gemm.hpp"
#include "wave_ops.hpp"

namespace npamd {

constexpr int kStripColumns = 64, kStripShares = 16;  // of a block

// Columns 64 `block` .. + 63, by WAVES waves.  Strips in sixteen shares, whose sums are added in their order whatever the number of waves; `meet` holds 64 values for each share.
template <int ACT, int WAVES>
__device__ __forceinline__ void add_strips(const StripSums& s, int block, float* meet) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = block * kStripColumns + lane;
#pragma unroll
  for (int k = 0; k < kStripShares / WAVES; ++k) {
    const int share = WAVES * k + wave, first = s.strips * share / kStripShares, last = s.strips * (share + 1) / kStripShares;
    float v = 0.f;
    if (col < s.columns) {
#pragma unroll 8
      for (int i = first; i < last; ++i) v += s.partials[(int64_t)i * s.columns + col];
    }
    meet[share * kStripColumns + lane] = v;
  }
  __syncthreads();
  if (wave || col >= s.columns) return;
  float v = meet[lane];
#pragma unroll
  for (int i = 1; i < kStripShares; ++i) v += meet[i * kStripColumns + lane];
  if (s.out_f32) ((float*)s.out)[col] = v;
  else store_from_f32<ACT>(s.out, col, v);
}

inline int strip_blocks(const StripSums& s) { return (s.columns + kStripColumns - 1) / kStripColumns; }

}  // namespace npamd
