// The arguments of the dense product's kernels (dense_gemm.hip, wide_gemm.hpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace npamd {

// What becomes of a sum before it is rounded: act(sum + bias) + residual.  Null: none.
struct DenseEpilogue {
  const void* bias;      // [N], f32 or (bias_16) of the activations' type
  const void* residual;  // [M][N] of the activations' type, rows ldr apart
  int64_t ldr;
  int act, bias_16;
};

struct DenseShape {
  const void* x;
  const void* w;
  const float* bias;
  void* y;
  int64_t ldx, ldw, ldy;
  int M, N, steps;   // 64-k steps of a row
  int row_tiles, col_tiles, splits, units_per_die;  // unit: a part of K of one tile
  float* partials;   // splits > 1: [splits][M][N]
  int pieces;        // 16-byte pieces of a row: K / 8
  int group;         // row tiles of a group (wide tiles)
  DenseEpilogue ep;  // of the kernels that have one
};

// The product on wide tile `tile` of the plan's list; splits > 1: its parts, without their sum.
int launch_wide(const DenseShape& s, int act, int tile, hipStream_t st);
int launch_wide_epilogue(const DenseShape& s, int act, int tile, hipStream_t st);

// The product with an epilogue, on the tile and parts of K that are planned for the shape without one: x and w 16-byte aligned, K and rows' distances multiples of 8.
int dense_gemm_epilogue(const char* what, const DenseShape& s, int K, int act, int64_t workspace_bytes, hipStream_t st);

}  // namespace npamd
