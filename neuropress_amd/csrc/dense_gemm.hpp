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
  // Of the gated product act(gate sum) * up sum, N columns of each, gate rows of w before up rows: null, or where the two sums go, [M][2 N], rows ldp apart.
  void* pre;
  int64_t ldp;
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
  int K;             // of the kernels with an operand whose rows are the contracted ones
};

// Values of a row of the parts of the gated products and those with turned operands: whole 16 bytes.
__host__ __device__ constexpr int parts_row(int N) { return (N + 3) / 4 * 4; }

// The product on wide tile `tile` of the plan's list; splits > 1: its parts, without their sum.
int launch_wide(const DenseShape& s, int act, int tile, hipStream_t st);
int launch_wide_epilogue(const DenseShape& s, int act, int tile, hipStream_t st);

// The product with an epilogue, on the tile and parts of K that are planned for the shape without one: x and w 16-byte aligned, K and rows' distances multiples of 8.
int dense_gemm_epilogue(const char* what, const DenseShape& s, int K, int act, int64_t workspace_bytes, hipStream_t st);

// The gated product (s.N: columns of y), x and w as above; its bytes of workspace.
int dense_gemm_gated(const char* what, const DenseShape& s, int K, int act, int64_t workspace_bytes, hipStream_t st);
int64_t dense_gemm_gated_workspace_bytes(int M, int N, int K);

// y[m][n] = sum over k of x w with w as [K][N] and, with x_too, x as [K][M]: rows 16-byte aligned, their distances multiples of 8, readable up to a multiple of eight columns; x
// as [M][K] up to a multiple of eight k.  Any K: what lies past it counts for nothing.
int dense_gemm_turned(const char* what, const DenseShape& s, int K, bool x_too, int act, int64_t workspace_bytes, hipStream_t st);
int64_t dense_gemm_turned_workspace_bytes(int M, int N, int K, bool x_too);

// Sums over strips of rows, [strips][columns] in f32, that are still to be added up, in their order: out in f32 or the activations' type.  columns 0: none.
struct StripSums {
  const float* partials;
  int strips, columns;
  void* out;
  int out_f32;
};

// The two products behind a gradient dp [M][K2] in one launch: dx [M][N] = dp w, w [K2][N], and dw [K2][N] = dp^T x, x [M][N] (`one` and `both` as for dense_gemm_turned), and the sums.
// The plan says whether that takes less time than one after the other.
struct PairPlan {
  bool together, both_first;
  int tile, splits;
};
PairPlan plan_pair(int M, int N, int K2);
int64_t dense_gemm_pair_workspace_bytes(const PairPlan& p, int M, int N);
int dense_gemm_pair(const char* what, const PairPlan& p, const DenseShape& one, const DenseShape& both, const StripSums& sums, int act, hipStream_t st);

int launch_wide_pair(const DenseShape& one, const DenseShape& both, const StripSums& sums, int act, int tile, bool both_first, hipStream_t st);
int launch_wide_gated(const DenseShape& s, int act, int tile, hipStream_t st);
int launch_wide_turned(const DenseShape& s, int act, int tile, bool x_too, hipStream_t st);

}  // namespace npamd
