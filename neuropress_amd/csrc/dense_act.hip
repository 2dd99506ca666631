// Dense product with an epilogue: y = act(x @ W^T + bias) + residual, f32 up to the one rounding at the store.
//
// For few tokens W is all that counts.  One and two: every wave streams whole rows of it into registers.  Up to 16, 32 or 64: whole lines into LDS, MFMAs.  More: the tiles of the
// dense product, with an epilogue of their own (wide_gemm.hpp, dense_gemm.hip).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "dense_gemm.hpp"
#include "dense_rows.hpp"

using namespace npamd;

namespace {

template <int ACT, int MT, int R>
int launch_some_tile(const FewArgs& a, int waves, hipStream_t st, const char* what) {
  using T = SomeTile<MT, R>;
  const int lds = T::lds(waves);
  static LdsLatch latch;
  const auto kernel = dense_some_kernel<ACT, MT, R>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
  launch(kernel, (unsigned)((a.N + 16 * R - 1) / (16 * R)), 64 * waves, lds, st, a);
  return check_launch(what);
}

// Row tiles of a block and its waves, us at eight tokens: 8192 x 2048 with one / two 11.3 / 9.5, 4096 x 4096 9.5 / 12.3; with four waves 4096 x 4096 11.1.
template <int ACT>
int launch_some(const FewArgs& a, hipStream_t st, const char* what) {
  const int steps = (a.K / 8 + 15) / 16, mt = (a.M + 15) / 16, r = a.N >= 8192 && mt <= 2 ? 2 : 1;
  const int waves = std::min(std::min(8, steps), 160 * 1024 / ((mt + r) * 8192));
  if (mt == 1) return r == 1 ? launch_some_tile<ACT, 1, 1>(a, waves, st, what) : launch_some_tile<ACT, 1, 2>(a, waves, st, what);
  if (mt == 2) return r == 1 ? launch_some_tile<ACT, 2, 1>(a, waves, st, what) : launch_some_tile<ACT, 2, 2>(a, waves, st, what);
  return mt == 3 ? launch_some_tile<ACT, 3, 1>(a, waves, st, what) : launch_some_tile<ACT, 4, 1>(a, waves, st, what);
}

// Rows of a wave: two from two tokens on, which then share a read of x.  Four waves to a row where there are few rows and each wave has
// columns to read (one token, one wave / four 1024 x 4096 4.1 / 3.7 us, 2048 x 8192 8.3 / 8.4, two tokens 10.5 / 8.9; but 4096 x 2048 5.4 / 6.1, 5488 x 311 3.7 / 5.9).
template <int ACT>
int launch_few(const FewArgs& a, hipStream_t st, const char* what) {
#define NPAMD_FEW(R, TB, KS)                                                                                                 \
  launch(dense_few_kernel<ACT, R, TB, KS, 4>, dim3((unsigned)((a.N + R * (4 / KS) - 1) / (R * (4 / KS))), (unsigned)((a.M + TB - 1) / TB)), 256, 0, st, a)
  const bool together = a.N <= 2048 && a.K > 1024;
  if (a.M == 1) {
    if (together) NPAMD_FEW(1, 1, 4);
    else NPAMD_FEW(1, 1, 1);
  } else if (a.M == 2) {
    if (together) NPAMD_FEW(2, 2, 4);
    else NPAMD_FEW(2, 2, 1);
  } else {
    if (together) NPAMD_FEW(2, 4, 4);
    else NPAMD_FEW(2, 4, 1);
  }
#undef NPAMD_FEW
  return check_launch(what);
}

// Which kernel takes a call; aligned: rows that the tiles can read.  Us with dense_few_kernel / dense_some_kernel / the tiles, silu and a residual: two tokens 4096 x 4096 9.1 /
// 9.3 / 13.9, 640 x 2048 3.3 / 3.9 / 8.9; eight 4096 x 4096 - / 9.5 / 13.9, 4096 x 14336 - / 23.7 / 28.1, 1024 x 4096 - / 5.3 / 9.5; 32 tokens 8192 x 2048 - / 14.0 / 14.7,
// 4096 x 4096 - / 14.0 / 19.7, 4096 x 14336 - / 35 / 29.  Past 32 tokens a block has few waves and reads many tokens: it needs a compute unit of its own and K no longer
// than that lasts: 64 tokens 4096 x 4096 16.0 / 18.0, 2048 x 2048 8.4 / 9.1, 3003 x 2184 11.7 / 15.8; but 8192 x 2048 19.9 / 13.6, 1024 x 4096 11.6 / 9.9, 2048 x 8192 24 / 15.
enum Path { kFew, kSome, kTiles };
Path path_of(int M, int N, int K, bool aligned) {
  if (M <= 2) return kFew;
  if (!aligned) return M <= NPAMD_GEMV_MAX_M ? kFew : kTiles;
  if (M <= 16 || (M <= 32 && (int64_t)N * K <= 1 << 24)) return kSome;
  return M <= 64 && N <= 4096 && K <= std::max(N, 2560) ? kSome : kTiles;
}

}  // namespace

extern "C" int64_t npamd_dense_gemm_act_workspace_bytes(int M, int N, int K) {
  return M < 1 || N < 1 || K < 1 || N > kMaxRows || K > kMaxColumns || path_of(M, N, K, true) != kTiles ? 0 : npamd_dense_gemm_workspace_bytes(M, N, (K + 63) / 64 * 64);
}

extern "C" int npamd_dense_gemm_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int activation,
                                    const void* residual, int64_t ldr, void* y, int64_t ldy, int M, int N, int K, int act_dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_dense_gemm_act";
  NPAMD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
  if (N > kMaxRows || K > kMaxColumns) return fail(NPAMD_ERR_UNSUPPORTED, "%s: N=%d and K=%d have to be at most 2^25 and 2^30", what, N, K);
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(!bias || bias_dtype == NPAMD_F32 || bias_dtype == act_dtype, "%s: the bias is f32 or of x's dtype", what);
  NPAMD_REQUIRE(activation >= NPAMD_ACT_NONE && activation <= NPAMD_ACT_SILU, "%s: unknown activation %d", what, activation);
  NPAMD_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), "%s: bad row stride", what);
  if (M == 0 || N == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && w && y, "%s: null pointer", what);
  hipStream_t st = (hipStream_t)stream;
  const DenseEpilogue ep{bias, residual, ldr, activation, bias_dtype != NPAMD_F32};
  const bool tiles = tiles_take(x, ldx, w, ldw, K);
  const FewArgs a{x, w, y, ldx, ldw, ldy, M, N, K, ep};
  const Path path = path_of(M, N, K, tiles);
  if (path == kSome) return act_dtype == NPAMD_BF16 ? launch_some<NPAMD_BF16>(a, st, what) : launch_some<NPAMD_F16>(a, st, what);
  if (path == kFew) {
    return act_dtype == NPAMD_BF16 ? launch_few<NPAMD_BF16>(a, st, what) : launch_few<NPAMD_F16>(a, st, what);
  }
  NPAMD_REQUIRE(tiles, "%s: past %d tokens x and w have to lie at 16-byte addresses, K=%d and rows' distances have to be multiples of 8", what, NPAMD_GEMV_MAX_M, K);
  NPAMD_REQUIRE(!workspace || ((uintptr_t)workspace & 15) == 0, "%s: the workspace has to lie at a 16-byte address", what);
  const DenseShape s{x, w, nullptr, y, ldx, ldw, ldy, M, N, 0, 0, 0, 1, 0, (float*)workspace, 0, 0, ep};
  return dense_gemm_epilogue(what, s, K, act_dtype, workspace_bytes, st);
}
