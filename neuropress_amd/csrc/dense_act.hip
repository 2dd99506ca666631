// Dense product with an epilogue: y = act(x @ W^T + bias) + residual, f32 up to the one rounding at the store.
//
// Up to four tokens W is all that counts: every wave streams whole rows of it, 16 bytes a lane, into registers, x comes from the L1.  Past that the tiles of the dense
// product take it, with an epilogue of their own (wide_gemm.hpp, dense_gemm.hip).
#include "activation.hpp"
#include "common.hpp"
#include "dense_gemm.hpp"
#include "wave_ops.hpp"

using namespace npamd;

namespace {

struct FewArgs {
  const void *x, *w;
  void* y;
  int64_t ldx, ldw, ldy;
  int M, N, K;
  DenseEpilogue ep;
};

template <int ACT>
__device__ __forceinline__ void finish(const FewArgs& a, int m, int n, float v) {
  if (a.ep.bias) v += a.ep.bias_16 ? load_as_f32<ACT>(a.ep.bias, n) : ((const float*)a.ep.bias)[n];
  v = activate(a.ep.act, v);
  if (a.ep.residual) v += load_as_f32<ACT>(a.ep.residual, (int64_t)m * a.ep.ldr + n);
  store_from_f32<ACT>(a.y, (int64_t)m * a.ldy + n, v);
}

template <int ACT>
__device__ __forceinline__ float dot8(const u32x4& a, const u32x4& b, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum = __builtin_fmaf(act_bits_to_f32<ACT>(a[i] & 0xFFFFu), act_bits_to_f32<ACT>(b[i] & 0xFFFFu), sum);
    sum = __builtin_fmaf(act_bits_to_f32<ACT>(a[i] >> 16), act_bits_to_f32<ACT>(b[i] >> 16), sum);
  }
  return sum;
}

// R rows of W and TB tokens to a wave, KS of a block's four waves to a row, U pieces of each row on their way; tokens past TB in further blocks.  Any K and any
// addresses: a row that does not end with a piece of eight has its last one end with the row, and the values that the piece before has too are zeroed in x.
template <int ACT, int R, int TB, int KS, int U>
__global__ void __launch_bounds__(256) dense_few_kernel(const FewArgs a) {
  __shared__ float sums[4][R * TB];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % KS;
  const int64_t n0 = ((int64_t)blockIdx.x * (4 / KS) + wave / KS) * R;
  const int m0 = blockIdx.y * TB, pieces = (a.K + 7) / 8, tail = pieces * 8 - a.K;
  const uint16_t *wr[R], *xr[TB];
#pragma unroll
  for (int r = 0; r < R; ++r) wr[r] = (const uint16_t*)a.w + min(n0 + r, (int64_t)a.N - 1) * a.ldw;  // past the end: the last row, not stored
#pragma unroll
  for (int t = 0; t < TB; ++t) xr[t] = (const uint16_t*)a.x + (int64_t)min(m0 + t, a.M - 1) * a.ldx;
  float acc[R][TB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[r][t] = 0.f;
  // pieces [first, last) of the part, whole turns of 64 of them dealt out
  const int turns = (pieces + 63) / 64, first = turns * part / KS * 64, last = min(turns * (part + 1) / KS * 64, pieces);
  auto at = [&](int p) { return min(p * 8, a.K - 8); };
  auto tile = [&](int p, const u32x4 (&wv)[R]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      u32x4 xv = *reinterpret_cast<const u32x4_any*>(xr[t] + at(p));
      if (p == pieces - 1 && tail) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < tail) xv[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r][t] = dot8<ACT>(wv[r], xv, acc[r][t]);
    }
  };
  if (a.K >= 8) {
    int p = first + lane;
    for (; p + (U - 1) * 64 < last; p += U * 64) {
      u32x4 wv[U][R];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) wv[u][r] = *reinterpret_cast<const u32x4_any*>(wr[r] + at(p + u * 64));
#pragma unroll
      for (int u = 0; u < U; ++u) tile(p + u * 64, wv[u]);
    }
    for (; p < last; p += 64) {
      u32x4 wv[R];
#pragma unroll
      for (int r = 0; r < R; ++r) wv[r] = *reinterpret_cast<const u32x4_any*>(wr[r] + at(p));
      tile(p, wv);
    }
  } else if (part == 0 && lane < a.K) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < TB; ++t) acc[r][t] = load_as_f32<ACT>(wr[r], lane) * load_as_f32<ACT>(xr[t], lane);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const float v = wave_sum_last(acc[r][t]);
      if (lane == 63) sums[wave][r * TB + t] = v;
    }
  __syncthreads();
  if (part != 0 || lane >= R * TB) return;
  const int r = lane / TB, t = lane % TB;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < KS; ++i) v += sums[wave + i][lane];
  if (n0 + r < a.N && m0 + t < a.M) finish<ACT>(a, m0 + t, (int)(n0 + r), v);
}

constexpr int kFewTokens = 4;

template <int ACT>
int launch_few(const FewArgs& a, hipStream_t st, const char* what) {
#define NPAMD_FEW(R, TB, KS, U)                                                                                             \
  launch(dense_few_kernel<ACT, R, TB, KS, U>, dim3((unsigned)((a.N + R * (4 / KS) - 1) / (R * (4 / KS))), (unsigned)((a.M + TB - 1) / TB)), 256, 0, st, a)
  const int tb = a.M == 1 ? 1 : a.M == 2 ? 2 : 4;
  static const int ks_ = getenv("KS") ? atoi(getenv("KS")) : 0, r_ = getenv("RR") ? atoi(getenv("RR")) : 0;
  const int ks = ks_ ? ks_ : a.N < 8192 ? 4 : 1, rr = r_ ? r_ : tb == 1 ? 1 : 2;
  if (tb == 1) {
    if (rr == 1) { if (ks == 1) NPAMD_FEW(1, 1, 1, 4); else NPAMD_FEW(1, 1, 4, 4); }
    else { if (ks == 1) NPAMD_FEW(2, 1, 1, 4); else NPAMD_FEW(2, 1, 4, 4); }
  } else if (tb == 2) {
    if (rr == 1) { if (ks == 1) NPAMD_FEW(1, 2, 1, 4); else NPAMD_FEW(1, 2, 4, 4); }
    else { if (ks == 1) NPAMD_FEW(2, 2, 1, 4); else NPAMD_FEW(2, 2, 4, 4); }
  } else {
    if (rr == 1) { if (ks == 1) NPAMD_FEW(1, 4, 1, 4); else NPAMD_FEW(1, 4, 4, 4); }
    else { if (ks == 1) NPAMD_FEW(2, 4, 1, 4); else NPAMD_FEW(2, 4, 4, 4); }
  }
#undef NPAMD_FEW
  return check_launch(what);
}

bool tiles_take(const void* x, int64_t ldx, const void* w, int64_t ldw, int K) {
  return K % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && (((uintptr_t)x | (uintptr_t)w) & 15) == 0 && ldx < NPAMD_TILE_MAX_STRIDE && ldw < NPAMD_TILE_MAX_STRIDE;
}

}  // namespace

extern "C" int64_t npamd_dense_gemm_act_workspace_bytes(int M, int N, int K) {
  return M <= kFewTokens ? 0 : npamd_dense_gemm_workspace_bytes(M, N, (K + 63) / 64 * 64);
}

extern "C" int npamd_dense_gemm_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int activation,
                                    const void* residual, int64_t ldr, void* y, int64_t ldy, int M, int N, int K, int act_dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_dense_gemm_act";
  NPAMD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(!bias || bias_dtype == NPAMD_F32 || bias_dtype == act_dtype, "%s: the bias is f32 or of x's dtype", what);
  NPAMD_REQUIRE(activation >= NPAMD_ACT_NONE && activation <= NPAMD_ACT_SILU, "%s: unknown activation %d", what, activation);
  NPAMD_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), "%s: bad row stride", what);
  if (M == 0 || N == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && w && y, "%s: null pointer", what);
  hipStream_t st = (hipStream_t)stream;
  const DenseEpilogue ep{bias, residual, ldr, activation, bias_dtype != NPAMD_F32};
  const bool tiles = tiles_take(x, ldx, w, ldw, K);
  if (M <= kFewTokens || (M <= NPAMD_GEMV_MAX_M && !tiles)) {
    const FewArgs a{x, w, y, ldx, ldw, ldy, M, N, K, ep};
    return act_dtype == NPAMD_BF16 ? launch_few<NPAMD_BF16>(a, st, what) : launch_few<NPAMD_F16>(a, st, what);
  }
  NPAMD_REQUIRE(tiles, "%s: past %d tokens x and w have to lie at 16-byte addresses, K=%d and rows' distances have to be multiples of 8", what, NPAMD_GEMV_MAX_M, K);
  NPAMD_REQUIRE(!workspace || ((uintptr_t)workspace & 15) == 0, "%s: the workspace has to lie at a 16-byte address", what);
  const DenseShape s{x, w, nullptr, y, ldx, ldw, ldy, M, N, 0, 0, 0, 1, 0, (float*)workspace, 0, 0, ep};
  return dense_gemm_epilogue(what, s, K, act_dtype, workspace_bytes, st);
}
