// Dense product with an epilogue: y = act(x @ W^T + bias) + residual, f32 up to the one rounding at the store.
#include "activation.hpp"
#include "common.hpp"

using namespace npamd;

namespace {

struct DenseActArgs {
  const void *x, *w, *bias, *residual;
  void* y;
  int64_t ldx, ldw, ldr, ldy;
  int M, N, K, act, bias_f32;
};

// 16 x 16 outputs to a block, a thread each; any shape and alignment.
template <int ACT>
__global__ void __launch_bounds__(256) dense_act_kernel(const DenseActArgs a) {
  __shared__ float xs[16][33], ws[16][33];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16;
  float acc = 0.f;
  for (int k0 = 0; k0 < a.K; k0 += 32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = threadIdx.x + 256 * i, row = at >> 5, k = at & 31;
      const bool in = k0 + k < a.K;
      xs[row][k] = in && m0 + row < a.M ? load_as_f32<ACT>(a.x, (m0 + row) * a.ldx + k0 + k) : 0.f;
      ws[row][k] = in && n0 + row < a.N ? load_as_f32<ACT>(a.w, (n0 + row) * a.ldw + k0 + k) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; ++k) acc = __builtin_fmaf(xs[r][k], ws[c][k], acc);
    __syncthreads();
  }
  const int64_t m = m0 + r, n = n0 + c;
  if (m >= a.M || n >= a.N) return;
  if (a.bias) acc += a.bias_f32 ? ((const float*)a.bias)[n] : load_as_f32<ACT>(a.bias, n);
  acc = activate(a.act, acc);
  if (a.residual) acc += load_as_f32<ACT>(a.residual, m * a.ldr + n);
  store_from_f32<ACT>(a.y, m * a.ldy + n, acc);
}

}  // namespace

extern "C" int64_t npamd_dense_gemm_act_workspace_bytes(int, int, int) { return 0; }

extern "C" int npamd_dense_gemm_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int activation,
                                    const void* residual, int64_t ldr, void* y, int64_t ldy, int M, int N, int K, int act_dtype, void*, int64_t,
                                    void* stream) {
  const char* what = "npamd_dense_gemm_act";
  NPAMD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(!bias || bias_dtype == NPAMD_F32 || bias_dtype == act_dtype, "%s: the bias is f32 or of x's dtype", what);
  NPAMD_REQUIRE(activation >= NPAMD_ACT_NONE && activation <= NPAMD_ACT_SILU, "%s: unknown activation %d", what, activation);
  NPAMD_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), "%s: bad row stride", what);
  if (M == 0 || N == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && w && y, "%s: null pointer", what);
  const DenseActArgs a{x, w, bias, residual, y, ldx, ldw, ldr, ldy, M, N, K, activation, bias_dtype == NPAMD_F32};
  const dim3 grid((N + 15) / 16, (M + 15) / 16);
  launch(act_dtype == NPAMD_BF16 ? dense_act_kernel<NPAMD_BF16> : dense_act_kernel<NPAMD_F16>, grid, 256, 0, (hipStream_t)stream, a);
  return check_launch(what);
}
