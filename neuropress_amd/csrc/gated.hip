// The gated product of a feed-forward block, h = act(x Wg^T + bg) * (x Wu^T + bu), W's gate rows before its up rows, forward and backward.
//
// Forward: one launch per product as in the dense product with an epilogue (dense_rows.hpp for few tokens, wide_gemm.hpp past them), in forms whose waves have both sums of each of their
// values; sums, bias, activation and product in f32, one rounding.  Where the backward pass follows, both sums are left as well, rounded to x's type: it is what a training step in 16 bits
// keeps of them, half of what f32 would take.
// Backward, from those sums g and u and the gradient dh: dg = dh u act'(g), du = dh act(g) in f32, rounded to x's type as the matrix pipes' operands (one rounding of 2^-9 or
// 2^-12 of each of the terms that dx and dW add up, as in a training step whose pointwise part stands by itself; two parts of each would double the products, which are nearly
// all of the time; past 65504 they are infinite with fp16); then dx = [dg du] W and dW = [dg du]^T x on the wide tiles whose operands lie with the contracted index as their rows (nothing
// is transposed in memory), both in one launch where that is estimated to take less time (dense_gemm.hip), and the bias's gradient as f32 sums of the f32 values over strips of rows, added in
// their order.
#include <algorithm>
#include <type_traits>

#include "activation.hpp"
#include "common.hpp"
#include "dense_gemm.hpp"
#include "dense_rows.hpp"
#include "row_pieces.hpp"
#include "strip_sums.hpp"
#include "wave_ops.hpp"

using namespace npamd;

namespace {

template <int ACT, int MT, int R>
int launch_some_tile(const FewArgs& a, int waves, hipStream_t st, const char* what) {
  const int lds = SomeTile<MT, R>::lds(waves);
  static LdsLatch latch;
  const auto kernel = dense_some_kernel<ACT, MT, R, true>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
  launch(kernel, (unsigned)((a.N + 8 * R - 1) / (8 * R)), 64 * waves, lds, st, a);
  return check_launch(what);
}

// A tile of gate rows and one of up rows to a block; two of each past 4096 columns, where one leaves a second round of blocks mostly empty (us at four tokens, one / two: 4864 x 896 7.6 / 5.9,
// 5504 x 2048 12.8 / 11.6, 14336 x 4096 49 / 45; 4096 x 1024 5.3 / -).
template <int ACT>
int launch_some(const FewArgs& a, hipStream_t st, const char* what) {
  const int steps = (a.K / 8 + 15) / 16, mt = (a.M + 15) / 16, r = mt <= 2 && a.N > 4096 ? 4 : 2, waves = std::min(std::min(8, steps), 160 * 1024 / ((mt + r) * 8192));
  if (mt == 1) return r == 4 ? launch_some_tile<ACT, 1, 4>(a, waves, st, what) : launch_some_tile<ACT, 1, 2>(a, waves, st, what);
  if (mt == 2) return r == 4 ? launch_some_tile<ACT, 2, 4>(a, waves, st, what) : launch_some_tile<ACT, 2, 2>(a, waves, st, what);
  return launch_some_tile<ACT, 3, 2>(a, waves, st, what);
}

// A gate row and its up row to a wave, or (few and long) to a block's four.
template <int ACT>
int launch_few(const FewArgs& a, hipStream_t st, const char* what) {
#define NPAMD_FEW(TB, KS) launch(dense_few_kernel<ACT, 2, TB, KS, 4, true>, dim3((unsigned)((a.N + 4 / KS - 1) / (4 / KS)), (unsigned)((a.M + TB - 1) / TB)), 256, 0, st, a)
  const bool together = a.N <= 1024 && a.K > 1024;
  if (a.M == 1) {
    if (together) NPAMD_FEW(1, 4);
    else NPAMD_FEW(1, 1);
  } else if (a.M == 2) {
    if (together) NPAMD_FEW(2, 4);
    else NPAMD_FEW(2, 1);
  } else {
    if (together) NPAMD_FEW(4, 4);
    else NPAMD_FEW(4, 1);
  }
#undef NPAMD_FEW
  return check_launch(what);
}

// Which kernel takes a call; aligned: rows that the tiles can read.  One and two tokens: dense_few_kernel (us, silu, with it / dense_some_kernel / the tiles: 14336 x 4096 43.5 / 44.2 / 54.5,
// 1024 x 1024 3.6 / 4.0 / 7.1).  From three on dense_some_kernel, whose blocks have all of K, or the tiles, which may have parts of it.  Up to 4096 columns K has to be long for so few of them before the tiles are
// ahead; past them blocks of dense_some_kernel have 32 columns, and what decides is how full their last round is and, past 16 tokens, whether rows of W lie a multiple of 4096 bytes apart, which the tiles read more
// slowly.  Us, dense_some_kernel / the tiles: 16 tokens 512 x 2560 5.8 / 7.9, 512 x 14336 26.4 / 13.9, 8192 x 2048 15.8 / 18.0, 9728 x 512 9.7 / 8.2; 24 tokens 1024 x 2560 8.9 / 9.7, 1024 x 8192 18.9 / 12.8,
// 3584 x 3584 13.4 / 16.2, 4288 x 1024 8.4 / 8.0, 8192 x 2560 19.2 / 18.9, 8192 x 4096 29.3 / 31.3, 9728 x 4096 44.2 / 40.3, 14336 x 4096 49.5 / 57.2; 40 tokens 2048 x 2048 9.3 / 11.8, 2048 x 4096 14.5 / 12.9,
// 4096 x 4096 17.2 / 21.4, 8192 x 4096 32.1 / 31.6.  Over 180 shapes of 512 to 28672 columns and K of 512 to 14336, at nine numbers of tokens from 3 to 48, the kernel taken is 0.2 to 1.2 % slower than the better
// one in the mean, 26 % at most; over 110 others 0.3 to 1.8 %, 35 % at most.  far: outputs whose rows are too far apart for the tiles.
enum Path { kFew, kSome, kTiles };
Path path_of(int M, int N, int K, bool aligned, bool far) {
  if (M <= 2) return kFew;
  if (!aligned) return M <= NPAMD_GEMV_MAX_M ? kFew : kTiles;
  if (far && M <= NPAMD_GEMV_MAX_M) return kSome;
  if (N <= 4096) return M <= 48 && K <= std::max(M <= 16 ? 4096 : 2560, N * N >> (M <= 16 ? 9 : M <= 32 ? 10 : 11)) ? kSome : kTiles;
  const int blocks = (N + 31) / 32, rounds = (blocks + 255) / 256;
  return (M <= 16 && N <= 8192) || (M <= 32 && K % 2048 == 0 && 6 * blocks >= 5 * 256 * rounds) ? kSome : kTiles;
}

bool bad_shape(int M, int N, int K) { return M < 0 || N < 0 || K < 1; }
bool past_kernels(int M, int N, int K) { return N > kMaxRows / 2 || K > kMaxColumns; }

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------

struct GatedPointwise {
  const void *dh, *pre;
  void* dpre;  // [M][2 N], rows ldd apart
  int64_t lddh, ldp, ldd;
  float* partials;  // null, or [strips][2 N]
  int M, N, strips;
};

// act(g) and act'(g); both are NaN where g is.
template <int KIND>
__device__ __forceinline__ void activation_and_slope(float g, float& value, float& slope) {
  if constexpr (KIND == NPAMD_ACT_RELU) {
    value = g < 0.f ? 0.f : g;
    slope = g > 0.f ? 1.f : g <= 0.f ? 0.f : g;
  } else if constexpr (KIND == NPAMD_ACT_GELU) {
    const float cdf = gelu_cdf_f32(g);
    value = g * cdf;
    slope = __builtin_fmaf(g * 0.3989422804f, __builtin_amdgcn_exp2f(g * g * -0.72134752f), cdf);
  } else if constexpr (KIND == NPAMD_ACT_GELU_TANH) {
    // (1 + tanh(w)) / 2 = s: the slope is s + g s (1 - s) 2 w'(g), whose second term is zero in f32 from 13 on
    const float c = fminf(fmaxf(g, -16.f), 16.f), w = c * __builtin_fmaf(0.044715f * c, c, 1.f);
    const float e = __expf(-1.5957691216f * w), s = __builtin_amdgcn_rcpf(1.f + e);
    value = gelu_tanh_f32(g);
    slope = __builtin_fmaf(c * s * (1.f - s), 1.5957691216f * __builtin_fmaf(0.134145f * c, c, 1.f), s);
    slope = g == g ? slope : g;  // fmaxf drops a NaN
  } else if constexpr (KIND == NPAMD_ACT_SILU) {
    const float p = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    value = g * p;
    slope = __builtin_fmaf(value, 1.f - p, p);
  } else {
    value = g;
    slope = 1.f;
  }
}

// [dg du] of a strip of rows, a quarter of it to each of a block's waves: a lane has eight columns (rows that do not end with a piece: the last eight), which it adds up over its rows.  Bound by
// HBM: it reads three values and writes two of every one of dh; 4096 x 14336 103 us, 5.7 TB/s.
template <int ACT, int KIND>
__global__ void __launch_bounds__(256) gated_pointwise_kernel(const GatedPointwise a) {
  using P = Pieces<ACT>;
  __shared__ float sums[4][16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, piece = blockIdx.x * 64 + lane;
  const int at = min(piece * 8, a.N - 8);  // past the end: the last piece again, which stores the same
  const int64_t strip = (int64_t)blockIdx.y * 4 + wave, first = a.M * strip / (4 * a.strips), last = a.M * (strip + 1) / (4 * a.strips);
  float sum[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[0][e] = sum[1][e] = 0.f;
  constexpr int U = 4;  // rows on their way
  for (int64_t row0 = first; row0 < last; row0 += U) {
    u32x4 dv[U], gv[U], uv[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t row = row0 + i;
      if (row >= last) break;
      const uint8_t* const pr = P::row_of(a.pre, row, a.ldp);
      dv[i] = P::load(P::row_of(a.dh, row, a.lddh), at);
      gv[i] = P::load(pr, at);
      uv[i] = P::load(pr + (int64_t)a.N * 2, at);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (row0 + i >= last) break;
      float dh[8], g[8], u[8];
      P::unpack(dv[i], dh);
      P::unpack(gv[i], g);
      P::unpack(uv[i], u);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float value, slope;
        activation_and_slope<KIND>(g[e], value, slope);
        g[e] = dh[e] * u[e] * slope;
        u[e] = dh[e] * value;
        sum[0][e] += g[e];
        sum[1][e] += u[e];
      }
      uint8_t* const to = const_cast<uint8_t*>(P::row_of(a.dpre, row0 + i, a.ldd));
      P::store(to, at, P::pack(g));
      P::store(to + (int64_t)a.N * 2, at, P::pack(u));
    }
  }
  if (!a.partials) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[wave][e][lane] = sum[0][e], sums[wave][8 + e][lane] = sum[1][e];
  __syncthreads();
  float* const to = a.partials + (int64_t)blockIdx.y * 2 * a.N + at;
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // a wave adds up four of a lane's sixteen sums
    const int e = 4 * wave + i;
    to[(e >> 3) * (int64_t)a.N + (e & 7)] = sums[0][e][lane] + sums[1][e][lane] + sums[2][e][lane] + sums[3][e][lane];
  }
}

// Fewer than eight columns: a value to a thread.
template <int ACT, int KIND>
__global__ void __launch_bounds__(64) gated_pointwise_narrow_kernel(const GatedPointwise a) {
  const int n = threadIdx.x;
  if (n >= a.N) return;
  const int64_t first = (int64_t)a.M * blockIdx.y / a.strips, last = (int64_t)a.M * (blockIdx.y + 1) / a.strips;
  float sum_g = 0.f, sum_u = 0.f;
  for (int64_t row = first; row < last; ++row) {
    float value, slope;
    activation_and_slope<KIND>(load_as_f32<ACT>(a.pre, row * a.ldp + n), value, slope);
    const float dh = load_as_f32<ACT>(a.dh, row * a.lddh + n), dg = dh * load_as_f32<ACT>(a.pre, row * a.ldp + a.N + n) * slope, du = dh * value;
    store_from_f32<ACT>(a.dpre, row * a.ldd + n, dg);
    store_from_f32<ACT>(a.dpre, row * a.ldd + a.N + n, du);
    sum_g += dg;
    sum_u += du;
  }
  if (!a.partials) return;
  a.partials[(int64_t)blockIdx.y * 2 * a.N + n] = sum_g;
  a.partials[(int64_t)blockIdx.y * 2 * a.N + a.N + n] = sum_u;
}

// The strips' sums.  5478 columns of 250 strips 4.7 us, latency.
template <int ACT>
__global__ void __launch_bounds__(1024) gated_bias_kernel(const StripSums s) {
  __shared__ float meet[kStripShares * kStripColumns];
  add_strips<ACT, 16>(s, blockIdx.x, meet);
}

// Strips of rows: some 8192 waves where there are as many rows; 256 strips at most where their sums are kept.
int strips_of(int M, int N, bool sums) {
  const int columns = (N + 511) / 512;
  return std::min((M + 3) / 4, std::clamp(2048 / columns, 1, sums ? 256 : 2048));
}

struct BackSpace {
  int64_t ldd, dpre, partials, parts;  // row distance and bytes
  PairPlan pair{false, false, 0, 1};
  int64_t bytes() const { return dpre + partials + parts; }
  BackSpace(int M, int N, int K, bool dx, bool dw, bool db) {
    ldd = (2 * (int64_t)N + 7) / 8 * 8;
    dpre = (int64_t)M * ldd * 2;
    dpre = (dpre + 15) / 16 * 16;
    partials = db ? ((int64_t)strips_of(M, N, true) * 2 * N * 4 + 15) / 16 * 16 : 0;
    if (dx && dw) pair = plan_pair(M, K, 2 * N);
    parts = pair.together ? dense_gemm_pair_workspace_bytes(pair, M, K)
                          : std::max(dx ? dense_gemm_turned_workspace_bytes(M, K, 2 * N, false) : 0, dw ? dense_gemm_turned_workspace_bytes(2 * N, K, M, true) : 0);
  }
};

template <int ACT>
void launch_pointwise(const GatedPointwise& a, int act, hipStream_t st) {
  const dim3 grid((unsigned)(((a.N + 7) / 8 + 63) / 64), (unsigned)a.strips);
#define NPAMD_POINTWISE(KIND)                                                                                  \
  case KIND:                                                                                                   \
    if (a.N < 8) launch(gated_pointwise_narrow_kernel<ACT, KIND>, dim3(1, (unsigned)a.strips), 64, 0, st, a);  \
    else launch(gated_pointwise_kernel<ACT, KIND>, grid, 256, 0, st, a);                                       \
    break
  switch (act) {
    NPAMD_POINTWISE(NPAMD_ACT_RELU);
    NPAMD_POINTWISE(NPAMD_ACT_GELU);
    NPAMD_POINTWISE(NPAMD_ACT_GELU_TANH);
    NPAMD_POINTWISE(NPAMD_ACT_SILU);
    NPAMD_POINTWISE(NPAMD_ACT_NONE);
  }
#undef NPAMD_POINTWISE
}

}  // namespace

extern "C" int64_t npamd_gated_linear_workspace_bytes(int M, int N, int K) {
  return M < 1 || N < 1 || K < 1 || past_kernels(M, N, K) || path_of(M, N, K, true, false) != kTiles ? 0 : dense_gemm_gated_workspace_bytes(M, N, K);
}

extern "C" int npamd_gated_linear(const void* x, int64_t ldx, const void* gate_up, int64_t ldw, const void* bias, int bias_dtype, int activation, void* y, int64_t ldy,
                                  void* pre, int64_t ldp, int M, int N, int K, int act_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_gated_linear";
  NPAMD_REQUIRE(!bad_shape(M, N, K), "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
  if (past_kernels(M, N, K)) return fail(NPAMD_ERR_UNSUPPORTED, "%s: N=%d and K=%d have to be at most 2^24 and 2^30", what, N, K);
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(!bias || bias_dtype == NPAMD_F32 || bias_dtype == act_dtype, "%s: the bias is f32 or of x's dtype", what);
  NPAMD_REQUIRE(activation >= NPAMD_ACT_NONE && activation <= NPAMD_ACT_SILU, "%s: unknown activation %d", what, activation);
  NPAMD_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!pre || ldp >= 2 * (int64_t)N), "%s: bad row stride", what);
  if (M == 0 || N == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && gate_up && y, "%s: null pointer", what);
  hipStream_t st = (hipStream_t)stream;
  const DenseEpilogue ep{bias, nullptr, 0, activation, bias_dtype != NPAMD_F32, pre, ldp};
  const bool tiles = tiles_take(x, ldx, gate_up, ldw, K);
  const FewArgs a{x, gate_up, y, ldx, ldw, ldy, M, N, K, ep};
  const bool far = ldy >= NPAMD_TILE_MAX_STRIDE || (pre && ldp >= NPAMD_TILE_MAX_STRIDE);
  const Path path = path_of(M, N, K, tiles, far);
  if (path == kSome) return act_dtype == NPAMD_BF16 ? launch_some<NPAMD_BF16>(a, st, what) : launch_some<NPAMD_F16>(a, st, what);
  if (path == kFew) return act_dtype == NPAMD_BF16 ? launch_few<NPAMD_BF16>(a, st, what) : launch_few<NPAMD_F16>(a, st, what);
  NPAMD_REQUIRE(tiles, "%s: past %d tokens x and gate_up have to lie at 16-byte addresses, K=%d and rows' distances have to be multiples of 8", what, NPAMD_GEMV_MAX_M, K);
  NPAMD_REQUIRE(!workspace || ((uintptr_t)workspace & 15) == 0, "%s: the workspace has to lie at a 16-byte address", what);
  if (far)
    return fail(NPAMD_ERR_UNSUPPORTED, "%s: past %d tokens the outputs' rows have to be less than 2^22 apart", what, NPAMD_GEMV_MAX_M);
  DenseShape s{};
  s.x = x, s.w = gate_up, s.y = y, s.ldx = ldx, s.ldw = ldw, s.ldy = ldy, s.M = M, s.N = N, s.partials = (float*)workspace, s.ep = ep;
  return dense_gemm_gated(what, s, K, act_dtype, workspace_bytes, st);
}

extern "C" int64_t npamd_gated_linear_backward_workspace_bytes(int M, int N, int K, int dx, int dgate_up, int dbias) {
  if (M < 1 || N < 1 || K < 1 || past_kernels(M, N, K)) return 0;
  return BackSpace(M, N, K, dx, dgate_up, dbias).bytes();
}

extern "C" int npamd_gated_linear_backward(const void* dh, int64_t lddh, const void* x, int64_t ldx, const void* gate_up, int64_t ldw, const void* pre, int64_t ldp, int activation,
                                           void* dx, int64_t lddx, void* dgate_up, int64_t lddw, void* dbias, int bias_dtype, int M, int N, int K, int act_dtype,
                                           void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_gated_linear_backward";
  NPAMD_REQUIRE(M >= 1 && N >= 1 && K >= 1, "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
  if (past_kernels(M, N, K)) return fail(NPAMD_ERR_UNSUPPORTED, "%s: N=%d and K=%d have to be at most 2^24 and 2^30", what, N, K);
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(!dbias || bias_dtype == NPAMD_F32 || bias_dtype == act_dtype, "%s: the bias is f32 or of x's dtype", what);
  NPAMD_REQUIRE(activation >= NPAMD_ACT_NONE && activation <= NPAMD_ACT_SILU, "%s: unknown activation %d", what, activation);
  NPAMD_REQUIRE(lddh >= N && ldp >= 2 * (int64_t)N && (!dgate_up || (ldx >= K && lddw >= K)) && (!dx || (ldw >= K && lddx >= K)), "%s: bad row stride", what);
  NPAMD_REQUIRE(dh && pre && (!dx || gate_up) && (!dgate_up || x), "%s: null pointer", what);
  auto whole_pieces = [](const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld < NPAMD_TILE_MAX_STRIDE; };
  NPAMD_REQUIRE((!dx || whole_pieces(gate_up, ldw)) && (!dgate_up || whole_pieces(x, ldx)),
                "%s: x and gate_up have to lie at 16-byte addresses, rows' distances have to be multiples of 8 and below 2^22", what);
  const BackSpace space(M, N, K, dx != nullptr, dgate_up != nullptr, dbias != nullptr);
  if (space.ldd >= NPAMD_TILE_MAX_STRIDE || (dx && lddx >= NPAMD_TILE_MAX_STRIDE) || (dgate_up && lddw >= NPAMD_TILE_MAX_STRIDE) || K >= NPAMD_TILE_MAX_STRIDE)
    return fail(NPAMD_ERR_UNSUPPORTED, "%s: rows of 2 N=%d and K=%d values have to be less than 2^22 apart", what, N, K);
  NPAMD_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= space.bytes(), "%s: needs %lld bytes of 16-byte aligned workspace", what, (long long)space.bytes());
  hipStream_t st = (hipStream_t)stream;
  uint8_t* const at = (uint8_t*)workspace;
  float* const partials = dbias ? (float*)(at + space.dpre) : nullptr;
  const GatedPointwise a{dh, pre, at, lddh, ldp, space.ldd, partials, M, N, strips_of(M, N, dbias != nullptr)};
  if (act_dtype == NPAMD_BF16) launch_pointwise<NPAMD_BF16>(a, activation, st);
  else launch_pointwise<NPAMD_F16>(a, activation, st);
  DenseShape one{}, both{};
  one.partials = both.partials = (float*)(at + space.dpre + space.partials);
  one.x = both.x = at, one.ldx = both.ldx = space.ldd;
  one.w = gate_up, one.ldw = ldw, one.y = dx, one.ldy = lddx, one.M = M, one.N = K;
  both.w = x, both.ldw = ldx, both.y = dgate_up, both.ldy = lddw, both.M = 2 * N, both.N = K;
  const StripSums sums{partials, a.strips, dbias ? 2 * N : 0, dbias, bias_dtype == NPAMD_F32};
  if (space.pair.together) {
    const int rc = check_launch(what);
    return rc != NPAMD_OK ? rc : dense_gemm_pair(what, space.pair, one, both, sums, act_dtype, st);
  }
  if (dbias) {
    if (act_dtype == NPAMD_BF16) launch(gated_bias_kernel<NPAMD_BF16>, (unsigned)strip_blocks(sums), 1024, 0, st, sums);
    else launch(gated_bias_kernel<NPAMD_F16>, (unsigned)strip_blocks(sums), 1024, 0, st, sums);
  }
  int rc = check_launch(what);
  if (rc == NPAMD_OK && dx) rc = dense_gemm_turned(what, one, 2 * N, false, act_dtype, space.parts, st);
  if (rc == NPAMD_OK && dgate_up) rc = dense_gemm_turned(what, both, M, true, act_dtype, space.parts, st);
  return rc;
}
