// Dense product with an epilogue: y = act(x @ W^T + bias) + residual, f32 up to the one rounding at the store.
//
// For few tokens W is all that counts.  One and two: every wave streams whole rows of it into registers.  Up to 16, 32 or 64: whole lines into LDS, MFMAs.  More: the tiles of the
// dense product, with an epilogue of their own (wide_gemm.hpp, dense_gemm.hip).
#include <algorithm>
#include <type_traits>

#include "activation.hpp"
#include "common.hpp"
#include "dense_gemm.hpp"
#include "lds_transfer.hpp"
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

// R rows of W and TB tokens to a wave, KS of a block's four waves to a row, U pieces of each row on their way; tokens past TB in further blocks.  Any K and any
// addresses: a row that does not end with a piece of eight has its last one end with the row, and the values that the piece before has too are zeroed in both
// (an infinite one times zero would be NaN).  x comes from the L1.  4096 x 14336, one token: 22.1 us, 5.3 TB/s, the rate of reads; 640 x 2048 2.9 us.
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
  auto blank = [&](u32x4& v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < tail) v[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
  };
  auto tile = [&](int p, u32x4 (&wv)[R]) __attribute__((always_inline)) {
    const bool ends = p == pieces - 1 && tail;
    if (ends) {
#pragma unroll
      for (int r = 0; r < R; ++r) blank(wv[r]);
    }
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      u32x4 xv = *reinterpret_cast<const u32x4_any*>(xr[t] + at(p));
      if (ends) blank(xv);
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r][t] = add_dot8<ACT>(wv[r], xv, acc[r][t]);
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

// Up to 16 MT tokens: an MFMA 16x16x32 takes 16 tokens and 16 rows of W, a block 16 R rows and all of K, which its waves share in steps of 128 columns.  x and W come
// straight into LDS in whole lines, a step ahead, into two places of a wave's own (rows of 256 bytes, 16-byte piece p of row r in place p ^ (r & 15)); the waves' sums meet
// in LDS.  One launch, where the tiles of the dense product would split K over blocks and add its parts in a second.  8192 x 2048, 17 tokens: 9.0 us
// (gelu), 4.0 TB/s, where the bytes of a large copy would take 6.5; 4096 x 14336, eight: 22.2 us.
template <int MT, int R>
struct SomeTile {
  static constexpr int kPlace = (MT + R) * 4096, kSums = 16 * MT * 16 * R * 4;
  static constexpr int lds(int waves) { return waves * (2 * kPlace > kSums ? 2 * kPlace : kSums); }
};

template <int ACT, int MT, int R>
__global__ void __launch_bounds__(512) dense_some_kernel(const FewArgs a) {
  using T = SomeTile<MT, R>;
  extern __shared__ __attribute__((aligned(16))) uint8_t some_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, c = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * R;
  const int pieces = a.K / 8, steps = (pieces + 15) / 16, first = steps * wave / waves, last = steps * (wave + 1) / waves;
  uint8_t* const mine = some_lds + wave * 2 * T::kPlace;
  const uint32_t mine_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
  const uint8_t* const wb = uniform_ptr((const uint8_t*)a.w + n0 * a.ldw * 2);
  const uint8_t* const xb = uniform_ptr((const uint8_t*)a.x);
  // Load i brings rows 4 i .. 4 i + 3 of its operand: a lane's row and piece.
  const int row4 = lane >> 4, last_row = (int)min((int64_t)(16 * R - 1), a.N - 1 - n0);
  uint32_t x_off[4 * MT], w_off[4 * R];
#pragma unroll
  for (int i = 0; i < 4 * MT; ++i) x_off[i] = (uint32_t)min(4 * i + row4, a.M - 1) * (uint32_t)(a.ldx * 2);
#pragma unroll
  for (int i = 0; i < 4 * R; ++i) w_off[i] = (uint32_t)min(4 * i + row4, last_row) * (uint32_t)(a.ldw * 2);
  auto load = [&](int step, int place) __attribute__((always_inline)) {
    const int end = pieces - step * 16 - 1;  // pieces past the rows' end: the last one again
    const uint32_t to = mine_at + (uint32_t)(place * T::kPlace);
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) {
      if (4 * i >= a.M) break;
      lds_load16(to + i * 1024, x_off[i] + (uint32_t)min((lane & 15) ^ ((4 * i + row4) & 15), end) * 16u, xb + (int64_t)step * 256);
    }
#pragma unroll
    for (int i = 0; i < 4 * R; ++i)
      lds_load16(to + MT * 4096 + i * 1024, w_off[i] + (uint32_t)min((lane & 15) ^ ((4 * i + row4) & 15), end) * 16u, wb + (int64_t)step * 256);
  };
  f32x4 acc[MT][R];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[t][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (first < last) load(first, 0);
  for (int step = first, place = 0; step < last; ++step, place ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (step + 1 < last) load(step + 1, place ^ 1);
    const uint8_t* const at = mine + place * T::kPlace;
    const int there = pieces - step * 16;
    auto one = [&](auto ragged, int i) __attribute__((always_inline)) {
      u32x4 xo[MT], wo[R];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int row = min(16 * t + c, a.M - 1);  // rows past the tokens: one that nobody stores again
        xo[t] = *reinterpret_cast<const u32x4*>(at + row * 256 + (((4 * i + q) ^ (row & 15)) << 4));
      }
#pragma unroll
      for (int r = 0; r < R; ++r) wo[r] = *reinterpret_cast<const u32x4*>(at + MT * 4096 + (16 * r + c) * 256 + (((4 * i + q) ^ c) << 4));
      if constexpr (decltype(ragged)::value) {  // what lies past the rows' end counts for nothing, whatever it is
        const bool dead = 4 * i + q >= there;
#pragma unroll
        for (int t = 0; t < MT; ++t) xo[t] = dead ? u32x4{0, 0, 0, 0} : xo[t];
#pragma unroll
        for (int r = 0; r < R; ++r) wo[r] = dead ? u32x4{0, 0, 0, 0} : wo[r];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[t][r] = mfma16<ACT>(xo[t], wo[r], acc[t][r]);
    };
    if (there >= 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) one(std::false_type{}, i);
    } else {
#pragma unroll 1
      for (int i = 0; 4 * i < there; ++i) one(std::true_type{}, i);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the place may be loaded again
  }
  // D[m = 16 t + 4 q + i][n = 16 r + c]
  float* const sums = reinterpret_cast<float*>(some_lds);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = 16 * t + 4 * q + i;
        if (m < a.M) sums[(wave * a.M + m) * 16 * R + 16 * r + c] = acc[t][r][i];
      }
  __syncthreads();
  for (int o = threadIdx.x; o < a.M * 16 * R; o += blockDim.x) {
    const int m = o / (16 * R);
    const int64_t n = n0 + o % (16 * R);
    if (n >= a.N) continue;
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += sums[w * a.M * 16 * R + o];
    finish<ACT>(a, m, (int)n, v);
  }
}

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

constexpr int kMaxRows = 1 << 25, kMaxColumns = 1 << 30;  // of W: a launch has fewer than 2^32 threads

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

bool tiles_take(const void* x, int64_t ldx, const void* w, int64_t ldw, int K) {
  return K % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && (((uintptr_t)x | (uintptr_t)w) & 15) == 0 && ldx < NPAMD_TILE_MAX_STRIDE && ldw < NPAMD_TILE_MAX_STRIDE;
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
