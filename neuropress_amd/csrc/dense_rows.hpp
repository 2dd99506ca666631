// Dense products of a few tokens, whose time is W's: rows of W streamed into registers, or in whole lines into LDS (dense_act.hip and gated.hip launch them).
#pragma once

#include <type_traits>

#include "activation.hpp"
#include "common.hpp"
#include "dense_gemm.hpp"
#include "lds_transfer.hpp"
#include "wave_ops.hpp"

namespace npamd {

constexpr int kMaxRows = 1 << 25, kMaxColumns = 1 << 30;  // of W: a launch has fewer than 2^32 threads

struct FewArgs {  // gated: N columns of y, 2 N rows of w
  const void *x, *w;
  void* y;
  int64_t ldx, ldw, ldy;
  int M, N, K;
  DenseEpilogue ep;
};

// The gated product's two sums of a value of y.
template <int ACT>
__device__ __forceinline__ void finish_gated(const FewArgs& a, int m, int n, float gate, float up) {
  if (a.ep.bias) {
    gate += a.ep.bias_16 ? load_as_f32<ACT>(a.ep.bias, n) : ((const float*)a.ep.bias)[n];
    up += a.ep.bias_16 ? load_as_f32<ACT>(a.ep.bias, (int64_t)a.N + n) : ((const float*)a.ep.bias)[(int64_t)a.N + n];
  }
  if (a.ep.pre) {
    store_from_f32<ACT>(a.ep.pre, (int64_t)m * a.ep.ldp + n, gate);
    store_from_f32<ACT>(a.ep.pre, (int64_t)m * a.ep.ldp + a.N + n, up);
  }
  store_from_f32<ACT>(a.y, (int64_t)m * a.ldy + n, activate(a.ep.act, gate) * up);
}

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
// GATED: half of a wave's rows are gate rows, the others the up rows of the same columns of y.
template <int ACT, int R, int TB, int KS, int U, bool GATED = false>
__global__ void __launch_bounds__(256) dense_few_kernel(const FewArgs a) {
  __shared__ float sums[4][R * TB];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % KS;
  constexpr int RN = GATED ? R / 2 : R;  // columns of y
  const int64_t n0 = ((int64_t)blockIdx.x * (4 / KS) + wave / KS) * RN;
  const int m0 = blockIdx.y * TB, pieces = (a.K + 7) / 8, tail = pieces * 8 - a.K;
  const uint16_t *wr[R], *xr[TB];
#pragma unroll
  for (int r = 0; r < R; ++r) wr[r] = (const uint16_t*)a.w + (min(n0 + r % RN, (int64_t)a.N - 1) + r / RN * (int64_t)a.N) * a.ldw;  // past the end: the last row, not stored
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
  if (part != 0 || lane >= RN * TB) return;
  const int r = lane / TB, t = lane % TB;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < KS; ++i) v += sums[wave + i][lane];
  if constexpr (GATED) {
    float up = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) up += sums[wave + i][RN * TB + lane];
    if (n0 + r < a.N && m0 + t < a.M) finish_gated<ACT>(a, m0 + t, (int)(n0 + r), v, up);
    return;
  }
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

// GATED: half of a block's row tiles are gate rows, the others the up rows of the same columns of y.
template <int ACT, int MT, int R, bool GATED = false>
__global__ void __launch_bounds__(512) dense_some_kernel(const FewArgs a) {
  using T = SomeTile<MT, R>;
  extern __shared__ __attribute__((aligned(16))) uint8_t some_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, c = lane & 15, q = lane >> 4;
  constexpr int RN = GATED ? R / 2 : R;  // row tiles of columns of y
  const int64_t n0 = (int64_t)blockIdx.x * 16 * RN;
  const int pieces = a.K / 8, steps = (pieces + 15) / 16, first = steps * wave / waves, last = steps * (wave + 1) / waves;
  uint8_t* const mine = some_lds + wave * 2 * T::kPlace;
  const uint32_t mine_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
  const uint8_t* const wb = uniform_ptr((const uint8_t*)a.w + n0 * a.ldw * 2);
  const uint8_t* const wb_up = GATED ? uniform_ptr((const uint8_t*)a.w + (n0 + a.N) * a.ldw * 2) : wb;
  const uint8_t* const xb = uniform_ptr((const uint8_t*)a.x);
  // Load i brings rows 4 i .. 4 i + 3 of its operand: a lane's row and piece.
  const int row4 = lane >> 4, last_row = (int)min((int64_t)(16 * RN - 1), a.N - 1 - n0);
  uint32_t x_off[4 * MT], w_off[4 * R];
#pragma unroll
  for (int i = 0; i < 4 * MT; ++i) x_off[i] = (uint32_t)min(4 * i + row4, a.M - 1) * (uint32_t)(a.ldx * 2);
#pragma unroll
  for (int i = 0; i < 4 * R; ++i) w_off[i] = (uint32_t)min(4 * (i % (4 * RN)) + row4, last_row) * (uint32_t)(a.ldw * 2);
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
      lds_load16(to + MT * 4096 + i * 1024, w_off[i] + (uint32_t)min((lane & 15) ^ ((4 * i + row4) & 15), end) * 16u, (i >= 4 * RN ? wb_up : wb) + (int64_t)step * 256);
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
  if constexpr (GATED) {
    for (int o = threadIdx.x; o < a.M * 16 * RN; o += blockDim.x) {
      const int m = o / (16 * RN), c = o % (16 * RN);
      if (n0 + c >= a.N) continue;
      float gate = 0.f, up = 0.f;
      for (int w = 0; w < waves; ++w) {
        const float* const of = sums + (w * a.M + m) * 16 * R + c;
        gate += of[0], up += of[16 * RN];
      }
      finish_gated<ACT>(a, m, (int)(n0 + c), gate, up);
    }
    return;
  }
  for (int o = threadIdx.x; o < a.M * 16 * R; o += blockDim.x) {
    const int m = o / (16 * R);
    const int64_t n = n0 + o % (16 * R);
    if (n >= a.N) continue;
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += sums[w * a.M * 16 * R + o];
    finish<ACT>(a, m, (int)n, v);
  }
}

// Whether the tiles can read these operands.
inline bool tiles_take(const void* x, int64_t ldx, const void* w, int64_t ldw, int K) {
  return K % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && (((uintptr_t)x | (uintptr_t)w) & 15) == 0 && ldx < NPAMD_TILE_MAX_STRIDE && ldw < NPAMD_TILE_MAX_STRIDE;
}

}  // namespace npamd
