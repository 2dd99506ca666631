// Layer norm over the last dimension, forward and backward.
//   mean = sum(x) / H,  rstd = 1 / sqrt(sum((x - mean)^2) / H + eps),  xh = (x - mean) rstd
//   y = xh w + b
//   backward, g = dy w:  dx = rstd (g - sum(g) / H - xh sum(g xh) / H),  dw = sum over rows of dy xh,  db = sum over rows of dy
// All arithmetic in f32, one rounding at the store; the variance is taken around the mean, in a second pass over the row.
#include "common.hpp"

using namespace npamd;

namespace {

// The sum over a block of 256 threads, in every one of them.  `part`: four floats of the block's own for this sum.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = wave_reduce_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

// Any H, any alignment: a block per row, which it reads three times.
template <int DT>
__global__ void __launch_bounds__(256)
layer_norm_block_kernel(const void* __restrict__ x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, void* __restrict__ out,
                        int64_t ldo, float* __restrict__ mean_out, float* __restrict__ rstd_out, int H, float eps) {
  __shared__ float part[2][4];
  const int64_t row = blockIdx.x;
  float s = 0.f;
  for (int i = threadIdx.x; i < H; i += 256) s += load_as_f32<DT>(x, row * ldx + i);
  const float mean = block_sum(s, part[0]) / (float)H;
  float ss = 0.f;
  for (int i = threadIdx.x; i < H; i += 256) {
    const float d = load_as_f32<DT>(x, row * ldx + i) - mean;
    ss = __builtin_fmaf(d, d, ss);
  }
  const float rstd = 1.0f / __builtin_sqrtf(block_sum(ss, part[1]) / (float)H + eps);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
  for (int i = threadIdx.x; i < H; i += 256) {
    float v = (load_as_f32<DT>(x, row * ldx + i) - mean) * rstd;
    if (w) v *= load_as_f32<DT>(w, i);
    if (b) v += load_as_f32<DT>(b, i);
    store_from_f32<DT>(out, row * ldo + i, v);
  }
}

struct LayerNormBack {
  const void *dy, *x, *w;
  const float *mean, *rstd;
  void* dx;
  int64_t lddy, ldx, lddx;
  int M, H;
};

// The gradient of the input, any H and alignment: a block per row.
template <int DT>
__global__ void __launch_bounds__(256)
layer_norm_back_block_kernel(const LayerNormBack a) {
  __shared__ float part[2][4];
  const int64_t row = blockIdx.x;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int i = threadIdx.x; i < a.H; i += 256) {
    const float g = load_as_f32<DT>(a.dy, row * a.lddy + i) * (a.w ? load_as_f32<DT>(a.w, i) : 1.f);
    s1 += g;
    s2 = __builtin_fmaf(g, (load_as_f32<DT>(a.x, row * a.ldx + i) - mean) * rstd, s2);
  }
  const float c1 = block_sum(s1, part[0]) / (float)a.H, c2 = block_sum(s2, part[1]) / (float)a.H;
  for (int i = threadIdx.x; i < a.H; i += 256) {
    const float g = load_as_f32<DT>(a.dy, row * a.lddy + i) * (a.w ? load_as_f32<DT>(a.w, i) : 1.f);
    const float xh = (load_as_f32<DT>(a.x, row * a.ldx + i) - mean) * rstd;
    store_from_f32<DT>(a.dx, row * a.lddx + i, (g - c1 - xh * c2) * rstd);
  }
}

// Sums over strips of rows for the gradients of weight and bias: partials [parts][2][H], a lane per column.
template <int DT>
__global__ void __launch_bounds__(256)
layer_norm_back_columns_kernel(const LayerNormBack a, float* __restrict__ partials, int parts) {
  __shared__ float sums[4][2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  const int first = (int)((int64_t)a.M * blockIdx.y / parts), last = (int)((int64_t)a.M * (blockIdx.y + 1) / parts);
  float dw = 0.f, db = 0.f;
  if (col < a.H)
    for (int64_t row = first + wave; row < last; row += 4) {
      const float d = load_as_f32<DT>(a.dy, row * a.lddy + col);
      dw = __builtin_fmaf(d, (load_as_f32<DT>(a.x, row * a.ldx + col) - a.mean[row]) * a.rstd[row], dw);
      db += d;
    }
  sums[wave][0][lane] = dw;
  sums[wave][1][lane] = db;
  __syncthreads();
  if (wave < 2 && col < a.H)
    partials[((int64_t)blockIdx.y * 2 + wave) * a.H + col] = sums[0][wave][lane] + sums[1][wave][lane] + sums[2][wave][lane] + sums[3][wave][lane];
}

// The parts' sums, in the order of the parts: 64 columns of one of the two gradients (blockIdx.y) to a block, its 16 waves each a sixteenth of the parts.
template <int DT>
__global__ void __launch_bounds__(1024)
layer_norm_back_sum_kernel(const float* __restrict__ partials, int parts, int H, void* __restrict__ dw, void* __restrict__ db) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  void* const out = blockIdx.y ? db : dw;
  if (!out) return;
  const int first = parts * wave / 16, last = parts * (wave + 1) / 16;
  float v = 0.f;
  if (col < H) {
    const float* p = partials + ((int64_t)first * 2 + blockIdx.y) * H + col;
#pragma unroll 8
    for (int i = first; i < last; ++i, p += 2 * (int64_t)H) v += *p;
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave || col >= H) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += sums[i][lane];
  store_from_f32<DT>(out, col, v);
}

// Strips of rows whose sums the backward pass keeps apart.
int back_parts(int M) { return M <= 0 ? 0 : M < 64 * 64 ? (M + 63) / 64 : 64; }

template <int DT>
int launch_forward(const void* x, int64_t ldx, const void* w, const void* b, void* out, int64_t ldo, float* mean, float* rstd, int M, int H, float eps,
                   hipStream_t st) {
  launch(layer_norm_block_kernel<DT>, M, 256, 0, st, x, ldx, w, b, out, ldo, mean, rstd, H, eps);
  return check_launch("npamd_layer_norm");
}

template <int DT>
int launch_backward(const LayerNormBack& a, void* dw, void* db, float* partials, hipStream_t st) {
  const char* what = "npamd_layer_norm_backward";
  if (a.M && a.dx) launch(layer_norm_back_block_kernel<DT>, a.M, 256, 0, st, a);
  if (dw || db) {
    const int parts = back_parts(a.M);
    const unsigned columns = (unsigned)(a.H + 63) / 64;
    if (parts) launch(layer_norm_back_columns_kernel<DT>, dim3(columns, parts), 256, 0, st, a, partials, parts);
    launch(layer_norm_back_sum_kernel<DT>, dim3(columns, 2), 1024, 0, st, partials, parts, a.H, dw, db);
  }
  return check_launch(what);
}

}  // namespace

extern "C" int npamd_layer_norm(const void* x, int64_t ldx, const void* weight, const void* bias, void* out, int64_t ldo, float* mean, float* rstd,
                                int M, int H, float eps, int dtype, void* stream) {
  const char* what = "npamd_layer_norm";
  NPAMD_REQUIRE(M >= 0 && H >= 1, "%s: bad shape M=%d H=%d", what, M, H);
  NPAMD_REQUIRE(dtype == NPAMD_F16 || dtype == NPAMD_BF16 || dtype == NPAMD_F32, "%s: bad dtype %d", what, dtype);
  NPAMD_REQUIRE(ldx >= H && ldo >= H, "%s: bad row stride", what);
  if (M == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && out, "%s: null pointer", what);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NPAMD_F16) return launch_forward<NPAMD_F16>(x, ldx, weight, bias, out, ldo, mean, rstd, M, H, eps, st);
  if (dtype == NPAMD_BF16) return launch_forward<NPAMD_BF16>(x, ldx, weight, bias, out, ldo, mean, rstd, M, H, eps, st);
  return launch_forward<NPAMD_F32>(x, ldx, weight, bias, out, ldo, mean, rstd, M, H, eps, st);
}

extern "C" int64_t npamd_layer_norm_workspace_bytes(int M, int H) {
  if (M < 1 || H < 1) return 0;
  return (int64_t)back_parts(M) * 2 * H * 4;
}

extern "C" int npamd_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, const float* mean,
                                         const float* rstd, void* dx, int64_t lddx, void* dweight, void* dbias, int M, int H, int dtype,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_layer_norm_backward";
  NPAMD_REQUIRE(M >= 0 && H >= 1, "%s: bad shape M=%d H=%d", what, M, H);
  NPAMD_REQUIRE(dtype == NPAMD_F16 || dtype == NPAMD_BF16 || dtype == NPAMD_F32, "%s: bad dtype %d", what, dtype);
  NPAMD_REQUIRE(lddy >= H && ldx >= H && (!dx || lddx >= H), "%s: bad row stride", what);
  NPAMD_REQUIRE(M == 0 || (dy && x && mean && rstd), "%s: null pointer", what);
  if (M && (dweight || dbias)) {
    const int64_t need = npamd_layer_norm_workspace_bytes(M, H);
    NPAMD_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need,
                  "%s: the gradients of weight and bias need %lld bytes of 16-byte aligned workspace", what, (long long)need);
  }
  const LayerNormBack a{dy, x, weight, mean, rstd, dx, lddy, ldx, lddx, M, H};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NPAMD_F16) return launch_backward<NPAMD_F16>(a, dweight, dbias, (float*)workspace, st);
  if (dtype == NPAMD_BF16) return launch_backward<NPAMD_BF16>(a, dweight, dbias, (float*)workspace, st);
  return launch_backward<NPAMD_F32>(a, dweight, dbias, (float*)workspace, st);
}
