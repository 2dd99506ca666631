// Layer norm over the last dimension, forward and backward.
//   mean = sum(x) / H,  rstd = 1 / sqrt(sum((x - mean)^2) / H + eps),  xh = (x - mean) rstd
//   y = xh w + b
//   backward, g = dy w:  dx = rstd (g - sum(g) / H - xh sum(g xh) / H),  dw = sum over rows of dy xh,  db = sum over rows of dy
// All arithmetic in f32 (but f64 in the sums over rows that do not fit the registers), one rounding at the store; the variance is taken around the mean, in a second pass over the row.
#include <algorithm>

#include "common.hpp"
#include "row_pieces.hpp"
#include "wave_ops.hpp"

using namespace npamd;

namespace {

// Below so many waves a row gets more of them: 1100 x 4096 7.3 -> 6.7 us, 300 x 2048 4.0 -> 2.8.
constexpr int kFewWaves = 4096;

// RW waves to a row, 4 / RW rows to a block, NV pieces to a lane, so that x is read once.  Bound by HBM: 4096 x 4096 bf16 14.7 us (a copy of x 12.7; one wave to a row, eight
// pieces to a lane 15.4: too few waves for the registers), 8192 x 2048 14.1 (12.9); by the launch and one round trip below that: 300 x 2048 2.8, one row 2.2.
template <int DT, int NV, int RW>
__global__ void __launch_bounds__(256)
layer_norm_row_kernel(const void* x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, void* out, int64_t ldo,
                      float* __restrict__ mean_out, float* __restrict__ rstd_out, int M, int H, float eps) {
  using P = Pieces<DT>;
  constexpr int V = P::V, kLanes = 64 * RW;
  __shared__ float part[2][4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (kLanes - 1);
  const int64_t row_of_wave = (int64_t)blockIdx.x * (4 / RW) + wave / RW, row = min(row_of_wave, (int64_t)M - 1);  // past the end: the last row, not stored
  const int pieces = (H + V - 1) / V;
  const uint8_t* const xr = P::row_of(x, row, ldx);
  u32x4 xv[NV], wv[NV], bv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + kLanes * i;
    xv[i] = u32x4{0, 0, 0, 0};
    if (p < pieces) xv[i] = P::load(xr, min(p * V, H - V));
  }
  auto parameters = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + kLanes * i, at = min(p * V, H - V);
      wv[i] = bv[i] = u32x4{0, 0, 0, 0};
      if (w && p < pieces) wv[i] = P::load((const uint8_t*)w, at);
      if (b && p < pieces) bv[i] = P::load((const uint8_t*)b, at);
    }
  };
  // Few rows wait for memory once: w and b are requested with x.  Many need the registers for waves: w and b come from the L1 when they are used.
  constexpr bool kEarly = NV <= 2;
  if constexpr (kEarly) parameters();
  // f(value) for the lane's values of the row, each once.
  auto values = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + kLanes * i;
      if (p >= pieces) continue;
      float v[V];
      P::forget(xv[i]);
      P::unpack(xv[i], v);
      if (p * V + V <= H) {
#pragma unroll
        for (int e = 0; e < V; ++e) f(v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e >= p * V + V - H) f(v[e]);
      }
    }
  };
  auto over_row = [&](float v, float* meet) __attribute__((always_inline)) {
    v = wave_sum(v);
    if constexpr (RW > 1) {
      if ((threadIdx.x & 63) == 0) meet[wave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < RW; ++i) v += meet[wave / RW * RW + i];
    }
    return v;
  };
  float s = 0.f, ss = 0.f;
  values([&](float v) __attribute__((always_inline)) { s += v; });
  const float mean = over_row(s, part[0]) / (float)H;
  values([&](float v) __attribute__((always_inline)) { ss = __builtin_fmaf(v - mean, v - mean, ss); });
  const float rstd = 1.0f / __builtin_sqrtf(over_row(ss, part[1]) / (float)H + eps);
  if constexpr (!kEarly) parameters();
  if (row_of_wave >= M) return;
  if (lane == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + kLanes * i;
    if (p >= pieces) continue;
    float f[V], g[V];
    P::forget(xv[i]);
    P::unpack(xv[i], f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (f[e] - mean) * rstd;
    if (w) {
      P::unpack(wv[i], g);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= g[e];
    }
    if (b) {
      P::unpack(bv[i], g);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] += g[e];
    }
    P::store(const_cast<uint8_t*>(P::row_of(out, row, ldo)), min(p * V, H - V), P::pack(f));
  }
}

// Rows too short for a piece or too long for the registers: a block per row, which it reads three times.
template <int DT>
__global__ void __launch_bounds__(256)
layer_norm_block_kernel(const void* x, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, void* out,
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

// Rows too short for a piece or too long for the registers.  The gradient of the input: a block per row.
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

// And sums over strips of rows for the gradients of weight and bias: partials [parts][2][H], a lane per column.  A strip may have any number of rows: in f64, so that
// the error does not grow with them.
template <int DT>
__global__ void __launch_bounds__(256)
layer_norm_back_columns_kernel(const LayerNormBack a, float* __restrict__ partials, int parts) {
  __shared__ double sums[4][2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  const int first = (int)((int64_t)a.M * blockIdx.y / parts), last = (int)((int64_t)a.M * (blockIdx.y + 1) / parts);
  double dw = 0., db = 0.;
  if (col < a.H)
    for (int64_t row = first + wave; row < last; row += 4) {
      const float d = load_as_f32<DT>(a.dy, row * a.lddy + col);
      dw = __builtin_fma((double)d, (double)((load_as_f32<DT>(a.x, row * a.ldx + col) - a.mean[row]) * a.rstd[row]), dw);
      db += (double)d;
    }
  sums[wave][0][lane] = dw;
  sums[wave][1][lane] = db;
  __syncthreads();
  if (wave < 2 && col < a.H)
    partials[((int64_t)blockIdx.y * 2 + wave) * a.H + col] = (float)(sums[0][wave][lane] + sums[1][wave][lane] + sums[2][wave][lane] + sums[3][wave][lane]);
}

constexpr int kManyGroups = 8;

// All of it in one pass over x and dy, 8192 x 4096 bf16 41.7 us in all, 4.8 TB/s, as fast as a copy (with masks for every value and pieces unpacked twice, 48: the vector
// instructions were the limit): RW waves to a row, G rows to a block at a time, a lane has NV pieces of every row that its group meets, the weight's at hand, and adds up
// its columns' part of the weight's and bias's gradients in registers.  The next rows are requested before the two sums of these meet in LDS (one barrier a turn).
template <int DT, int NV>
__global__ void __launch_bounds__(1024)
layer_norm_back_kernel(const LayerNormBack a, float* __restrict__ partials, void* __restrict__ dw_out, void* __restrict__ db_out, int RW, int G) {
  using P = Pieces<DT>;
  constexpr int V = P::V;
  extern __shared__ __attribute__((aligned(16))) float back_lds[];
  __shared__ float meet[2][16][2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave / RW, lanes = 64 * RW;
  const int lane = (int)threadIdx.x - group * lanes, pieces = (a.H + V - 1) / V;
  const float inv = 1.f / (float)a.H;
  u32x4 xv[NV], dv[NV], wv[NV];
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + lanes * i;
    xv[i] = dv[i] = wv[i] = u32x4{0, 0, 0, 0};
    if (a.w && p < pieces) wv[i] = P::load((const uint8_t*)a.w, min(p * V, a.H - V));
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  float next_mean = 0.f, next_rstd = 0.f;
  auto request = [&](int64_t row) __attribute__((always_inline)) {
    if (row >= a.M) return;
    int64_t at_row = row;  // by vector loads: scalar ones would be waited for in front of the barrier
    asm volatile("" : "+v"(at_row));
    next_mean = a.mean[at_row];
    next_rstd = a.rstd[at_row];
    const uint8_t* const xr = P::row_of(a.x, row, a.ldx);
    const uint8_t* const dr = P::row_of(a.dy, row, a.lddy);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + lanes * i, at = min(p * V, a.H - V);
      if (p >= pieces) continue;
      xv[i] = P::load(xr, at);
      dv[i] = P::load(dr, at);
    }
  };
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + group;
  request(row);
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * G; first < a.M; first += step, row += step, turn ^= 1) {
    const bool live = row < a.M;
    const float mean = next_mean, rstd = next_rstd;
    u32x4 xc[NV], dc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) xc[i] = xv[i], dc[i] = dv[i];
    request(row + step);
    float s1 = 0.f, s2 = 0.f, xh[NV][V], g[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + lanes * i;
      if (!live || p >= pieces) continue;
      float wf[V], d[V];
      P::unpack(xc[i], xh[i]);
      P::unpack(dc[i], d);
      P::unpack(wv[i], wf);
      auto value = [&](int e) __attribute__((always_inline)) {
        dw[i][e] = __builtin_fmaf(d[e], xh[i][e], dw[i][e]);
        db[i][e] += d[e];
        s1 += g[i][e];
        s2 = __builtin_fmaf(g[i][e], xh[i][e], s2);
      };
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xh[i][e] = (xh[i][e] - mean) * rstd;
        g[i][e] = a.w ? d[e] * wf[e] : d[e];
      }
      if (p * V + V <= a.H) {
#pragma unroll
        for (int e = 0; e < V; ++e) value(e);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e >= p * V + V - a.H) value(e);
      }
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (RW > 1) {
      if ((threadIdx.x & 63) == 0) meet[turn][wave][0] = s1, meet[turn][wave][1] = s2;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the loads stay on their way
      s1 = s2 = 0.f;
      for (int i = 0; i < RW; ++i) s1 += meet[turn][group * RW + i][0], s2 += meet[turn][group * RW + i][1];
    }
    if (!live || !a.dx) continue;
    const float c1 = -s1 * inv * rstd, c2 = -s2 * inv * rstd;
    uint8_t* const to = const_cast<uint8_t*>(P::row_of(a.dx, row, a.lddx));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + lanes * i;
      if (p >= pieces) continue;
      if constexpr (NV > 1) {  // not kept
        float wf[V];
        P::forget(xc[i]);
        P::forget(dc[i]);
        P::forget(wv[i]);
        P::unpack(xc[i], xh[i]);
        P::unpack(dc[i], g[i]);
        P::unpack(wv[i], wf);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          xh[i][e] = (xh[i][e] - mean) * rstd;
          if (a.w) g[i][e] *= wf[e];
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) g[i][e] = __builtin_fmaf(xh[i][e], c2, __builtin_fmaf(g[i][e], rstd, c1));
      P::store(to, min(p * V, a.H - V), P::pack(g[i]));
    }
  }
  if (!partials && !dw_out && !db_out) return;
  // The groups' sums meet in LDS and are added in their order: by the first group, or by all threads where there are many (8 x 320 4.2 -> 2.9 us, 64 x 768
  // 7.9 -> 7.1; but 64 x 2048, four groups, 7.7 -> 8.3).  Rows of whole pieces: a row's last piece lies behind those before, whole.
  const int width = pieces * V;
  float* const to = partials + (int64_t)blockIdx.x * 2 * width;
  if (G >= kManyGroups) {
    float* const mine = back_lds + (int64_t)group * 2 * width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + lanes * i;
      if (p >= pieces) continue;
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        *reinterpret_cast<f32x4*>(mine + p * V + e) = f32x4{dw[i][e], dw[i][e + 1], dw[i][e + 2], dw[i][e + 3]};
        *reinterpret_cast<f32x4*>(mine + width + p * V + e) = f32x4{db[i][e], db[i][e + 1], db[i][e + 2], db[i][e + 3]};
      }
    }
    __syncthreads();
    for (int o = threadIdx.x; o < 2 * width; o += blockDim.x) {
      float v = 0.f;
      for (int g = 0; g < G; ++g) v += back_lds[g * 2 * width + o];
      if (partials) {
        to[o] = v;
        continue;
      }
      void* const out = o < width ? dw_out : db_out;
      const int at = o < width ? o : o - width, whole = a.H / V * V, column = at < whole ? at : at + a.H - width;
      if (out && (at < whole || column >= whole)) store_from_f32<DT>(out, column, v);
    }
    return;
  }
  float* const mine = back_lds + (int64_t)(group - 1) * 2 * NV * V * lanes + lane;
  if (group > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) mine[(2 * (i * V + e)) * lanes] = dw[i][e], mine[(2 * (i * V + e) + 1) * lanes] = db[i][e];
  }
  __syncthreads();
  if (group > 0) return;
  for (int o = 0; o < G - 1; ++o) {
    const float* const theirs = back_lds + (int64_t)o * 2 * NV * V * lanes + lane;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) dw[i][e] += theirs[(2 * (i * V + e)) * lanes], db[i][e] += theirs[(2 * (i * V + e) + 1) * lanes];
  }
  if (!partials) {  // the only block: its sums are all there is
    auto leave = [&](void* out, const float (&sum)[NV][V]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int p = lane + lanes * i, at = min(p * V, a.H - V);
        if (p >= pieces) continue;
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (at + e >= p * V) store_from_f32<DT>(out, at + e, sum[i][e]);  // the others are the piece's before
      }
    };
    if (dw_out) leave(dw_out, dw);
    if (db_out) leave(db_out, db);
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + lanes * i;
    if (p >= pieces) continue;
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      *reinterpret_cast<f32x4*>(to + p * V + e) = f32x4{dw[i][e], dw[i][e + 1], dw[i][e + 2], dw[i][e + 3]};
      *reinterpret_cast<f32x4*>(to + width + p * V + e) = f32x4{db[i][e], db[i][e + 1], db[i][e + 2], db[i][e + 3]};
    }
  }
}

// The parts' sums, in the order of the parts: 64 columns of one of the two gradients (blockIdx.y) to a block, its 16 waves each a sixteenth of the parts.  A part has `width`
// columns for each, whole pieces: the last one's lie at its end.
template <int DT>
__global__ void __launch_bounds__(1024)
layer_norm_back_sum_kernel(const float* __restrict__ partials, int parts, int H, int width, int last, void* __restrict__ dw, void* __restrict__ db) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  void* const out = blockIdx.y ? db : dw;
  if (!out) return;
  const int first = parts * wave / 16, end = parts * (wave + 1) / 16;
  float v = 0.f;
  if (col < H) {
    const float* p = partials + ((int64_t)first * 2 + blockIdx.y) * width + (col < last ? col : col + width - H);
#pragma unroll 8
    for (int i = first; i < end; ++i, p += 2 * (int64_t)width) v += *p;
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave || col >= H) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += sums[i][lane];
  store_from_f32<DT>(out, col, v);
}

// A block's turns, where rows are few: a turn takes 1.3 us, but every block leaves sums of two rows' bytes in f32, so two where those would be more than kMaxSums bytes (one /
// two / four turns 509 x 3003, 6 MB with one, 12.3 / 10.5 / 13.8 us, 512 x 2048, 2 MB, 8.2 / 9.6 / 11.3, 104 x 176 5.5 / 6.7 / 8.5) or where one block then takes all rows,
// without a second launch (16 x 768 6.0 / 5.2); and no more blocks than compute units (8192 x 4096 with 192 / 256 / 512 55 / 48 / 54 us).
constexpr int64_t kMaxSums = 4 << 20;
// Which kernel the backward pass takes.  parts: sums over rows that it leaves to be added.
struct BackPlan {
  int nv = 0, row_waves = 0, groups = 0, parts = 0;  // nv 0: rows that do not fit the registers
  // Bytes of LDS where the groups' sums meet: 64 KiB at most (rows of two pieces to a lane have one group).
  int lds(int pieces, int V) const { return (groups >= kManyGroups ? groups * pieces : (groups - 1) * nv * 64 * row_waves) * 2 * V * 4; }
  BackPlan(int M, int H, int dtype) {
    const int V = dtype == NPAMD_F32 ? 4 : 8, pieces = (H + V - 1) / V;
    if (H < V || pieces > 64 * 16 * 2) {
      // strips of 64 rows, 1024 of them where their sums are small (64 / 1024: 2^20 x 2 f32 1336 / 726 us, 100000 x 5 fp16 146 / 89, dx among them)
      parts = (int)std::min<int64_t>(std::clamp<int64_t>(kMaxSums / (8 * (int64_t)H), 64, 1024), ((int64_t)M + 63) / 64);
      return;
    }
    nv = pieces <= 1024 ? 1 : 2;
    row_waves = 1;
    while (row_waves * 64 * nv < pieces) row_waves *= 2;
    groups = std::min(16 / row_waves, std::max(1, M));
    auto blocks = [&](int turns) { return std::min<int64_t>(256, ((int64_t)M + groups * turns - 1) / (groups * turns)); };
    parts = (int)blocks(blocks(2) > 1 && blocks(1) * H * 8 <= kMaxSums ? 1 : 2);
  }
};

template <int DT>
int launch_forward_rows(const void* x, int64_t ldx, const void* w, const void* b, void* out, int64_t ldo, float* mean, float* rstd, int M, int H, float eps,
                        hipStream_t st) {
  constexpr int V = Pieces<DT>::V;
  const int pieces = (H + V - 1) / V;
  if (H < V || pieces > 256 * 16) {
    launch(layer_norm_block_kernel<DT>, M, 256, 0, st, x, ldx, w, b, out, ldo, mean, rstd, H, eps);
    return check_launch("npamd_layer_norm");
  }
#define NPAMD_LN(NV, RW) launch(layer_norm_row_kernel<DT, NV, RW>, (unsigned)((M + 4 / RW - 1) / (4 / RW)), 256, 0, st, x, ldx, w, b, out, ldo, mean, rstd, M, H, eps)
  int rw = 1;
  while (rw < 4 && (pieces > 64 * 4 * rw || (pieces > 64 * rw && (int64_t)M * rw < kFewWaves))) rw *= 2;
  const int nv = (pieces + 64 * rw - 1) / (64 * rw);
  if (rw == 1) {
    if (nv <= 1) NPAMD_LN(1, 1);
    else if (nv <= 2) NPAMD_LN(2, 1);
    else NPAMD_LN(4, 1);
  } else if (rw == 2) {
    if (nv <= 1) NPAMD_LN(1, 2);
    else if (nv <= 2) NPAMD_LN(2, 2);
    else NPAMD_LN(4, 2);
  } else {
    if (nv <= 1) NPAMD_LN(1, 4);
    else if (nv <= 2) NPAMD_LN(2, 4);
    else if (nv <= 4) NPAMD_LN(4, 4);
    else if (nv <= 8) NPAMD_LN(8, 4);
    else NPAMD_LN(16, 4);
  }
#undef NPAMD_LN
  return check_launch("npamd_layer_norm");
}

template <int DT>
int launch_forward(const void* x, int64_t ldx, const void* w, const void* b, void* out, int64_t ldo, float* mean, float* rstd, int M, int H, float eps,
                   hipStream_t st) {
  using P = Pieces<DT>;
  for (int64_t at = 0; at < M; at += kRowsAtOnce) {
    const int rc = launch_forward_rows<DT>(P::row_of(x, at, ldx), ldx, w, b, const_cast<uint8_t*>(P::row_of(out, at, ldo)), ldo, mean ? mean + at : nullptr,
                                           rstd ? rstd + at : nullptr, (int)std::min<int64_t>(kRowsAtOnce, M - at), H, eps, st);
    if (rc != NPAMD_OK) return rc;
  }
  return NPAMD_OK;
}

template <int DT>
int launch_backward(const LayerNormBack& a, void* dw, void* db, float* partials, hipStream_t st) {
  const char* what = "npamd_layer_norm_backward";
  const bool sums = dw || db;
  const BackPlan p(a.M, a.H, DT);
  const unsigned columns = (unsigned)(a.H + 63) / 64;
  if (a.M && p.nv) {
    constexpr int V = Pieces<DT>::V;
    const int lds = sums ? p.lds((a.H + V - 1) / V, V) : 0;
    const auto kernel = p.nv == 1 ? layer_norm_back_kernel<DT, 1> : layer_norm_back_kernel<DT, 2>;
    static LdsLatch latch[2];
    const hipError_t e = enable_dynamic_lds(latch[p.nv - 1], reinterpret_cast<const void*>(kernel), lds);
    if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
    const bool alone = p.parts == 1;
    if (sums || a.dx)
      launch(kernel, p.parts, 64 * p.row_waves * p.groups, lds, st, a, sums && !alone ? partials : nullptr, alone ? dw : nullptr, alone ? db : nullptr, p.row_waves, p.groups);
    if (alone) return check_launch(what);
  } else if (a.M) {
    // The columns' sums first: dx may take the place of dy or x.
    if (sums) launch(layer_norm_back_columns_kernel<DT>, dim3(columns, p.parts), 256, 0, st, a, partials, p.parts);
    if (a.dx) {
      LayerNormBack part = a;
      for (int64_t at = 0; at < a.M; at += kRowsAtOnce) {
        part.dy = Pieces<DT>::row_of(a.dy, at, a.lddy), part.x = Pieces<DT>::row_of(a.x, at, a.ldx);
        part.dx = const_cast<uint8_t*>(Pieces<DT>::row_of(a.dx, at, a.lddx)), part.mean = a.mean + at, part.rstd = a.rstd + at;
        launch(layer_norm_back_block_kernel<DT>, (unsigned)std::min<int64_t>(kRowsAtOnce, a.M - at), 256, 0, st, part);
      }
    }
  }
  constexpr int V = Pieces<DT>::V;
  const int width = p.nv ? (a.H + V - 1) / V * V : a.H, last = p.nv ? a.H / V * V : a.H;
  if (sums) launch(layer_norm_back_sum_kernel<DT>, dim3(columns, 2), 1024, 0, st, partials, p.parts, a.H, width, last, dw, db);
  return check_launch(what);
}

}  // namespace

extern "C" int npamd_layer_norm(const void* x, int64_t ldx, const void* weight, const void* bias, void* out, int64_t ldo, float* mean, float* rstd,
                                int M, int H, float eps, int dtype, void* stream) {
  const char* what = "npamd_layer_norm";
  NPAMD_REQUIRE(M >= 0 && H >= 1 && H <= kMaxWidth, "%s: bad shape M=%d H=%d", what, M, H);
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
  if (M < 1 || H < 1 || H > kMaxWidth) return 0;
  return (int64_t)std::max(BackPlan(M, H, NPAMD_F16).parts, BackPlan(M, H, NPAMD_F32).parts) * 2 * ((H + 7) / 8 * 8) * 4;
}

extern "C" int npamd_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, const float* mean,
                                         const float* rstd, void* dx, int64_t lddx, void* dweight, void* dbias, int M, int H, int dtype,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_layer_norm_backward";
  NPAMD_REQUIRE(M >= 0 && H >= 1 && H <= kMaxWidth, "%s: bad shape M=%d H=%d", what, M, H);
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
