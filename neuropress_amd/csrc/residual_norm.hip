// Where one half of a decoder block ends and the next begins, forward and backward:
//   b = y rstd_y wp (RMS norm behind the half; without wp: y),  r = x + scale gate b,  z = r rstd w (RMS norm in front of the next half),
//   rstd_y = 1 / sqrt(sum(y^2) / H + eps),  rstd = 1 / sqrt(sum(r^2) / H + eps).  The norm takes r as it is before it is rounded.
// Backward, from the gradients ds of r and dz of z, with rh = r rstd, yh = y rstd_y, v = dz w:
//   dr = ds + rstd (v - rh sum(v rh) / H) = dx,  dw = sum over rows of dz rh,  dgate = sum over the gate's rows of scale dr b,
//   u = scale gate dr:  without wp dy = u;  with it dwp = sum over rows of u yh,  dy = rstd_y (u wp - yh sum(u wp yh) / H).
// All arithmetic in f32 (but f64 in the sums over rows that do not fit the registers), one rounding at the store.  The backward pass takes r as the forward pass rounded it, which is what a
// training step keeps of it, next to the rstd of the unrounded one: rh is then off by half a step of r's type, as dz and ds are.  Sums over rows that fit the registers are chains of M / 128 additions and
// fewer, as many as a team has rows (129 to 256 gates have a block each), then those over teams and blocks.
#include <algorithm>

#include "common.hpp"
#include "row_pieces.hpp"
#include "wave_ops.hpp"

using namespace npamd;

namespace {

struct ResidualNorm {
  const void *x, *y, *w, *wp, *gate;
  void *stream, *normed;
  float *post_rstd, *rstd;
  int64_t ldx, ldy, ldg, lds, ldn;
  int M, H, gate_every;  // rows that share a row of the gate
  float scale, eps;
};

__device__ __forceinline__ float rsqrt_mean(float sum, int H, float eps) { return 1.0f / __builtin_sqrtf(sum / (float)H + eps); }

// RW waves to a row, NV pieces to a lane: x and y are read once, r stays in registers between its sum and its norm.  x and y are read by all of a row's waves before the first of
// them stores, so that r and z may take their places.  Bound by HBM: 4096 x 4096 bf16 with both norms 23.4 us, 5.7 TB/s of 134 MB (a copy: 4.9), one row 2.0.
template <int DT, int NV, int RW>
__global__ void __launch_bounds__(RW < 4 ? 256 : 64 * RW) residual_norm_row_kernel(const ResidualNorm a, int64_t first) {
  using P = Pieces<DT>;
  constexpr int V = P::V, kLanes = 64 * RW, kWaves = RW < 4 ? 4 : RW;
  __shared__ float part[2][kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (kLanes - 1);
  const int64_t row_of_wave = first + (int64_t)blockIdx.x * (kWaves / RW) + wave / RW, row = min(row_of_wave, (int64_t)a.M - 1);  // past the end: the last row, not stored
  const int H = a.H, pieces = (H + V - 1) / V;
  const uint8_t* const xr = P::row_of(a.x, row, a.ldx);
  const uint8_t* const yr = P::row_of(a.y, row, a.ldy);
  const uint8_t* const gr = a.gate ? P::row_of(a.gate, row / a.gate_every, a.ldg) : nullptr;
  u32x4 xv[NV], yv[NV], gv[NV], pv[NV], wv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + kLanes * i, at = min(p * V, H - V);
    xv[i] = yv[i] = gv[i] = pv[i] = wv[i] = u32x4{0, 0, 0, 0};
    if (p >= pieces) continue;
    yv[i] = P::load(yr, at);
    xv[i] = P::load(xr, at);
    if (gr) gv[i] = P::load(gr, at);
    if (a.wp) pv[i] = P::load((const uint8_t*)a.wp, at);
    wv[i] = P::load((const uint8_t*)a.w, at);
  }
  // The sum of the squares of the lane's values of a row, each once.
  auto squares = [&](const float (&v)[V], int p, float s) __attribute__((always_inline)) {
    if (p * V + V <= H) {
#pragma unroll
      for (int e = 0; e < V; ++e) s = __builtin_fmaf(v[e], v[e], s);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e >= p * V + V - H) s = __builtin_fmaf(v[e], v[e], s);
    }
    return s;
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
  float r[NV][V], post_rstd = 1.f, ss = 0.f;
  if (a.wp) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + kLanes * i;
      if (p >= pieces) continue;
      P::unpack(yv[i], r[i]);
      s = squares(r[i], p, s);
    }
    post_rstd = rsqrt_mean(over_row(s, part[0]), H, a.eps);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + kLanes * i;
    if (p >= pieces) continue;
    float f[V];
    P::forget(yv[i]);
    P::unpack(yv[i], r[i]);
    if (a.wp) {
      P::unpack(pv[i], f);
#pragma unroll
      for (int e = 0; e < V; ++e) r[i][e] = r[i][e] * post_rstd * f[e];
    }
    if (gr) {
      P::unpack(gv[i], f);
#pragma unroll
      for (int e = 0; e < V; ++e) r[i][e] *= f[e];
    }
    P::unpack(xv[i], f);
#pragma unroll
    for (int e = 0; e < V; ++e) r[i][e] = __builtin_fmaf(a.scale, r[i][e], f[e]);
    ss = squares(r[i], p, ss);
  }
  const float rstd = rsqrt_mean(over_row(ss, part[1]), H, a.eps);
  if (row_of_wave >= a.M) return;
  if (lane == 0) {
    if (a.post_rstd) a.post_rstd[row] = post_rstd;
    if (a.rstd) a.rstd[row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + kLanes * i, at = min(p * V, H - V);
    if (p >= pieces) continue;
    float f[V];
    P::store(const_cast<uint8_t*>(P::row_of(a.stream, row, a.lds)), at, P::pack(r[i]));
    P::unpack(wv[i], f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] *= r[i][e] * rstd;
    P::store(const_cast<uint8_t*>(P::row_of(a.normed, row, a.ldn)), at, P::pack(f));
  }
}

// Rows too short for a piece or too long for the registers: a block per row, which it reads two or three times, each value by one thread.
template <int DT>
__global__ void __launch_bounds__(256) residual_norm_block_kernel(const ResidualNorm a, int64_t first) {
  __shared__ float part[2][4];
  const int64_t row = first + blockIdx.x, gate_row = a.gate ? row / a.gate_every : 0;
  float post_rstd = 1.f, s = 0.f;
  if (a.wp) {
    for (int i = threadIdx.x; i < a.H; i += 256) {
      const float v = load_as_f32<DT>(a.y, row * a.ldy + i);
      s = __builtin_fmaf(v, v, s);
    }
    post_rstd = rsqrt_mean(block_sum(s, part[0]), a.H, a.eps);
  }
  auto stream = [&](int i) __attribute__((always_inline)) {
    float v = load_as_f32<DT>(a.y, row * a.ldy + i);
    if (a.wp) v = v * post_rstd * load_as_f32<DT>(a.wp, i);
    if (a.gate) v *= load_as_f32<DT>(a.gate, gate_row * a.ldg + i);
    return __builtin_fmaf(a.scale, v, load_as_f32<DT>(a.x, row * a.ldx + i));
  };
  s = 0.f;
  for (int i = threadIdx.x; i < a.H; i += 256) {
    const float v = stream(i);
    s = __builtin_fmaf(v, v, s);
  }
  const float rstd = rsqrt_mean(block_sum(s, part[1]), a.H, a.eps);
  if (threadIdx.x == 0) {
    if (a.post_rstd) a.post_rstd[row] = post_rstd;
    if (a.rstd) a.rstd[row] = rstd;
  }
  for (int i = threadIdx.x; i < a.H; i += 256) {
    const float v = stream(i);
    store_from_f32<DT>(a.stream, row * a.lds + i, v);
    store_from_f32<DT>(a.normed, row * a.ldn + i, v * rstd * load_as_f32<DT>(a.w, i));
  }
}

struct ResidualNormBack {
  const void *ds, *dz, *y, *r, *w, *wp, *gate;  // ds or dz null: zero
  const float *post_rstd, *rstd;
  void *dx, *dy, *dgate;  // dgate: of a row, where every row has a gate of its own
  int64_t ldds, lddz, ldy, ldr, ldg, lddx, lddy;
  int M, H, gate_every, groups, parts;  // groups of rows that share a gate (one where none do), parts of a group's rows
  float scale;
};

// Sums over rows: a part's in f32, or (partial null) all of them, rounded.
struct ColumnSums {
  float* partial;
  void* out;
};

// Four values of a piece, the first or the second: what is made of a whole piece at a time does not fit the registers next to a row that is on its way.
template <int DT>
__device__ __forceinline__ void four(const u32x4& v, int half, float (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == NPAMD_F32) f[e] = __builtin_bit_cast(float, (uint32_t)v[e]);
    else f[e] = act_bits_to_f32<DT>(e & 1 ? v[2 * half + e / 2] >> 16 : v[2 * half + e / 2] & 0xFFFFu);
  }
}
template <int DT>
__device__ __forceinline__ void put_four(u32x4& v, int half, const float (&f)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == NPAMD_F32) v[e] = __builtin_bit_cast(uint32_t, f[e]);
    else if (e & 1) continue;
    else if constexpr (DT == NPAMD_BF16) v[2 * half + e / 2] = f32_to_bf16_bits(f[e]) | (f32_to_bf16_bits(f[e + 1]) << 16);
    else v[2 * half + e / 2] = f32_to_f16_bits(f[e]) | (f32_to_f16_bits(f[e + 1]) << 16);
  }
}

// The piece has been read when this has been passed: what stands behind it, a barrier too, may let others overwrite where it came from.
__device__ __forceinline__ void arrived(const u32x4& v) { asm volatile("; arrived %0" ::"v"(v) : "memory"); }

// Whether the registers hold a team's next rows too.
constexpr bool rows_ahead(int dt, int nv, bool post, int gate) { return dt == NPAMD_F32 ? nv < 4 : nv < (post && gate ? 2 : 3); }

enum Gate { kNoGate, kSharedGate, kOwnGate };  // own: of a row

// One pass over the four rows: RW waves to a row, `teams` rows to a block at a time, a lane has NV pieces of every row that its team meets and adds up its columns' part of the
// weights' and the gate's gradients in registers.  sum(u wp yh) is taken apart so that it needs no dr: with c = scale gate wp yh it is sum(c (ds + rstd v)) - rstd sum(v rh) / H
// sum(c rh), so a row's sums meet in LDS once.  Blocks take parts of a group's rows, so that a shared gate's sums have one place; a team's next row is on its way while
// this one's sums meet where the registers hold it (rows_ahead: one piece to a lane; two of 16 bits but with both norms and a gate, three of f32).  Bound by HBM: 8192 x 4096 bf16 with both norms and a gate 82 us,
// 4.9 TB/s of 403 MB.  Few rows: by the sums over rows, column by column through LDS and then a second launch (513 x 3003 fp16 with a gate of each sequence 13.8 us in both launches, 8.2 when neither dweight nor dgate is
// asked for; two rows of 8192 with both norms and a gate 15.2, 6.2 without any of its three sums).
template <int DT, int NV, bool POST, int GATE>
__global__ void __launch_bounds__(NV == 1 ? 1024 : 512) residual_norm_back_kernel(const ResidualNormBack a, const ColumnSums sum_w, const ColumnSums sum_p, const ColumnSums sum_g, int RW, int teams) {
  using P = Pieces<DT>;
  constexpr int V = P::V;
  constexpr bool kAhead = rows_ahead(DT, NV, POST, GATE);
  extern __shared__ __attribute__((aligned(16))) float team_sums[];
  __shared__ float meet[2][16][3];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = wave / RW, lanes = 64 * RW;
  const int lane = (int)threadIdx.x - team * lanes, H = a.H, pieces = (H + V - 1) / V;
  const float inv = 1.f / (float)H;
  constexpr bool kHeld = NV < 4 || !POST;  // the weights and a shared gate stay in registers; else they come from the L1 when they are used (2048 x 12288 bf16, shared gate: 254 / 127 us)
  u32x4 dsv[NV], dzv[NV], yv[NV], rv[NV], wv[NV], pv[NV], gv[NV];
  float dw[NV][V], dp[NV][V], dg[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = lane + lanes * i, at = min(p * V, H - V);
    dsv[i] = dzv[i] = yv[i] = rv[i] = wv[i] = pv[i] = gv[i] = u32x4{0, 0, 0, 0};
    if (kHeld && p < pieces) {
      wv[i] = P::load((const uint8_t*)a.w, at);
      if (POST) pv[i] = P::load((const uint8_t*)a.wp, at);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = dp[i][e] = dg[i][e] = 0.f;
  }
  float next_stats = 0.f;  // rstd in even lanes, post_rstd in odd ones
  const float* const stats = POST && threadIdx.x % 2 ? a.post_rstd : a.rstd;
  auto request = [&](int64_t row, int64_t end) __attribute__((always_inline)) {
    if (row >= end) return;
    int64_t at_row = row;  // by vector loads: scalar ones would be waited for in front of the barrier
    asm volatile("" : "+v"(at_row));
    next_stats = stats[at_row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + lanes * i, at = min(p * V, H - V);
      if (p >= pieces) continue;
      if (a.dz) dzv[i] = P::load(P::row_of(a.dz, row, a.lddz), at);
      rv[i] = P::load(P::row_of(a.r, row, a.ldr), at);
      if (a.ds) dsv[i] = P::load(P::row_of(a.ds, row, a.ldds), at);
      yv[i] = P::load(P::row_of(a.y, row, a.ldy), at);
      if (GATE == kOwnGate) gv[i] = P::load(P::row_of(a.gate, row, a.ldg), at);
    }
  };
  // The teams' sums meet in LDS and are added in their order.  Rows of whole pieces: a row's last piece lies behind those before, whole.
  const int width = pieces * V;
  auto leave = [&](const ColumnSums& to, float (&sum)[NV][V], int64_t place, int64_t out_row) __attribute__((always_inline)) {
    if (!to.partial && !to.out) return;
    __syncthreads();  // who adds up the sums before has read them
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = lane + lanes * i;
      if (p < pieces) {
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<f32x4*>(team_sums + team * width + p * V + e) = f32x4{sum[i][e], sum[i][e + 1], sum[i][e + 2], sum[i][e + 3]};
      }
#pragma unroll
      for (int e = 0; e < V; ++e) sum[i][e] = 0.f;
    }
    __syncthreads();
    const int whole = H / V * V;
    for (int o = threadIdx.x; o < width; o += blockDim.x) {
      float v = 0.f;
      for (int t = 0; t < teams; ++t) v += team_sums[t * width + o];
      const int column = o < whole ? o : o + H - width;
      if (to.partial) to.partial[place * width + o] = v;
      else if (o < whole || column >= whole) store_from_f32<DT>(to.out, out_row * H + column, v);
    }
  };
  int turn = 0;
  for (int unit = blockIdx.x; unit < a.groups * a.parts; unit += gridDim.x) {
    const int group = unit / a.parts, part = unit - group * a.parts;
    const int64_t from = GATE == kSharedGate ? (int64_t)group * a.gate_every : 0, rows = GATE == kSharedGate ? min((int64_t)a.gate_every, a.M - from) : a.M;
    // The parts' rows in turn: neighbouring blocks read neighbouring rows, where strips of rows would start a power of two of bytes apart (8192 x 4096: 92 / 83 us).
    const int64_t begin = from + (int64_t)part * teams, end = from + rows;
    const int step = a.parts * teams;
    if (GATE == kSharedGate && kHeld) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int p = lane + lanes * i;
        if (p < pieces) gv[i] = P::load(P::row_of(a.gate, group, a.ldg), min(p * V, H - V));
      }
    }
    auto bring = [&](int i, int at) __attribute__((always_inline)) {  // what is not held
      if (kHeld) return;
      wv[i] = P::load((const uint8_t*)a.w, at);
      if (POST) pv[i] = P::load((const uint8_t*)a.wp, at);
      if (GATE == kSharedGate) gv[i] = P::load(P::row_of(a.gate, group, a.ldg), at);
    };
    int64_t row = begin + team;
    if (kAhead) request(row, end);
    for (int64_t first = begin; first < end; first += step, row += step, turn ^= 1) {
      if (!kAhead) request(row, end);
      const bool live = row < end;
      const int stats_bits = __builtin_bit_cast(int, next_stats);
      const float rstd = __builtin_bit_cast(float, __builtin_amdgcn_readlane(stats_bits, 0)), post = __builtin_bit_cast(float, __builtin_amdgcn_readlane(stats_bits, 1));
      u32x4 ds_[NV], dz_[NV], y_[NV], r_[NV], g_[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) ds_[i] = dsv[i], dz_[i] = dzv[i], y_[i] = yv[i], r_[i] = rv[i], g_[i] = gv[i];
      if (kAhead) request(row + step, end);
      float s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int p = lane + lanes * i, skip = p * V + V <= H ? 0 : p * V + V - H;  // values that the piece before has too
        if (!live || p >= pieces) continue;
        bring(i, min(p * V, H - V));
        if (GATE == kSharedGate && !kHeld) g_[i] = gv[i];
#pragma unroll
        for (int half = 0; half < V / 4; ++half) {
          float dz[4], rh[4], w[4], ds[4], yh[4], wp[4], g[4];
          four<DT>(dz_[i], half, dz);
          four<DT>(r_[i], half, rh);
          four<DT>(wv[i], half, w);
          if (POST) {
            four<DT>(ds_[i], half, ds);
            four<DT>(y_[i], half, yh);
            four<DT>(pv[i], half, wp);
            if (GATE) four<DT>(g_[i], half, g);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float z = 4 * half + e >= skip ? dz[e] : 0.f, h = rh[e] * rstd, v = z * w[e];
            dw[i][4 * half + e] = __builtin_fmaf(z, h, dw[i][4 * half + e]);
            s1 = __builtin_fmaf(v, h, s1);
            if (POST) {
              float c = a.scale * wp[e] * (yh[e] * post);
              if (GATE) c *= g[e];
              c = 4 * half + e >= skip ? c : 0.f;
              s2 = __builtin_fmaf(c, __builtin_fmaf(rstd, v, ds[e]), s2);
              s3 = __builtin_fmaf(c, h, s3);
            }
          }
        }
      }
      s1 = wave_sum(s1);
      if (POST) s2 = wave_sum(s2), s3 = wave_sum(s3);
      if (RW > 1) {
        // dx and dy may take the places of ds and y, and a row's last two pieces overlap, also where they are two waves': every value of the row has to be here before any is stored.  The sums
        // have used dz and, with POST, these two.
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (!POST) arrived(ds_[i]), arrived(y_[i]);
        if ((threadIdx.x & 63) == 0) {
          meet[turn][wave][0] = s1;
          if (POST) meet[turn][wave][1] = s2, meet[turn][wave][2] = s3;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the loads stay on their way
        s1 = s2 = s3 = 0.f;
        for (int i = 0; i < RW; ++i) {
          s1 += meet[turn][team * RW + i][0];
          if (POST) s2 += meet[turn][team * RW + i][1], s3 += meet[turn][team * RW + i][2];
        }
      }
      if (!live) continue;
      const float c1 = s1 * inv, c2 = POST ? (s2 - rstd * c1 * s3) * inv : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int p = lane + lanes * i, at = min(p * V, H - V);
        if (p >= pieces) continue;
        const int skip = p * V + V <= H ? 0 : p * V + V - H;
        bring(i, at);
        if (GATE == kSharedGate && !kHeld) g_[i] = gv[i];
        P::forget(ds_[i]);
        P::forget(dz_[i]);
        P::forget(r_[i]);
        P::forget(y_[i]);
        u32x4 to_dx, to_dy, to_gate;
#pragma unroll
        for (int half = 0; half < V / 4; ++half) {
          float dr[4], f[4], g[4], y[4], wp[4], own[4];
          four<DT>(ds_[i], half, dr);
          four<DT>(dz_[i], half, f);
          four<DT>(wv[i], half, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] *= g[e];
          four<DT>(r_[i], half, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) dr[e] = __builtin_fmaf(rstd, f[e] - g[e] * rstd * c1, dr[e]);
          put_four<DT>(to_dx, half, dr);
          four<DT>(y_[i], half, y);
          if (POST) four<DT>(pv[i], half, wp);
          if (GATE) four<DT>(g_[i], half, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float d = a.scale * dr[e], u = GATE ? d * g[e] : d, yh = POST ? y[e] * post : y[e];
            if (GATE == kOwnGate) own[e] = d * (POST ? yh * wp[e] : yh);
            if (4 * half + e >= skip) {
              if (GATE == kSharedGate) dg[i][4 * half + e] = __builtin_fmaf(d, POST ? yh * wp[e] : yh, dg[i][4 * half + e]);
              if (POST) dp[i][4 * half + e] = __builtin_fmaf(u, yh, dp[i][4 * half + e]);
            }
            f[e] = POST ? post * __builtin_fmaf(u, wp[e], -yh * c2) : u;
          }
          put_four<DT>(to_dy, half, f);
          if (GATE == kOwnGate) put_four<DT>(to_gate, half, own);
        }
        if (a.dx) P::store(const_cast<uint8_t*>(P::row_of(a.dx, row, a.lddx)), at, to_dx);
        if (a.dy) P::store(const_cast<uint8_t*>(P::row_of(a.dy, row, a.lddy)), at, to_dy);
        if (GATE == kOwnGate && a.dgate) P::store(const_cast<uint8_t*>(P::row_of(a.dgate, row, H)), at, to_gate);
      }
    }
    if (GATE == kSharedGate) leave(sum_g, dg, unit, group);
  }
  leave(sum_w, dw, blockIdx.x, 0);
  if (POST) leave(sum_p, dp, blockIdx.x, 0);
}

// Rows too short for a piece or too long for the registers, a block per row: first the two factors of the rows' sums, which the columns need too ([M][2]), then, when
// the columns have been added up (dx and dy may take the place of what they read), dx and dy and the gradient of a row's own gate.
template <int DT>
struct BackValues {
  const ResidualNormBack& a;
  int64_t row, gate_row;
  float rstd, post;
  __device__ BackValues(const ResidualNormBack& a_, int64_t row_) : a(a_), row(row_), gate_row(a_.gate ? row_ / a_.gate_every : 0) {
    rstd = a.rstd[row];
    post = a.wp ? a.post_rstd[row] : 1.f;
  }
  __device__ float dz(int i) const { return a.dz ? load_as_f32<DT>(a.dz, row * a.lddz + i) : 0.f; }
  __device__ float ds(int i) const { return a.ds ? load_as_f32<DT>(a.ds, row * a.ldds + i) : 0.f; }
  __device__ float v(int i) const { return dz(i) * load_as_f32<DT>(a.w, i); }
  __device__ float rh(int i) const { return load_as_f32<DT>(a.r, row * a.ldr + i) * rstd; }
  __device__ float yh(int i) const { return load_as_f32<DT>(a.y, row * a.ldy + i) * post; }
  __device__ float wp(int i) const { return a.wp ? load_as_f32<DT>(a.wp, i) : 1.f; }
  __device__ float gate(int i) const { return a.gate ? load_as_f32<DT>(a.gate, gate_row * a.ldg + i) : 1.f; }
  __device__ float dr(int i, float c1) const { return __builtin_fmaf(rstd, v(i) - rh(i) * c1, ds(i)); }
};

template <int DT>
__global__ void __launch_bounds__(256) residual_norm_back_rows_kernel(const ResidualNormBack a, float* __restrict__ factors, int64_t first) {
  __shared__ float part[2][4];
  const BackValues<DT> of(a, first + blockIdx.x);
  float s = 0.f;
  for (int i = threadIdx.x; i < a.H; i += 256) s = __builtin_fmaf(of.v(i), of.rh(i), s);
  const float c1 = block_sum(s, part[0]) / (float)a.H;
  s = 0.f;
  if (a.wp)
    for (int i = threadIdx.x; i < a.H; i += 256) s = __builtin_fmaf(a.scale * of.gate(i) * of.wp(i) * of.yh(i), of.dr(i, c1), s);
  const float c2 = block_sum(s, part[1]) / (float)a.H;
  if (threadIdx.x == 0) factors[2 * of.row] = c1, factors[2 * of.row + 1] = c2;
}

template <int DT>
__global__ void __launch_bounds__(256) residual_norm_back_block_kernel(const ResidualNormBack a, const float* __restrict__ factors, int64_t first) {
  const BackValues<DT> of(a, first + blockIdx.x);
  const float c1 = factors[2 * of.row], c2 = factors[2 * of.row + 1];
  for (int i = threadIdx.x; i < a.H; i += 256) {
    const float dr = of.dr(i, c1), d = a.scale * dr, u = d * of.gate(i), yh = of.yh(i), wp = of.wp(i);
    if (a.dx) store_from_f32<DT>(a.dx, of.row * a.lddx + i, dr);
    if (a.dy) store_from_f32<DT>(a.dy, of.row * a.lddy + i, a.wp ? of.post * __builtin_fmaf(u, wp, -yh * c2) : u);
    if (a.dgate) store_from_f32<DT>(a.dgate, of.row * a.H + i, d * yh * wp);
  }
}

// The columns' sums over a part of a group's rows, a lane per column, in f64: a part may have any number of rows.
template <int DT>
__global__ void __launch_bounds__(256)
residual_norm_back_columns_kernel(const ResidualNormBack a, const float* __restrict__ factors, const ColumnSums sum_w, const ColumnSums sum_p, const ColumnSums sum_g) {
  __shared__ double sums[4][3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  double acc_w = 0., acc_p = 0.;
  auto leave = [&](const ColumnSums& to, int k, double v, int64_t place, int64_t out_row) {
    __syncthreads();
    sums[wave][k][lane] = v;
    __syncthreads();
    if (wave || col >= a.H) return;
    v = sums[0][k][lane] + sums[1][k][lane] + sums[2][k][lane] + sums[3][k][lane];
    if (to.partial) to.partial[place * a.H + col] = (float)v;
    else if (to.out) store_from_f32<DT>(to.out, out_row * a.H + col, (float)v);
  };
  for (int unit = blockIdx.y; unit < a.groups * a.parts; unit += gridDim.y) {
    const int group = unit / a.parts, part = unit - group * a.parts;
    const int64_t from = a.groups > 1 ? (int64_t)group * a.gate_every : 0, rows = a.groups > 1 ? min((int64_t)a.gate_every, a.M - from) : a.M;
    const int64_t begin = from + rows * part / a.parts, end = from + rows * (part + 1) / a.parts;
    double acc_g = 0.;
    if (col < a.H)
      for (int64_t row = begin + wave; row < end; row += 4) {
        const BackValues<DT> of(a, row);
        const float d = a.scale * of.dr(col, factors[2 * row]), yh = of.yh(col);
        acc_w = __builtin_fma((double)of.dz(col), (double)of.rh(col), acc_w);
        acc_p = __builtin_fma((double)(d * of.gate(col)), (double)yh, acc_p);
        acc_g = __builtin_fma((double)d, (double)(yh * of.wp(col)), acc_g);
      }
    if (sum_g.partial || sum_g.out) leave(sum_g, 2, acc_g, unit, group);
  }
  leave(sum_w, 0, acc_w, blockIdx.y, 0);
  leave(sum_p, 1, acc_p, blockIdx.y, 0);
}

// The parts' sums, in the order of the parts: 64 columns of one vector (blockIdx.y: the first weight's, the other's, the gates') to a block, its 16 waves each a sixteenth of the parts.
// A part has `width` columns, whole pieces: the last one's lie at its end.  Three vectors of 4096 in 256 parts 5.3 us, latency.
struct SumParts {
  ColumnSums w, p, g;
  int parts, gate_parts, H, width, last;
};
template <int DT>
__global__ void __launch_bounds__(1024) residual_norm_back_sum_kernel(const SumParts s) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane, which = min((int)blockIdx.y, 2), gate = (int)blockIdx.y - 2;
  const ColumnSums to = which == 0 ? s.w : which == 1 ? s.p : s.g;
  if (!to.partial) return;
  const int parts = which == 2 ? s.gate_parts : s.parts, first = parts * wave / 16, end = parts * (wave + 1) / 16;
  float v = 0.f;
  if (col < s.H) {
    const float* p = to.partial + ((which == 2 ? (int64_t)gate * parts : 0) + first) * s.width + (col < s.last ? col : col + s.width - s.H);
#pragma unroll 8
    for (int i = first; i < end; ++i, p += s.width) v += *p;
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave || col >= s.H) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += sums[i][lane];
  store_from_f32<DT>(to.out, (which == 2 ? (int64_t)gate * s.H : 0) + col, v);
}

constexpr int64_t kRows = 1 << 21;  // of a launch: it has fewer than 2^32 threads
constexpr int64_t kMaxSums = 4 << 20;

// Which kernels the backward pass takes.  Blocks have `parts` parts of each group's rows; their sums over rows are left to be added where there are several.
struct BackPlan {
  int nv = 0, row_waves = 0, teams = 0, groups = 1, parts = 1, blocks = 1;  // nv 0: rows that do not fit the registers
  int64_t width = 0;                                                       // of a part's sums
  int lds() const { return nv ? teams * (int)width * 4 : 0; }
  int64_t floats_w() const { return blocks > 1 ? blocks * width : 0; }
  int64_t floats_g() const { return parts > 1 ? groups * (int64_t)parts * width : 0; }
  int64_t factors(int M) const { return nv ? 0 : ((int64_t)2 * M + 3) / 4 * 4; }
  BackPlan(int M, int H, int gate_every, bool shared, int dtype) {
    const int V = dtype == NPAMD_F32 ? 4 : 8, pieces = (H + V - 1) / V;
    groups = shared ? (int)(((int64_t)M + gate_every - 1) / gate_every) : 1;
    const int64_t rows = shared ? std::min(M, gate_every) : M;  // of a group
    if (H < V || pieces > 2048) {
      width = H;
      const int64_t strips = std::min<int64_t>(std::clamp<int64_t>(kMaxSums / (8 * (int64_t)H), 64, 1024), ((int64_t)M + 63) / 64);
      parts = (int)std::clamp<int64_t>(strips / groups, 1, (rows + 63) / 64);
      blocks = (int)std::min<int64_t>((int64_t)groups * parts, 1024);
      return;
    }
    width = (int64_t)pieces * V;
    nv = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
    row_waves = 1;
    while (row_waves * 64 * nv < pieces) row_waves *= 2;
    teams = std::min((nv == 1 ? 16 : 8) / row_waves, std::max(1, M));
    auto count = [&](int turns) { return std::min<int64_t>(256, ((int64_t)M + teams * turns - 1) / (teams * turns)); };
    // A second launch for the sums costs what a turn of 4096 values does (two rows of 8192 bf16 in one block / in two 18.3 / 15.6 us, f32 22 / 18; four of 4096 12.9 / 11.9; four of 2048 f32 8.6 / 9.1).
    const int64_t most = count((count(2) > 1 || H >= 4096) && count(1) * H * 8 <= kMaxSums ? 1 : 2);
    parts = (int)std::clamp<int64_t>(most / groups, 1, std::max<int64_t>(1, (rows + teams - 1) / teams));
    blocks = (int)std::min<int64_t>((int64_t)groups * parts, 256);
  }
};

template <int DT>
int launch_forward(const ResidualNorm& a, hipStream_t st) {
  const char* what = "npamd_residual_norm";
  constexpr int V = Pieces<DT>::V;
  const int pieces = (a.H + V - 1) / V;
  for (int64_t at = 0; at < a.M; at += kRows) {
    const int64_t rows = std::min<int64_t>(kRows, a.M - at);
    if (a.H < V || pieces > 2048) {
      launch(residual_norm_block_kernel<DT>, (unsigned)rows, 256, 0, st, a, at);
      continue;
    }
#define NPAMD_RN(NV, RW) launch(residual_norm_row_kernel<DT, NV, RW>, (unsigned)((rows + (RW < 4 ? 4 / RW : 1) - 1) / (RW < 4 ? 4 / RW : 1)), RW < 4 ? 256 : 64 * RW, 0, st, a, at)
    if (pieces <= 64) NPAMD_RN(1, 1);
    else if (pieces <= 128) NPAMD_RN(1, 2);
    else if (pieces <= 256) NPAMD_RN(1, 4);
    else if (pieces <= 512) NPAMD_RN(1, 8);
    else if (pieces <= 1024) NPAMD_RN(1, 16);
    else NPAMD_RN(2, 16);
#undef NPAMD_RN
  }
  return check_launch(what);
}

template <int DT, int NV, bool POST>
const void* back_kernel(int gate) {
  return gate == kNoGate ? (const void*)residual_norm_back_kernel<DT, NV, POST, kNoGate>
                         : gate == kSharedGate ? (const void*)residual_norm_back_kernel<DT, NV, POST, kSharedGate> : (const void*)residual_norm_back_kernel<DT, NV, POST, kOwnGate>;
}

template <int DT>
int launch_backward(ResidualNormBack a, void* dw, void* dwp, void* dgate, float* space, hipStream_t st) {
  const char* what = "npamd_residual_norm_backward";
  const int gate = !a.gate ? kNoGate : a.gate_every == 1 ? kOwnGate : kSharedGate;
  const BackPlan p(a.M, a.H, a.gate_every, gate == kSharedGate, DT);
  a.groups = p.groups, a.parts = p.parts;
  a.dgate = gate == kOwnGate ? dgate : nullptr;
  if (gate != kSharedGate) dgate = nullptr;
  float* const factors = space;
  float* const pw = space + p.factors(a.M);
  float* const pp = pw + p.floats_w();
  float* const pg = pp + p.floats_w();
  const ColumnSums sw{dw && p.blocks > 1 ? pw : nullptr, dw}, sp{dwp && p.blocks > 1 ? pp : nullptr, dwp}, sg{dgate && p.parts > 1 ? pg : nullptr, dgate};
  if (p.nv) {
    using Kernel = void (*)(const ResidualNormBack, const ColumnSums, const ColumnSums, const ColumnSums, int, int);
    const void* const k = p.nv == 1   ? (a.wp ? back_kernel<DT, 1, true>(gate) : back_kernel<DT, 1, false>(gate))
                          : p.nv == 2 ? (a.wp ? back_kernel<DT, 2, true>(gate) : back_kernel<DT, 2, false>(gate))
                                      : (a.wp ? back_kernel<DT, 4, true>(gate) : back_kernel<DT, 4, false>(gate));
    static LdsLatch latch[3][2][3];
    const hipError_t e = enable_dynamic_lds(latch[p.nv / 2][a.wp ? 1 : 0][gate], k, p.lds());
    if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, p.lds(), hipGetErrorString(e));
    launch((Kernel)k, (unsigned)p.blocks, 64 * p.row_waves * p.teams, (unsigned)p.lds(), st, a, sw, sp, sg, p.row_waves, p.teams);
  } else {
    for (int64_t at = 0; at < a.M; at += kRows) launch(residual_norm_back_rows_kernel<DT>, (unsigned)std::min<int64_t>(kRows, a.M - at), 256, 0, st, a, factors, at);
    if (dw || dwp || dgate) launch(residual_norm_back_columns_kernel<DT>, dim3((unsigned)(a.H + 63) / 64, (unsigned)p.blocks), 256, 0, st, a, factors, sw, sp, sg);
    if (a.dx || a.dy || a.dgate)
      for (int64_t at = 0; at < a.M; at += kRows) launch(residual_norm_back_block_kernel<DT>, (unsigned)std::min<int64_t>(kRows, a.M - at), 256, 0, st, a, factors, at);
  }
  if (sw.partial || sp.partial || sg.partial) {
    constexpr int V = Pieces<DT>::V;
    const SumParts s{sw, sp, sg, p.blocks, p.parts, a.H, (int)p.width, p.nv ? a.H / V * V : a.H};
    launch(residual_norm_back_sum_kernel<DT>, dim3((unsigned)(a.H + 63) / 64, (unsigned)(2 + (sg.partial ? p.groups : 0))), 1024, 0, st, s);  // groups in parts: 512 at most
  }
  return check_launch(what);
}

bool bad_dtype(int dtype) { return dtype != NPAMD_F16 && dtype != NPAMD_BF16 && dtype != NPAMD_F32; }

}  // namespace

extern "C" int npamd_residual_norm(const void* x, int64_t ldx, const void* y, int64_t ldy, const void* weight, const void* post_weight, const void* gate, int64_t ldg,
                                   int gate_every, float scale, void* stream_out, int64_t lds, void* normed, int64_t ldn, float* post_rstd, float* rstd, int M, int H,
                                   float eps, int dtype, void* stream) {
  const char* what = "npamd_residual_norm";
  NPAMD_REQUIRE(M >= 0 && H >= 1 && H <= kMaxWidth, "%s: bad shape M=%d H=%d", what, M, H);
  NPAMD_REQUIRE(!bad_dtype(dtype), "%s: bad dtype %d", what, dtype);
  NPAMD_REQUIRE(ldx >= H && ldy >= H && lds >= H && ldn >= H && (!gate || ldg >= H), "%s: bad row stride", what);
  NPAMD_REQUIRE(!gate || gate_every >= 1, "%s: gate_every has to be at least 1, got %d", what, gate_every);
  if (M == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && y && weight && stream_out && normed, "%s: null pointer", what);
  const ResidualNorm a{x, y, weight, post_weight, gate, stream_out, normed, post_weight ? post_rstd : nullptr, rstd, ldx, ldy, ldg, lds, ldn, M, H, gate ? gate_every : 1, scale, eps};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NPAMD_F16) return launch_forward<NPAMD_F16>(a, st);
  if (dtype == NPAMD_BF16) return launch_forward<NPAMD_BF16>(a, st);
  return launch_forward<NPAMD_F32>(a, st);
}

extern "C" int64_t npamd_residual_norm_workspace_bytes(int M, int H, int gate_every, int dtype) {
  if (M < 1 || H < 1 || H > kMaxWidth || gate_every < 0 || bad_dtype(dtype)) return 0;
  const BackPlan p(M, H, std::max(1, gate_every), gate_every > 1, dtype);
  return 4 * (p.factors(M) + 2 * p.floats_w() + p.floats_g());
}

extern "C" int npamd_residual_norm_backward(const void* dstream, int64_t ldds, const void* dnormed, int64_t lddz, const void* y, int64_t ldy, const void* stream_in, int64_t ldr,
                                            const void* weight, const void* post_weight, const void* gate, int64_t ldg, int gate_every, float scale,
                                            const float* post_rstd, const float* rstd, void* dx, int64_t lddx, void* dy, int64_t lddy, void* dweight, void* dpost_weight,
                                            void* dgate, int M, int H, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_residual_norm_backward";
  NPAMD_REQUIRE(M >= 1 && H >= 1 && H <= kMaxWidth, "%s: bad shape M=%d H=%d", what, M, H);
  NPAMD_REQUIRE(!bad_dtype(dtype), "%s: bad dtype %d", what, dtype);
  NPAMD_REQUIRE((!dstream || ldds >= H) && (!dnormed || lddz >= H) && ldy >= H && ldr >= H && (!gate || ldg >= H) && (!dx || lddx >= H) && (!dy || lddy >= H), "%s: bad row stride", what);
  NPAMD_REQUIRE(!gate || gate_every >= 1, "%s: gate_every has to be at least 1, got %d", what, gate_every);
  NPAMD_REQUIRE((dstream || dnormed) && y && stream_in && weight && rstd && (!post_weight || post_rstd), "%s: null pointer", what);
  const int64_t need = npamd_residual_norm_workspace_bytes(M, H, gate ? gate_every : 0, dtype);
  NPAMD_REQUIRE(!need || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need), "%s: needs %lld bytes of 16-byte aligned workspace", what, (long long)need);
  const ResidualNormBack a{dstream, dnormed, y, stream_in, weight, post_weight, gate, post_rstd, rstd, dx, dy, nullptr, ldds, lddz, ldy, ldr, ldg, lddx, lddy,
                           M, H, gate ? gate_every : 1, 1, 1, scale};
  void* const dwp = post_weight ? dpost_weight : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NPAMD_F16) return launch_backward<NPAMD_F16>(a, dweight, dwp, gate ? dgate : nullptr, (float*)workspace, st);
  if (dtype == NPAMD_BF16) return launch_backward<NPAMD_BF16>(a, dweight, dwp, gate ? dgate : nullptr, (float*)workspace, st);
  return launch_backward<NPAMD_F32>(a, dweight, dwp, gate ? dgate : nullptr, (float*)workspace, st);
}
