// Low-rank adapters of many requests beside a projection that they share: y = base + scale[a] (x A_a^T) B_a^T, a = ids[m] the adapter of a token, none where it is outside the list.
//
// Two products whose weights depend on the token.  Tokens of one adapter meet its weights as the columns of MFMAs (16x16x32), so both kernels work on entries: an adapter and some of its
// tokens.  Up to 64 tokens every wave finds its entry's tokens by itself from the ids (one comparison of all of them and a count of bits), so a call is two launches; past that a
// block of one launch more sorts tokens by adapter and lists the entries.
//   down: t = x A^T, f32.  A block takes 16, 32 or 64 tokens of an entry, up to 64 ranks and a part of K; x and A come into LDS in whole lines, each wave with steps of its own, and the waves'
//         sums meet in LDS.
//   up:   y = base + scale t B^T.  A block brings its entry's t into LDS once, as two parts of B's type, for an MFMA each (t is not rounded to 16 bits: 2^-16 of it is left with bf16; fp16, scaled
//         by a power of two to the row's largest, 2^-21 of it and 2^-37 of the largest), and its waves take 64 or 128 columns each.  Column 8 c + b of a wave is row c of MFMA b, so that a lane ends up with eight neighbouring columns
//         of four tokens and 16 lanes with 256 bytes of a row of base and y, side by side.  (With four tokens' rows in every quarter of the lanes instead, as the MFMAs' own layout
//         has them, a load touches 64 places: 64 to 86 us in the place of 52 for 4096 tokens through 14336 columns of bf16, rank 64.)
// Bound by the latency of two dependent launches for a decode step, by the bytes of base and y for prompts.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "gemm_tile.hpp"
#include "lds_transfer.hpp"
#include "wave_ops.hpp"

using namespace npamd;

namespace {

constexpr int kBallotTokens = 64;  // as many as a wave compares at once
constexpr int kMaxAdapters = 8192, kMaxRank = 256;
constexpr int kDownTokens = 32, kDownMost = 64;  // of a listed entry's part in the down kernel
constexpr int kManyWaves = 1024;   // of the up kernel: four for each compute unit
constexpr int kGridRows = 65535;   // of a launch

struct Entry {
  int adapter, first, count, unused;  // tokens: order[first .. first + count)
};

struct AdapterArgs {
  const void *x, *ids, *a, *b, *base;
  const float* scale;
  void* y;
  int64_t ldx, ldbase, ldy;
  int M, N, K, rank, rank8, adapters, ids_64, parts;
  float* t;              // [parts][M][rank8]
  const int* order;      // listed entries
  const Entry* entries;
  const int* count;
  int entry_tokens;      // at most
};

// The adapter of a token; -1: none.
__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int m) {
  const int64_t id = a.ids_64 ? ((const int64_t*)a.ids)[m] : ((const int*)a.ids)[m];
  return id >= 0 && id < a.adapters ? (int)id : -1;
}

// An entry as a wave holds it.
struct Tokens {
  int adapter, first, count;  // count 0: no entry
  int mine;                   // of up to 64 tokens: the entry's token number lane % 16, valid below count
};

// Block `e` of up to 64 tokens has an entry if token e is the first, 17th, 33rd ... of its adapter.
__device__ __forceinline__ Tokens ballot_entry(const AdapterArgs& a, int e) {
  const int lane = threadIdx.x & 63;
  const int id = lane < a.M ? adapter_of(a, lane) : -2;
  const int wanted = __builtin_amdgcn_readlane(id, e);
  const uint64_t same = __ballot(id == wanted);
  const int before = __popcll(same & ((1ull << e) - 1)), count = min(16, __popcll(same) - before);
  if (before % 16) return {wanted, 0, 0, 0};
  const int slot = __popcll(same & ((1ull << lane) - 1)) - before;
  const int to = (same >> lane & 1) && slot >= 0 && slot < 16 ? slot : 63;  // lane 63 is nobody's slot
  const int token = __builtin_amdgcn_ds_permute(to * 4, lane);
  return {wanted, 0, count, __builtin_amdgcn_ds_bpermute((lane & 15) * 4, token)};
}

__device__ __forceinline__ Tokens listed_entry(const AdapterArgs& a, int e) {
  const Entry v = a.entries[e];  // there for every block, whether it has been written or not: one round trip to memory, not two
  if (e >= *a.count) return {-1, 0, 0, 0};
  return {__builtin_amdgcn_readfirstlane(v.adapter), __builtin_amdgcn_readfirstlane(v.first), __builtin_amdgcn_readfirstlane(v.count), 0};
}

// TG groups of 16 tokens, RG of 16 ranks; blockIdx.x: entry (listed: and its part of 32 or 64 tokens), .y: ranks, .z: part of K.  A wave takes every so manieth 64-k step of the part, in two places of its
// own in LDS: rows of 128 bytes, 16-byte piece p of row r in place p ^ ((r >> 1) & 7).  Tokens' rows come from wherever they are.
template <int TG, int RG>
struct DownTile {
  static constexpr int kTokens = 16 * TG, kRows = kTokens + 16 * RG, kPlace = kRows * 128, kSums = TG * RG * 1024;
  static constexpr int kWaves = kLdsPerBlockMax / (2 * kPlace) < 8 ? kLdsPerBlockMax / (2 * kPlace) : 8;
  static constexpr int lds(int waves) { return waves * 2 * kPlace; }
  static_assert(2 * kPlace >= kSums);
};

template <int ACT, int TG, int RG, bool LISTED>
__global__ void __launch_bounds__(512) adapter_down_kernel(const AdapterArgs a) {
  using T = DownTile<TG, RG>;
  constexpr int L = T::kRows / 8;
  extern __shared__ __attribute__((aligned(16))) uint8_t down_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, c = lane & 15, h = lane >> 4;
  Tokens e;
  if constexpr (LISTED) {
    const int parts_of_entry = a.entry_tokens / T::kTokens, part = blockIdx.x % parts_of_entry;
    e = listed_entry(a, blockIdx.x / parts_of_entry);
    e.first += part * T::kTokens;
    e.count = min(e.count - part * T::kTokens, T::kTokens);
  } else {
    e = ballot_entry(a, blockIdx.x);
  }
  auto token = [&](int at) __attribute__((always_inline)) { return LISTED ? a.order[e.first + at] : __builtin_amdgcn_ds_bpermute(at * 4, e.mine); };  // by all lanes at once
  if (e.count <= 0 || e.adapter < 0) return;
  const int r0 = blockIdx.y * 16 * RG, pieces = a.K / 8, steps = (pieces + 7) / 8;
  const int from = (int)((int64_t)steps * blockIdx.z / a.parts), till = (int)((int64_t)steps * (blockIdx.z + 1) / a.parts);
  // Load i brings rows 8 i .. 8 i + 7: tokens (past the entry's end its last one, or what was there), then ranks (past the last: it again); what comes of those is not stored.
  const int row8 = lane >> 3;
  const uint8_t* row[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int r = 8 * i + row8;
    if (8 * i < T::kTokens) row[i] = (const uint8_t*)a.x + (int64_t)token(min(r, e.count - 1)) * a.ldx * 2;
    else row[i] = (const uint8_t*)a.a + ((int64_t)e.adapter * a.rank + min(r0 + r - T::kTokens, a.rank - 1)) * a.K * 2;
  }
  uint8_t* const mine = down_lds + wave * 2 * T::kPlace;
  const uint32_t mine_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
  auto load = [&](int step, int place) __attribute__((always_inline)) {
    const int end = pieces - step * 8 - 1;  // pieces past the rows' end: the last one again
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (8 * i < T::kTokens && 8 * i >= e.count) continue;
      const int p = min((lane & 7) ^ (((8 * i + row8) >> 1) & 7), end);
      lds_load16_from(mine_at + (uint32_t)(place * T::kPlace + i * 1024), row[i] + (int64_t)step * 128 + p * 16);
    }
  };
  f32x4 acc[TG][RG];
#pragma unroll
  for (int g = 0; g < TG; ++g)
#pragma unroll
    for (int q = 0; q < RG; ++q) acc[g][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  int place = 0;
  if (from + wave < till) load(from + wave, 0);
  for (int step = from + wave; step < till; step += waves, place ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (step + waves < till) load(step + waves, place ^ 1);
    const uint8_t* const at = mine + place * T::kPlace;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4 xo[TG], ao[RG];
      const int spot = ((4 * j + h) ^ ((c >> 1) & 7)) << 4;
#pragma unroll
      for (int g = 0; g < TG; ++g) xo[g] = *reinterpret_cast<const u32x4*>(at + (16 * g + c) * 128 + spot);
#pragma unroll
      for (int q = 0; q < RG; ++q) ao[q] = *reinterpret_cast<const u32x4*>(at + (T::kTokens + 16 * q + c) * 128 + spot);
      if (step * 8 + 4 * j + h >= pieces) {  // past the rows' end: counts for nothing, whatever it is
#pragma unroll
        for (int g = 0; g < TG; ++g) xo[g] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < RG; ++q) ao[q] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int g = 0; g < TG; ++g)
#pragma unroll
        for (int q = 0; q < RG; ++q) acc[g][q] = mfma16<ACT>(ao[q], xo[g], acc[g][q]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the place may be loaded again
  }
  // A lane has the ranks 16 q + 4 h .. + 3 of token 16 g + c.
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(down_lds);
#pragma unroll
  for (int g = 0; g < TG; ++g)
#pragma unroll
    for (int q = 0; q < RG; ++q) *reinterpret_cast<f32x4*>(sums + (((wave * TG + g) * RG + q) * 64 + lane) * 4) = acc[g][q];
  __syncthreads();
  for (int o = wave; o < TG * RG; o += waves) {
    const int g = o / RG, q = o % RG, r = r0 + 16 * q + 4 * h, m = token(min(16 * g + c, e.count - 1));
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < waves; ++w) v += *reinterpret_cast<const f32x4*>(sums + ((w * TG * RG + o) * 64 + lane) * 4);
    if (16 * g + c >= e.count || r >= a.rank8) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r + i < a.rank ? v[i] : 0.f;  // what only fills B's rows up
    *reinterpret_cast<f32x4*>(a.t + ((int64_t)blockIdx.z * a.M + m) * a.rank8 + r) = v;
  }
}

// Eight values as two parts of the operands' type, both of the value's sign: the first cut off, the second what is left.  A part that would be zero where the value is not is the smallest
// number there is instead (bf16: the smallest normal one), so that a product with an infinite weight is infinite and not NaN.  The matrix pipes take fp16's subnormal numbers as they are: of a row
// whose largest value is 2^14 and more, two parts are off by 2 x 2^-24 at most where they are that small, 2^-37 of the largest (with the smallest normal number, 2^-14, in both parts 2^-27).
template <int ACT>
__device__ __forceinline__ void two_parts(const float (&v)[8], u32x4& hi, u32x4& lo) {
  constexpr float kTiny = ACT == NPAMD_BF16 ? 1.17549435e-38f : 5.9604644775390625e-8f;
  uint32_t h16[8], l16[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v[i]);
    const float tiny = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, kTiny) | (bits & 0x80000000u));
    float first;
    if constexpr (ACT == NPAMD_BF16) first = __builtin_bit_cast(float, bits & 0xFFFF0000u);
    else first = (float)__builtin_amdgcn_cvt_pkrtz(v[i], 0.f)[0];
    float left = fabsf(v[i]) == __builtin_inff() ? 0.f : v[i] - first;
    first = (v[i] != 0.f && fabsf(first) < kTiny) ? tiny : first;
    left = (v[i] != 0.f && fabsf(left) < kTiny) ? tiny : left;
    h16[i] = ACT == NPAMD_BF16 ? f32_to_bf16_bits(first) : f32_to_f16_bits(first);
    l16[i] = ACT == NPAMD_BF16 ? f32_to_bf16_bits(left) : f32_to_f16_bits(left);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) hi[i] = h16[2 * i] | (h16[2 * i + 1] << 16), lo[i] = l16[2 * i] | (l16[2 * i + 1] << 16);
}

// RC chunks of 32 ranks, CT columns to a lane; blockIdx.x: 16 CT columns to each of the block's waves, .y and .z: entry.  LDS: t's two parts, rows of 64 RC + 16 bytes, then what each token's sums are
// multiplied with, and the tokens.
template <int RC>
struct UpTile {
  static constexpr int kRow = 64 * RC + 16;
  static constexpr int lds(int tokens) { return tokens * (2 * kRow + 8); }
};

template <int ACT, int RC, int CT, bool LISTED>
__global__ void __launch_bounds__(256, RC == 1 ? 4 : 2) adapter_up_kernel(const AdapterArgs a) {
  using T = UpTile<RC>;
  constexpr int kPieces = 4 * RC;  // of a row of t, eight values each
  typedef uint32_t Columns __attribute__((ext_vector_type(CT / 2)));
  typedef uint32_t ColumnsAny __attribute__((ext_vector_type(CT / 2), aligned(2)));
  extern __shared__ __attribute__((aligned(16))) uint8_t up_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
  const Tokens e = LISTED ? listed_entry(a, blockIdx.z * gridDim.y + blockIdx.y) : ballot_entry(a, blockIdx.y);
  if (e.count <= 0) return;
  const int groups = (e.count + 15) / 16;
  const int64_t col0 = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * 16 * CT, n0 = col0 + CT * c;
  u32x4 bo[RC][CT];
  if (e.adapter >= 0) {
#pragma unroll
    for (int b = 0; b < CT; ++b) {
      const uint16_t* const row = (const uint16_t*)a.b + ((int64_t)e.adapter * a.N + min(n0 + b, (int64_t)a.N - 1)) * a.rank8;
#pragma unroll
      for (int q = 0; q < RC; ++q) {
        const int r = 32 * q + 8 * h;
        bo[q][b] = u32x4{0, 0, 0, 0};
        if (r < a.rank8) bo[q][b] = *reinterpret_cast<const u32x4*>(row + r);
      }
    }
  }
  // Columns of a row: as they lie, a row's last ones one by one.
  auto base_of = [&](int m) __attribute__((always_inline)) {
    Columns v;
#pragma unroll
    for (int i = 0; i < CT / 2; ++i) v[i] = 0;
    if (!a.base || n0 >= a.N) return v;
    const uint16_t* const row = (const uint16_t*)a.base + m * a.ldbase;
    if (n0 + CT <= a.N) return (Columns) * reinterpret_cast<const ColumnsAny*>(row + n0);
#pragma unroll
    for (int i = 0; i < CT; ++i)
      if (n0 + i < a.N) v[i >> 1] |= (uint32_t)row[n0 + i] << (16 * (i & 1));
    return v;
  };
  int next_m[4];
  Columns next[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // the first group's, on their way while t comes
    const int at = min(4 * h + i, e.count - 1);
    next_m[i] = LISTED ? a.order[e.first + at] : __builtin_amdgcn_ds_bpermute(at * 4, e.mine);
    next[i] = base_of(next_m[i]);
  }
  uint8_t* const first_part = up_lds;
  uint8_t* const second_part = up_lds + groups * 16 * T::kRow;
  float* const factors = reinterpret_cast<float*>(second_part + groups * 16 * T::kRow);
  int* const tokens = reinterpret_cast<int*>(factors + groups * 16);
  const float scale = e.adapter < 0 ? 0.f : a.scale ? a.scale[e.adapter] : 1.f;
  for (int o = threadIdx.x; o < groups * 16 * kPieces; o += blockDim.x) {
    const int at = o / kPieces, r = o % kPieces * 8;
    const int m = LISTED ? a.order[e.first + min(at, e.count - 1)] : __builtin_amdgcn_ds_bpermute(min(at, e.count - 1) * 4, e.mine);
    if (r == 0) tokens[at] = m;
    if (e.adapter < 0) continue;
    f32x4 sum[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    if (at < e.count && r < a.rank8) {
      const float* const from = a.t + (int64_t)m * a.rank8 + r;
      const int64_t part = (int64_t)a.M * a.rank8;
      for (int z0 = 0; z0 < a.parts; z0 += 4) {  // four parts on their way
        f32x4 got[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (z0 + i >= a.parts) break;
          const f32x4* const of = reinterpret_cast<const f32x4*>(from + (z0 + i) * part);
          got[i][0] = of[0];
          got[i][1] = of[1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (z0 + i < a.parts) sum[0] += got[i][0], sum[1] += got[i][1];
      }
    }
    float v[8], back = 1.f;  // a power of two
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = sum[i >> 2][i & 3];
    if constexpr (ACT == NPAMD_F16) {
      // The row's largest finite value to 2^14 .. 2^15.
      int top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = __builtin_bit_cast(int, v[i]) >> 23 & 255;
        top = max(top, x == 255 ? 0 : x);
      }
#pragma unroll
      for (int far = 1; far < kPieces; far *= 2) top = max(top, __shfl_xor(top, far, 64));
      top = max(top, 15);
      const float up = __builtin_bit_cast(float, (268 - top) << 23);
      back = __builtin_bit_cast(float, (top - 14) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= up;
    }
    u32x4 hi, lo;
    two_parts<ACT>(v, hi, lo);
    *reinterpret_cast<u32x4*>(first_part + at * T::kRow + r * 2) = hi;
    *reinterpret_cast<u32x4*>(second_part + at * T::kRow + r * 2) = lo;
    if (r == 0) factors[at] = scale * back;
  }
  __syncthreads();
  if (col0 >= a.N) return;
  for (int g = 0; g < groups; ++g) {
    int m[4];
    Columns base[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = next_m[i], base[i] = next[i];
    if (g + 1 < groups) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        next_m[i] = tokens[16 * (g + 1) + 4 * h + i];
        next[i] = base_of(next_m[i]);
      }
    }
    f32x4 acc[CT];  // token 16 g + 4 h + i, column n0 + b
    float factor[4];
    if (e.adapter >= 0) {
#pragma unroll
      for (int b = 0; b < CT; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < RC; ++q) {
        const uint32_t at = (16 * g + c) * T::kRow + q * 64 + h * 16;
        const u32x4 hi = *reinterpret_cast<const u32x4*>(first_part + at), lo = *reinterpret_cast<const u32x4*>(second_part + at);
#pragma unroll
        for (int b = 0; b < CT; ++b) acc[b] = mfma16<ACT>(hi, bo[q][b], mfma16<ACT>(lo, bo[q][b], acc[b]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) factor[i] = factors[16 * g + 4 * h + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (16 * g + 4 * h + i >= e.count) continue;
      Columns out = base[i];  // without an adapter: as it is, whatever it is
      if (e.adapter >= 0) {
#pragma unroll
        for (int k = 0; k < CT / 2; ++k) {
          uint32_t bits[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float v = __builtin_fmaf(factor[i], acc[2 * k + u][i], act_bits_to_f32<ACT>(u ? base[i][k] >> 16 : base[i][k] & 0xFFFFu));
            bits[u] = ACT == NPAMD_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
          }
          out[k] = bits[0] | (bits[1] << 16);
        }
      }
      uint16_t* const to = (uint16_t*)a.y + m[i] * a.ldy;
      if (n0 + CT <= a.N) {
        *reinterpret_cast<ColumnsAny*>(to + n0) = out;
      } else {
#pragma unroll
        for (int k = 0; k < CT; ++k)
          if (n0 + k < a.N) to[n0 + k] = (uint16_t)(out[k >> 1] >> (16 * (k & 1)));
      }
    }
  }
}

// Tokens by adapter, those without one last, and the entries.  One block: counts in LDS, their running sums, then every token to its place.  Where all of a wave's tokens have one
// adapter, as a prompt's have, they are counted and placed side by side with one atomic addition; else each by itself.  A token's results do not depend on its place.  5.6 us for 4096 tokens of
// five prompts, 6.4 for 4096 of 1024 adapters in any order (with a wave's adapters one after the other 8.4 and 91).
__global__ void __launch_bounds__(1024) adapter_list_kernel(const AdapterArgs a, int* __restrict__ order, Entry* __restrict__ entries, int* __restrict__ count) {
  extern __shared__ int places[];  // [adapters + 1]
  __shared__ int sums[2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, buckets = a.adapters + 1;
  // f(the lane's token, its bucket, whether there is one) for all tokens.  The first turns' ids are read once, all at a time.
  constexpr int kKept = 8;
  int kept[kKept];
  auto bucket_of = [&](int64_t id) __attribute__((always_inline)) { return id >= 0 && id < a.adapters ? (int)id : a.adapters; };
  auto bucket_at = [&](int64_t m) __attribute__((always_inline)) {  // past the end: the last one's
    m = min(m, (int64_t)a.M - 1);
    return bucket_of(a.ids_64 ? ((const int64_t*)a.ids)[m] : ((const int*)a.ids)[m]);
  };
  // All of them on their way at a time: without a branch between them.
  auto keep = [&](const auto* ids) __attribute__((always_inline)) {
    std::remove_cv_t<std::remove_reference_t<decltype(*ids)>> raw[kKept];
#pragma unroll
    for (int i = 0; i < kKept; ++i) raw[i] = ids[min(i * 1024 + (int)threadIdx.x, a.M - 1)];
#pragma unroll
    for (int i = 0; i < kKept; ++i) kept[i] = bucket_of(raw[i]);
  };
  if (a.ids_64) keep((const int64_t*)a.ids);
  else keep((const int*)a.ids);
  for (int i = threadIdx.x; i < buckets; i += 1024) places[i] = 0;
  __syncthreads();
  auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kKept; ++i)
      if (i * 1024 < a.M) f(i * 1024 + (int)threadIdx.x, kept[i]);
    int next = bucket_at(kKept * 1024 + threadIdx.x);
    for (int64_t at = kKept * 1024; at < a.M; at += 1024) {
      const int bucket = next;
      next = bucket_at(at + 1024 + threadIdx.x);
      f((int)at + (int)threadIdx.x, bucket);
    }
  };
  each([&](int m, int bucket) __attribute__((always_inline)) {
    const bool there = m < a.M;
    const uint64_t all = __ballot(there);
    if (__ballot(there && bucket == __builtin_amdgcn_readfirstlane(bucket)) == all) {
      if (lane == 0) atomicAdd(&places[bucket], __popcll(all));
    } else if (there) {
      atomicAdd(&places[bucket], 1);
    }
  });
  __syncthreads();
  // A thread's neighbouring buckets: tokens and entries in them, then in those before.
  const int per = (buckets + 1023) / 1024, first = min((int)threadIdx.x * per, buckets), last = min(first + per, buckets);
  int tokens = 0, parts = 0;
  for (int i = first; i < last; ++i) {
    tokens += places[i];
    parts += (places[i] + a.entry_tokens - 1) / a.entry_tokens;
  }
  int before[2] = {tokens, parts};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    for (int o = 1; o < 64; o <<= 1) {
      const int from = __shfl_up(before[k], o, 64);
      if (lane >= o) before[k] += from;
    }
    if (lane == 63) sums[k][wave] = before[k];
  }
  __syncthreads();
  int token = before[0] - tokens, entry = before[1] - parts, all_entries = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    token += w < wave ? sums[0][w] : 0;
    entry += w < wave ? sums[1][w] : 0;
    all_entries += sums[1][w];
  }
  for (int i = first; i < last; ++i) {
    const int n = places[i];
    places[i] = token;
    for (int at = 0; at < n; at += a.entry_tokens) entries[entry++] = Entry{i < a.adapters ? i : -1, token + at, min(a.entry_tokens, n - at), 0};
    token += n;
  }
  if (threadIdx.x == 0) *count = all_entries;
  __syncthreads();
  each([&](int m, int bucket) __attribute__((always_inline)) {
    const bool there = m < a.M;
    const uint64_t all = __ballot(there);
    int at = 0;
    if (__ballot(there && bucket == __builtin_amdgcn_readfirstlane(bucket)) == all) {
      if (lane == 0) at = atomicAdd(&places[bucket], __popcll(all));
      at = __builtin_amdgcn_readfirstlane(at) + lane;
    } else if (there) {
      at = atomicAdd(&places[bucket], 1);
    }
    if (there) order[at] = m;
  });
}

// Whether a lane of the up kernel has eight columns of listed tokens, not four: past rank 64, where they leave the registers of a wave two blocks to a compute unit, with blocks enough (us of a call of
// rank 128, four / eight: 4096 tokens through 14336 columns 135 / 112, 2000 through 14336 68 / 62, 1024 47.5 / 44.5; 4096 through 4096 65 / 67, 300 through 4096 22.6 / 25.0).
bool eight_columns(int M, int N, int rank8) { return rank8 <= 64 || (rank8 <= 128 && ((int64_t)N + 511) / 512 * ((M + kDownTokens - 1) / kDownTokens) >= 512); }

// Tokens of a listed entry: as many as leave two rounds of the up kernel's blocks, B being read once for each.
int entry_tokens_of(int M, int N, int rank8) {
  const int most = eight_columns(M, N, rank8) ? 128 : rank8 <= 128 ? 64 : 32;
  const int64_t columns = ((int64_t)N + 511) / 512;
  int tokens = most;
  while (tokens > kDownTokens && columns * ((M + tokens - 1) / tokens) < 512) tokens /= 2;
  return tokens;
}

struct AdapterSpace {
  bool listed;
  int rank8, parts, tokens, down_tokens, most, layers;  // entries at most, whole layers of a grid's rows
  int64_t t, entries, order, bytes;
  AdapterSpace(int M, int N, int K, int rank, int adapters) {
    listed = M > kBallotTokens;
    rank8 = (rank + 7) / 8 * 8;
    tokens = listed ? entry_tokens_of(M, N, rank8) : 16;
    most = listed ? (int)std::min<int64_t>(M, ((int64_t)M + tokens - 1) / tokens + adapters + 1) : M;
    layers = (most + kGridRows - 1) / kGridRows;
    most = (most + layers - 1) / layers * layers;
    // Parts of K of the down kernel: as many as there are compute units for its blocks, of which an eighth more are counted, as entries end inside; few tokens: two steps for each of a
    // block's waves.  64 tokens to a block, which A's rows are read for once, where there are blocks enough (us of a call, 32 tokens / 64, 4096 tokens of five prompts through 4096 columns: rank
    // 64, K = 4096 53.7 / 50.1; rank 32, K = 14336 70.5 / 56.9; five prompts through 14336 columns, rank 64, K = 4096 91.1 / 88.4).
    const int ranks = (rank8 + 63) / 64, parts_most = std::max(1, K / 1024);
    down_tokens = tokens >= kDownMost && (int64_t)(M / kDownMost) * ranks * parts_most >= 128 ? kDownMost : kDownTokens;
    const int blocks = (M + down_tokens - 1) / down_tokens * ranks, counted = blocks + blocks / 8;
    parts = listed ? std::clamp(std::min(256 / counted, parts_most), 1, 8) : std::clamp((K + 1023) / 1024, 1, 8);
    t = (int64_t)parts * M * rank8 * 4;
    entries = listed ? 16 + (int64_t)most * sizeof(Entry) : 0;
    order = listed ? ((int64_t)M * 4 + 15) / 16 * 16 : 0;
    bytes = t + entries + order;
  }
};

template <int ACT, int TG, int RG, bool LISTED>
int launch_down(const AdapterArgs& a, unsigned blocks, hipStream_t st, const char* what) {
  using T = DownTile<TG, RG>;
  const int steps = (a.K + 63) / 64, waves = std::clamp((steps + a.parts - 1) / a.parts, 1, T::kWaves), lds = T::lds(waves);
  static LdsLatch latch;
  const auto kernel = adapter_down_kernel<ACT, TG, RG, LISTED>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
  launch(kernel, dim3(blocks, (unsigned)((a.rank8 + 16 * RG - 1) / (16 * RG)), (unsigned)a.parts), 64 * waves, lds, st, a);
  return check_launch(what);
}

template <int ACT, int RC, int CT, bool LISTED>
int launch_up_tile(const AdapterArgs& a, int entries, int layers, hipStream_t st, const char* what) {
  using T = UpTile<RC>;
  // Four waves to a block, which bring t in together; one where that is next to nothing and blocks are few.
  const int64_t strips = ((int64_t)a.N + 16 * CT - 1) / (16 * CT);
  const int waves = LISTED || strips * entries >= kManyWaves ? 4 : 1, lds = T::lds(a.entry_tokens);
  static LdsLatch latch;
  const auto kernel = adapter_up_kernel<ACT, RC, CT, LISTED>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
  launch(kernel, dim3((unsigned)((strips + waves - 1) / waves), (unsigned)(entries / layers), (unsigned)layers), 64 * waves, lds, st, a);
  return check_launch(what);
}

// Four columns to a lane where registers allow no more and, of up to 64 tokens, where waves are few: there is less to a wave then (us of a call, eight / four: one token 4096 x 4096 of rank 16 7.3 / 6.9,
// 16 of rank 64 8.8 / 8.0; but 32 tokens of as many adapters 14336 x 4096 9.8 / 11.5).
template <int ACT, bool LISTED>
int launch_up(const AdapterArgs& a, int entries, int layers, hipStream_t st, const char* what) {
  if (a.rank8 > 128) return launch_up_tile<ACT, 8, 4, LISTED>(a, entries, layers, st, what);
  if constexpr (LISTED) {
    if (a.rank8 > 64 && eight_columns(a.M, a.N, a.rank8)) return launch_up_tile<ACT, 4, 8, true>(a, entries, layers, st, what);
  }
  if (a.rank8 > 64) return launch_up_tile<ACT, 4, 4, LISTED>(a, entries, layers, st, what);
  if constexpr (!LISTED) {
    if (((int64_t)a.N + 127) / 128 * entries < kManyWaves)
      return a.rank8 <= 32 ? launch_up_tile<ACT, 1, 4, false>(a, entries, layers, st, what) : launch_up_tile<ACT, 2, 4, false>(a, entries, layers, st, what);
  }
  return a.rank8 <= 32 ? launch_up_tile<ACT, 1, 8, LISTED>(a, entries, layers, st, what) : launch_up_tile<ACT, 2, 8, LISTED>(a, entries, layers, st, what);
}

template <int ACT, int TG>
int launch_listed_down(const AdapterArgs& a, unsigned blocks, hipStream_t st, const char* what) {
  // Up to 64 ranks to a block, so that the tokens' rows are read once.
  if (a.rank8 <= 16) return launch_down<ACT, TG, 1, true>(a, blocks, st, what);
  return a.rank8 <= 32 ? launch_down<ACT, TG, 2, true>(a, blocks, st, what) : launch_down<ACT, TG, 4, true>(a, blocks, st, what);
}

template <int ACT>
int launch_adapters(AdapterArgs a, const AdapterSpace& space, uint8_t* at, hipStream_t st, const char* what) {
  a.t = (float*)at;
  if (!space.listed) {
    const int rc = launch_down<ACT, 1, 1, false>(a, (unsigned)a.M, st, what);
    return rc != NPAMD_OK ? rc : launch_up<ACT, false>(a, a.M, 1, st, what);
  }
  int* const count = (int*)(at + space.t);
  Entry* const entries = (Entry*)(at + space.t + 16);
  int* const order = (int*)(at + space.t + space.entries);
  launch(adapter_list_kernel, 1, 1024, (unsigned)(a.adapters + 1) * 4, st, a, order, entries, count);
  a.order = order, a.entries = entries, a.count = count;
  const unsigned blocks = (unsigned)(space.most * (space.tokens / space.down_tokens));
  const int rc = space.down_tokens == kDownMost ? launch_listed_down<ACT, kDownMost / 16>(a, blocks, st, what) : launch_listed_down<ACT, kDownTokens / 16>(a, blocks, st, what);
  return rc != NPAMD_OK ? rc : launch_up<ACT, true>(a, space.most, space.layers, st, what);
}

}  // namespace

extern "C" int64_t npamd_adapter_linear_workspace_bytes(int M, int N, int K, int rank, int adapters) {
  if (M < 1 || N < 1 || K < 1 || rank < 1 || rank > kMaxRank || adapters < 1 || adapters > kMaxAdapters) return 0;
  return AdapterSpace(M, N, K, rank, adapters).bytes;
}

extern "C" int npamd_adapter_linear(const void* x, int64_t ldx, const void* ids, int ids_bits, const void* a, const void* b, const float* scale, const void* base, int64_t ldbase,
                                    void* y, int64_t ldy, int M, int N, int K, int rank, int adapters, int act_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_adapter_linear";
  NPAMD_REQUIRE(M >= 0 && N >= 0 && K >= 1 && rank >= 1 && adapters >= 1, "%s: bad shape M=%d N=%d K=%d rank=%d adapters=%d", what, M, N, K, rank, adapters);
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(ids_bits == 32 || ids_bits == 64, "%s: ids of 32 or 64 bits, got %d", what, ids_bits);
  if (rank > kMaxRank || adapters > kMaxAdapters || M > 1 << 22 || N > 1 << 24)
    return fail(NPAMD_ERR_UNSUPPORTED, "%s: at most 2^22 tokens, 2^24 columns of y, rank %d and %d adapters", what, kMaxRank, kMaxAdapters);
  NPAMD_REQUIRE(ldx >= K && ldy >= N && (!base || ldbase >= N), "%s: bad row stride", what);
  if (M == 0 || N == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && ids && a && b && y, "%s: null pointer", what);
  NPAMD_REQUIRE((((uintptr_t)a | (uintptr_t)b) & 15) == 0, "%s: a and b have to lie at 16-byte addresses", what);
  NPAMD_REQUIRE(((uintptr_t)x & 15) == 0 && ldx % 8 == 0 && K % 8 == 0, "%s: x has to lie at a 16-byte address, K=%d and its rows' distance have to be multiples of 8", what, K);
  const AdapterSpace space(M, N, K, rank, adapters);
  NPAMD_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= space.bytes, "%s: needs %lld bytes of 16-byte aligned workspace", what, (long long)space.bytes);
  const AdapterArgs args{x, ids, a, b, base, scale, y, ldx, ldbase, ldy, M, N, K, rank, space.rank8, adapters, ids_bits == 64, space.parts, nullptr, nullptr, nullptr, nullptr, space.tokens};
  hipStream_t st = (hipStream_t)stream;
  if (act_dtype == NPAMD_BF16) return launch_adapters<NPAMD_BF16>(args, space, (uint8_t*)workspace, st, what);
  return launch_adapters<NPAMD_F16>(args, space, (uint8_t*)workspace, st, what);
}
