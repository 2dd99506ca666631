// Low-rank adapters of many requests beside a projection that they share: y = base + scale[a] (x A_a^T) B_a^T, a = ids[m] the adapter of a token, none where it is outside the list.
//
// Two products whose weights depend on the token.  Tokens of one adapter meet its weights as the columns of MFMAs (16x16x32), so both kernels work on entries: an adapter and some of its
// tokens.  Up to 64 tokens every wave finds its entry's tokens by itself from the ids (one comparison of all of them and a count of bits), so a call is two launches; past that a
// block of one launch more sorts tokens by adapter and lists the entries.
//   down: t = x A^T, f32.  A block takes an entry's tokens, 16 to 64 ranks and (where rows are long) a part of K, which its waves share; their sums meet in LDS.
//   up:   y = base + scale t B^T.  A wave takes 64 columns: B's rows are dealt to the MFMAs' rows so that a lane ends up with 16 neighbouring columns of one token, whose base it reads and whose y
//         it writes as they lie.  t is not rounded to 16 bits: it is two parts of B's type (2^-16 of it left with bf16; fp16, scaled by a power of two to the row's largest, 2^-21), an MFMA each.
// Bound by the latency of two dependent launches for a decode step, by the bytes of base and y for prompts.
#include <algorithm>

#include "common.hpp"
#include "wave_ops.hpp"

using namespace npamd;

namespace {

constexpr int kBallotTokens = 64;  // as many as a wave compares at once
constexpr int kMaxAdapters = 8192, kMaxRank = 256;
constexpr int kDownTokens = 32;    // of a listed entry's part in the down kernel

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

// An entry as a wave holds it: lane c of each 16 lanes knows tokens c, 16 + c, ... of it.
struct Tokens {
  int adapter, first, count;  // count 0: no entry
  int mine;                   // ballot: the lane's token, valid below count
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
  if (e >= *a.count) return {-1, 0, 0, 0};
  const Entry v = a.entries[e];
  return {__builtin_amdgcn_readfirstlane(v.adapter), __builtin_amdgcn_readfirstlane(v.first), __builtin_amdgcn_readfirstlane(v.count), 0};
}

// TG groups of 16 tokens, RG of 16 ranks; blockIdx.x: entry (and its part of 32 tokens), .y: ranks, .z: part of K.  Any K of at least eight and any address: a row that does not end with a
// piece of eight has its last one end with the row, and the values that the piece before has too are zeroed in both operands.
template <int ACT, int TG, int RG, bool LISTED>
__global__ void __launch_bounds__(1024) adapter_down_kernel(const AdapterArgs a) {
  extern __shared__ __attribute__((aligned(16))) float down_sums[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, c = lane & 15, h = lane >> 4;
  Tokens e;
  if constexpr (LISTED) {
    const int pieces = a.entry_tokens / kDownTokens, part = blockIdx.x % pieces;
    e = listed_entry(a, blockIdx.x / pieces);
    e.first += part * kDownTokens;
    e.count = min(e.count - part * kDownTokens, kDownTokens);
  } else {
    e = ballot_entry(a, blockIdx.x);
  }
  if (e.count <= 0 || e.adapter < 0) return;
  int token[TG];
#pragma unroll
  for (int g = 0; g < TG; ++g) {  // past the entry's end: its last token, not stored
    const int at = min(16 * g + c, e.count - 1);
    token[g] = LISTED ? a.order[e.first + at] : __builtin_amdgcn_ds_bpermute(at * 4, e.mine);
  }
  const int r0 = blockIdx.y * 16 * RG;
  const uint16_t *xr[TG], *ar[RG];
#pragma unroll
  for (int g = 0; g < TG; ++g) xr[g] = (const uint16_t*)a.x + token[g] * a.ldx;
#pragma unroll
  for (int q = 0; q < RG; ++q) ar[q] = (const uint16_t*)a.a + ((int64_t)e.adapter * a.rank + min(r0 + 16 * q + c, a.rank - 1)) * a.K;
  const int pieces = (a.K + 7) / 8, tail = pieces * 8 - a.K, steps = (pieces + 3) / 4;
  const int from = (int)((int64_t)steps * blockIdx.z / a.parts), till = (int)((int64_t)steps * (blockIdx.z + 1) / a.parts);
  const int first = from + (till - from) * wave / waves, last = from + (till - from) * (wave + 1) / waves;
  f32x4 acc[TG][RG];
#pragma unroll
  for (int g = 0; g < TG; ++g)
#pragma unroll
    for (int q = 0; q < RG; ++q) acc[g][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = TG * RG > 4 ? 2 : 4;  // steps on their way
  auto get = [&](const uint16_t* row, int step) __attribute__((always_inline)) {
    const int p = step * 4 + h;
    u32x4 v{0, 0, 0, 0};
    if (p < pieces && step < last) v = *reinterpret_cast<const u32x4_any*>(row + min(p * 8, a.K - 8));
    return v;
  };
  for (int step = first; step < last; step += U) {
    u32x4 xo[U][TG], ao[U][RG];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int g = 0; g < TG; ++g) xo[u][g] = get(xr[g], step + u);
#pragma unroll
      for (int q = 0; q < RG; ++q) ao[u][q] = get(ar[q], step + u);
    }
    if (tail && step + U >= steps) {  // the last piece's first values are the piece's before
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool ends = (step + u) * 4 + h == pieces - 1;
        auto blank = [&](u32x4& v) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (ends && i < tail) v[i >> 1] &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        };
#pragma unroll
        for (int g = 0; g < TG; ++g) blank(xo[u][g]);
#pragma unroll
        for (int q = 0; q < RG; ++q) blank(ao[u][q]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < TG; ++g)
#pragma unroll
        for (int q = 0; q < RG; ++q) acc[g][q] = mfma16<ACT>(ao[u][q], xo[u][g], acc[g][q]);
  }
  // A lane has the ranks 16 q + 4 h .. + 3 of token 16 g + c.
#pragma unroll
  for (int g = 0; g < TG; ++g)
#pragma unroll
    for (int q = 0; q < RG; ++q) *reinterpret_cast<f32x4*>(down_sums + (((wave * TG + g) * RG + q) * 64 + lane) * 4) = acc[g][q];
  __syncthreads();
  for (int o = wave; o < TG * RG; o += waves) {
    const int g = o / RG, q = o % RG, r = r0 + 16 * q + 4 * h;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < waves; ++w) v += *reinterpret_cast<const f32x4*>(down_sums + ((w * TG * RG + o) * 64 + lane) * 4);
    if (16 * g + c >= e.count || r >= a.rank8) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r + i < a.rank ? v[i] : 0.f;  // what only fills B's rows up
    int m = token[0];
#pragma unroll
    for (int i = 1; i < TG; ++i) m = g == i ? token[i] : m;
    *reinterpret_cast<f32x4*>(a.t + ((int64_t)blockIdx.z * a.M + m) * a.rank8 + r) = v;
  }
}

// Eight values as two parts of the operands' type, both of the value's sign: the first cut off, the second what is left.  A part that would be zero where the value is not is the smallest
// normal number instead, so that a product with an infinite weight is infinite and not NaN.
template <int ACT>
__device__ __forceinline__ void two_parts(const float (&v)[8], u32x4& hi, u32x4& lo) {
  constexpr float kTiny = ACT == NPAMD_BF16 ? 1.17549435e-38f : 6.103515625e-5f;
  uint32_t h16[8], l16[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v[i]);
    const float tiny = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, kTiny) | (bits & 0x80000000u));
    float first;
    if constexpr (ACT == NPAMD_BF16) first = __builtin_bit_cast(float, bits & 0xFFFF0000u);
    else first = (float)__builtin_amdgcn_cvt_pkrtz(v[i], 0.f)[0];
    float left = fabsf(v[i]) == __builtin_inff() ? 0.f : v[i] - first;
    first = (v[i] != 0.f) & (fabsf(first) < kTiny) ? tiny : first;
    left = (v[i] != 0.f) & (fabsf(left) < kTiny) ? tiny : left;
    h16[i] = ACT == NPAMD_BF16 ? f32_to_bf16_bits(first) : f32_to_f16_bits(first);
    l16[i] = ACT == NPAMD_BF16 ? f32_to_bf16_bits(left) : f32_to_f16_bits(left);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) hi[i] = h16[2 * i] | (h16[2 * i + 1] << 16), lo[i] = l16[2 * i] | (l16[2 * i + 1] << 16);
}

// RC chunks of 32 ranks; blockIdx.x: 64 columns to each of the block's waves, .y: entry.
template <int ACT, int RC, bool LISTED>
__global__ void __launch_bounds__(256) adapter_up_kernel(const AdapterArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, h = lane >> 4;
  const int64_t col0 = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * 64;
  if (col0 >= a.N) return;
  const Tokens e = LISTED ? listed_entry(a, blockIdx.y) : ballot_entry(a, blockIdx.y);
  if (e.count <= 0) return;
  const int groups = (e.count + 15) / 16;
  const int64_t n0 = col0 + 16 * h;  // the lane's 16 columns
  struct Row {
    int m;
    u32x4 base[2];
    f32x4 t[RC][2];
  };
  // Pieces of eight columns: whole ones as they lie, a row's last values one by one.
  auto piece = [&](const uint16_t* row, int64_t n) __attribute__((always_inline)) {
    u32x4 v{0, 0, 0, 0};
    if (n + 8 <= a.N) return (u32x4) * reinterpret_cast<const u32x4_any*>(row + n);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < a.N) v[i >> 1] |= (uint32_t)row[n + i] << (16 * (i & 1));
    return v;
  };
  auto request = [&](int g) __attribute__((always_inline)) {
    Row row;
    const int at = min(16 * g + c, e.count - 1);  // past the entry's end: its last token, not stored
    row.m = LISTED ? a.order[e.first + at] : __builtin_amdgcn_ds_bpermute(at * 4, e.mine);
    row.base[0] = row.base[1] = u32x4{0, 0, 0, 0};
    if (a.base) {
      const uint16_t* const from = (const uint16_t*)a.base + row.m * a.ldbase;
      row.base[0] = piece(from, n0);
      row.base[1] = piece(from, n0 + 8);
    }
#pragma unroll
    for (int q = 0; q < RC; ++q) {
      row.t[q][0] = row.t[q][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int r = 32 * q + 8 * h;
      if (e.adapter < 0 || r >= a.rank8) continue;
      for (int z = 0; z < a.parts; ++z) {
        const f32x4* const from = reinterpret_cast<const f32x4*>(a.t + ((int64_t)z * a.M + row.m) * a.rank8 + r);
        row.t[q][0] += from[0];
        row.t[q][1] += from[1];
      }
    }
    return row;
  };
  u32x4 bo[RC][4];
  float scale = 0.f;
  if (e.adapter >= 0) {
    scale = a.scale ? a.scale[e.adapter] : 1.f;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      // Row 4 h' + i of MFMA b is column 16 h' + 4 b + i.
      const int64_t n = min(col0 + 16 * (c >> 2) + 4 * b + (c & 3), (int64_t)a.N - 1);
      const uint16_t* const row = (const uint16_t*)a.b + ((int64_t)e.adapter * a.N + n) * a.rank8;
#pragma unroll
      for (int q = 0; q < RC; ++q) {
        const int r = 32 * q + 8 * h;
        bo[q][b] = u32x4{0, 0, 0, 0};
        if (r < a.rank8) bo[q][b] = *reinterpret_cast<const u32x4*>(row + r);
      }
    }
  }
  Row next = request(0);
  for (int g = 0; g < groups; ++g) {
    Row row = next;
    if (g + 1 < groups) next = request(g + 1);
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] = act_bits_to_f32<ACT>(row.base[i >> 2][i & 3] & 0xFFFFu);
      v[2 * i + 1] = act_bits_to_f32<ACT>(row.base[i >> 2][i & 3] >> 16);
    }
    if (e.adapter >= 0) {
      float up = 1.f, down = 1.f;  // powers of two
      if constexpr (ACT == NPAMD_F16) {
        // The row's largest finite value to 2^14 .. 2^15.
        int top = 0;
#pragma unroll
        for (int q = 0; q < RC; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float value = row.t[q][i >> 2][i & 3];  // a copy: the cast of an element itself takes the first one's bits
            const int x = __builtin_bit_cast(int, value) >> 23 & 255;
            top = max(top, x == 255 ? 0 : x);
          }
        top = max(top, __shfl_xor(top, 16, 64));
        top = max(max(top, __shfl_xor(top, 32, 64)), 15);
        up = __builtin_bit_cast(float, (268 - top) << 23);
        down = __builtin_bit_cast(float, (top - 14) << 23);
      }
      f32x4 acc[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < RC; ++q) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = row.t[q][i >> 2][i & 3] * up;
        u32x4 hi, lo;
        two_parts<ACT>(t, hi, lo);
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[b] = mfma16<ACT>(bo[q][b], hi, mfma16<ACT>(bo[q][b], lo, acc[b]));
      }
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * b + i] = __builtin_fmaf(scale, acc[b][i] * down, v[4 * b + i]);
    }
    if (16 * g + c >= e.count) continue;
    uint32_t bits[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) bits[i] = ACT == NPAMD_BF16 ? f32_to_bf16_bits(v[i]) : f32_to_f16_bits(v[i]);
    uint16_t* const to = (uint16_t*)a.y + row.m * a.ldy;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t n = n0 + 8 * p;
      u32x4 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = bits[8 * p + 2 * i] | (bits[8 * p + 2 * i + 1] << 16);
      if (e.adapter < 0) out = row.base[p];  // as it is, whatever it is
      if (n + 8 <= a.N) {
        *reinterpret_cast<u32x4_any*>(to + n) = out;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n + i < a.N) to[n + i] = (uint16_t)(out[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// Tokens by adapter, those without one last, and the entries.  One block: counts in LDS, their running sums, then every token to its place; a wave's tokens of one adapter are placed
// side by side with one atomic addition, so that a prompt's stay together.  A token's results do not depend on its place.
__global__ void __launch_bounds__(1024) adapter_list_kernel(const AdapterArgs a, int* __restrict__ order, Entry* __restrict__ entries, int* __restrict__ count) {
  extern __shared__ int places[];  // [adapters + 1]
  __shared__ int sums[2][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, buckets = a.adapters + 1;
  for (int i = threadIdx.x; i < buckets; i += 1024) places[i] = 0;
  __syncthreads();
  // f(bucket of the lane's token, its place among the wave's of that bucket, how many those are, first lane?) for every token, once.
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    for (int64_t at = 0; at < a.M; at += 1024) {
      const int64_t m = at + threadIdx.x;
      const int id = m < a.M ? adapter_of(a, (int)m) : -2;
      uint64_t open = __ballot(id != -2);
      while (open) {
        const int chosen = __builtin_amdgcn_readlane(id, __ffsll((unsigned long long)open) - 1);
        const uint64_t same = __ballot(id == chosen);
        f(chosen < 0 ? a.adapters : chosen, same, id == chosen, (int)m);
        open &= ~same;
      }
    }
  };
  each([&](int bucket, uint64_t same, bool, int) __attribute__((always_inline)) {
    if (lane == 0) atomicAdd(&places[bucket], __popcll(same));
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
  if (threadIdx.x < 2) {
    int v = 0;
    for (int w = 0; w < 16; ++w) {
      const int next = sums[threadIdx.x][w];
      sums[threadIdx.x][w] = v;
      v += next;
    }
    sums[threadIdx.x][16] = v;
  }
  __syncthreads();
  int token = sums[0][wave] + before[0] - tokens, entry = sums[1][wave] + before[1] - parts;
  for (int i = first; i < last; ++i) {
    const int n = places[i];
    places[i] = token;
    for (int at = 0; at < n; at += a.entry_tokens) entries[entry++] = Entry{i < a.adapters ? i : -1, token + at, min(a.entry_tokens, n - at), 0};
    token += n;
  }
  if (threadIdx.x == 0) *count = sums[1][16];
  __syncthreads();
  each([&](int bucket, uint64_t same, bool mine, int m) __attribute__((always_inline)) {
    int at = 0;
    if (lane == 0) at = atomicAdd(&places[bucket], __popcll(same));
    at = __builtin_amdgcn_readfirstlane(at);
    if (mine) order[at + __popcll(same & ((1ull << lane) - 1))] = m;
  });
}

// Tokens of a listed entry: as many as leave two rounds of the up kernel's blocks, B being read once for each.
int entry_tokens_of(int M, int N) {
  const int64_t columns = ((int64_t)N + 255) / 256;
  int tokens = 128;
  while (tokens > kDownTokens && columns * ((M + tokens - 1) / tokens) < 512) tokens /= 2;
  return tokens;
}

struct AdapterSpace {
  bool listed;
  int rank8, parts, tokens, most;  // entries at most
  int64_t t, entries, order, bytes;
  AdapterSpace(int M, int N, int K, int rank, int adapters) {
    listed = M > kBallotTokens;
    rank8 = (rank + 7) / 8 * 8;
    parts = listed ? 1 : std::clamp((K + 4095) / 4096, 1, 16);
    tokens = listed ? entry_tokens_of(M, N) : 16;
    most = listed ? (int)std::min<int64_t>(M, ((int64_t)M + tokens - 1) / tokens + adapters + 1) : M;
    t = (int64_t)parts * M * rank8 * 4;
    entries = listed ? 16 + (int64_t)most * sizeof(Entry) : 0;
    order = listed ? ((int64_t)M * 4 + 15) / 16 * 16 : 0;
    bytes = t + entries + order;
  }
};

template <int ACT, int TG, int RG, bool LISTED>
int launch_down(const AdapterArgs& a, unsigned blocks, hipStream_t st, const char* what) {
  const int steps = ((a.K + 7) / 8 + 3) / 4, waves = std::clamp((steps + a.parts - 1) / a.parts, 1, 16), lds = waves * TG * RG * 1024;
  static LdsLatch latch;
  const auto kernel = adapter_down_kernel<ACT, TG, RG, LISTED>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
  launch(kernel, dim3(blocks, (unsigned)((a.rank8 + 16 * RG - 1) / (16 * RG)), (unsigned)a.parts), 64 * waves, lds, st, a);
  return check_launch(what);
}

template <int ACT, bool LISTED>
int launch_up(const AdapterArgs& a, unsigned entries, hipStream_t st, const char* what) {
  // A wave to a block where columns and entries are few.
  const int64_t strips = ((int64_t)a.N + 63) / 64;
  const int waves = strips * entries >= 2048 ? 4 : 1;
  const dim3 grid((unsigned)((strips + waves - 1) / waves), entries);
  if (a.rank8 <= 32) launch(adapter_up_kernel<ACT, 1, LISTED>, grid, 64 * waves, 0, st, a);
  else if (a.rank8 <= 64) launch(adapter_up_kernel<ACT, 2, LISTED>, grid, 64 * waves, 0, st, a);
  else if (a.rank8 <= 128) launch(adapter_up_kernel<ACT, 4, LISTED>, grid, 64 * waves, 0, st, a);
  else launch(adapter_up_kernel<ACT, 8, LISTED>, grid, 64 * waves, 0, st, a);
  return check_launch(what);
}

template <int ACT>
int launch_adapters(AdapterArgs a, const AdapterSpace& space, uint8_t* at, hipStream_t st, const char* what) {
  a.t = (float*)at;
  if (!space.listed) {
    const int rc = launch_down<ACT, 1, 1, false>(a, (unsigned)a.M, st, what);
    return rc != NPAMD_OK ? rc : launch_up<ACT, false>(a, (unsigned)a.M, st, what);
  }
  int* const count = (int*)(at + space.t);
  Entry* const entries = (Entry*)(at + space.t + 16);
  int* const order = (int*)(at + space.t + space.entries);
  launch(adapter_list_kernel, 1, 1024, (unsigned)(a.adapters + 1) * 4, st, a, order, entries, count);
  a.order = order, a.entries = entries, a.count = count;
  const unsigned blocks = (unsigned)(space.most * (space.tokens / kDownTokens));
  // Up to 64 ranks to a block, so that the tokens' rows are read once.
  const int rc = a.rank8 <= 16   ? launch_down<ACT, 2, 1, true>(a, blocks, st, what)
                 : a.rank8 <= 32 ? launch_down<ACT, 2, 2, true>(a, blocks, st, what)
                                 : launch_down<ACT, 2, 4, true>(a, blocks, st, what);
  return rc != NPAMD_OK ? rc : launch_up<ACT, true>(a, (unsigned)space.most, st, what);
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
  if (K < 8 || rank > kMaxRank || adapters > kMaxAdapters || M > 1 << 22 || N > 1 << 24)
    return fail(NPAMD_ERR_UNSUPPORTED, "%s: at least 8 columns of x, at most 2^22 tokens, 2^24 columns of y, rank %d and %d adapters", what, kMaxRank, kMaxAdapters);
  NPAMD_REQUIRE(ldx >= K && ldy >= N && (!base || ldbase >= N), "%s: bad row stride", what);
  if (M == 0 || N == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && ids && a && b && y, "%s: null pointer", what);
  NPAMD_REQUIRE(((uintptr_t)b & 15) == 0, "%s: b has to lie at a 16-byte address", what);
  const AdapterSpace space(M, N, K, rank, adapters);
  NPAMD_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= space.bytes, "%s: needs %lld bytes of 16-byte aligned workspace", what, (long long)space.bytes);
  const AdapterArgs args{x, ids, a, b, base, scale, y, ldx, ldbase, ldy, M, N, K, rank, space.rank8, adapters, ids_bits == 64, space.parts, nullptr, nullptr, nullptr, nullptr, space.tokens};
  hipStream_t st = (hipStream_t)stream;
  if (act_dtype == NPAMD_BF16) return launch_adapters<NPAMD_BF16>(args, space, (uint8_t*)workspace, st, what);
  return launch_adapters<NPAMD_F16>(args, space, (uint8_t*)workspace, st, what);
}
