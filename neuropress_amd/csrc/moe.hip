// A mixture-of-experts layer for a few tokens:
//   logits = x router^T,  p = softmax(logits) over all experts,  the top_k largest (ties to the lower index), divided by their sum on request
//   y = sum over them of p_e down_e(silu(gate_e(x)) * up_e(x))
// Expert weights are dense or group-quantized codes, w = (q - zero) scale, which is not rounded.  What is rounded to the activation type on the way is
// silu(gate) * up, the operand of the second product: sums and p stay in f32 up to the store of y.
//
// Three launches: the logits (a block per expert), up (every block first picks each token's experts from the logits, then walks (expert, 16 gate rows and their
// 16 up rows)), down (a block per 16 rows of y, all its experts one behind the other).  The experts' weights are all that counts: each byte is read once, an expert's
// tokens share it as the 16 columns of an MFMA.
//
// Codes: an MFMA 16x16x32 sees 32 columns of one scale group, so a group's scale multiplies the f32 sum behind it, four multiply-adds for 512 weights, instead of the
// weights in front of it; nothing is rounded to 16 bits that way.  The codes become operands as they are, their bits under an exponent: q + 128, + 1024 or + 64
// exactly; the offset and the symmetric zero point go out by the MFMA's own addend, -(offset + zero) sum(x), itself an MFMA on a constant operand that the row
// tiles share.  (Sums of x (q + 1024) in f32 are off by 2^-24 1024 / 8 of a group's sum, some 1e-5: far below half a step of fp16.)
#include <algorithm>

#include "activation.hpp"
#include "common.hpp"
#include "gemm_tile.hpp"
#include "lds_transfer.hpp"

using namespace npamd;

namespace {

constexpr int kMoeMaxTokens = NPAMD_GEMV_MAX_M, kMoeMaxExperts = 512, kMoeMaxTopK = 16, kMoeMaxPairs = kMoeMaxTokens * kMoeMaxTopK;
constexpr int kMoeMaxWaves = 8;  // of a block

struct MoeArgs {
  const void *x, *router;
  const uint8_t *gate_up, *down;
  const uint16_t *gate_up_scale, *gate_up_zero, *down_scale, *down_zero;
  void* y;
  int64_t ldx, ldy;
  int M, E, top_k, H, I, shift, renormalize;  // shift: log2(group / 32)
  float* logits;   // [M][E]
  int32_t* ids;    // [M][top_k]
  float* share;    // [M][top_k]
  uint16_t* xs;    // [M][H], rows as the up kernel reads them
  uint16_t* h;     // [M][top_k][I]
};

// Eight 16-bit values at any even address.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// int4 operands hold the columns of an octet in the order 0 4 1 5 2 6 3 7 (the nibbles 4 i and 4 i + 16 of a dword are a pair): where column k of it lies.
__device__ __forceinline__ int octet_place(int k) { return ((k & 3) << 1) | ((k >> 2) & 1); }
__device__ __forceinline__ u32x4 octet_order(const u32x4& v) {  // (0 1) (2 3) (4 5) (6 7) -> (0 4) (1 5) (2 6) (3 7)
  return u32x4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u), __builtin_amdgcn_perm(v.w, v.y, 0x05040100u),
               __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
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

// The logits of one expert, TB tokens at a time; and every row of x, copied to where the up kernel reads it (NIBBLES: each octet in int4's order), by one block each.
template <int ACT, int TB, bool NIBBLES>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a) {
  __shared__ float part[4][kMoeMaxTokens];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x, octets = a.H / 8;
  const auto* x = reinterpret_cast<const uint16_t*>(a.x);
  const u32x4* const router = reinterpret_cast<const u32x4*>(a.router) + (int64_t)e * octets;
  for (int m0 = 0; m0 < a.M; m0 += TB) {
    float v[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) v[t] = 0.f;
    for (int k = threadIdx.x; k < octets; k += 256) {
      const u32x4 r = router[k];
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        const u32x4 xv = *reinterpret_cast<const u32x4_any*>(x + min(m0 + t, a.M - 1) * a.ldx + 8 * k);
        v[t] = dot8<ACT>(xv, r, v[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const float s = wave_reduce_sum(v[t]);
      if (lane == 0 && m0 + t < a.M) part[wave][m0 + t] = s;
    }
  }
  for (int m = e; m < a.M; m += a.E)
    for (int k = threadIdx.x; k < octets; k += 256) {
      const u32x4 xv = *reinterpret_cast<const u32x4_any*>(x + m * a.ldx + 8 * k);
      reinterpret_cast<u32x4*>(a.xs)[(int64_t)m * octets + k] = NIBBLES ? octet_order(xv) : xv;
    }
  __syncthreads();
  if ((int)threadIdx.x < a.M) a.logits[threadIdx.x * a.E + e] = part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
}

// The routing of all tokens in a block's LDS.
struct MoeRoute {
  int32_t ids[kMoeMaxPairs];  // [M][top_k]
  float share[kMoeMaxPairs];
  uint32_t met[kMoeMaxExperts / 32];  // bit e: some token meets expert e
  uint16_t experts[kMoeMaxExperts];   // those, in order
  int n_experts;
};

// One wave picks the experts of token m.
__device__ __forceinline__ void pick_experts(const MoeArgs& a, int m, int lane, MoeRoute& route) {
  constexpr int kPer = kMoeMaxExperts / 64;
  float v[kPer];
  float most = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    v[i] = -INFINITY;
    if (64 * i < a.E) v[i] = lane + 64 * i < a.E ? a.logits[m * a.E + lane + 64 * i] : -INFINITY;
    most = fmaxf(most, v[i]);
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (64 * i < a.E && lane + 64 * i < a.E) sum += expf(v[i] - most);
  sum = wave_reduce_sum(sum);
  uint32_t taken = 0;
  float mine = 0.f, total = 0.f;
  int id = 0;
  for (int t = 0; t < a.top_k; ++t) {
    // the largest of what is left, NaN above all: an order of (value, -index) as one 64-bit number
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (64 * i >= a.E) break;
      if (lane + 64 * i >= a.E || (taken >> i & 1)) continue;
      const float l = v[i];
      const uint32_t bits = __builtin_bit_cast(uint32_t, l + 0.f);  // minus zero is zero
      const uint32_t order = l != l ? 0xFFFFFFFFu : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
      const uint64_t key = ((uint64_t)order << 32) | (uint32_t)(0xFFFFFFFFu - (lane + 64 * i));
      best = key > best ? key : best;
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, off, 64);
      best = other > best ? other : best;
    }
    const int e = (int)(0xFFFFFFFFu - (uint32_t)best);
    if ((e & 63) == lane) taken |= 1u << (e >> 6);
    const uint32_t order = (uint32_t)(best >> 32), bits = order & 0x80000000u ? order & 0x7FFFFFFFu : ~order;
    const float l = order == 0xFFFFFFFFu ? NAN : __builtin_bit_cast(float, bits);
    const float p = expf(l - most) / sum;
    total += p;
    if (lane == t) mine = p, id = e;
  }
  if (lane < a.top_k) {
    route.ids[m * a.top_k + lane] = id;
    route.share[m * a.top_k + lane] = a.renormalize ? mine / total : mine;
  }
}

// The list of the experts that are met, from the pairs; all threads of the block, behind a barrier that follows the ids.
__device__ __forceinline__ void list_experts(const MoeArgs& a, MoeRoute& route) {
  constexpr int kWords = kMoeMaxExperts / 32;
  if (threadIdx.x < kWords) route.met[threadIdx.x] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < a.M * a.top_k; p += blockDim.x) atomicOr(&route.met[route.ids[p] >> 5], 1u << (route.ids[p] & 31));
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    if (!(route.met[e >> 5] >> (e & 31) & 1)) continue;
    int before = __popc(route.met[e >> 5] & ((1u << (e & 31)) - 1u));
    for (int w = 0; w < e >> 5; ++w) before += __popc(route.met[w]);
    route.experts[before] = (uint16_t)e;
  }
  if (threadIdx.x == 0) {
    int n = 0;
    for (int w = 0; w < kWords; ++w) n += __popc(route.met[w]);
    route.n_experts = n;
  }
  __syncthreads();
}

// The pairs of expert e in their order, into a wave's own list; returns how many.
__device__ __forceinline__ int list_pairs(const MoeArgs& a, const MoeRoute& route, int e, int lane, uint16_t* list) {
  int n = 0;
  for (int p0 = 0; p0 < a.M * a.top_k; p0 += 64) {
    const bool is = p0 + lane < a.M * a.top_k && route.ids[p0 + lane] == e;
    const uint64_t all = __ballot(is);
    if (is) list[n + __popcll(all & ((1ull << lane) - 1ull))] = (uint16_t)(p0 + lane);
    n += __popcll(all);
  }
  return n;
}

// A step: KSTEP columns of 16 R rows of weights and of an expert's tokens, in a wave's own LDS: its tokens, 1024 / kXRow to a KiB (16-byte piece p of
// token j in place p ^ (j & 15) of its row), then for each of the R row tiles its 16 rows (piece p of row r in place p ^ (r >> 1 & 7) of eight or p ^ r of 16) and its
// scales and zero points, a dword for each row and 64 columns.
template <int FMT, bool ASYM>
struct MoeStep {
  static constexpr int kColumns = FMT == 16 ? 128 : 256, kMfmas = kColumns / 32;
  static constexpr int kRow = kColumns * FMT / 8, kSlots = kRow / 16, kRowsPerLoad = 64 / kSlots, kCodeLoads = 16 * kRow / 1024;
  static constexpr int kScales = FMT == 16 ? 0 : ASYM ? 512 : 256;
  static constexpr int kItem = 16 * kRow + kScales;
  static constexpr int kXRow = kColumns * 2, kXSlots = kXRow / 16, kTokensPerLoad = 1024 / kXRow;
  static constexpr int kWords = FMT == 4 ? 1 : FMT == 8 ? 2 : 4;  // dwords of a lane's octet
  static constexpr int x_loads(int tokens) { return (tokens + kTokensPerLoad - 1) / kTokensPerLoad; }
};

template <int ACT, int FMT, bool ASYM, int MT, int R>
struct MoeWalk {
  using S = MoeStep<FMT, ASYM>;
  static constexpr int kXLoads = S::x_loads(16 * MT);
  uint8_t* mine;
  uint32_t mine_lds;
  int lane, c, q, K, chunks, groups, shift, x_bytes;  // x_bytes: LDS of the tokens
  const uint8_t *w[R], *x;
  const uint16_t *scale[R], *zero[R];
  int count;  // tokens
  uint32_t x_off[kXLoads];
  f32x4 acc[R][MT];

  __device__ __forceinline__ MoeWalk(uint8_t* lds, int x_loads, int columns, int shift_) : mine(lds), K(columns), shift(shift_) {
    lane = threadIdx.x & 63;
    c = lane & 15, q = lane >> 4;
    mine_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    chunks = K / 64;
    groups = (K / 32) >> shift;
    x_bytes = x_loads * 1024;
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Row tile r: 16 rows from `row` on.
  __device__ __forceinline__ void rows(int r, const uint8_t* weights, const uint16_t* scales, const uint16_t* zeros, int64_t row) {
    w[r] = weights + row * (int64_t)(K / 8 * FMT);
    if constexpr (FMT != 16) scale[r] = scales + row * groups;
    if constexpr (ASYM) zero[r] = zeros + row * groups;
  }
  // The tokens: row list[j] / divide of x.
  __device__ __forceinline__ void tokens(const uint16_t* rows_of_x, const uint16_t* list, int n, int divide) {
    x = reinterpret_cast<const uint8_t*>(rows_of_x);
    count = __builtin_amdgcn_readfirstlane(n);
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
      const int j = min(i * S::kTokensPerLoad + lane / S::kXSlots, n - 1);
      x_off[i] = (uint32_t)((int)list[j] / divide) * (uint32_t)(K * 2);
    }
  }
  __device__ __forceinline__ void load(int step) {
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
      if (i * S::kTokensPerLoad >= count) break;
      const int j = i * S::kTokensPerLoad + lane / S::kXSlots;
      const int p = step * S::kXSlots + ((lane % S::kXSlots) ^ (j & 15));
      lds_load16(mine_lds + (uint32_t)(i * 1024), x_off[i] + (uint32_t)(min(p, K / 8 - 1) * 16), uniform_ptr(x));
    }
    const uint32_t row_bytes = (uint32_t)(K / 8 * FMT);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t dst = mine_lds + (uint32_t)(x_bytes + r * S::kItem);
#pragma unroll
      for (int t = 0; t < S::kCodeLoads; ++t) {
        const int row = t * S::kRowsPerLoad + lane / S::kSlots;
        const int p = step * S::kSlots + ((lane % S::kSlots) ^ (S::kSlots == 8 ? (row >> 1) & 7 : row));
        lds_load16(dst + (uint32_t)(t * 1024), (uint32_t)row * row_bytes + (uint32_t)min(p, (int)row_bytes / 16 - 1) * 16u, uniform_ptr(w[r]));
      }
      if constexpr (FMT != 16) {
        const int kc = min(step * 4 + (lane & 3), chunks - 1);
        const uint32_t at = (((uint32_t)(lane >> 2) * (uint32_t)groups + (uint32_t)((2 * kc) >> shift)) * 2u) & ~3u;
        lds_load4(dst + 16 * S::kRow, at, uniform_ptr(reinterpret_cast<const uint8_t*>(scale[r])));
        if constexpr (ASYM) lds_load4(dst + 16 * S::kRow + 256, at, uniform_ptr(reinterpret_cast<const uint8_t*>(zero[r])));
      }
    }
  }
  // A constant operand: `even` and `odd` dwords.
  static __device__ __forceinline__ u32x4 constant(uint32_t even, uint32_t odd) { return u32x4{even, odd, even, odd}; }

  static __device__ __forceinline__ u32x4 operand(const uint32_t (&v)[S::kWords]) {
    if constexpr (FMT == 16) {
      return u32x4{v[0], v[1], v[2], v[3]};
    } else if constexpr (FMT == 8 && ACT == NPAMD_F16) {  // 1024 + q
      return u32x4{__builtin_amdgcn_perm(0x64646464u, v[0], 0x04010400u), __builtin_amdgcn_perm(0x64646464u, v[0], 0x04030402u),
                   __builtin_amdgcn_perm(0x64646464u, v[1], 0x04010400u), __builtin_amdgcn_perm(0x64646464u, v[1], 0x04030402u)};
    } else if constexpr (FMT == 8) {  // q: eight bits are a bf16's
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t d = v[i >> 1] >> (16 * (i & 1));
        const uint32_t lo = __builtin_bit_cast(uint32_t, (float)(d & 0xFFu)), hi = __builtin_bit_cast(uint32_t, (float)((d >> 8) & 0xFFu));
        o[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
      }
      return u32x4{o[0], o[1], o[2], o[3]};
    } else if constexpr (ACT == NPAMD_F16) {  // 1024 + q, 64 + q
      return u32x4{(v[0] & 0x000F000Fu) | 0x64006400u, (v[0] & 0x00F000F0u) | 0x54005400u, ((v[0] >> 8) & 0x000F000Fu) | 0x64006400u,
                   ((v[0] >> 8) & 0x00F000F0u) | 0x54005400u};
    } else {  // 128 + q
      return u32x4{(v[0] & 0x000F000Fu) | 0x43004300u, ((v[0] >> 4) & 0x000F000Fu) | 0x43004300u, ((v[0] >> 8) & 0x000F000Fu) | 0x43004300u,
                   ((v[0] >> 12) & 0x000F000Fu) | 0x43004300u};
    }
  }
  static constexpr bool kOffset = FMT == 4 || (FMT == 8 && (ACT == NPAMD_F16 || !ASYM));
  // Minus what operand() adds to q, and minus the symmetric zero point.
  static __device__ __forceinline__ u32x4 offset() {
    if constexpr (FMT == 4) {
      if constexpr (ACT == NPAMD_F16) return ASYM ? constant(0xE400E400u, 0xD400D400u) : constant(0xE408E408u, 0xD480D480u);  // -1024, -64; -1032, -72
      else return ASYM ? constant(0xC300C300u, 0xC300C300u) : constant(0xC308C308u, 0xC308C308u);                             // -128; -136
    } else {
      if constexpr (ACT == NPAMD_F16) return ASYM ? constant(0xE400E400u, 0xE400E400u) : constant(0xE480E480u, 0xE480E480u);  // -1024; -1152
      else return constant(0xC300C300u, 0xC300C300u);                                                                         // -128
    }
  }
  static __device__ __forceinline__ u32x4 ones() { return ACT == NPAMD_F16 ? constant(0x3C003C00u, 0x3C003C00u) : constant(0x3F803F80u, 0x3F803F80u); }

  // The step that has been loaded; `next` issues the loads of the one behind it, as soon as this one is in registers.
  template <class Next>
  __device__ __forceinline__ void compute(int step, Next&& next) {
    const int in_lds = count;  // next() may go on to other tokens
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    u32x4 xa[MT][S::kMfmas];
    uint32_t raw[R][S::kMfmas][S::kWords];
    u32x4 sc[R], zp[R];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int j = min(16 * t + c, in_lds - 1);  // rows past the tokens: one that nobody stores again
      const uint8_t* const row = mine + j * S::kXRow;
#pragma unroll
      for (int i = 0; i < S::kMfmas; ++i) xa[t][i] = *reinterpret_cast<const u32x4*>(row + (((4 * i + q) ^ (j & 15)) << 4));
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint8_t* const item = mine + x_bytes + r * S::kItem;
      const uint8_t* const row = item + c * S::kRow;
      const int swizzle = S::kSlots == 8 ? (c >> 1) & 7 : c;
#pragma unroll
      for (int i = 0; i < S::kMfmas; ++i) {
        if constexpr (FMT == 4) {
          raw[r][i][0] = *reinterpret_cast<const uint32_t*>(row + ((i ^ swizzle) << 4) + 4 * q);
        } else if constexpr (FMT == 8) {
          const u32x2 v = *reinterpret_cast<const u32x2*>(row + (((2 * i + (q >> 1)) ^ swizzle) << 4) + 8 * (q & 1));
          raw[r][i][0] = v.x, raw[r][i][1] = v.y;
        } else {
          const u32x4 v = *reinterpret_cast<const u32x4*>(row + (((4 * i + q) ^ swizzle) << 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[r][i][e] = v[e];
        }
      }
      if constexpr (FMT != 16) sc[r] = *reinterpret_cast<const u32x4*>(item + 16 * S::kRow + 16 * c);
      if constexpr (ASYM) zp[r] = *reinterpret_cast<const u32x4*>(item + 16 * S::kRow + 256 + 16 * c);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    next();
    const int live = min(S::kMfmas, (K - step * S::kColumns) / 32);  // MFMAs in front of the rows' end
#pragma unroll
    for (int i = 0; i < S::kMfmas; ++i) {
      if (i >= live) break;
      f32x4 from[MT], sum[MT];
      if constexpr (FMT != 16) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          from[t] = f32x4{0.f, 0.f, 0.f, 0.f};
          if constexpr (kOffset) from[t] = mfma16<ACT>(xa[t][i], offset(), from[t]);
          if constexpr (ASYM) sum[t] = mfma16<ACT>(xa[t][i], ones(), f32x4{0.f, 0.f, 0.f, 0.f});
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const u32x4 b = operand(raw[r][i]);
        if constexpr (FMT == 16) {
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[r][t] = mfma16<ACT>(xa[t][i], b, acc[r][t]);
        } else {
          // groups of 32: a dword has both scales of its 64 columns; larger: the one scale, in either half of it
          const uint32_t index = (uint32_t)c * (uint32_t)groups + (uint32_t)((2 * (step * 4 + (i >> 1))) >> shift);
          const uint32_t half = shift ? index & 1u : (uint32_t)(i & 1);
          const float s = f16_bits_to_f32((sc[r][i >> 1] >> (16u * half)) & 0xFFFFu);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            f32x4 d = mfma16<ACT>(xa[t][i], b, from[t]);
            if constexpr (ASYM) {
              const float z = f16_bits_to_f32((zp[r][i >> 1] >> (16u * half)) & 0xFFFFu);
#pragma unroll
              for (int e = 0; e < 4; ++e) d[e] = __builtin_fmaf(-z, sum[t][e], d[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][t][e] = __builtin_fmaf(s, d[e], acc[r][t][e]);
          }
        }
      }
    }
  }
};

constexpr int kMoeRedRow = 36;  // floats of a token's row where the waves' sums meet: 32 and some to spread the banks

template <int ACT, int FMT, bool ASYM, int MT>
__global__ void __launch_bounds__(64 * kMoeMaxWaves) moe_up_kernel(const MoeArgs a, int x_loads) {
  using Walk = MoeWalk<ACT, FMT, ASYM, MT, 2>;
  using S = typename Walk::S;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ MoeRoute route;
  __shared__ uint16_t lists[kMoeMaxWaves][2][kMoeMaxTokens];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  float* const red = reinterpret_cast<float*>(lds + waves * (x_loads * 1024 + 2 * S::kItem));

  for (int m = wave; m < a.M; m += waves) pick_experts(a, m, lane, route);
  __syncthreads();
  if (blockIdx.x == 0)  // for the down kernel
    for (int p = threadIdx.x; p < a.M * a.top_k; p += blockDim.x) a.ids[p] = route.ids[p], a.share[p] = route.share[p];
  list_experts(a, route);

  const int tiles = a.I / 16, items = route.n_experts * tiles, steps = (a.H + S::kColumns - 1) / S::kColumns;
  const int first = steps * wave / waves, last = steps * (wave + 1) / waves;  // this wave's steps of an item
  Walk walk(lds + wave * (x_loads * 1024 + 2 * S::kItem), x_loads, a.H, a.shift);
  int parity = 0;
  auto begin = [&](int item) {
    const int e = route.experts[item / tiles], tile = item % tiles;
    uint16_t* const list = lists[wave][parity];
    const int n = list_pairs(a, route, e, lane, list);
    walk.rows(0, a.gate_up, a.gate_up_scale, a.gate_up_zero, (int64_t)e * 2 * a.I + tile * 16);
    walk.rows(1, a.gate_up, a.gate_up_scale, a.gate_up_zero, (int64_t)e * 2 * a.I + a.I + tile * 16);
    walk.tokens(a.xs, list, n, a.top_k);
  };
  int item = blockIdx.x;
  if (item < items) {
    begin(item);
    if (first < last) walk.load(first);
  }
  for (; item < items; item += gridDim.x) {
    const int count = walk.count;
    const uint16_t* const list = lists[wave][parity];
    const int following = item + gridDim.x;
    auto go_on = [&] {
      if (following >= items) return;
      parity ^= 1;
      begin(following);
      if (first < last) walk.load(first);
    };
    walk.clear();
    for (int step = first; step < last - 1; ++step) walk.compute(step, [&] { walk.load(step + 1); });
    // The last step of an item brings the next item's first on its way; `count` tokens are this one's.
    if (first < last) walk.compute(last - 1, go_on);
    else go_on();
    block_sync_lds();  // nobody reads the sums of the item before any more
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 16 * t + 4 * (lane >> 4) + i;
          if (j < count) red[(wave * 16 * MT + j) * kMoeRedRow + r * 16 + (lane & 15)] = walk.acc[r][t][i];
        }
    block_sync_lds();
    const int tile = item % tiles;
    for (int o = threadIdx.x; o < count * 16; o += blockDim.x) {
      const int j = o >> 4, n = o & 15;
      float gate = 0.f, up = 0.f;
      for (int w = 0; w < waves; ++w) {
        gate += red[(w * 16 * MT + j) * kMoeRedRow + n];
        up += red[(w * 16 * MT + j) * kMoeRedRow + 16 + n];
      }
      const int k = tile * 16 + n;
      const int at = FMT == 4 ? (k & ~7) | octet_place(k & 7) : k;
      store_from_f32<ACT>(a.h, (int64_t)list[j] * a.I + at, silu_f32(gate) * up);
    }
  }
}

template <int ACT, int FMT, bool ASYM, int MT>
__global__ void __launch_bounds__(64 * kMoeMaxWaves) moe_down_kernel(const MoeArgs a, int x_loads) {
  using Walk = MoeWalk<ACT, FMT, ASYM, MT, 1>;
  using S = typename Walk::S;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ MoeRoute route;
  __shared__ uint16_t lists[kMoeMaxWaves][2][kMoeMaxTokens];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  float* const sums = reinterpret_cast<float*>(lds + waves * (x_loads * 1024 + S::kItem));  // [wave][M][16]
  for (int p = threadIdx.x; p < a.M * a.top_k; p += blockDim.x) route.ids[p] = a.ids[p], route.share[p] = a.share[p];
  for (int o = threadIdx.x; o < waves * a.M * 16; o += blockDim.x) sums[o] = 0.f;
  __syncthreads();
  list_experts(a, route);
  const int n0 = blockIdx.x * 16, steps = (a.I + S::kColumns - 1) / S::kColumns, all = route.n_experts * steps;
  const int first = (int)((int64_t)all * wave / waves), last = (int)((int64_t)all * (wave + 1) / waves);
  Walk walk(lds + wave * (x_loads * 1024 + S::kItem), x_loads, a.I, a.shift);
  int parity = 0;
  auto begin = [&](int at) {
    const int e = route.experts[at / steps];
    const int n = list_pairs(a, route, e, lane, lists[wave][parity]);
    walk.rows(0, a.down, a.down_scale, a.down_zero, (int64_t)e * a.H + n0);
    walk.tokens(a.h, lists[wave][parity], n, 1);
  };
  if (first < last) {
    begin(first);
    walk.load(first % steps);
  }
  float* const mine = sums + wave * a.M * 16;
  for (int at = first; at < last; ++at) {
    const int step = at % steps, count = walk.count;
    const uint16_t* const list = lists[wave][parity];
    const bool ends = step == steps - 1 || at == last - 1;
    walk.compute(step, [&] {
      if (at == last - 1) return;
      if (ends) {
        parity ^= 1;
        begin(at + 1);
      }
      walk.load(ends ? 0 : step + 1);
    });
    if (!ends) continue;
    // the expert's tokens, each times its share: a token's place is written by one lane
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 16 * t + 4 * (lane >> 4) + i;
        if (j < count) {
          const int pair = list[j];
          float* const to = mine + pair / a.top_k * 16 + (lane & 15);
          *to = __builtin_fmaf(route.share[pair], walk.acc[0][t][i], *to);
        }
      }
    walk.clear();
  }
  __syncthreads();
  for (int o = threadIdx.x; o < a.M * 16; o += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += sums[w * a.M * 16 + o];
    store_from_f32<ACT>(a.y, (o >> 4) * a.ldy + n0 + (o & 15), v);
  }
}

struct MoeSpace {
  int64_t logits, ids, share, xs, h, bytes;
  MoeSpace(int M, int E, int top_k, int H, int I) {
    int64_t at = 0;
    auto take = [&](int64_t n) {
      const int64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    logits = take((int64_t)M * E * 4);
    ids = take((int64_t)M * top_k * 4);
    share = take((int64_t)M * top_k * 4);
    xs = take((int64_t)M * H * 2);
    h = take((int64_t)M * top_k * I * 2);
    bytes = at;
  }
};

template <int ACT, int FMT, bool ASYM, int MT>
int launch_moe_mt(const MoeArgs& a, hipStream_t st) {
  const char* what = "npamd_moe_layer";
  using S = MoeStep<FMT, ASYM>;
  constexpr bool kNibbles = FMT == 4;
  const int x_loads = S::x_loads(a.M);
  auto up_lds_of = [&](int waves) { return waves * (x_loads * 1024 + 2 * S::kItem) + waves * 16 * MT * kMoeRedRow * 4; };
  auto down_lds_of = [&](int waves) { return waves * (x_loads * 1024 + S::kItem) + waves * a.M * 16 * 4; };
  constexpr int kRoom = 160 * 1024 - 8192;  // next to what the kernels have of their own
  static const int env_up = getenv("UPW") ? atoi(getenv("UPW")) : 4, env_down = getenv("DNW") ? atoi(getenv("DNW")) : 8, env_cu = getenv("UPC") ? atoi(getenv("UPC")) : 4;
  int up_waves = env_up, down_waves = env_down;
  while (up_lds_of(up_waves) > kRoom) --up_waves;
  while (down_lds_of(down_waves) > kRoom) --down_waves;
  const int up_lds = up_lds_of(up_waves), down_lds = down_lds_of(down_waves);
  static LdsLatch up_latch, down_latch;
  const auto up = moe_up_kernel<ACT, FMT, ASYM, MT>;
  const auto down = moe_down_kernel<ACT, FMT, ASYM, MT>;
  hipError_t e = enable_dynamic_lds(up_latch, reinterpret_cast<const void*>(up), up_lds);
  if (e == hipSuccess) e = enable_dynamic_lds(down_latch, reinterpret_cast<const void*>(down), down_lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve LDS: %s", what, hipGetErrorString(e));
  const auto logits = a.M == 1 ? moe_logits_kernel<ACT, 1, kNibbles> : a.M <= 4 ? moe_logits_kernel<ACT, 4, kNibbles> : moe_logits_kernel<ACT, 8, kNibbles>;
  launch(logits, a.E, 256, 0, st, a);
  const int most = a.E < a.M * a.top_k ? a.E : a.M * a.top_k;  // experts that can be met
  const int64_t items = (int64_t)most * (a.I / 16);
  const int per_cu = std::min(env_cu, (160 * 1024) / (up_lds + 8192));
  launch(up, (unsigned)std::min<int64_t>(items, 256 * std::max(per_cu, 1)), 64 * up_waves, up_lds, st, a, x_loads);
  launch(down, a.H / 16, 64 * down_waves, down_lds, st, a, x_loads);
  return check_launch(what);
}

template <int ACT>
int launch_moe(const MoeArgs& a, int nbits, hipStream_t st) {
  const bool two = a.M > 16;
#define NPAMD_MOE(FMT, ASYM) return two ? launch_moe_mt<ACT, FMT, ASYM, 2>(a, st) : launch_moe_mt<ACT, FMT, ASYM, 1>(a, st)
  if (nbits == 16) NPAMD_MOE(16, false);
  if (nbits == 8 && a.gate_up_zero) NPAMD_MOE(8, true);
  if (nbits == 8) NPAMD_MOE(8, false);
  if (a.gate_up_zero) NPAMD_MOE(4, true);
  NPAMD_MOE(4, false);
#undef NPAMD_MOE
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int64_t npamd_moe_workspace_bytes(int M, int E, int top_k, int H, int I) {
  if (M < 1 || E < 1 || top_k < 1 || H < 1 || I < 1) return 0;
  return MoeSpace(M, E, top_k, H, I).bytes;
}

extern "C" int npamd_moe_layer(const void* x, int64_t ldx, const void* router, const void* gate_up, const void* gate_up_scale_f16,
                               const void* gate_up_zero_f16, const void* down, const void* down_scale_f16, const void* down_zero_f16, void* y,
                               int64_t ldy, int M, int E, int top_k, int H, int I, int nbits, int group_size, int renormalize, int act_dtype,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "npamd_moe_layer";
  NPAMD_REQUIRE(act_dtype == NPAMD_F16 || act_dtype == NPAMD_BF16, "%s: f16 or bf16 only", what);
  NPAMD_REQUIRE(nbits == 4 || nbits == 8 || nbits == 16, "%s: nbits must be 4, 8 or 16 (dense), got %d", what, nbits);
  NPAMD_REQUIRE(M >= 0 && E >= 1 && H >= 1 && I >= 1 && top_k >= 1 && top_k <= E, "%s: bad shape M=%d E=%d top_k=%d H=%d I=%d", what, M, E, top_k, H, I);
  if (M > kMoeMaxTokens || E > kMoeMaxExperts || top_k > kMoeMaxTopK)
    return fail(NPAMD_ERR_UNSUPPORTED, "%s: at most %d tokens, %d experts and top_k %d, got %d, %d and %d", what, kMoeMaxTokens, kMoeMaxExperts, kMoeMaxTopK, M, E, top_k);
  if (H % 64 || I % 64) return fail(NPAMD_ERR_UNSUPPORTED, "%s: H=%d and I=%d have to be multiples of 64", what, H, I);
  if (nbits != 16) {
    const bool power = group_size >= 32 && (group_size & (group_size - 1)) == 0;
    if (!power || H % group_size || I % group_size)
      return fail(NPAMD_ERR_UNSUPPORTED, "%s: group_size has to be 32, 64, 128, ... and divide H=%d and I=%d, got %d", what, H, I, group_size);
    NPAMD_REQUIRE(gate_up_scale_f16 && down_scale_f16, "%s: codes without scales", what);
    NPAMD_REQUIRE(!gate_up_zero_f16 == !down_zero_f16, "%s: zero points for both weights or for neither", what);
  }
  if (I > (1 << 20) || H > (1 << 20)) return fail(NPAMD_ERR_UNSUPPORTED, "%s: H=%d and I=%d have to be at most 2^20", what, H, I);
  NPAMD_REQUIRE(ldx >= H && ldy >= H, "%s: bad row stride", what);
  if (M == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && router && gate_up && down && y, "%s: null pointer", what);
  NPAMD_REQUIRE(aligned16(router) && aligned16(gate_up) && aligned16(down), "%s: router and weights have to lie at 16-byte addresses", what);
  const uintptr_t halves = nbits == 16 ? 0 : (uintptr_t)gate_up_scale_f16 | (uintptr_t)gate_up_zero_f16 | (uintptr_t)down_scale_f16 | (uintptr_t)down_zero_f16;
  NPAMD_REQUIRE((halves & 3) == 0, "%s: scales and zero points have to lie at 4-byte addresses", what);
  const MoeSpace space(M, E, top_k, H, I);
  NPAMD_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= space.bytes, "%s: needs %lld bytes of 16-byte aligned workspace", what, (long long)space.bytes);
  auto* at = (uint8_t*)workspace;
  const bool codes = nbits != 16;
  auto half = [&](const void* p) { return codes ? (const uint16_t*)p : nullptr; };
  int shift = 0;
  while (codes && (32 << shift) < group_size) ++shift;
  const MoeArgs a{x, router, (const uint8_t*)gate_up, (const uint8_t*)down, half(gate_up_scale_f16), half(gate_up_zero_f16), half(down_scale_f16),
                  half(down_zero_f16), y, ldx, ldy, M, E, top_k, H, I, shift, renormalize, (float*)(at + space.logits), (int32_t*)(at + space.ids),
                  (float*)(at + space.share), (uint16_t*)(at + space.xs), (uint16_t*)(at + space.h)};
  return act_dtype == NPAMD_BF16 ? launch_moe<NPAMD_BF16>(a, nbits, (hipStream_t)stream) : launch_moe<NPAMD_F16>(a, nbits, (hipStream_t)stream);
}
