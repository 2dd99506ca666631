// A mixture-of-experts layer for a few tokens:
//   logits = x router^T,  p = softmax(logits) over all experts,  the top_k largest (ties to the lower index), divided by their sum on request
//   y = sum over them of p_e down_e(silu(gate_e(x)) * up_e(x))
// Expert weights are dense or group-quantized codes, w = (q - zero) scale, which is not rounded.  Sums and p stay in f32 up to the store of y.  silu(gate) * up, the operand
// of the second product, is kept as the sum of two bf16: to 2^-16, in the range of f32 whatever the activations' type (in fp16 it would be infinite past 65504).
//
// Three launches: the logits (a block per expert), up (every block first picks each token's experts from the logits, then walks (expert, 16 gate rows and their
// 16 up rows)), down (a block per 32 rows of y and part of all their experts' columns).  The experts' weights are all that counts: each byte is read once for up to 16
// of an expert's tokens (eight in the down kernel), which share it as the columns of an MFMA.  One token through two of eight int4 experts of 4096 x 14336: 5.0, 31.4 and 20.6 us by
// themselves, 50 in a row, 4.0 TB/s of 198 MB; 16 tokens fp16 with zero points 181-186 us, 4.0 TB/s.  Bound by HBM inside the walks, by round trips in front of and behind them.
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
#include "wave_ops.hpp"

using namespace npamd;

namespace {

constexpr int kMoeMaxTokens = NPAMD_GEMV_MAX_M, kMoeMaxExperts = 512, kMoeMaxTopK = 16;
constexpr int kMoeMaxWaves = 8;  // of a block

struct MoeArgs {
  const void *x, *router;
  const uint8_t *gate_up, *down;
  const uint16_t *gate_up_scale, *gate_up_zero, *down_scale, *down_zero;
  void* y;
  int64_t ldx, ldy;
  int M, E, top_k, H, I, shift, renormalize;  // shift: log2(group / 32)
  float* logits;   // [M][E]
  uint16_t* ids;   // [M][top_k]
  float* share;    // [M][top_k]
  uint32_t* entries;  // [M * top_k], and how many there are
  uint32_t* done;  // [H / 32] blocks of the down kernel that have left their part
  float* parts;    // [part][H / 32][M * 32]
  uint16_t* xs;    // [M][H], rows as the up kernel reads them
  uint16_t* h;     // [M][top_k][2][I], bf16: silu(gate) * up, and what is left of it
};

// int4 operands hold the columns of an octet in the order 0 4 1 5 2 6 3 7 (the nibbles 4 i and 4 i + 16 of a dword are a pair): where column k of it lies.
__device__ __forceinline__ int octet_place(int k) { return ((k & 3) << 1) | ((k >> 2) & 1); }
__device__ __forceinline__ u32x4 octet_order(const u32x4& v) {  // (0 1) (2 3) (4 5) (6 7) -> (0 4) (1 5) (2 6) (3 7)
  return u32x4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u), __builtin_amdgcn_perm(v.w, v.y, 0x05040100u),
               __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}

// The logits of one expert for TB tokens (blockIdx.y); and every row of x, copied to where the up kernel reads it (NIBBLES: each octet in int4's order), by one block
// each.  It clears the down kernel's counters.
template <int ACT, int TB, bool NIBBLES>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a) {
  __shared__ float part[4][TB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x, octets = a.H / 8, m0 = blockIdx.y * TB;
  const auto* x = reinterpret_cast<const uint16_t*>(a.x);
  const u32x4* const router = reinterpret_cast<const u32x4*>(a.router) + (int64_t)e * octets;
  if (e == 0 && m0 == 0)
    for (int i = threadIdx.x; i < a.H / 32; i += 256) a.done[i] = 0;
  float v[TB];
#pragma unroll
  for (int t = 0; t < TB; ++t) v[t] = 0.f;
#pragma unroll 2
  for (int k = threadIdx.x; k < octets; k += 256) {
    const u32x4 r = router[k];
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const u32x4 xv = *reinterpret_cast<const u32x4_any*>(x + min(m0 + t, a.M - 1) * a.ldx + 8 * k);
      v[t] = add_dot8<ACT>(xv, r, v[t]);
      if ((m0 + t) % a.E == e && m0 + t < a.M) reinterpret_cast<u32x4*>(a.xs)[(int64_t)(m0 + t) * octets + k] = NIBBLES ? octet_order(xv) : xv;
    }
  }
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    const float s = wave_sum_last(v[t]);
    if (lane == 63) part[wave][t] = s;
  }
  __syncthreads();
  const int t = threadIdx.x;
  if (t < TB && m0 + t < a.M) a.logits[(m0 + t) * a.E + e] = part[0][t] + part[1][t] + part[2][t] + part[3][t];
}

// The routing of all tokens, in a block's LDS.  An entry is an expert and up to `cap` of its pairs.
struct MoeRoute {
  uint32_t* entries;  // [pairs] expert, and from bit 16 on the number of its first pair
  uint32_t* met;      // [E] pairs of each expert, while the entries are made
  int* counts;        // [wave][2] how many pairs the wave's lists hold
  int* n_entries;
  uint16_t* lists;    // [wave][2][16] the pairs of the entries that a wave is at
  uint16_t* ids;      // [M][top_k]
  static __host__ __device__ int bytes(int pairs, int waves) { return pairs * 4 + waves * 2 * (4 + 32) + 16 + (pairs + 1) / 2 * 4; }
  // `met` lies where weights will.
  __device__ __forceinline__ MoeRoute(uint8_t* at, int pairs, int waves, uint8_t* scratch) {
    entries = reinterpret_cast<uint32_t*>(at);
    counts = reinterpret_cast<int*>(entries + pairs);
    n_entries = counts + waves * 2;
    lists = reinterpret_cast<uint16_t*>(n_entries + 4);
    ids = lists + waves * 32;
    met = reinterpret_cast<uint32_t*>(scratch);
  }
};

// One wave picks the experts of token m; `first`: and writes them down for the down kernel.
__device__ __forceinline__ void pick_experts(const MoeArgs& a, int m, int lane, const MoeRoute& route, bool first) {
  constexpr int kPer = kMoeMaxExperts / 64;
  float v[kPer];
  uint32_t key[kPer];  // in the order of the logits, NaN above all; 0: none
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = 0;
    if (64 * i >= a.E) continue;
    v[i] = lane + 64 * i < a.E ? a.logits[m * a.E + lane + 64 * i] : -INFINITY;
    const uint32_t bits = __builtin_bit_cast(uint32_t, v[i] + 0.f);  // minus zero is zero
    if (lane + 64 * i < a.E) key[i] = v[i] != v[i] ? 0xFFFFFFFFu : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  }
  // A lane's expert is as many places behind the first as there are larger keys: three instructions for each, where a turn below waits for some 20 one after the other.
  if (a.E <= 64 && a.E <= 16 * a.top_k) {
    int place = 0;
    for (int e = 0; e < a.E; ++e) {
      const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)key[0], e);
      place += other > key[0] || (other == key[0] && e < lane);
    }
    const bool picked = lane < a.E && place < a.top_k;
    if (picked) route.ids[m * a.top_k + place] = (uint16_t)lane;
    if (!first) return;
    const uint32_t top = wave_max(key[0]);
    const float most = top == 0xFFFFFFFFu ? NAN : __builtin_bit_cast(float, top & 0x80000000u ? top & 0x7FFFFFFFu : ~top);
    const float power = lane < a.E ? __expf(v[0] - most) : 0.f, p = power / wave_sum(power), total = wave_sum(picked ? p : 0.f);
    if (picked) {
      a.ids[m * a.top_k + place] = (uint16_t)lane;
      a.share[m * a.top_k + place] = a.renormalize ? p / total : p;
    }
    return;
  }
  float most = 0.f, sum = 0.f, mine = 0.f, total = 0.f;
  int id = 0;
  for (int t = 0; t < a.top_k; ++t) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (64 * i < a.E) top = max(top, key[i]);
    top = wave_max(top);
    int e = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (64 * i >= a.E || found) continue;
      const uint64_t with = __ballot(key[i] == top);
      if (!with) continue;
      found = true;
      const int at = __ffsll((unsigned long long)with) - 1;
      e = 64 * i + at;
      if (lane == at) key[i] = 0;
    }
    const float l = top == 0xFFFFFFFFu ? NAN : __builtin_bit_cast(float, top & 0x80000000u ? top & 0x7FFFFFFFu : ~top);
    if (t == 0) {
      most = l;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (64 * i < a.E && lane + 64 * i < a.E) sum += __expf(v[i] - most);
      sum = wave_sum(sum);
    }
    const float p = __expf(l - most) / sum;
    total += p;
    if (lane == t) mine = p, id = e;
  }
  if (lane < a.top_k) {
    route.ids[m * a.top_k + lane] = (uint16_t)id;
    if (first) {
      a.ids[m * a.top_k + lane] = (uint16_t)id;
      a.share[m * a.top_k + lane] = a.renormalize ? mine / total : mine;
    }
  }
}

// The entries, from the pairs; all threads of the block, behind a barrier that follows the ids.
__device__ __forceinline__ void list_entries(const MoeArgs& a, const MoeRoute& route, int cap) {
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) route.met[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < a.M * a.top_k; p += blockDim.x) atomicAdd(&route.met[route.ids[p]], 1u);
  __syncthreads();
  if (threadIdx.x < 64) {
    int before = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + threadIdx.x, mine = e < a.E ? ((int)route.met[e] + cap - 1) / cap : 0;
      int upto = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int other = __shfl_up(upto, off, 64);
        if ((int)threadIdx.x >= off) upto += other;
      }
      for (int i = 0; i < mine; ++i) route.entries[before + upto - mine + i] = (uint32_t)(e | (i * cap) << 16);
      before += __shfl(upto, 63, 64);
    }
    if (threadIdx.x == 0) *route.n_entries = before;
  }
  __syncthreads();
}

// The pairs of an entry in their order, into a wave's list; returns how many.
__device__ __forceinline__ int list_pairs(const MoeArgs& a, const MoeRoute& route, uint32_t entry, int cap, int lane, uint16_t* list) {
  const int e = entry & 0xFFFF, first = entry >> 16;
  int n = 0;
  for (int p0 = 0; p0 < a.M * a.top_k; p0 += 64) {
    const bool is = p0 + lane < a.M * a.top_k && route.ids[p0 + lane] == e;
    const uint64_t all = __ballot(is);
    const int at = n + __popcll(all & ((1ull << lane) - 1ull)) - first;
    if (is && at >= 0 && at < cap) list[at] = (uint16_t)(p0 + lane);
    n += __popcll(all);
  }
  return min(n - first, cap);
}

// A step: kColumns columns of 16 R rows of weights and of an entry's tokens, in LDS in one of two places: the tokens, 1024 / kXRow to a KiB (16-byte piece p of
// token j in place p ^ j of its row), and for each of a wave's R row tiles its 16 rows (piece p of row r in place p ^ (r >> 1 & 7) of eight or p ^ r of 16) and its
// scales and zero points, a dword for each row and 64 columns.  All of it comes in whole lines, straight into LDS, a step ahead of the MFMAs.
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

// (v & MASK) | BITS in one instruction, which takes constants from registers only: one of them scalar.
template <uint32_t MASK, uint32_t BITS>
__device__ __forceinline__ uint32_t masked_or(uint32_t v) {
  uint32_t mask = MASK, bits = BITS;
  asm("" : "+s"(mask));
  asm("" : "+v"(bits));
  return (v & mask) | bits;
}

// ACT: the type of the tokens and so of the operands; DENSE: of dense weights.  GROUP: MFMAs that see one scale group, one after the other into one sum.
template <int ACT, int FMT, bool ASYM, int R, int GROUP, int DENSE>
struct MoeWalk {
  using S = MoeStep<FMT, ASYM>;
  static constexpr int kXLoads = S::x_loads(16), kPlace = R * S::kItem;
  uint8_t *own, *shared;  // LDS: the weights (two places of kPlace), the tokens (two of x_bytes)
  int lane, c, q, K, groups, shift, x_bytes;
  int x_first, x_stride;  // the loads of the tokens that this wave makes
  const uint8_t *w[R], *x;
  const uint8_t *scale[R], *zero[R];
  int x_loads;
  uint32_t x_row[kXLoads], w_off[S::kCodeLoads];
  f32x4 acc[R];

  __device__ __forceinline__ MoeWalk(uint8_t* weights_lds, uint8_t* tokens_lds, int most_x_loads, int columns, int shift_, int x_first_, int x_stride_)
      : own(weights_lds), shared(tokens_lds), K(columns), shift(shift_), x_first(x_first_), x_stride(x_stride_) {
    lane = threadIdx.x & 63;
    c = lane & 15, q = lane >> 4;
    groups = (K / 32) >> shift;
    x_bytes = most_x_loads * 1024;
#pragma unroll
    for (int t = 0; t < S::kCodeLoads; ++t) {
      const int row = t * S::kRowsPerLoad + lane / S::kSlots;
      w_off[t] = (uint32_t)row * (uint32_t)(K / 8 * FMT);
    }
    clear();
  }
  static __device__ __forceinline__ uint32_t lds_address(const uint8_t* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Row tile r: 16 rows from `row` on.
  __device__ __forceinline__ void rows(int r, const uint8_t* weights, const uint16_t* scales, const uint16_t* zeros, int64_t row) {
    w[r] = uniform_ptr(weights + row * (int64_t)(K / 8 * FMT));
    if constexpr (FMT != 16) scale[r] = uniform_ptr((const uint8_t*)(scales + row * groups));
    if constexpr (ASYM) zero[r] = uniform_ptr((const uint8_t*)(zeros + row * groups));
  }
  // The n tokens: rows row_of(j) of rows_of_x.
  template <class Row>
  __device__ __forceinline__ void tokens(const uint16_t* rows_of_x, int n, Row&& row_of) {
    x = reinterpret_cast<const uint8_t*>(rows_of_x);
    x_loads = __builtin_amdgcn_readfirstlane(S::x_loads(n));
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
      const int j = min(i * S::kTokensPerLoad + lane / S::kXSlots, n - 1);
      x_row[i] = (uint32_t)row_of(j) * (uint32_t)(K * 2);
    }
  }
  __device__ __forceinline__ void load(int step, int place) {
    int lane = this->lane;
    asm volatile("" : "+v"(lane));  // as in multiply()
    // pieces past the rows' end: the last one again
    const int last_x = (K - step * S::kColumns) / 8 - 1, last_w = (K - step * S::kColumns) / 8 * FMT / 16 - 1;
    const uint8_t* const xs = x + (int64_t)step * S::kXRow;
    const uint32_t to_x = lds_address(shared) + (uint32_t)(place * x_bytes), to = lds_address(own) + (uint32_t)(place * kPlace);
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
      if (i >= x_loads) break;
      if (i % x_stride != x_first) continue;
      const int p = (lane % S::kXSlots) ^ (i * S::kTokensPerLoad + lane / S::kXSlots);
      lds_load16(to_x + (uint32_t)(i * 1024), x_row[i] + (uint32_t)(min(p, last_x) * 16), xs);
    }
    uint32_t at_scale = 0;
    if constexpr (FMT != 16) {
      const int kc = min(step * 4 + (lane & 3), K / 64 - 1);
      at_scale = (((uint32_t)(lane >> 2) * (uint32_t)groups + (uint32_t)((2 * kc) >> shift)) * 2u) & ~3u;
    }
    uint32_t at[S::kCodeLoads];
#pragma unroll
    for (int t = 0; t < S::kCodeLoads; ++t) {
      const int row = t * S::kRowsPerLoad + lane / S::kSlots, p = (lane % S::kSlots) ^ (S::kSlots == 8 ? (row >> 1) & 7 : row);
      at[t] = w_off[t] + (uint32_t)min(p, last_w) * 16u;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t dst = to + (uint32_t)(r * S::kItem);
#pragma unroll
      for (int t = 0; t < S::kCodeLoads; ++t) lds_load16(dst + (uint32_t)(t * 1024), at[t], w[r] + (int64_t)step * S::kRow);
      if constexpr (FMT != 16) lds_load4(dst + 16 * S::kRow, at_scale, scale[r]);
      if constexpr (ASYM) lds_load4(dst + 16 * S::kRow + 256, at_scale, zero[r]);
    }
  }
  // This wave's loads have arrived.
  static __device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
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
      return u32x4{masked_or<0x000F000Fu, 0x64006400u>(v[0]), masked_or<0x00F000F0u, 0x54005400u>(v[0]), masked_or<0x000F000Fu, 0x64006400u>(v[0] >> 8),
                   masked_or<0x00F000F0u, 0x54005400u>(v[0] >> 8)};
    } else {  // 128 + q
      return u32x4{masked_or<0x000F000Fu, 0x43004300u>(v[0]), masked_or<0x000F000Fu, 0x43004300u>(v[0] >> 4), masked_or<0x000F000Fu, 0x43004300u>(v[0] >> 8),
                   masked_or<0x000F000Fu, 0x43004300u>(v[0] >> 12)};
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
  // Dense fp16 weights as sums of two bf16, exactly: eight and three bits.  Both parts have the weight's sign and neither is zero where it is not (2^-100 of it is lost in any
  // other second part), so that what meets an infinite hidden value is not NaN; an infinite weight's second part is finite.
  static __device__ __forceinline__ void split_f16(const uint32_t (&v)[S::kWords], u32x4* first, u32x4* second) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t part[2], rest[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float w = f16_bits_to_f32((v[i] >> (16 * e)) & 0xFFFFu), finite = __builtin_amdgcn_fmed3f(w, -65504.f, 65504.f);
        part[e] = __builtin_bit_cast(uint32_t, w);
        rest[e] = __builtin_bit_cast(uint32_t, __builtin_fmaf(finite, 0x1p-100f, finite - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, finite) & 0xFFFF0000u)));
      }
      (*first)[i] = __builtin_amdgcn_perm(part[1], part[0], 0x07060302u);
      (*second)[i] = __builtin_amdgcn_perm(rest[1], rest[0], 0x07060302u);
    }
  }

  // The step in `place`, with `n` tokens.
  __device__ __forceinline__ void multiply(int step, int place, int n) {
    // Places in LDS are worked out anew every time: kept, they would take more registers than the waves that hide the waits can spare.
    int c = this->c;
    asm volatile("" : "+v"(c));
    const int j = min(c, n - 1);  // rows past the tokens: one that nobody stores again
    const uint8_t* const xrow = shared + place * x_bytes + j * S::kXRow;
    const uint8_t* const base = own + place * kPlace;
    const int swizzle = S::kSlots == 8 ? (c >> 1) & 7 : c;
    const f32x4 zero4{0.f, 0.f, 0.f, 0.f};
    auto group = [&](int g) __attribute__((always_inline)) {
      u32x4 xa[GROUP];
      f32x4 d[R], from = zero4, sum = zero4;
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        xa[i] = *reinterpret_cast<const u32x4*>(xrow + (((4 * (g * GROUP + i) + q) ^ j) << 4));
        if constexpr (FMT != 16 && kOffset) from = mfma16<ACT>(xa[i], offset(), from);
        if constexpr (ASYM) sum = mfma16<ACT>(xa[i], ones(), sum);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint8_t* const row = base + r * S::kItem + c * S::kRow;
        d[r] = from;
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
          const int at = g * GROUP + i;
          uint32_t raw[S::kWords];
          if constexpr (FMT == 4) {
            raw[0] = *reinterpret_cast<const uint32_t*>(row + ((at ^ swizzle) << 4) + 4 * q);
          } else if constexpr (FMT == 8) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(row + (((2 * at + (q >> 1)) ^ swizzle) << 4) + 8 * (q & 1));
            raw[0] = v.x, raw[1] = v.y;
          } else {
            const u32x4 v = *reinterpret_cast<const u32x4*>(row + (((4 * at + q) ^ swizzle) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = v[e];
          }
          if constexpr (FMT != 16) {
            d[r] = mfma16<ACT>(xa[i], operand(raw), d[r]);
          } else if constexpr (DENSE == ACT) {
            acc[r] = mfma16<ACT>(xa[i], operand(raw), acc[r]);
          } else {
            u32x4 first, second;
            split_f16(raw, &first, &second);
            acc[r] = mfma16<ACT>(xa[i], first, mfma16<ACT>(xa[i], second, acc[r]));
          }
        }
      }
      if constexpr (FMT != 16) {
        // groups of 32: a dword has both scales of its 64 columns; larger: the one scale, in either half of it
        const int chunk = g * GROUP / 2;
        uint32_t by = (uint32_t)(g & 1) * 16u;
        if constexpr (GROUP > 1) by = (((uint32_t)c * (uint32_t)groups + (uint32_t)((2 * (step * 4 + chunk)) >> shift)) & 1u) * 16u;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint8_t* const at = base + r * S::kItem + 16 * S::kRow + 16 * c + 4 * chunk;
          const float s = f16_bits_to_f32((*reinterpret_cast<const uint32_t*>(at) >> by) & 0xFFFFu);
          if constexpr (ASYM) {
            const float z = f16_bits_to_f32((*reinterpret_cast<const uint32_t*>(at + 256) >> by) & 0xFFFFu);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[r][e] = __builtin_fmaf(-z, sum[e], d[r][e]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][e] = __builtin_fmaf(s, d[r][e], acc[r][e]);
        }
      }
    };
    const int live = (K - step * S::kColumns) / 32;  // MFMAs in front of the rows' end: whole groups
    if (live >= S::kMfmas) {
#pragma unroll
      for (int g = 0; g < S::kMfmas / GROUP; ++g) group(g);
    } else {
#pragma unroll 1
      for (int g = 0; g < live / GROUP; ++g) group(g);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the place may be loaded again
  }
};

constexpr int kMoeRedRow = 36;  // floats of a token's row where the waves' sums meet: 32 and some to spread the banks

// Items: (entry, 16 gate rows and their 16 up rows for each wave or for all), dealt to the blocks in turn.  TOGETHER: the waves have row tiles of their own and share the
// tokens, a barrier per step; else they share the columns of one pair of row tiles, each with tokens of its own, and their sums meet at the item's end.  Tokens
// take LDS and come from the L2 once per wave or per block: few of them are best brought by each wave, many are not.
template <int ACT, int FMT, bool ASYM, int GROUP, bool TOGETHER>
__global__ void __launch_bounds__(64 * kMoeMaxWaves, FMT == 8 && ASYM ? 3 : 4) moe_up_kernel(const MoeArgs a, int cap, int down_cap, int own_lds) {
  using Walk = MoeWalk<ACT, FMT, ASYM, 2, GROUP, ACT>;
  using S = typename Walk::S;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const MoeRoute route(lds + own_lds, a.M * a.top_k, waves, lds);
  for (int m = wave; m < a.M; m += waves) pick_experts(a, m, lane, route, blockIdx.x == 0);
  __syncthreads();
  list_entries(a, route, blockIdx.x == 0 ? down_cap : cap);
  if (blockIdx.x == 0) {  // for the down kernel
    for (int p = threadIdx.x; p < *route.n_entries; p += blockDim.x) a.entries[p] = route.entries[p];
    if (threadIdx.x == 0) a.entries[a.M * a.top_k] = *route.n_entries;
    if (down_cap != cap) list_entries(a, route, cap);  // those are read before its first barrier
  }

  const int groups = TOGETHER ? waves : 1, tiles = a.I / 16 / groups, items = __builtin_amdgcn_readfirstlane(*route.n_entries) * tiles, steps = (a.H + S::kColumns - 1) / S::kColumns;
  const int first = TOGETHER ? 0 : steps * wave / waves, last = TOGETHER ? steps : steps * (wave + 1) / waves;  // this wave's steps of an item: one at least
  const int x_bytes = S::x_loads(cap) * 1024;
  uint8_t* const tokens = lds + waves * 2 * Walk::kPlace;
  Walk walk(lds + wave * 2 * Walk::kPlace, tokens + (TOGETHER ? 0 : wave * 2 * x_bytes), S::x_loads(cap), a.H, a.shift, TOGETHER ? wave : 0, groups);
  float* const red = reinterpret_cast<float*>(tokens + (TOGETHER ? 1 : waves) * 2 * x_bytes);

  // What is requested next: a step ahead of what is multiplied, so it may be the next item's.
  int ahead = blockIdx.x, ahead_step = first, ahead_entry = -1, ahead_slot = 1;
  auto request = [&](int place) __attribute__((always_inline)) {
    if (ahead >= items) return;
    if (ahead_step == first) {
      const int at = ahead / tiles;
      const uint32_t entry = __builtin_amdgcn_readfirstlane(route.entries[at]);
      if (at != ahead_entry) {  // the entries that a block meets take the two lists in turn
        ahead_entry = at;
        ahead_slot ^= 1;
        uint16_t* const list = route.lists + (wave * 2 + ahead_slot) * 16;
        const int n = list_pairs(a, route, entry, cap, lane, list);
        if (lane == 0) route.counts[wave * 2 + ahead_slot] = n;
        walk.tokens(a.xs, n, [&](int j) { return (int)list[j] / a.top_k; });
      }
      const int64_t row = (int64_t)(entry & 0xFFFF) * 2 * a.I + (ahead % tiles * groups + (TOGETHER ? wave : 0)) * 16;
      walk.rows(0, a.gate_up, a.gate_up_scale, a.gate_up_zero, row);
      walk.rows(1, a.gate_up, a.gate_up_scale, a.gate_up_zero, row + a.I);
    }
    walk.load(ahead_step, place);
    if (++ahead_step == last) {
      ahead_step = first;
      ahead += gridDim.x;
    }
  };
  request(0);
  int place = 0, slot = 1, entry_now = -1;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    if (item / tiles != entry_now) slot ^= 1;
    entry_now = item / tiles;
    const int count = __builtin_amdgcn_readfirstlane(route.counts[wave * 2 + slot]);
    const uint16_t* const list = route.lists + (wave * 2 + slot) * 16;
    walk.clear();
    for (int step = first; step < last; ++step) {
      Walk::arrived();
      if constexpr (TOGETHER) block_sync_lds();  // everybody's tokens are there, and nobody reads the other place any more
      request(place ^ 1);
      walk.multiply(step, place, count);
      place ^= 1;
    }
    const int tile = item % tiles;
    auto store = [&](int j, int k, float gate, float up) __attribute__((always_inline)) {
      const int to = FMT == 4 ? (k & ~7) | octet_place(k & 7) : k;
      // Cut, not rounded: both parts have the value's sign, and neither is zero where it is not, so that an infinite weight makes no NaN of them.
      const float v = silu_f32(gate) * up;
      const uint32_t bits = __builtin_bit_cast(uint32_t, v);
      const float rest = fabsf(v) < INFINITY ? v - __builtin_bit_cast(float, bits & 0xFFFF0000u) : 0.f;
      uint16_t* const at = a.h + (int64_t)list[j] * 2 * a.I + to;
      at[0] = (uint16_t)(bits >> 16);
      at[a.I] = (uint16_t)f32_to_bf16_bits(v != 0.f ? copysignf(fmaxf(fabsf(rest), 0x1p-126f), v) : 0.f);
    };
    if constexpr (TOGETHER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * (lane >> 4) + i;
        if (j < count) store(j, (tile * groups + wave) * 16 + (lane & 15), walk.acc[0][i], walk.acc[1][i]);
      }
    } else {
      block_sync_lds();  // nobody reads the sums of the item before any more
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 4 * (lane >> 4) + i;
          if (j < count) red[(wave * cap + j) * kMoeRedRow + r * 16 + (lane & 15)] = walk.acc[r][i];
        }
      block_sync_lds();
      for (int o = threadIdx.x; o < count * 16; o += blockDim.x) {
        const int j = o >> 4, n = o & 15;
        float gate = 0.f, up = 0.f;
        for (int w = 0; w < waves; ++w) {
          gate += red[(w * cap + j) * kMoeRedRow + n];
          up += red[(w * cap + j) * kMoeRedRow + 16 + n];
        }
        store(j, tile * 16 + n, gate, up);
      }
    }
  }
}

// A block per 32 rows of y and part of the columns of all entries, laid one behind the other; its waves share those.  A pair is two of an MFMA's 16 tokens, the two parts of
// its hidden values: as many MFMAs as with one part, for up to kMoeDownPairs pairs.  Codes are exact in bf16, dense fp16 weights are taken apart.  Parts leave their sums in the workspace, past the
// L2 (agent scope), and the last of a row tile's blocks to do so adds them in their order.
template <int ACT, int FMT, bool ASYM, int GROUP>
__global__ void __launch_bounds__(64 * kMoeMaxWaves, 4) moe_down_kernel(const MoeArgs a, int cap, int own_lds) {
  using Walk = MoeWalk<NPAMD_BF16, FMT, ASYM, 2, GROUP, ACT>;
  using S = typename Walk::S;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int x_loads = S::x_loads(2 * cap), x_bytes = x_loads * 1024;
  const MoeRoute route(lds + own_lds, a.M * a.top_k, waves, lds);
  uint8_t* const tokens = lds + waves * 2 * Walk::kPlace;
  Walk walk(lds + wave * 2 * Walk::kPlace, tokens + wave * 2 * x_bytes, x_loads, a.I, a.shift, 0, 1);
  float* const sums = reinterpret_cast<float*>(tokens + waves * 2 * x_bytes);  // [wave][M][32]
  for (int p = threadIdx.x; p < a.M * a.top_k; p += blockDim.x) route.ids[p] = a.ids[p], route.entries[p] = a.entries[p];  // those behind the last: never looked at
  if (threadIdx.x == 0) *route.n_entries = (int)a.entries[a.M * a.top_k];
  for (int o = threadIdx.x; o < waves * a.M * 32; o += blockDim.x) sums[o] = 0.f;
  __syncthreads();

  const int n0 = blockIdx.x * 32, steps = (a.I + S::kColumns - 1) / S::kColumns, all = __builtin_amdgcn_readfirstlane(*route.n_entries) * steps;
  const int shares = waves * gridDim.y, of = blockIdx.y * waves + wave;
  const int first = (int)((int64_t)all * of / shares), last = (int)((int64_t)all * (of + 1) / shares);
  int left_to_ask = last - first, ahead_entry = first / steps, ahead_step = first - ahead_entry * steps, ahead_slot = 1;
  bool ahead_new = true;
  auto request = [&](int place) __attribute__((always_inline)) {
    if (left_to_ask <= 0) return;
    --left_to_ask;
    if (ahead_new) {
      ahead_new = false;
      ahead_slot ^= 1;
      const uint32_t entry = __builtin_amdgcn_readfirstlane(route.entries[ahead_entry]);
      uint16_t* const list = route.lists + (wave * 2 + ahead_slot) * 16;
      const int n = list_pairs(a, route, entry, cap, lane, list);
      if (lane == 0) route.counts[wave * 2 + ahead_slot] = n;
      const int64_t row = (int64_t)(entry & 0xFFFF) * a.H + n0;
      walk.rows(0, a.down, a.down_scale, a.down_zero, row);
      walk.rows(1, a.down, a.down_scale, a.down_zero, row + 16);
      walk.tokens(a.h, 2 * n, [&](int j) { return (int)list[j >> 1] * 2 + (j & 1); });
    }
    walk.load(ahead_step, place);
    if (++ahead_step == steps) {
      ahead_step = 0;
      ++ahead_entry;
      ahead_new = true;
    }
  };
  request(0);
  int slot = 0, place = 0, step = first % steps;
  float* const mine = sums + wave * a.M * 32;
  for (int i = first; i < last; ++i) {
    const int count = __builtin_amdgcn_readfirstlane(route.counts[wave * 2 + slot]);
    Walk::arrived();
    request(place ^ 1);
    walk.multiply(step, place, 2 * count);
    place ^= 1;
    if (++step != steps && i != last - 1) continue;
    // the entry's tokens, each times its share: a token's place is written by one lane
    step = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * (lane >> 4) + e;
      if (j < count) {
        const int pair = route.lists[(wave * 2 + slot) * 16 + j];
        const float share = a.share[pair];
        float* const to = mine + pair / a.top_k * 32 + (lane & 15);
#pragma unroll
        for (int r = 0; r < 2; ++r) to[16 * r] = __builtin_fmaf(share, walk.acc[r][2 * e] + walk.acc[r][2 * e + 1], to[16 * r]);
      }
    }
    slot ^= 1;
    walk.clear();
  }
  __syncthreads();
  const int values = a.M * 32;
  float* const left = a.parts + (int64_t)blockIdx.x * values;
  const int64_t part_stride = (int64_t)gridDim.x * values;
  for (int o = threadIdx.x; o < values; o += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += sums[w * values + o];
    if (gridDim.y == 1) store_from_f32<ACT>(a.y, (o >> 5) * a.ldy + n0 + (o & 31), v);
    else __hip_atomic_store(left + blockIdx.y * part_stride + o, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (gridDim.y == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the part is where the others will read it
  __syncthreads();
  int* const order = route.n_entries;
  if (threadIdx.x == 0) *order = (int)__hip_atomic_fetch_add(a.done + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (*order != (int)gridDim.y - 1) return;
  for (int o = threadIdx.x; o < values; o += blockDim.x) {
    float v = 0.f;
    for (unsigned p = 0; p < gridDim.y; ++p) v += __hip_atomic_load(left + p * part_stride + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    store_from_f32<ACT>(a.y, (o >> 5) * a.ldy + n0 + (o & 31), v);
  }
}

// The down kernel's blocks: the columns are parted while all row tiles' parts are no more than compute units (row tiles alone may be).
constexpr int kMoeBlocks = 256;
int moe_max_parts(int H) { return std::max(1, kMoeBlocks / std::max(1, H / 32)); }

struct MoeSpace {
  int64_t logits, ids, share, entries, xs, h, done, parts, bytes;
  MoeSpace(int M, int E, int top_k, int H, int I) {
    int64_t at = 0;
    auto take = [&](int64_t n) {
      const int64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    logits = take((int64_t)M * E * 4);
    ids = take((int64_t)M * top_k * 2);
    share = take((int64_t)M * top_k * 4);
    entries = take(((int64_t)M * top_k + 1) * 4);
    xs = take((int64_t)M * H * 2);
    h = take((int64_t)M * top_k * 2 * I * 2);
    done = take((int64_t)H / 32 * 4);
    parts = take((int64_t)moe_max_parts(H) * M * H * 4);
    bytes = at;
  }
};

// Four waves to a block of the up kernel (us of the layer with two / four / eight: int4 4096 x 14336, one token 54 / 50 / 56; dense 2048 x 2048, four tokens 58 / 55 / 56), three
// where that many divide an item's steps better (nine steps, hidden size 2304, with four / three: int4 one token 31.2 / 30.9, four tokens 64.1 / 62.3, int8 39.2 / 39.5), and
// eight of the down kernel (four / eight: 54 / 50, 55.7 / 55.4), whose blocks split the columns (one part / two: int4 one token 57 / 50; hidden size 256, inner 13440, 14
// experts, one / eight / 16 / 32 parts 130 / 47 / 42 / 45; 384 and 1152, 12 experts 22 / 19 / 21 / 23).  From entries of five pairs on the up kernel's waves share them (each for
// itself / shared: 16 tokens int4 197 / 187, one token 50 / 53); unless that leaves compute units without a block (19 tokens through four of four, 3840 x 768, shared / each
// for itself 46 / 37).
constexpr int kMoeUpWaves = 4, kMoeDownWaves = 8, kMoeTogether = 5, kMoeWavesPerCu = 16, kMoeDownPairs = 8;

template <int ACT, int FMT, bool ASYM, int GROUP>
int launch_moe_format(const MoeArgs& a, hipStream_t st) {
  const char* what = "npamd_moe_layer";
  using S = MoeStep<FMT, ASYM>;
  constexpr int kRoom = 160 * 1024;
  // Pairs of an entry: their places in LDS keep blocks out, an expert that has more pairs is read again.  All that an MFMA takes; eight where an expert has four at the mean
  // (us with 16 / eight: 16 tokens int4 through two of eight 190 / 183, through eight of 64 88 / 70, 32 tokens through two of eight 199 / 231); four where it has one, of int8,
  // whose steps are the largest, two (with eight / four / two / one: eight tokens dense through eight of 64 129 / 112 / 112 / -; int8 through eight of 64, seven 67 / 71 / 64 / 73,
  // four 54 / 54 / 46 / 49; eight of 128, 12 tokens 92 / 100 / 87 / 98; four of 60, ten 73 / 74 / 67 / 73; one of 32, 32 tokens 138 / 121 / 114 / 140; two of eight 4096 x 14336, four
  // 201 / 201 / 203 / 230; with zero points eight of 128, 16 tokens 127 / 127 / 130 / 159).
  const int pairs = a.M * a.top_k, cap = std::min(a.M, pairs <= a.E ? (FMT == 8 ? 2 : 4) : pairs <= 4 * a.E ? 8 : 16), x_bytes = 2 * S::x_loads(cap) * 1024;
  // The down kernel's, whose pairs are two tokens each: eight, four up to a mean of two (us with four / eight: 16 tokens int4 through eight of 64 65 / 71, 24 through four of 60
  // 80 / 86, 20 through three of 32 106 / 112; 16 int8 through eight of 64 95 / 94, eight dense through four of 16 89 / 90; but at four 16 tokens int4 through two of
  // eight 197 / 186, 32 int8 through eight of 64 135 / 126, 32 dense through four of 16 137 / 117).
  const int down_cap = std::min(cap, pairs <= 2 * a.E ? 4 : kMoeDownPairs), down_x_bytes = 2 * S::x_loads(2 * down_cap) * 1024;
  const int most_entries = std::min(pairs, a.E + pairs / cap);
  const bool together = cap >= kMoeTogether && (int64_t)most_entries * (a.I / 16 / kMoeUpWaves) >= kMoeBlocks;
  auto up_own = [&](int waves) { return waves * 4 * S::kItem + (together ? x_bytes : waves * (x_bytes + cap * kMoeRedRow * 4)); };
  auto down_own = [&](int waves) { return waves * (down_x_bytes + 4 * S::kItem + a.M * 32 * 4); };
  const int up_steps = (a.H + S::kColumns - 1) / S::kColumns;
  auto idle = [&](int waves) { return (float)((up_steps + waves - 1) / waves * waves) / (float)up_steps; };
  const int up_waves = together ? kMoeUpWaves : up_steps < kMoeUpWaves ? up_steps : idle(3) * 1.1f < idle(kMoeUpWaves) ? 3 : kMoeUpWaves;
  int down_waves = kMoeDownWaves;
  while (down_own(down_waves) + MoeRoute::bytes(pairs, down_waves) > kRoom) --down_waves;
  const int up_lds = up_own(up_waves) + MoeRoute::bytes(pairs, up_waves), down_lds = down_own(down_waves) + MoeRoute::bytes(pairs, down_waves);
  static LdsLatch up_latch[2], down_latch;
  const auto up = together ? moe_up_kernel<ACT, FMT, ASYM, GROUP, true> : moe_up_kernel<ACT, FMT, ASYM, GROUP, false>;
  const auto down = moe_down_kernel<ACT, FMT, ASYM, GROUP>;
  hipError_t e = enable_dynamic_lds(up_latch[together], reinterpret_cast<const void*>(up), up_lds);
  if (e == hipSuccess) e = enable_dynamic_lds(down_latch, reinterpret_cast<const void*>(down), down_lds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "%s: cannot reserve LDS: %s", what, hipGetErrorString(e));
  if (a.M == 1) launch(moe_logits_kernel<ACT, 1, FMT == 4>, a.E, 256, 0, st, a);
  else launch(moe_logits_kernel<ACT, 4, FMT == 4>, dim3(a.E, (a.M + 3) / 4), 256, 0, st, a);
  const int64_t items = (int64_t)most_entries * (a.I / 16 / (together ? up_waves : 1));  // no more than that
  const int per_cu = std::max(1, std::min(kMoeWavesPerCu / up_waves, kRoom / up_lds));
  launch(up, (unsigned)std::min<int64_t>(items, kMoeBlocks * per_cu), 64 * up_waves, up_lds, st, a, cap, down_cap, up_own(up_waves));
  // Parts of the columns: a wave's steps, 2 us each, against 0.4 us for each part that meets the others.
  const int down_steps = std::min(pairs, a.E) * ((a.I + S::kColumns - 1) / S::kColumns);  // if every expert that can be met is
  auto down_cost = [&](int n) { return 5 * ((down_steps + n * down_waves - 1) / (n * down_waves)) + n; };
  int parts = 1;
  for (int n = 2; n <= moe_max_parts(a.H); ++n)
    if (down_cost(n) < down_cost(parts)) parts = n;
  launch(down, dim3(a.H / 32, parts), 64 * down_waves, down_lds, st, a, down_cap, down_own(down_waves));
  return check_launch(what);
}

template <int ACT, int FMT, bool ASYM>
int launch_moe_codes(const MoeArgs& a, hipStream_t st) {
  if (a.shift == 0) return launch_moe_format<ACT, FMT, ASYM, 1>(a, st);
  if (a.shift == 1) return launch_moe_format<ACT, FMT, ASYM, 2>(a, st);
  return launch_moe_format<ACT, FMT, ASYM, 4>(a, st);
}
template <int ACT>
int launch_moe(const MoeArgs& a, int nbits, hipStream_t st) {
  if (nbits == 16) return launch_moe_format<ACT, 16, false, 2>(a, st);
  if (nbits == 8) return a.gate_up_zero ? launch_moe_codes<ACT, 8, true>(a, st) : launch_moe_codes<ACT, 8, false>(a, st);
  return a.gate_up_zero ? launch_moe_codes<ACT, 4, true>(a, st) : launch_moe_codes<ACT, 4, false>(a, st);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int64_t npamd_moe_workspace_bytes(int M, int E, int top_k, int H, int I) {
  if (M < 1 || E < 1 || top_k < 1 || H < 1 || I < 1 || M > kMoeMaxTokens || E > kMoeMaxExperts || top_k > std::min(E, kMoeMaxTopK)) return 0;  // refused without any
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
                  half(down_zero_f16), y, ldx, ldy, M, E, top_k, H, I, shift, renormalize, (float*)(at + space.logits), (uint16_t*)(at + space.ids),
                  (float*)(at + space.share), (uint32_t*)(at + space.entries), (uint32_t*)(at + space.done), (float*)(at + space.parts), (uint16_t*)(at + space.xs), (uint16_t*)(at + space.h)};
  return act_dtype == NPAMD_BF16 ? launch_moe<NPAMD_BF16>(a, nbits, (hipStream_t)stream) : launch_moe<NPAMD_F16>(a, nbits, (hipStream_t)stream);
}
