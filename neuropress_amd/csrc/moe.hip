// A mixture-of-experts layer for a few tokens:
//   logits = x router^T,  p = softmax(logits) over all experts,  the top_k largest (ties to the lower index), divided by their sum on request
//   y = sum over them of p_e down_e(silu(gate_e(x)) * up_e(x))
// Expert weights are dense or group-quantized codes, w = (q - zero) scale, which is not rounded.  What is rounded to the activation type on the way is
// silu(gate) * up, the operand of the second product: sums and p stay in f32 up to the store of y.
#include "activation.hpp"
#include "common.hpp"

using namespace npamd;

namespace {

constexpr int kMoeMaxTokens = NPAMD_GEMV_MAX_M, kMoeMaxExperts = 512, kMoeMaxTopK = 16;

struct MoeArgs {
  const void *x, *router;
  const uint8_t *gate_up, *down;
  const uint16_t *gate_up_scale, *gate_up_zero, *down_scale, *down_zero;
  void* y;
  int64_t ldx, ldy;
  int M, E, top_k, H, I, nbits, group, renormalize;
  int32_t* ids;  // [M][top_k]
  float* share;  // [M][top_k]
  uint16_t* h;   // [M][top_k][I]
};

// A block per token: a wave per expert and turn, then the first wave picks.
template <int ACT>
__global__ void __launch_bounds__(256) moe_router_kernel(const MoeArgs a) {
  __shared__ float logits[kMoeMaxExperts];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = blockIdx.x;
  for (int e = wave; e < a.E; e += 4) {
    float v = 0.f;
    for (int k = lane; k < a.H; k += 64) v = __builtin_fmaf(load_as_f32<ACT>(a.x, m * a.ldx + k), load_as_f32<ACT>(a.router, (int64_t)e * a.H + k), v);
    v = wave_reduce_sum(v);
    if (lane == 0) logits[e] = v;
  }
  __syncthreads();
  if (wave) return;
  constexpr int kPer = kMoeMaxExperts / 64;
  float v[kPer];
  float most = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    v[i] = lane + 64 * i < a.E ? logits[lane + 64 * i] : -INFINITY;
    most = fmaxf(most, v[i]);
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 64 * i < a.E) sum += expf(v[i] - most);
  sum = wave_reduce_sum(sum);
  uint32_t taken = 0;
  float mine = 0.f, total = 0.f;
  int id = 0;
  for (int t = 0; t < a.top_k; ++t) {
    // the largest of what is left, NaN above all: an order of (value, -index) as one 64-bit number
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
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
    const float p = expf(logits[e] - most) / sum;
    total += p;
    if (lane == t) mine = p, id = e;
  }
  if (lane < a.top_k) {
    a.ids[m * a.top_k + lane] = id;
    a.share[m * a.top_k + lane] = a.renormalize ? mine / total : mine;
  }
}

// Weight (row, k) of an expert whose rows start at row 0.
template <int ACT>
__device__ __forceinline__ float moe_weight(const uint8_t* w, const uint16_t* scale, const uint16_t* zero, int64_t row, int k, int K, int nbits, int group) {
  if (nbits == 16) return load_as_f32<ACT>(w, row * K + k);
  const int64_t at = row * K + k, g = row * (K / group) + k / group;
  const int q = nbits == 8 ? w[at] : (w[at >> 1] >> (4 * (k & 1))) & 15;
  return ((float)q - (zero ? f16_bits_to_f32(zero[g]) : (float)(1 << (nbits - 1)))) * f16_bits_to_f32(scale[g]);
}

// A wave per value of silu(gate) * up of a (token, expert) pair.
template <int ACT>
__global__ void __launch_bounds__(256) moe_up_kernel(const MoeArgs a) {
  const int lane = threadIdx.x & 63, i = blockIdx.x * 4 + (threadIdx.x >> 6), pair = blockIdx.y, m = pair / a.top_k;
  if (i >= a.I) return;
  const int64_t row = (int64_t)a.ids[pair] * 2 * a.I + i;
  float gate = 0.f, up = 0.f;
  for (int k = lane; k < a.H; k += 64) {
    const float v = load_as_f32<ACT>(a.x, m * a.ldx + k);
    gate = __builtin_fmaf(v, moe_weight<ACT>(a.gate_up, a.gate_up_scale, a.gate_up_zero, row, k, a.H, a.nbits, a.group), gate);
    up = __builtin_fmaf(v, moe_weight<ACT>(a.gate_up, a.gate_up_scale, a.gate_up_zero, row + a.I, k, a.H, a.nbits, a.group), up);
  }
  gate = wave_reduce_sum(gate);
  up = wave_reduce_sum(up);
  if (lane == 0) store_from_f32<ACT>(a.h, (int64_t)pair * a.I + i, silu_f32(gate) * up);
}

// A wave per output of a token.
template <int ACT>
__global__ void __launch_bounds__(256) moe_down_kernel(const MoeArgs a) {
  const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6), m = blockIdx.y;
  if (n >= a.H) return;
  float y = 0.f;
  for (int t = 0; t < a.top_k; ++t) {
    const int pair = m * a.top_k + t;
    const int64_t row = (int64_t)a.ids[pair] * a.H + n;
    float v = 0.f;
    for (int k = lane; k < a.I; k += 64)
      v = __builtin_fmaf(load_as_f32<ACT>(a.h, (int64_t)pair * a.I + k), moe_weight<ACT>(a.down, a.down_scale, a.down_zero, row, k, a.I, a.nbits, a.group), v);
    y = __builtin_fmaf(a.share[pair], wave_reduce_sum(v), y);
  }
  if (lane == 0) store_from_f32<ACT>(a.y, m * a.ldy + n, y);
}

struct MoeSpace {
  int64_t ids, share, h, bytes;
  MoeSpace(int M, int top_k, int I) {
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    ids = 0;
    share = up((int64_t)M * top_k * 4);
    h = share + up((int64_t)M * top_k * 4);
    bytes = h + up((int64_t)M * top_k * I * 2);
  }
};

template <int ACT>
int launch_moe(const MoeArgs& a, hipStream_t st) {
  launch(moe_router_kernel<ACT>, a.M, 256, 0, st, a);
  launch(moe_up_kernel<ACT>, dim3((a.I + 3) / 4, a.M * a.top_k), 256, 0, st, a);
  launch(moe_down_kernel<ACT>, dim3((a.H + 3) / 4, a.M), 256, 0, st, a);
  return check_launch("npamd_moe_layer");
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int64_t npamd_moe_workspace_bytes(int M, int E, int top_k, int H, int I) {
  if (M < 1 || E < 1 || top_k < 1 || H < 1 || I < 1) return 0;
  return MoeSpace(M, top_k, I).bytes;
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
  NPAMD_REQUIRE(ldx >= H && ldy >= H && ldx % 8 == 0, "%s: bad row stride", what);
  if (M == 0) return NPAMD_OK;
  NPAMD_REQUIRE(x && router && gate_up && down && y, "%s: null pointer", what);
  NPAMD_REQUIRE(aligned16(x) && aligned16(router) && aligned16(gate_up) && aligned16(down), "%s: x, router and weights have to lie at 16-byte addresses", what);
  const MoeSpace space(M, top_k, I);
  NPAMD_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= space.bytes, "%s: needs %lld bytes of 16-byte aligned workspace", what, (long long)space.bytes);
  auto* at = (uint8_t*)workspace;
  const bool codes = nbits != 16;
  auto half = [&](const void* p) { return codes ? (const uint16_t*)p : nullptr; };
  const MoeArgs a{x, router, (const uint8_t*)gate_up, (const uint8_t*)down, half(gate_up_scale_f16), half(gate_up_zero_f16), half(down_scale_f16),
                  half(down_zero_f16), y, ldx, ldy, M, E, top_k, H, I, nbits, codes ? group_size : 1, renormalize,
                  (int32_t*)(at + space.ids), (float*)(at + space.share), (uint16_t*)(at + space.h)};
  return act_dtype == NPAMD_BF16 ? launch_moe<NPAMD_BF16>(a, (hipStream_t)stream) : launch_moe<NPAMD_F16>(a, (hipStream_t)stream);
}
