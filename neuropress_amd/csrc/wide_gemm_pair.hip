// Two products with turned operands (wide_gemm.hpp) in one launch: x W with W turned and x^T W with both turned, on tiles of one size.  Neither waits for the other, so the blocks of
// the one that comes second take the compute units that the last round of the other leaves empty,
// and sums over strips of rows, which are a few us of latency, have a place next to them.
#include "strip_sums.hpp"
#include "wide_gemm.hpp"

namespace npamd {

namespace {

// The sums' blocks lie behind the products', of which `blocks`, a whole number for each die, are those of whichever comes first.
template <int ACT, class T>
__global__ void __launch_bounds__(T::kThreads, T::kThreads == 256 ? 2 : 1)
wide_gemm_pair_kernel(const DenseShape one, const DenseShape both, const StripSums sums, int blocks, int all_blocks, int both_first) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  if ((int)blockIdx.x >= all_blocks) return add_strips<ACT, T::kWaves>(sums, (int)blockIdx.x - all_blocks, reinterpret_cast<float*>(lds));
  const bool first = (int)blockIdx.x < blocks;
  const int block = first ? blockIdx.x : (int)blockIdx.x - blocks;
  if (first != (both_first != 0)) wide_gemm_block<ACT, T, kWidePlain, false, true>(one, block);
  else wide_gemm_block<ACT, T, kWidePlain, true, true>(both, block);
}

template <int ACT, class T>
int launch_pair_tile(DenseShape one, DenseShape both, const StripSums& sums, bool both_first, hipStream_t st) {
  const int64_t first = count_units<T, kWidePlain>(one), second = count_units<T, kWidePlain>(both);
  const int64_t extra = strip_blocks(sums);
  if (first + second + extra > 0x7FFFFFFF) return fail(NPAMD_ERR_UNSUPPORTED, "npamd_dense_gemm: too many tiles");
  static LdsLatch latch;
  const auto kernel = wide_gemm_pair_kernel<ACT, T>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), T::kLds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "npamd_dense_gemm: cannot reserve %d bytes of LDS: %s", T::kLds, hipGetErrorString(e));
  launch(kernel, (unsigned)(first + second + extra), T::kThreads, T::kLds, st, one, both, sums, (int)(both_first ? second : first), (int)(first + second), (int)both_first);
  return check_launch("npamd_dense_gemm");
}

template <int ACT>
int launch_pair_on(const DenseShape& one, const DenseShape& both, const StripSums& sums, int tile, bool both_first, hipStream_t st) {
  switch (tile) {  // numbered as in launch_wide_on
    case 1: return launch_pair_tile<ACT, WideTile<2, 2, 2, 2, 6, 4>>(one, both, sums, both_first, st);    // 64 x 64
    case 2: return launch_pair_tile<ACT, WideTile<2, 2, 2, 4, 5, 12>>(one, both, sums, both_first, st);   // 64 x 128
    case 3: return launch_pair_tile<ACT, WideTile<2, 2, 4, 4, 4, 24>>(one, both, sums, both_first, st);   // 128 x 128
    case 5: return launch_pair_tile<ACT, WideTile<4, 2, 4, 4, 3, 24>>(one, both, sums, both_first, st);   // 256 x 128
    default: return launch_pair_tile<ACT, WideTile<2, 4, 8, 4, 2, 24>>(one, both, sums, both_first, st);  // 256 x 256
  }
}

}  // namespace

int launch_wide_pair(const DenseShape& one, const DenseShape& both, const StripSums& sums, int act, int tile, bool both_first, hipStream_t st) {
  return act == NPAMD_BF16 ? launch_pair_on<NPAMD_BF16>(one, both, sums, tile, both_first, st) : launch_pair_on<NPAMD_F16>(one, both, sums, tile, both_first, st);
}

}  // namespace npamd
