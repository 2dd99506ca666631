// Two products with turned operands (wide_gemm.hpp) in one launch: x W with W turned and x^T W with both turned, on tiles of one size.  Neither waits for the other, so the blocks of
// the one that comes second take the compute units that the last round of the other leaves empty.
#include "wide_gemm.hpp"

namespace npamd {

namespace {

// `blocks`, a whole number for each die, are those of whichever comes first.
template <int ACT, class T>
__global__ void __launch_bounds__(T::kThreads, T::kThreads == 256 ? 2 : 1)
wide_gemm_pair_kernel(const DenseShape one, const DenseShape both, int blocks, int both_first) {
  const bool first = (int)blockIdx.x < blocks;
  const int block = first ? blockIdx.x : (int)blockIdx.x - blocks;
  if (first != (both_first != 0)) wide_gemm_block<ACT, T, kWidePlain, false, true>(one, block);
  else wide_gemm_block<ACT, T, kWidePlain, true, true>(both, block);
}

template <int ACT, class T>
int launch_pair_tile(DenseShape one, DenseShape both, bool both_first, hipStream_t st) {
  const int64_t first = count_units<T, kWidePlain>(one), second = count_units<T, kWidePlain>(both);
  if (first + second > 0x7FFFFFFF) return fail(NPAMD_ERR_UNSUPPORTED, "npamd_dense_gemm: too many tiles");
  static LdsLatch latch;
  const auto kernel = wide_gemm_pair_kernel<ACT, T>;
  const hipError_t e = enable_dynamic_lds(latch, reinterpret_cast<const void*>(kernel), T::kLds);
  if (e != hipSuccess) return fail(NPAMD_ERR_LAUNCH, "npamd_dense_gemm: cannot reserve %d bytes of LDS: %s", T::kLds, hipGetErrorString(e));
  launch(kernel, (unsigned)(first + second), T::kThreads, T::kLds, st, one, both, (int)(both_first ? second : first), (int)both_first);
  return check_launch("npamd_dense_gemm");
}

template <int ACT>
int launch_pair_on(const DenseShape& one, const DenseShape& both, int tile, bool both_first, hipStream_t st) {
  switch (tile) {  // numbered as in launch_wide_on
    case 1: return launch_pair_tile<ACT, WideTile<2, 2, 2, 2, 6, 4>>(one, both, both_first, st);    // 64 x 64
    case 2: return launch_pair_tile<ACT, WideTile<2, 2, 2, 4, 5, 12>>(one, both, both_first, st);   // 64 x 128
    case 3: return launch_pair_tile<ACT, WideTile<2, 2, 4, 4, 4, 24>>(one, both, both_first, st);   // 128 x 128
    case 5: return launch_pair_tile<ACT, WideTile<4, 2, 4, 4, 3, 24>>(one, both, both_first, st);   // 256 x 128
    default: return launch_pair_tile<ACT, WideTile<2, 4, 8, 4, 2, 24>>(one, both, both_first, st);  // 256 x 256
  }
}

}  // namespace

int launch_wide_pair(const DenseShape& one, const DenseShape& both, int act, int tile, bool both_first, hipStream_t st) {
  return act == NPAMD_BF16 ? launch_pair_on<NPAMD_BF16>(one, both, tile, both_first, st) : launch_pair_on<NPAMD_F16>(one, both, tile, both_first, st);
}

}  // namespace npamd
