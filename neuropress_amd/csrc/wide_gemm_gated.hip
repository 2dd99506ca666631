// The wide tiles of the gated product (wide_gemm.hpp): those with an even number of column groups to a wave.  Bound by the matrix pipes, busy
// 76 % of all cycles: 4096 x 28672 x 4096 bf16 with SiLU 705 to 713 us, 1.36 PFLOP/s.
#include "wide_gemm.hpp"

namespace npamd {

namespace {

template <int ACT>
int launch_gated_on(const DenseShape& s, int tile, hipStream_t st) {
  switch (tile) {  // numbered as in launch_wide_on
    case 1: return launch_wide_tile<ACT, WideTile<2, 2, 2, 2, 6, 4>, kWideGated>(s, st);    // 64 x 64
    case 2: return launch_wide_tile<ACT, WideTile<2, 2, 2, 4, 5, 12>, kWideGated>(s, st);   // 64 x 128
    case 3: return launch_wide_tile<ACT, WideTile<2, 2, 4, 4, 4, 24>, kWideGated>(s, st);   // 128 x 128
    case 5: return launch_wide_tile<ACT, WideTile<4, 2, 4, 4, 3, 24>, kWideGated>(s, st);   // 256 x 128
    case 6: return launch_wide_tile<ACT, WideTile<4, 2, 3, 4, 3, 20>, kWideGated>(s, st);   // 192 x 128
    case 7: return launch_wide_tile<ACT, WideTile<2, 2, 3, 4, 4, 20>, kWideGated>(s, st);   // 96 x 128
    case 8: return launch_wide_tile<ACT, WideTile<2, 4, 5, 4, 3, 24>, kWideGated>(s, st);   // 160 x 256
    case 9: return launch_wide_tile<ACT, WideTile<2, 4, 6, 4, 2, 20>, kWideGated>(s, st);   // 192 x 256
    default: return launch_wide_tile<ACT, WideTile<2, 4, 8, 4, 2, 24>, kWideGated>(s, st);  // 256 x 256
  }
}

}  // namespace

int launch_wide_gated(const DenseShape& s, int act, int tile, hipStream_t st) {
  return act == NPAMD_BF16 ? launch_gated_on<NPAMD_BF16>(s, tile, st) : launch_gated_on<NPAMD_F16>(s, tile, st);
}

}  // namespace npamd
