// The wide tiles of the dense product whose operands lie with the contracted index as their rows (wide_gemm.hpp): W, or W and x.  A turned operand has 64, 128 or 256 columns to a tile.
// Bound by the matrix pipes, busy 72 to 78 % of all cycles: 4096 x 4096 x 28672 (W turned) 677 to 756 us, 28672 x 4096 x 4096 (both) 714 to 806 with the clock, 1.2 to 1.4 PFLOP/s.
#include "wide_gemm.hpp"

namespace npamd {

namespace {

template <int ACT, bool XK>
int launch_turned_on(const DenseShape& s, int tile, hipStream_t st) {
  switch (tile) {  // numbered as in launch_wide_on
    case 1: return launch_wide_tile<ACT, WideTile<2, 2, 2, 2, 6, 4>, kWidePlain, XK, true>(s, st);    // 64 x 64
    case 2: return launch_wide_tile<ACT, WideTile<2, 2, 2, 4, 5, 12>, kWidePlain, XK, true>(s, st);   // 64 x 128
    case 3: return launch_wide_tile<ACT, WideTile<2, 2, 4, 4, 4, 24>, kWidePlain, XK, true>(s, st);   // 128 x 128
    case 5: return launch_wide_tile<ACT, WideTile<4, 2, 4, 4, 3, 24>, kWidePlain, XK, true>(s, st);   // 256 x 128
    default: return launch_wide_tile<ACT, WideTile<2, 4, 8, 4, 2, 24>, kWidePlain, XK, true>(s, st);  // 256 x 256
  }
}

}  // namespace

int launch_wide_turned(const DenseShape& s, int act, int tile, bool x_too, hipStream_t st) {
  if (x_too) return act == NPAMD_BF16 ? launch_turned_on<NPAMD_BF16, true>(s, tile, st) : launch_turned_on<NPAMD_F16, true>(s, tile, st);
  return act == NPAMD_BF16 ? launch_turned_on<NPAMD_BF16, false>(s, tile, st) : launch_turned_on<NPAMD_F16, false>(s, tile, st);
}

}  // namespace npamd
