// The wide tiles of the dense product (wide_gemm.hpp).
#include "wide_gemm.hpp"

namespace npamd {

int launch_wide(const DenseShape& s, int act, int tile, hipStream_t st) {
  return act == NPAMD_BF16 ? launch_wide_on<NPAMD_BF16, false>(s, tile, st) : launch_wide_on<NPAMD_F16, false>(s, tile, st);
}

}  // namespace npamd
