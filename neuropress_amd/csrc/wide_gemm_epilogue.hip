// The wide tiles of the dense product with an epilogue (wide_gemm.hpp).
#include "wide_gemm.hpp"

namespace npamd {

int launch_wide_epilogue(const DenseShape& s, int act, int tile, hipStream_t st) {
  return act == NPAMD_BF16 ? launch_wide_on<NPAMD_BF16, true>(s, tile, st) : launch_wide_on<NPAMD_F16, true>(s, tile, st);
}

}  // namespace npamd
