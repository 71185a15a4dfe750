// The matrix products of the linear layer for f16 operands (gemm_tile.h); a file of its own per
// storage type so that the kernels compile side by side.
#include "gemm_tile.h"

int sf_gemm_f16(const SfGemmArgs &a, int layout, int tile, hipStream_t st) {
  return sf_gemm_any<_Float16>(a, layout, tile, st);
}
int sf_gradients_f16(const SfGemmArgs &dx, const SfGemmArgs &dw, const SfColumnSums &db, hipStream_t st) {
  return sf_gradients_go<_Float16>(dx, dw, db, st);
}
int sf_tiny_gradients_f16(const SfGradients &g, bool direct, hipStream_t st) {
  return sf_tiny_gradients_go<_Float16>(g, direct, st);
}
