// The matrix products of the linear layer for f32 operands (gemm_tile.h); a file of its own per
// storage type so that the kernels compile side by side.
#include "gemm_tile.h"

int sf_gemm_f32(const SfGemmArgs &a, int layout, int tile, hipStream_t st) {
  return sf_gemm_any<float>(a, layout, tile, st);
}
int sf_gradients_f32(const SfGemmArgs &dx, const SfGemmArgs &dw, const SfColumnSums &db, hipStream_t st) {
  return sf_gradients_go<float>(dx, dw, db, st);
}
int sf_tiny_gradients_f32(const SfGradients &g, bool direct, hipStream_t st) {
  return sf_tiny_gradients_go<float>(g, direct, st);
}
