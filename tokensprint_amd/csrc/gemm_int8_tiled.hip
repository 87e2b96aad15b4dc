// Products in 8 bits for many rows: the LDS-tiled kernel's 8-bit form (gemm_tiled_kernel.h).
#include "gemm_tiled_kernel.h"

bool gemm_int8_tiled_fits(int M, int N, int row, bool pair) {
  const int64_t rows_w = pair ? 2 * (int64_t)N : N;
  return M > 0 && N > 0 && row >= 512 && row % 128 == 0 && (int64_t)M * row < (1ll << 32) && rows_w * row < (1ll << 32);
}

int gemm_int8_tiled(const Int8Args& a, int c_type, bool pair, int tile, hipStream_t stream) {
  TiledInt8Args g{};
  g.a = (const bf16_t*)a.a, g.w = (const bf16_t*)a.w, g.c = a.c;
  g.M = a.M, g.N = a.N, g.K = a.row / 2;
  g.a_scale = a.a_scale, g.w_scale = a.w_scale, g.limit = a.limit;
  if (pair)
    return c_type == TS_BF16 ? choose_tile<true, bf16_t, kInt8>(g, tile, stream) : choose_tile<true, float, kInt8>(g, tile, stream);
  return c_type == TS_BF16 ? choose_tile<false, bf16_t, kInt8>(g, tile, stream) : choose_tile<false, float, kInt8>(g, tile, stream);
}
