// Products in 8 bits for many rows: the LDS-tiled kernel's 8-bit form (gemm_tiled_kernel.h).
#include "gemm_tiled_kernel.h"

bool gemm_int8_tiled_fits(int M, int N, int row, bool pair) {
  const int64_t rows_w = pair ? 2 * (int64_t)N : N;
  return M > 0 && N > 0 && row >= 512 && row % 128 == 0 && (int64_t)M * row < (1ll << 32) && rows_w * row < (1ll << 32);
}

// Where tiles of 64 rows leave units without one, K is split until every unit has a part, of eight steps of 128 bytes at
// least: 64 columns a tile from rows of 8,192 bytes on, else 32.  The parts' sums are whole numbers, so their order
// is of no consequence.  64 rows, W in memory: [4096, 12288] 27 us whole (128 tiles of 32 columns), 18 in four parts of 64
// columns, 20 in two of 32; [4096, 8192] 19, 14 and 15; [4096, 4096] 11, 10.6 and 9.2; in twice as many parts as
// there are units 21, 17 and 10.  [6144, 4096] has 192 tiles and is not split: 12.0, in two parts 12.7.
Int8Split gemm_int8_split(int M, int N, int row, bool pair) {
  Int8Split s{1, 0, 0, 0};
  if (M > kSplitRows || !gemm_int8_tiled_fits(M, N, row, pair)) return s;
  const int64_t cols = pair ? 2 * (int64_t)N : N;
  const int steps = row / 128, units = compute_units(), rows = (M + 63) / 64;
  const int bn = steps >= 64 && (cols + 63) / 64 * rows * 8 >= units ? 64 : 32;
  const int64_t tiles = (cols + bn - 1) / bn * rows;
  if (tiles * 2 > units) return s;
  int splits = units / (int)tiles;
  if (splits > steps / 8) splits = steps / 8;
  if (splits > 8) splits = 8;
  while (splits > 1 && steps - (steps + splits - 1) / splits * (splits - 1) < 4) --splits;    // a tile's ring of buffers
  if (splits < 2) return s;
  return Int8Split{splits, bn == 32 ? 8 : 7, (int)tiles, tiles * splits * 64 * bn * 4};
}

int gemm_int8_tiled(const Int8Args& a, int c_type, bool pair, int tile, int* partial, unsigned* arrivals, hipStream_t stream) {
  TiledInt8Args g{};
  g.a = (const bf16_t*)a.a, g.w = (const bf16_t*)a.w, g.c = a.c;
  g.M = a.M, g.N = a.N, g.K = a.row / 2;
  g.a_scale = a.a_scale, g.w_scale = a.w_scale, g.limit = a.limit;
  g.splits = 1;
  if (tile == 0 && partial) {
    const Int8Split s = gemm_int8_split(a.M, a.N, a.row, pair);
    if (s.splits > 1) g.splits = s.splits, g.partial = partial, g.arrivals = arrivals, tile = s.tile;
  }
  if (pair)
    return c_type == TS_BF16 ? choose_tile<true, bf16_t, kInt8>(g, tile, stream) : choose_tile<true, float, kInt8>(g, tile, stream);
  return c_type == TS_BF16 ? choose_tile<false, bf16_t, kInt8>(g, tile, stream) : choose_tile<false, float, kInt8>(g, tile, stream);
}
