// Products of rows and weights in 8 bits: what the kernels for few and for many rows share.
//     C[m][n] = scale_a[m] scale_w[n] sum over k of A[m][k] W[n][k]
// The sum is a whole number in 32 bits, exact and the same in whatever order it is made (K up to 131,072:
// 127 x 127 x K < 2^31); it becomes a float32 number, then the weight's
// scale follows, then the row's (rows near float32's largest number stay finite where the result is).  PAIR: W is [2, N, K], gate
// rows, then up rows, and C = unit(gate, up) (gated_unit) of the scaled sums, which are not rounded to the output's type first.
#pragma once
#include "gemm_common.h"

typedef __attribute__((ext_vector_type(4))) int i32x4;

struct Int8Args {
  const signed char* a;      // [M, row]
  const signed char* w;      // [N, row] (pair: [2 N, row])
  const float* a_scale;      // [M]
  const float* w_scale;      // [N] (pair: [2 N])
  void* c;                   // [M, N]
  int M, N, row;             // row: bytes of a row, a multiple of 256, zeros behind K
  float limit;               // pair: gated_unit's
};

// The kernel for many rows (gemm_int8_tiled.hip); whether it takes these sizes; into how many parts it would rather have K
// split, and what memory that takes (bytes of partial sums, tiles).
struct Int8Split {
  int splits, tile, tiles;
  int64_t bytes;
};
constexpr int kSplitRows = 128;
bool gemm_int8_tiled_fits(int M, int N, int row, bool pair);
Int8Split gemm_int8_split(int M, int N, int row, bool pair);
int gemm_int8_tiled(const Int8Args& a, int c_type, bool pair, int tile, int* partial, unsigned* arrivals, hipStream_t stream);
