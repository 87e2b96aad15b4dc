// Products of rows and weights in 8 bits: what the kernels for few and for many rows share.
//     C[m][n] = scale_a[m] scale_w[n] sum over k of A[m][k] W[n][k]
// The sum is a whole number in 32 bits, exact and the same in whatever order it is made (K up to 131,072:
// 127 x 127 x K < 2^31); it becomes a float32 number, then the weight's
// scale follows, then the row's (rows near float32's largest number stay finite where the result is).  PAIR: W is [2, N, K], gate
// rows, then up rows, and C = unit(gate, up) (Int8Unit) of the scaled sums, which are not rounded to the output's type first.
#pragma once
#include "gemm_common.h"

typedef __attribute__((ext_vector_type(4))) int i32x4;

// A scale as products take it: of a row with an infinity (an infinite scale, and numbers that say nothing) NaN, so that
// what it gives is no number behind a clamp either.
__device__ __forceinline__ float int8_scale(float s) { return s + (s - s); }

// The gated unit of all these products: gated_unit's three forms in one, by the hardware's exp2 and reciprocal (an ulp each),
// the same instructions whichever kernel a row's product comes from, so that its bits do not depend on the rows beside it.
// (The clamps change nothing without a limit, and NaN stays NaN.)
struct Int8Unit {
  float top, lift, slope, cubic;
  __device__ __forceinline__ explicit Int8Unit(float limit) {
    const bool clamped = limit > 0.f, gelu = limit < 0.f;
    top = clamped ? limit : INFINITY, lift = clamped ? 1.f : 0.f;
    // the weight exp2(g (slope + cubic g^2)): of the sigmoid, or for gelu_tanh(g) = g sigmoid(2 sqrt(2 / pi) (g + 0.044715 g^3))
    slope = (clamped ? -1.702f : gelu ? -2.f * 0.79788456080286536f : -1.f) * 1.44269504f;
    cubic = gelu ? 0.044715f * slope : 0.f;
  }
  __device__ __forceinline__ float operator()(float gate, float up) const {
    const float g = __builtin_elementwise_minimum(gate, top);
    const float u = __builtin_elementwise_minimum(__builtin_elementwise_maximum(up, -top), top) + lift;
    // (from 10^4 on the weight is 0 or 1; a gate of 2e19 has no square, and 0 times that is no number)
    const float e = __builtin_amdgcn_fmed3f(g, -1e4f, 1e4f);
    return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(e * fmaf(cubic, e * e, slope))) * u;
  }
};

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
