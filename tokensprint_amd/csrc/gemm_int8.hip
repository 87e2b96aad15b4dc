// Products in 8 bits for few rows, where streaming the weight once is the whole cost, and the entry point of all.
//
// A workgroup owns 16 rows of W (16 of each half with PAIR) and up to 64 rows of A; its waves share K out. Both operands go
// from memory into the layout of v_mfma_i32_16x16x64_i8: a lane takes 64 contiguous bytes of its row
// an iteration, so four lanes cover 256 and a wave 4 KB of W; the k that a register slot stands for is permuted the
// same way in both, which a sum of whole numbers does not notice.
#include "gemm_int8.h"

// MT: 16-row tiles of A; NW: waves along K.
template <int MT, int NW, typename TC, bool PAIR>
__global__ __launch_bounds__(NW * kWave) void gemm_int8_kernel(Int8Args a) {
  constexpr int HALVES = PAIR ? 2 : 1;
  __shared__ i32x4 red[NW - 1][HALVES][MT][kWave];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (MT * 16);
  const signed char* w = a.w + (int64_t)min(n0 + r, a.N - 1) * a.row + g * 64;
  const signed char* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = a.a + (int64_t)min(m0 + t * 16 + r, a.M - 1) * a.row + g * 64;
  i32x4 acc[HALVES][MT];
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[h][t] = i32x4{0, 0, 0, 0};
#pragma unroll 2
  for (int k = wave * 256; k < a.row; k += NW * 256) {
    i32x4 wv[HALVES][4];
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int s = 0; s < 4; ++s) wv[h][s] = *(const i32x4*)(w + (int64_t)h * a.N * a.row + k + s * 16);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      i32x4 xv[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) xv[s] = *(const i32x4*)(x[t] + k + s * 16);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          acc[h][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[h][s], xv[s], acc[h][t], 0, 0, 0);
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int t = 0; t < MT; ++t) red[wave - 1][h][t][lane] = acc[h][t];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int o = 0; o < NW - 1; ++o)
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[h][t] += red[o][h][t][lane];
  // lane holds the sums of columns n0 + 4 g + i of row m0 + 16 t + r
  const int n = n0 + g * 4;
  if (n >= a.N) return;
  float scale[HALVES][4];
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[h][i] = a.w_scale[h * a.N + min(n + i, a.N - 1)];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = m0 + t * 16 + r;
    if (m >= a.M) continue;
    const float row = a.a_scale[m];
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = (float)acc[0][t][i] * scale[0][i] * row;
      if constexpr (PAIR) v[i] = gated_unit(v[i], (float)acc[1][t][i] * scale[1][i] * row, a.limit);
    }
    store4<TC>((TC*)a.c + (int64_t)m * a.N + n, v, a.N - n);
  }
}

template <typename TC, bool PAIR>
static int launch_int8(const Int8Args& a, hipStream_t stream) {
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  const dim3 grid((a.N + 15) / 16, (a.M + mt * 16 - 1) / (mt * 16));
  if (grid.y > 65535) TS_FAIL("gemm_int8: M=%d rows of %d bytes", a.M, a.row);
#define TS_INT8(MT) hipLaunchKernelGGL((gemm_int8_kernel<MT, 4, TC, PAIR>), grid, dim3(4 * kWave), 0, stream, a)
  if (mt == 1) TS_INT8(1);
  else if (mt == 2) TS_INT8(2);
  else TS_INT8(4);
#undef TS_INT8
  TS_CHECK_LAUNCH("gemm_int8");
  return 0;
}

// `tile`: 0 lets the sizes choose the kernel; 1 to 8 name a tile of the kernel for many rows, 9 the one for few (for
// measuring; the result is the same to the bit).
extern "C" int ts_gemm_int8(const void* x, const float* a_scale, const void* w, const float* w_scale, void* c,
                            int c_type, int M, int N, int row, int pair, float limit, int tile, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (row <= 0 || row % 256 || row > 131072) TS_FAIL("gemm_int8: rows of %d bytes", row);
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)c) & 15) TS_FAIL("gemm_int8: operands must be 16-byte aligned");
  if (c_type != TS_F32 && c_type != TS_BF16) TS_FAIL("gemm_int8: output type %d", c_type);
  if (tile < 0 || tile > 9) TS_FAIL("gemm_int8: no tile %d", tile);
  const Int8Args a{(const signed char*)x, (const signed char*)w, a_scale, w_scale, c, M, N, row, limit};
  const bool many = gemm_int8_tiled_fits(M, N, row, pair != 0);
  if (tile > 0 && tile < 9 && !many) TS_FAIL("gemm_int8: M=%d N=%d rows of %d bytes not taken in tiles", M, N, row);
  if (tile == 0 ? M > 64 && many : tile < 9) return gemm_int8_tiled(a, c_type, pair != 0, tile, stream);
  if (pair) return c_type == TS_BF16 ? launch_int8<bf16_t, true>(a, stream) : launch_int8<float, true>(a, stream);
  return c_type == TS_BF16 ? launch_int8<bf16_t, false>(a, stream) : launch_int8<float, false>(a, stream);
}

extern "C" int ts_quantize_rows(const void* x, int type, void* codes, float* scales, int M, int K, int row,
                                hipStream_t stream);
extern "C" int ts_norm_quantize_rows(const float* resid, const void* delta, int delta_type, const float* norm_w, float eps,
                                     float* resid_out, void* codes, float* scales, int M, int K, int row,
                                     hipStream_t stream);

// Rows into 8 bits and their product.  `norm_w` null: x as it is; else x is the float32 stream, `delta` (or null) is
// added to it, the sum goes into `resid_out` and the rows are normed.  `rows`: M (row + 4) bytes of scratch memory.
extern "C" int ts_linear_int8(const void* x, int x_type, const void* delta, int delta_type, const float* norm_w, float eps,
                              float* resid_out, void* rows, const void* w, const float* w_scale, void* c, int c_type,
                              int M, int N, int K, int row, int pair, float limit, hipStream_t stream) {
  if (M <= 0) return 0;
  float* scales = (float*)((char*)rows + (int64_t)M * row);
  const int rc = norm_w ? ts_norm_quantize_rows((const float*)x, delta, delta_type, norm_w, eps, resid_out, rows, scales, M,
                                                K, row, stream)
                        : ts_quantize_rows(x, x_type, rows, scales, M, K, row, stream);
  return rc ? rc : ts_gemm_int8(rows, scales, w, w_scale, c, c_type, M, N, row, pair, limit, 0, stream);
}
