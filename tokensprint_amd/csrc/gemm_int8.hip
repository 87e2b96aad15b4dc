// Products in 8 bits for few rows, where streaming the weight once is the whole cost, and the entry point of all.
//
// A workgroup owns 16 rows of W (16 of each half with PAIR) and 16 rows of A; its eight waves share K out.  Both operands
// go from memory into the layout of v_mfma_i32_16x16x64_i8: of a row, four lanes take 64 contiguous bytes a load, and
// four loads 256.  (A lane taking 64 contiguous bytes over four loads, which the products' order of k would allow,
// touched four times as many pieces of memory a load: 16 rows of [2 x 12288, 4096] took 29 us against 20.)
// W of 16.8 MB that no cache holds takes 6 us for 1 row, 8 for 16 (2.8 and 2.1 TB/s); 50 MB as [4096, 12288] 13 and 18;
// 100 MB as [2 x 12288, 4096] 24 and 28 (4.2 and 3.6 TB/s).  Four waves lose 10 % in the first two.
#include "gemm_int8.h"
#include "rows_int8.h"

constexpr int kWavesAlongK = 8;

// What the waves summed along K, added up and out: lane 16 g + r has columns n0 + 4 g + i of row m (`row`: its scale).
template <typename TC, bool PAIR, int HALVES>
__device__ __forceinline__ void finish_few(const Int8Args& a, i32x4 (&acc)[HALVES], i32x4 (&red)[kWavesAlongK - 1][HALVES][kWave],
                                           int wave, int lane, int n0, int m, const float* scales) {
  constexpr int NW = kWavesAlongK;
  if (wave > 0) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h) red[wave - 1][h][lane] = acc[h];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int o = 0; o < NW - 1; ++o)
#pragma unroll
    for (int h = 0; h < HALVES; ++h) acc[h] += red[o][h][lane];
  const int n = n0 + lane / 16 * 4;
  if (n >= a.N || m >= a.M) return;
  const float row = int8_scale(scales[m]);
  const Int8Unit unit(a.limit);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int column = min(n + i, a.N - 1);
    v[i] = (float)acc[0][i] * int8_scale(a.w_scale[column]) * row;
    if constexpr (PAIR) v[i] = unit(v[i], (float)acc[1][i] * int8_scale(a.w_scale[a.N + column]) * row);
  }
  store4<TC>((TC*)a.c + (int64_t)m * a.N + n, v, a.N - n);
}

template <typename TC, bool PAIR>
__global__ __launch_bounds__(kWavesAlongK* kWave) void gemm_int8_kernel(Int8Args a) {
  constexpr int HALVES = PAIR ? 2 : 1, NW = kWavesAlongK;
  __shared__ i32x4 red[NW - 1][HALVES][kWave];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16;
  const int n0 = blockIdx.x * 16, m = blockIdx.y * 16 + r;
  const signed char* w = a.w + (int64_t)min(n0 + r, a.N - 1) * a.row + g * 16;
  const signed char* x = a.a + (int64_t)min(m, a.M - 1) * a.row + g * 16;
  i32x4 acc[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) acc[h] = i32x4{0, 0, 0, 0};
  for (int k = wave * 256; k < a.row; k += NW * 256) {
    i32x4 wv[HALVES][4], xv[4];
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int s = 0; s < 4; ++s) wv[h][s] = *(const i32x4*)(w + (int64_t)h * a.N * a.row + k + s * 64);
#pragma unroll
    for (int s = 0; s < 4; ++s) xv[s] = *(const i32x4*)(x + k + s * 64);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int h = 0; h < HALVES; ++h) acc[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[h][s], xv[s], acc[h], 0, 0, 0);
  }
  finish_few<TC, PAIR, HALVES>(a, acc, red, wave, lane, n0, m, a.a_scale);
}

// The same for one row that is made on the way: every workgroup turns the row into numbers itself, in LDS, its first two
// pieces of W already sent for.  The row's sums are made as quant_rows_kernel makes them, so the numbers are the same to
// the bit.  One row with [4096, 4096] from memory 7.4 us, as two kernels 10.0 (with the norm 7.9 and 10.1), with [24576,
// 4096] 23.5 and 27.0; from 1,536 workgroups on, whose rows take turns, the row costs more than a launch ([150000,
// 1024] 50 and 39, with the norm 75 and 38), and so it does for two rows and more (2 rows of [4096, 4096]: 11.1 and 10.3).
struct RowInt8Args {
  Int8Args g;
  const void* x;             // [K]
  const void* delta;         // NORM: [K] of TD, or null
  const float* norm_w;       // NORM: [K]
  float* resid_out;          // NORM: x + delta [K], or null
  int K;
  float eps;
};
constexpr int kRowLongest = 8192;            // elements: a piece of eight for each of 1,024 threads there, two a thread here

template <typename T, typename TD, bool NORM, typename TC, bool PAIR>
__global__ __launch_bounds__(kWavesAlongK* kWave) void row_gemm_int8_kernel(RowInt8Args args) {
  const Int8Args& a = args.g;
  constexpr int HALVES = PAIR ? 2 : 1, NW = kWavesAlongK, GROUPS = kRowLongest / 8 / kWave, CH = GROUPS / NW;
  typedef T eight __attribute__((ext_vector_type(8)));
  typedef TD eight_d __attribute__((ext_vector_type(8)));
  typedef float eight_f __attribute__((ext_vector_type(8)));
  __shared__ i32x4 red[NW - 1][HALVES][kWave];
  __shared__ __attribute__((aligned(16))) signed char codes[kRowLongest];
  __shared__ float sums[GROUPS], tops[NW], row_scales[1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16, n0 = blockIdx.x * 16;
  const int K = args.K;
  auto at = [&](int c) { return ((c * NW + wave) * kWave + lane) * 8; };
  float v[CH][8];
  {
    eight raw[CH];
    eight_d more[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      raw[c] = *(const eight*)((const T*)args.x + min(at(c), K - 8));
      if (NORM && args.delta) more[c] = *(const eight_d*)((const TD*)args.delta + min(at(c), K - 8));
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[c][j] = at(c) < K ? to_f32(raw[c][j]) : 0.f;
        if (NORM && args.delta) v[c][j] += at(c) < K ? to_f32(more[c][j]) : 0.f;
      }
  }
  const signed char* w = a.w + (int64_t)min(n0 + r, a.N - 1) * a.row + g * 16;
  auto load = [&](int k, i32x4 (&wv)[HALVES][4]) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int s = 0; s < 4; ++s) wv[h][s] = *(const i32x4*)(w + (int64_t)h * a.N * a.row + k + s * 64);
  };
  const int k0 = wave * 256, k1 = k0 + NW * 256;
  i32x4 w0[HALVES][4], w1[HALVES][4];
  if (k0 < a.row) load(k0, w0);
  if (k1 < a.row) load(k1, w1);
  if constexpr (NORM) {
    eight_f nw[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) nw[c] = *(const eight_f*)(args.norm_w + min(at(c), K - 8));
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float sq = 0.f;
      eight_f sum;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(v[c][j], v[c][j], sq), sum[j] = v[c][j];
      if (args.resid_out && blockIdx.x == 0 && at(c) < K) *(eight_f*)(args.resid_out + at(c)) = sum;
      sq = wave_sum(sq);
      if (lane == 0) sums[c * NW + wave] = sq;
    }
    __syncthreads();
    float total = 0.f;
    for (int i = 0; i * kWave * 8 < K; ++i) total += sums[i];
    const float rstd = rsqrtf(total / (float)K + args.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] *= rstd * nw[c][j];
  }
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = larger(top, at(c) < K ? fabsf(v[c][j]) : 0.f);
  const float scale = block_largest(top, tops) / 127.f;
  const RowScale by = row_scale(scale);
  if (threadIdx.x == 0) row_scales[0] = scale;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (at(c) >= a.row) continue;
    uint2 packed = codes8(v[c], by);
    if (at(c) >= K) packed = make_uint2(0, 0);
    *(uint2*)(codes + at(c)) = packed;
  }
  __syncthreads();
  i32x4 acc[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) acc[h] = i32x4{0, 0, 0, 0};
  auto products = [&](int k, const i32x4 (&wv)[HALVES][4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const i32x4 xv = *(const i32x4*)(codes + k + s * 64 + g * 16);
#pragma unroll
      for (int h = 0; h < HALVES; ++h) acc[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[h][s], xv, acc[h], 0, 0, 0);
    }
  };
  if (k0 < a.row) products(k0, w0);
  if (k1 < a.row) products(k1, w1);
  for (int k = k1 + NW * 256; k < a.row; k += NW * 256) {
    load(k, w0);
    products(k, w0);
  }
  finish_few<TC, PAIR, HALVES>(a, acc, red, wave, lane, n0, r, row_scales);
}

template <typename TC, bool PAIR>
static int launch_int8(const Int8Args& a, hipStream_t stream) {
  const dim3 grid((a.N + 15) / 16, (a.M + 15) / 16);
  if (grid.y > 65535) TS_FAIL("gemm_int8: M=%d rows of %d bytes", a.M, a.row);
  hipLaunchKernelGGL((gemm_int8_kernel<TC, PAIR>), grid, dim3(kWavesAlongK * kWave), 0, stream, a);
  TS_CHECK_LAUNCH("gemm_int8");
  return 0;
}

// Tiles from 5 rows on where the kernel above would be more than two workgroups a unit, of which every one reads its
// rows of A for 16 rows of W alone (W [24576, 4096]: 1 row 24 us here, 26 in tiles; 16 rows 30 and 27.  [12288, 4096]:
// 8 rows 15 and 15, 16 rows 17 and 15.  [4096, 4096]: 16 rows 8 and 10), or from 17 rows more than one (tiles split
// along K: [4096, 4096] 32 rows 10.5 and 8.8; [4096, 12288] 26.6 and 17.0; [1024, 4096] 64 rows 6.0 and 6.7), or
// where rows are very long ([5120, 25600], 16 rows 56 and 35).
static bool takes_few(int M, int N, int row, bool pair) {
  const int64_t workgroups = ((pair ? 2ll * N : N) + 15) / 16 * ((M + 15) / 16);
  return M <= 4 || (row <= 16384 && workgroups <= (M <= 16 ? 512 : 256));
}

// `tile`: 0 lets the sizes choose the kernel; 1 to 8 name a tile of the kernel for many rows, 9 the one for few (for
// measuring; the result is the same to the bit).  `partial`: as much memory as ts_gemm_int8_split says, `arrivals` as many zeros;
// null: K is not split.
extern "C" int ts_gemm_int8(const void* x, const float* a_scale, const void* w, const float* w_scale, void* c,
                            int c_type, int M, int N, int row, int pair, float limit, int tile, void* partial,
                            unsigned* arrivals, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (row <= 0 || row % 256 || row > 131072) TS_FAIL("gemm_int8: rows of %d bytes", row);
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)c) & 15) TS_FAIL("gemm_int8: operands must be 16-byte aligned");
  if (c_type != TS_F32 && c_type != TS_BF16) TS_FAIL("gemm_int8: output type %d", c_type);
  if (tile < 0 || tile > 9) TS_FAIL("gemm_int8: no tile %d", tile);
  const Int8Args a{(const signed char*)x, (const signed char*)w, a_scale, w_scale, c, M, N, row, limit};
  const bool many = gemm_int8_tiled_fits(M, N, row, pair != 0);
  if (tile > 0 && tile < 9 && !many) TS_FAIL("gemm_int8: M=%d N=%d rows of %d bytes not taken in tiles", M, N, row);
  const bool few = takes_few(M, N, row, pair != 0);
  if (tile == 0 ? many && !few : tile < 9) return gemm_int8_tiled(a, c_type, pair != 0, tile, (int*)partial, arrivals, stream);
  if (pair) return c_type == TS_BF16 ? launch_int8<bf16_t, true>(a, stream) : launch_int8<float, true>(a, stream);
  return c_type == TS_BF16 ? launch_int8<bf16_t, false>(a, stream) : launch_int8<float, false>(a, stream);
}

extern "C" int ts_quantize_rows(const void* x, int type, void* codes, float* scales, int M, int K, int row,
                                hipStream_t stream);
extern "C" int ts_norm_quantize_rows(const float* resid, const void* delta, int delta_type, const float* norm_w, float eps,
                                     float* resid_out, void* codes, float* scales, int M, int K, int row,
                                     hipStream_t stream);

// Bytes of partial sums with which a product of these sizes is split along K, or 0, and the tiles that count themselves in.
extern "C" int64_t ts_gemm_int8_split(int M, int N, int row, int pair, int* tiles) {
  *tiles = 0;
  if (M <= 0 || N <= 0 || row <= 0 || takes_few(M, N, row, pair != 0)) return 0;
  const Int8Split s = gemm_int8_split(M, N, row, pair != 0);
  *tiles = s.tiles;
  return s.bytes;
}

// Rows into 8 bits and their product.  `norm_w` null: x as it is; else x is the float32 stream, `delta` (or null) is
// added to it, the sum goes into `resid_out` and the rows are normed.  `rows`: M (row + 4) bytes of scratch memory.
extern "C" int ts_linear_int8(const void* x, int x_type, const void* delta, int delta_type, const float* norm_w, float eps,
                              float* resid_out, void* rows, const void* w, const float* w_scale, void* c, int c_type,
                              int M, int N, int K, int row, int pair, float limit, void* partial, unsigned* arrivals,
                              hipStream_t stream) {
  if (M <= 0) return 0;
  const uintptr_t used = (uintptr_t)x | (uintptr_t)delta | (uintptr_t)norm_w | (uintptr_t)resid_out | (uintptr_t)w | (uintptr_t)c;
  if (M == 1 && N > 0 && (pair ? 2ll * N : N) <= 24576 && K >= 8 && K % 8 == 0 && row >= K && row % 256 == 0 && row <= kRowLongest &&
      used % 16 == 0 && (c_type == TS_F32 || c_type == TS_BF16)) {
    const RowInt8Args a{{nullptr, (const signed char*)w, nullptr, w_scale, c, M, N, row, limit}, x, delta, norm_w, resid_out, K, eps};
#define TS_ROW(T, TD, NORM, TC, PAIR) \
  hipLaunchKernelGGL((row_gemm_int8_kernel<T, TD, NORM, TC, PAIR>), dim3((N + 15) / 16), dim3(kWavesAlongK * kWave), 0, stream, a)
#define TS_ROW_OF(T, TD, NORM) \
  if (c_type == TS_BF16) { if (pair) TS_ROW(T, TD, NORM, bf16_t, true); else TS_ROW(T, TD, NORM, bf16_t, false); } \
  else { if (pair) TS_ROW(T, TD, NORM, float, true); else TS_ROW(T, TD, NORM, float, false); }
    if (norm_w) { TS_DISPATCH_TYPE(delta_type, TD, TS_ROW_OF(float, TD, true)) }
    else { TS_DISPATCH_TYPE(x_type, T, TS_ROW_OF(T, T, false)) }
#undef TS_ROW_OF
#undef TS_ROW
    TS_CHECK_LAUNCH("row_gemm_int8");
    return 0;
  }
  float* scales = (float*)((char*)rows + (int64_t)M * row);
  const int rc = norm_w ? ts_norm_quantize_rows((const float*)x, delta, delta_type, norm_w, eps, resid_out, rows, scales, M,
                                                K, row, stream)
                        : ts_quantize_rows(x, x_type, rows, scales, M, K, row, stream);
  return rc ? rc : ts_gemm_int8(rows, scales, w, w_scale, c, c_type, M, N, row, pair, limit, 0, partial, arrivals, stream);
}
