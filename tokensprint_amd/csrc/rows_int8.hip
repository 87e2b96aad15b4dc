// Rows in 8 bits: scale = the row's largest magnitude / 127, an element the nearest whole number of scales,
// ties to even.  Alone (weights too: a row is an output channel), or behind the residual add and the RMSNorm
// whose rows go into an 8-bit product: the normed row is quantised as it is in registers, never rounded to the activation
// type or written in it.  A row with an infinity or a NaN has a scale that is neither finite, and its products
// are NaN (int8_scale in gemm_int8.h).
//
// A workgroup takes a row, eight neighbouring elements a piece: bound by memory for many rows (8,192 of 5,120 28 us, 4.5
// TB/s; with the add and the norm 87 us, 5.3 TB/s), by one trip and two meetings of the workgroup for few (3.3 us).  Codes go into rows of `row` bytes (a multiple of 256, zeros behind the
// last element), which is what the products walk in.
#include "rows_int8.h"

struct QuantRowsArgs {
  const void* x;           // [M, K]
  const void* delta;       // NORM: [M, K] of TD, or null
  const float* norm_w;     // NORM: [K]
  float* resid_out;        // NORM: x + delta [M, K], or null
  signed char* codes;      // [M, row]
  float* scales;           // [M]
  int M, K, row;
  float eps;
};

// CH pieces of eight elements a thread, all in registers; CH = 0: rows of any length and alignment, an element at a
// time, walked once for each of the sums.
template <typename T, typename TD, bool NORM, int CH>
__global__ __launch_bounds__(CH > 4 ? 512 : 1024) void quant_rows_kernel(QuantRowsArgs a) {
  __shared__ float scratch[16], sums[16];
  const int64_t m = blockIdx.x;
  const T* x = (const T*)a.x + m * a.K;
  const TD* delta = NORM && a.delta ? (const TD*)a.delta + m * a.K : nullptr;
  signed char* codes = a.codes + m * a.row;
  if constexpr (CH > 0) {
    typedef T eight __attribute__((ext_vector_type(8)));
    typedef TD eight_d __attribute__((ext_vector_type(8)));
    typedef float eight_f __attribute__((ext_vector_type(8)));
    auto at = [&](int c) { return (c * (int)blockDim.x + (int)threadIdx.x) * 8; };
    eight raw[CH];
    float v[NORM ? CH : 1][8], top = 0.f;
    if constexpr (NORM) {
      eight_d more[CH];
      eight_f w[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int e = min(at(c), a.K - 8);                  // behind the row's end its last piece again, dropped
        raw[c] = *(const eight*)(x + e);
        if (delta) more[c] = *(const eight_d*)(delta + e);
        w[c] = *(const eight_f*)(a.norm_w + e);
      }
      float sq = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const bool there = at(c) < a.K;
        eight_f sum;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[c][j] = there ? to_f32(raw[c][j]) : 0.f;
          if (delta) v[c][j] += there ? to_f32(more[c][j]) : 0.f;
          sq = fmaf(v[c][j], v[c][j], sq);
          sum[j] = v[c][j];
        }
        if (a.resid_out && there) *(eight_f*)(a.resid_out + m * a.K + at(c)) = sum;
      }
      const float rstd = rsqrtf(block_sum(sq, sums) / (float)a.K + a.eps);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[c][j] *= rstd * w[c][j];
          top = larger(top, at(c) < a.K ? fabsf(v[c][j]) : 0.f);
        }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) raw[c] = *(const eight*)(x + min(at(c), a.K - 8));
#pragma unroll
      for (int c = 0; c < CH; ++c)                          // (the last piece again changes nothing)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = larger(top, fabsf(to_f32(raw[c][j])));
    }
    const float scale = block_largest(top, scratch) / 127.f;
    const RowScale by = row_scale(scale);
    if (threadIdx.x == 0) a.scales[m] = scale;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (at(c) >= a.row) continue;
      if constexpr (!NORM) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[0][j] = to_f32(raw[c][j]);
      }
      uint2 packed = codes8(v[NORM ? c : 0], by);
      if (at(c) >= a.K) packed = make_uint2(0, 0);          // zeros behind the row's end
      *(uint2*)(codes + at(c)) = packed;
    }
  } else {
    auto value = [&](int e) {
      float y = to_f32(x[e]);
      if (NORM && delta) y += to_f32(delta[e]);
      return y;
    };
    float rstd = 1.f;
    if constexpr (NORM) {
      float sq = 0.f;
      for (int e = threadIdx.x; e < a.K; e += blockDim.x) {
        const float y = value(e);
        sq = fmaf(y, y, sq);
        if (a.resid_out) a.resid_out[m * a.K + e] = y;
      }
      rstd = rsqrtf(block_sum(sq, sums) / (float)a.K + a.eps);
    }
    auto normed = [&](int e) { return NORM ? value(e) * (rstd * a.norm_w[e]) : value(e); };
    float top = 0.f;
    for (int e = threadIdx.x; e < a.K; e += blockDim.x) top = larger(top, fabsf(normed(e)));
    const float scale = block_largest(top, scratch) / 127.f;
    const RowScale by = row_scale(scale);
    if (threadIdx.x == 0) a.scales[m] = scale;
    for (int e = threadIdx.x; e < a.row; e += blockDim.x)
      codes[e] = e < a.K && scale > 0.f ? (signed char)code8(normed(e), by) : (signed char)0;
  }
}

template <typename T, typename TD, bool NORM>
static int launch_quant_rows(const QuantRowsArgs& a, hipStream_t stream) {
  const uintptr_t used = (uintptr_t)a.x | (uintptr_t)a.delta | (uintptr_t)a.norm_w | (uintptr_t)a.resid_out;
  const int pieces = a.row / 8;
#define TS_ROWS(CH, THREADS) \
  hipLaunchKernelGGL((quant_rows_kernel<T, TD, NORM, CH>), dim3((unsigned)a.M), dim3(THREADS), 0, stream, a)
  // Few rows, and rows with a norm: a thread a piece, up to 1,024 threads (16 rows of 4,096: 3.3 us, with 256 threads 4.0;
  // 16,384 with the norm 134 us, 5.5 TB/s, and 137).  Many rows without one: 256 threads and more loads in flight
  // for each, so that a unit holds more rows between their first load and their last store (8,192 rows
  // of 5,120: 28 us, 4.5 TB/s; with 640 threads 38; with 64 31).
  const int most = NORM || a.M <= 512 ? 1024 : pieces <= 1536 ? 256 : 512;
  const int each = (pieces + most - 1) / most, threads = ((pieces + each - 1) / each + 63) / 64 * 64;
  if (a.K % 8 || (used & 15) || pieces > 4096) TS_ROWS(0, a.K < 512 ? (a.K + 63) / 64 * 64 : 512);
  else if (each == 1) TS_ROWS(1, threads);
  else if (each == 2) TS_ROWS(2, threads);
  else if constexpr (NORM) TS_ROWS(4, threads);
  else if (each == 3) TS_ROWS(3, threads);
  else if (each == 4) TS_ROWS(4, threads);
  else if (each <= 6) TS_ROWS(6, threads);
  else TS_ROWS(8, threads);
#undef TS_ROWS
  TS_CHECK_LAUNCH("quantize_rows");
  return 0;
}

// Rows as they are.
extern "C" int ts_quantize_rows(const void* x, int type, void* codes, float* scales, int M, int K, int row,
                                hipStream_t stream) {
  if (M <= 0) return 0;
  if (K <= 0 || row < K || row % 256) TS_FAIL("quantize_rows: K=%d in rows of %d bytes", K, row);
  if ((uintptr_t)codes & 15) TS_FAIL("quantize_rows: codes must be 16-byte aligned");
  QuantRowsArgs a{};
  a.x = x, a.codes = (signed char*)codes, a.scales = scales, a.M = M, a.K = K, a.row = row;
  TS_DISPATCH_TYPE(type, T, return (launch_quant_rows<T, T, false>(a, stream)));
  return 0;
}

// RMSNorm(resid + delta) in 8 bits; resid + delta into `resid_out` (null: not kept; delta null: none).
extern "C" int ts_norm_quantize_rows(const float* resid, const void* delta, int delta_type, const float* norm_w, float eps,
                                     float* resid_out, void* codes, float* scales, int M, int K, int row,
                                     hipStream_t stream) {
  if (M <= 0) return 0;
  if (K <= 0 || row < K || row % 256) TS_FAIL("norm_quantize_rows: K=%d in rows of %d bytes", K, row);
  if (!norm_w) TS_FAIL("norm_quantize_rows: no norm weight");
  if ((uintptr_t)codes & 15) TS_FAIL("norm_quantize_rows: codes must be 16-byte aligned");
  QuantRowsArgs a{resid, delta, norm_w, resid_out, (signed char*)codes, scales, M, K, row, eps};
  TS_DISPATCH_TYPE(delta_type, TD, return (launch_quant_rows<float, TD, true>(a, stream)));
  return 0;
}
