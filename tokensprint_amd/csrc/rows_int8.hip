// Rows in 8 bits: scale = the row's largest magnitude / 127, an element the nearest whole number of scales,
// ties to even.  Alone (weights too: a row is an output channel), or behind the residual add and the RMSNorm
// whose rows go into an 8-bit product: the normed row is quantised as it is in registers, never rounded to the activation
// type or written in it.  A row with an infinity or a NaN has a scale that is neither finite, so its products
// are not numbers either.
//
// A workgroup takes a row, eight neighbouring elements a piece: bound by memory for many rows, by one trip and
// two meetings of the workgroup for few.  Codes go into rows of `row` bytes (a multiple of 256, zeros behind the
// last element), which is what the products walk in.
#include "common.h"

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

// The larger, or NaN if either is.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <int N>
__device__ __forceinline__ float block_largest(float v, float* scratch) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v = larger(v, __shfl_xor(v, o, kWave));
  const int waves = (blockDim.x + kWave - 1) / kWave;
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < waves; ++w) v = larger(v, scratch[w]);
  return v;
}

__device__ __forceinline__ int code8(float x, float scale, float inv) {
  return (int)fminf(fmaxf(nearest_whole(x, scale, inv), -127.f), 127.f);
}

// CH pieces of eight elements a thread, all in registers; CH = 0: rows of any length and alignment, an element at a
// time, walked once for each of the sums.
template <typename T, typename TD, bool NORM, int CH>
__global__ __launch_bounds__(1024) void quant_rows_kernel(QuantRowsArgs a) {
  __shared__ float scratch[16], sums[16];
  const int64_t m = blockIdx.x;
  const T* x = (const T*)a.x + m * a.K;
  const TD* delta = NORM && a.delta ? (const TD*)a.delta + m * a.K : nullptr;
  signed char* codes = a.codes + m * a.row;
  if constexpr (CH > 0) {
    typedef T eight __attribute__((ext_vector_type(8)));
    typedef TD eight_d __attribute__((ext_vector_type(8)));
    typedef float eight_f __attribute__((ext_vector_type(8)));
    float v[CH][8];
    eight raw[CH];
    eight_d more[CH];
    eight_f w[CH];
    auto at = [&](int c) { return (c * (int)blockDim.x + (int)threadIdx.x) * 8; };
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int e = min(at(c), a.K - 8);                    // behind the row's end its last piece again, dropped
      raw[c] = *(const eight*)(x + e);
      if (NORM && delta) more[c] = *(const eight_d*)(delta + e);
      if (NORM) w[c] = *(const eight_f*)(a.norm_w + e);
    }
    float sq = 0.f, top = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const bool there = at(c) < a.K;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[c][j] = there ? to_f32(raw[c][j]) : 0.f;
        if (NORM && delta) v[c][j] += there ? to_f32(more[c][j]) : 0.f;
        if (NORM) sq = fmaf(v[c][j], v[c][j], sq);
      }
      if (NORM && a.resid_out && there) {
        eight_f out;
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = v[c][j];
        *(eight_f*)(a.resid_out + m * a.K + at(c)) = out;
      }
    }
    if constexpr (NORM) {
      const float rstd = rsqrtf(block_sum(sq, sums) / (float)a.K + a.eps);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] *= rstd * w[c][j];
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = larger(top, at(c) < a.K ? fabsf(v[c][j]) : 0.f);
    const float scale = block_largest<0>(top, scratch) / 127.f, inv = scale > 0.f ? 1.f / scale : 0.f;
    if (threadIdx.x == 0) a.scales[m] = scale;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (at(c) >= a.row) continue;
      uint64_t packed = 0;                                  // zeros behind the row's end
      if (at(c) < a.K && scale > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) packed |= (uint64_t)(unsigned char)code8(v[c][j], scale, inv) << (8 * j);
      }
      *(uint64_t*)(codes + at(c)) = packed;
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
    const float scale = block_largest<0>(top, scratch) / 127.f, inv = scale > 0.f ? 1.f / scale : 0.f;
    if (threadIdx.x == 0) a.scales[m] = scale;
    for (int e = threadIdx.x; e < a.row; e += blockDim.x)
      codes[e] = e < a.K && scale > 0.f ? (signed char)code8(normed(e), scale, inv) : (signed char)0;
  }
}

template <typename T, typename TD, bool NORM>
static int launch_quant_rows(const QuantRowsArgs& a, hipStream_t stream) {
  const uintptr_t used = (uintptr_t)a.x | (uintptr_t)a.delta | (uintptr_t)a.norm_w | (uintptr_t)a.resid_out;
  const int pieces = a.row / 8;
#define TS_ROWS(CH, THREADS) \
  hipLaunchKernelGGL((quant_rows_kernel<T, TD, NORM, CH>), dim3((unsigned)a.M), dim3(THREADS), 0, stream, a)
  // rows of up to 8,192 elements one piece a thread; longer ones more
  if (a.K % 8 || (used & 15) || pieces > 4096) TS_ROWS(0, 512);
  else if (pieces <= 1024) TS_ROWS(1, (pieces + 63) / 64 * 64);
  else if (pieces <= 2048) TS_ROWS(2, 1024);
  else TS_ROWS(4, 1024);
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
