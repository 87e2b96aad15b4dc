// Rows in 8 bits: what the kernel that makes them alone (rows_int8.hip) and the one that makes them on the way into a
// product (gemm_int8.hip) share.
#pragma once
#include "common.h"

// The larger, or NaN if either is.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ float block_largest(float v, float* scratch) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v = larger(v, __shfl_xor(v, o, kWave));
  const int waves = blockDim.x / kWave;
  if (waves == 1) return v;
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < waves; ++w) v = larger(v, scratch[w]);
  return v;
}

// What turns a row's elements into numbers: about 1 / scale; of a scale so small that this would not be a float32
// number, scale and elements times 2^64 first.
struct RowScale {
  float scale, inv, lift;
  bool plain;              // the fast way is exact enough (see codes8)
};
__device__ __forceinline__ RowScale row_scale(float scale) {
  RowScale r;
  r.lift = scale < 0x1p-100f ? 0x1p64f : 1.f;
  r.scale = scale * r.lift;
  r.inv = scale > 0.f ? 1.f / r.scale : 0.f;
  r.plain = scale >= 0x1p-100f && scale < __builtin_inff();
  return r;
}
__device__ __forceinline__ int code8(float x, const RowScale& r) {
  return (int)fminf(fmaxf(nearest_whole(x * r.lift, r.scale, r.inv), -127.f), 127.f);
}

// Eight numbers in eight bytes.  The quotient by the product with 1 / scale is within 127 x 2^-23 of the right one (two
// roundings), and its sum with 1.5 x 2^23 is the nearest whole number in the lowest byte; where one of the wave's
// quotients is so near to a border between two numbers that this might be the other one (or the scale is not an
// ordinary number), nearest_whole decides for all: 4 % of the pieces of ordinary rows.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], const RowScale& r) {
  constexpr float kMagic = 12582912.f;
  unsigned b[8];
  float off = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = fmaf(v[j], r.inv, kMagic);
    off = fmaxf(off, fabsf(fmaf(v[j], r.inv, kMagic - t)));
    b[j] = __float_as_uint(t);
  }
  if (__builtin_amdgcn_ballot_w64(off > 0.49996f || !r.plain) != 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = r.scale > 0.f ? (unsigned)code8(v[j], r) : 0u;
  }
  auto four = [](unsigned x, unsigned y, unsigned z, unsigned w) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400u), __builtin_amdgcn_perm(y, x, 0x0c0c0400u), 0x05040100u);
  };
  return make_uint2(four(b[0], b[1], b[2], b[3]), four(b[4], b[5], b[6], b[7]));
}
