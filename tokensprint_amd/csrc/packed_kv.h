// Keys and values held in 4 bits: what a group is, and where its bits stand in a page.
//
// A group is up to 64 neighbouring elements of one head of one token (the head's last group may be
// shorter).  With lo the smaller of zero and its smallest element and hi the larger of zero and its largest:
//     step  = (hi - lo) / 15 in float16 (at most its largest number)
//     zero  = -lo / step, code = x / step + zero, both to the nearest whole number, ties to even, 0 .. 15
//     value = step (code - zero)
// A step of 0 (all elements zero, or too small for float16) gives codes of 0; NaN is held as 0, an
// infinity as the largest float32: what a cache holds is always finite, so a key that a mask hides
// (weight 0) adds nothing whatever it was.  The zero is a whole number, not a float like the step, so that a
// weight p of the softmax need be rounded once for a key's group: p step enters the products with codes and
// with the zero alike, and the rounding's error is one of the value, not of the distance to a corner
// of the group's range (with a bfloat16 corner and p rounded for it apart, twice the error of bfloat16's own
// rounding of the result).
//
// A block is 16 tokens of a page and one key/value head.  Its bytes lie as the wavefront of the
// attention kernels wants them (lane = 16 g + r): one load of 4 NB bytes a lane, NB = slices of 32 elements,
// for all codes of the block's keys, and one for its values':
//   keys    codes  [g][token r][NB] words: elements 32 b + 8 g + j of token r
//           scale  [g][G]{ step [4], bias [4] } of tokens 4 g + i (as the score product leaves the tokens): the step
//                  and -(16 + zero), all float16
//   values  codes  [g][r][NB] words: elements 32 b + r and 32 b + 16 + r of tokens 4 g + i
//           scale  the same of the values
// G: groups of a head rounded up to a power of two.  128 elements: 1,152 bytes for 16 keys, 16 values the same
// (bfloat16: 4,096), 4.5 bits an element.
//
// A code c becomes the bfloat16 number 16 + c by putting its bits behind the leading bit of 16, so a word
// gives eight operands in seven instructions: (word >> 4 i) & 0x00780078 | 0x41804180; values the same in float16 (0x03c003c0,
// 0x4c004c00), because a weight times a step is rounded to float16, an eighth of bfloat16's error, in the instruction that
// multiplies (weights are at most 1 and steps float16 numbers: nothing overflows).  For that a
// word of keys is kept turned left by three bits, one of values by six.  Code p of a word (before turning: bits 4 p .. 4 p + 3) is
// element j = 2 p of keys for p < 4, 2 (p - 4) + 1 else; of values, token i of the first element for p = i / 2 + 4
// (i % 2), of the second 2 further.
#pragma once
#include <type_traits>

#include "common.h"

constexpr int kPackGroup = 64;     // elements
constexpr int kPackTokens = 16;    // tokens of a block

__host__ __device__ constexpr int pack_slices(int hd) { return (hd + 31) / 32; }
__host__ __device__ constexpr int pack_groups(int hd) {     // rounded up to a power of two
  return hd <= 64 ? 1 : hd <= 128 ? 2 : 4;
}
__host__ __device__ constexpr int pack_block_bytes(int hd) {
  return 256 * pack_slices(hd) + 64 * pack_groups(hd);
}
// Where a block's scales begin.
__host__ __device__ constexpr int pack_codes_bytes(int hd) { return 256 * pack_slices(hd); }

// 1 if a cache of 4 bits is built for these sizes.
inline bool pack_fits(int hd, int page_size) {
  return hd >= 16 && hd <= 256 && hd % 16 == 0 && page_size >= kPackTokens && (page_size & (page_size - 1)) == 0;
}

// Byte at which a token's block of a head begins.
__device__ __forceinline__ int64_t pack_block(int page, int nkv, int kvh, int page_size, int slot, int bytes) {
  return (((int64_t)page * nkv + kvh) * (page_size / kPackTokens) + slot / kPackTokens) * bytes;
}

struct PackGroup {
  _Float16 step;
  float zero;
};

// The group of the eight lanes that hold 64 elements between them, eight each (`v`; elements that are not there are
// zeros), and this lane's codes.  A quotient by the estimate of 1 / step is off by less than 2^-18, so a code is the whole
// number next to it unless that is nearly half a step away; where one of a wavefront's is, all are worked out with what is
// left over (exactly: ties to even), and where one is no finite number, they are made one.
__device__ __forceinline__ PackGroup pack_eight(float (&v)[8], unsigned (&code)[8]) {
  constexpr float kMost = 3.4028234663852886e38f;
  float none = 0.f;                                            // NaN if an element is not finite
#pragma unroll
  for (int j = 0; j < 8; ++j) none = fmaf(v[j], 0.f, none);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(none != none) != 0, 0)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] == v[j] ? fminf(fmaxf(v[j], -kMost), kMost) : 0.f;
  }
  float lo = fminf(fminf(v[0], v[1]), 0.f), hi = fmaxf(fmaxf(v[0], v[1]), 0.f);
#pragma unroll
  for (int j = 2; j < 8; j += 2) {
    lo = fminf(fminf(lo, v[j]), v[j + 1]);
    hi = fmaxf(fmaxf(hi, v[j]), v[j + 1]);
  }
  // (the neighbour's, the other pair's, then the other four's: lane moves, not trips through LDS)
  auto from = [](float x, auto how) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(how)::value, 0xf, 0xf, true));
  };
  lo = fminf(lo, from(lo, std::integral_constant<int, 0xB1>{})), hi = fmaxf(hi, from(hi, std::integral_constant<int, 0xB1>{}));
  lo = fminf(lo, from(lo, std::integral_constant<int, 0x4E>{})), hi = fmaxf(hi, from(hi, std::integral_constant<int, 0x4E>{}));
  lo = fminf(lo, from(lo, std::integral_constant<int, 0x141>{})), hi = fmaxf(hi, from(hi, std::integral_constant<int, 0x141>{}));
  PackGroup p;
  p.step = (_Float16)fminf((hi - lo) / 15.f, 65504.f);
  const float step = (float)p.step, inv = step > 0.f ? __builtin_amdgcn_rcpf(step) : 0.f;
  float c[8], off;
  p.zero = rintf(-lo * inv);
  off = fabsf(fmaf(-lo, inv, -p.zero));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = v[j] * inv;
    c[j] = rintf(x);
    off = fmaxf(off, fabsf(x - c[j]));
  }
  if (__builtin_amdgcn_ballot_w64(off > 0.4999f || step >= 65504.f) != 0) {
    p.zero = nearest_whole(-lo, step, inv);
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = nearest_whole(v[j], step, inv);
  }
  p.zero = step > 0.f ? fminf(p.zero, 15.f) : 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) code[j] = (unsigned)__builtin_amdgcn_fmed3f(c[j] + p.zero, 0.f, 15.f);
  return p;
}

// How far a word of keys, and one of values, is turned.
constexpr int kPackTurnK = 3, kPackTurnV = 6;
template <int BY>
__device__ __forceinline__ unsigned pack_turned(unsigned word) { return __builtin_rotateleft32(word, BY); }
template <int BY>
__device__ __forceinline__ unsigned pack_unturned(unsigned word) { return __builtin_rotateright32(word, BY); }
