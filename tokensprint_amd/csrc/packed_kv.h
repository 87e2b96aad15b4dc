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
// multiplies (steps are brought up to stand high in float16's range first, so neither does it overflow nor do small
// weights lose bits: PackedLift in packed_attention_kernel.h).  For that a
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
// zeros), and this lane's codes, in the order that `place` gives: element j's in bits 4 place(j) on.  A quotient by the
// estimate of 1 / step is off by less than 2^-17 (two roundings of at most 15), so a code is the whole number next to it (which adding 1.5 x 2^23 leaves in
// the lowest bits) unless that is nearly half a step away; where one of a wavefront's is, all are worked out with what
// is left over (exactly: ties to even), and where one is no finite number, they are made one.
template <typename PLACE>
__device__ __forceinline__ PackGroup pack_eight(float (&v)[8], unsigned& word, PLACE place) {
  constexpr float kMost = 3.4028234663852886e38f, kMagic = 12582912.f;
  // (the neighbour's, the other pair's, then the other four's: lane moves, not trips through LDS)
  auto from = [](float x, auto how) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(how)::value, 0xf, 0xf, true));
  };
  float lo, hi;
  auto range = [&]() {                                         // NaN if an element is
    lo = hi = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      lo = __builtin_elementwise_minimum(__builtin_elementwise_minimum(lo, v[j]), v[j + 1]);
      hi = __builtin_elementwise_maximum(__builtin_elementwise_maximum(hi, v[j]), v[j + 1]);
    }
    auto both = [&](auto how) {
      lo = __builtin_elementwise_minimum(lo, from(lo, how)), hi = __builtin_elementwise_maximum(hi, from(hi, how));
    };
    both(std::integral_constant<int, 0xB1>{});
    both(std::integral_constant<int, 0x4E>{});
    both(std::integral_constant<int, 0x141>{});
  };
  range();
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(hi - lo <= kMost)) != 0, 0)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] == v[j] ? fminf(fmaxf(v[j], -kMost), kMost) : 0.f;
    range();
  }
  PackGroup p;
  // (hi - lo) / 15, rounded as a division rounds it (checked for every significand); of an infinite range NaN, so the most
  const float wide = hi - lo, about = wide * (1.f / 15.f);
  p.step = (_Float16)fminf(fmaf(fmaf(-15.f, about, wide), 1.f / 15.f, about), 65504.f);
  const float step = (float)p.step, inv = step > 0.f ? __builtin_amdgcn_rcpf(step) : 0.f;
  p.zero = rintf(-lo * inv);
  float off = fabsf(fmaf(-lo, inv, -p.zero)), c[8];
  p.zero = fminf(p.zero, 15.f);                                // (steps of few bits)
  const float one = kMagic + p.zero;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    c[j] = fmaf(v[j], inv, one);
    off = fmaxf(off, fabsf(fmaf(v[j], inv, one - c[j])));
  }
  if (__builtin_amdgcn_ballot_w64(off > 0.49999f || step >= 65504.f) != 0) {
    p.zero = nearest_whole(-lo, step, inv);
    p.zero = step > 0.f ? fminf(p.zero, 15.f) : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      c[j] = kMagic + (step > 0.f ? __builtin_amdgcn_fmed3f(nearest_whole(v[j], step, inv) + p.zero, 0.f, 15.f) : 0.f);
  }
  word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    word = (__float_as_uint(__builtin_amdgcn_fmed3f(c[j], kMagic, kMagic + 15.f)) << (4 * place(j))) + word;
    word -= __float_as_uint(kMagic) << (4 * place(j));         // (one constant for all eight)
  }
  return p;
}

// Eight codes of each of eight lanes that make up eight words of values between them, turned round: code e of lane q
// becomes code q of lane e, of the lanes' numbers (token's bit 1, sub's bit 1, token's bit 0), lane = 16 token + sub: the
// lowest bits of the words of packed_kv.h's order.  Its own inverse.
__device__ __forceinline__ unsigned pack_turned_round(unsigned x, int lane) {
  auto stage = [&](unsigned other, int bit, unsigned low, int shift) {
    const unsigned keep = bit ? ~low : low;
    return (x & keep) | (__builtin_rotateright32(other, bit ? shift : 32 - shift) & ~keep);
  };
  x = stage(__shfl_xor(x, 32, kWave), lane >> 5 & 1, 0x0F0F0F0Fu, 4);
  x = stage(__builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, true), lane >> 1 & 1, 0x00FF00FFu, 8);
  return stage(__shfl_xor(x, 16, kWave), lane >> 4 & 1, 0x0000FFFFu, 16);
}

// How far a word of keys, and one of values, is turned.
constexpr int kPackTurnK = 3, kPackTurnV = 6;
template <int BY>
__device__ __forceinline__ unsigned pack_turned(unsigned word) { return __builtin_rotateleft32(word, BY); }
template <int BY>
__device__ __forceinline__ unsigned pack_unturned(unsigned word) { return __builtin_rotateright32(word, BY); }
