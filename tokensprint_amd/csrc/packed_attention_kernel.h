// Paged attention over keys and values of 4 bits (packed_kv.h) on the matrix cores, as a template whose forms
// compile in translation units of their own.
//
// As over a wider cache (attention_core.h) a wavefront owns 16 query rows and takes 32 keys at a time,
//     S^T = K Q^T,    O^T = V^T P^T         (v_mfma_f32_16x16x32_bf16),
// a lane's scores being in place its part of the second product's operand.  Here the operands of K and V are
// codes, turned into the numbers 16 + c, which are exact, and steps stand outside the products:
//     q . k  =  sum over groups of  step (q . (16 + c) - (16 + zero) sum(q))
//     o      =  sum over keys of    (p step) (16 + c) - (p step) (16 + zero)
// Sums of q over a group are float32 numbers of a query row, that is of a lane, and start the group's product as
// -(16 + zero) sum(q); p step is rounded to float16 once and meets codes and -(16 + zero) (a product with the same numbers in
// every row) alike, so what its rounding costs is in proportion to the value.
// Float16 holds 11 bits from 2^-14 on only, and a key far below the row's largest score, or values far below 1, would
// lose them (of 4,000 keys 12 below one that has no value itself, with values of 0.02, a tenth of the result, while the
// row's sum of weights keeps them).  So steps are brought up first, by the power of two that puts the largest of the
// wavefront's keys so far below 2^15 (PackedLift): p step has all its bits from 2^-28 of that on, a
// weight of 4e-9 where steps are alike.  Three instructions more for 32 keys than without.
// A wavefront dequantises nothing: seven instructions make a word of eight codes operands, a score costs two
// multiplications a group and a weight one.
//
// WIDE (float32 activations): the whole numbers c - zero instead, so that nothing cancels but what does in exact
// arithmetic either (with 16 + c the sums of values are of up to 31 steps where the result is of a tenth of one, and were
// 2.7e-6 off where float32 sums are 3.5e-7), against q and p step in two float16 parts of 11 bits each.  A query row is
// scaled by a power of two first, to stand high in float16's range; the second part of p step counts 2,048 times in sums of
// its own.  (Three bfloat16 parts hold 24 bits, but whole numbers in bfloat16 are three more instructions for two: 26 us for 24
// requests of up to 1,024 keys of 64, most of it instructions met for the first time.)
#pragma once
#include "attention_core.h"
#include "packed_kv.h"

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

struct PackedArgs {
  AttentionArgs base;        // k_pages, v_pages: blocks
  const int* tiles;          // [num_tiles, 3]: batch entry, first flat token, tokens in tile; or null: tile = entry = token
  float* partial_o;          // [workgroups, 2, 16, 32 NB]
  float* partial_ml;         // [workgroups, 2, 16, 2]
  unsigned* arrivals;        // [items] zeros: the last workgroup of an item merges its parts and leaves a zero
  int num_tiles;
  int rows_per_token;        // query heads of a tile per token: min(group, 16)
  int head_blocks;           // ceil(group / 16)
  int workgroups;            // that share all items' keys out; 0: a workgroup per item
};

template <int NB>
struct PackedBlock {
  static constexpr int G = pack_groups(NB * 32);
  unsigned k[2][NB], v[2][NB];
  unsigned ks[2], vs[2];           // word r % (4 G) of the steps and biases of tokens 4 g + i
  unsigned kz[2][G];               // WIDE: the bias of token r (a word of its own: halves would go through LDS)
  int page[2];                     // below 0: no keys there (the context ends, or a window has let go)
};

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// Eight codes as the numbers 16 + c: codes 0 and 4, 1 and 5, 2 and 6, 3 and 7 of a word of keys (bfloat16) or of
// values (float16).
template <bool VALUES>
__device__ __forceinline__ void packed_codes(unsigned word, unsigned (&out)[4]) {
  // (one of the two constants in a vector register, one in a scalar: `and` and `or` are one instruction then)
  unsigned bits = VALUES ? 0x03c003c0u : 0x00780078u, lead = VALUES ? 0x4c004c00u : 0x41804180u;
  asm("" : "+v"(bits));
  asm("" : "+s"(lead));
  out[0] = (word & bits) | lead;
  out[1] = (word >> 4 & bits) | lead;
  out[2] = ((VALUES ? __builtin_amdgcn_alignbit(word, word, 8) : word >> 8) & bits) | lead;
  out[3] = (__builtin_amdgcn_alignbit(word, word, 12) & bits) | lead;
}
// The whole numbers code - zero of a word of keys in float16, with the bias of their token.
__device__ __forceinline__ void whole_keys(unsigned word, _Float16 bias, unsigned (&out)[4]) {
  unsigned c[4];
  packed_codes<true>(__builtin_amdgcn_alignbit(word, word, 32 - (kPackTurnV - kPackTurnK)), c);
  const f16x2 b = {bias, bias};
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, c[i]) + b);
}
// The same of a word of values, with the biases of tokens 0 and 1, 2 and 3.
__device__ __forceinline__ void whole_values(unsigned word, f16x2 b01, f16x2 b23, unsigned (&out)[4]) {
  unsigned c[4];
  packed_codes<true>(word, c);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, c[i]) + (i % 2 ? b23 : b01));
}

__device__ __forceinline__ bf16x8 as_bf16x8(unsigned a, unsigned b, unsigned c, unsigned d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(bf16x8, v);
}

// Number j of eight float16 in four words, and its product with a float32 in one instruction (of
// the form that adds a float32: a multiplication alone would convert first).
__device__ __forceinline__ _Float16 half_of(const u32x4& words, int j) {
  return __builtin_bit_cast(f16x8, words)[j];
}
__device__ __forceinline__ float half_times(_Float16 h, float x) { return __builtin_fmaf((float)h, x, 0.f); }

__device__ __forceinline__ f16x8 as_f16x8(unsigned a, unsigned b, unsigned c, unsigned d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(f16x8, v);
}

template <int N>
__device__ __forceinline__ void load_words(unsigned (&w)[N], const unsigned char* p) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = ((const unsigned*)p)[i];
}

// The 32 keys at walk coordinate `v`; calls come in steps of `stride` keys (the cursor holds this
// call's pages and then fetches those of v + stride).
template <int NB, bool WIDE>
__device__ __forceinline__ void load_packed(PackedBlock<NB>& b, const AttentionArgs& a, PageCursor& cur, int kvh, int v,
                                            int stride, int lane) {
  constexpr int G = PackedBlock<NB>::G, BYTES = pack_block_bytes(NB * 32), CODES = pack_codes_bytes(NB * 32);
  const int r = lane % 16, g = lane / 16, kb = cur.walk.real(v), P = a.page_size;
  const int page[2] = {cur.next0, cur.next1};
  // offsets of 32 bits beside scalar addresses (made known here: hoisted out of the walk they would be widened, and
  // every load would add 64 bits for itself)
  unsigned at_code = (unsigned)(lane * (NB * 4)), at_s = (unsigned)(CODES + g * G * 16 + r % (4 * G) * 4);
  unsigned at_z = (unsigned)(CODES + r / 4 * G * 16 + 8 + r % 4 * 2);
  asm volatile("" : "+v"(at_code), "+v"(at_s), "+v"(at_z));
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    const int64_t at = (((int64_t)max(page[blk], 0) * a.nkv + kvh) * P + ((kb + blk * 16) & (P - 1))) / 16 * BYTES;
    const unsigned char* kp = (const unsigned char*)a.k_pages + at;
    const unsigned char* vp = (const unsigned char*)a.v_pages + at;
    b.ks[blk] = *(const unsigned*)(kp + at_s);
    load_words<NB>(b.k[blk], kp + at_code);
    b.vs[blk] = *(const unsigned*)(vp + at_s);
    load_words<NB>(b.v[blk], vp + at_code);
#pragma unroll
    for (int i = 0; i < G; ++i)
      if constexpr (WIDE) b.kz[blk][i] = *(const unsigned short*)(kp + at_z + i * 16);
  }
  // (no load under a condition, which would put waits for those under way behind it: of a page that is not there, the
  // first page's, and the mask takes its keys out)
  b.page[0] = page[0], b.page[1] = page[1];
  cur.start(v + stride);
}

// A group's steps and biases, out of the sixteen lanes that hold a quarter's: one instruction a word.  (Loaded by every
// lane for itself they were eight loads of 16 bytes a lane for 32 keys, and what a compute unit takes of loads, a kilobyte in
// 7 ns, was two thirds of a walk.)
template <int I>
__device__ __forceinline__ u32x4 packed_scale(unsigned word) {
  return u32x4{(unsigned)__builtin_amdgcn_update_dpp(0, (int)word, 0x150 + 4 * I, 0xf, 0xf, false),
               (unsigned)__builtin_amdgcn_update_dpp(0, (int)word, 0x151 + 4 * I, 0xf, 0xf, false),
               (unsigned)__builtin_amdgcn_update_dpp(0, (int)word, 0x152 + 4 * I, 0xf, 0xf, false),
               (unsigned)__builtin_amdgcn_update_dpp(0, (int)word, 0x153 + 4 * I, 0xf, 0xf, false)};
}
template <int G>
__device__ __forceinline__ u32x4 packed_scale_of(unsigned word, int i) {      // i: known when unrolled
  if (G == 1 || i == 0) return packed_scale<0>(word);
  if (i == 1) return packed_scale<1>(word);
  if (i == 2) return packed_scale<2>(word);
  return packed_scale<3>(word);
}

// By how much a wavefront's steps are brought up: the power of two that takes the largest so far from below
// 2^(exponent - 14) to below 2^15, in two factors that float16 holds (a lane of biases: 1).  Steps are float16 numbers, so
// this is exact, and with it all that follows from it but the bits that small weights would lose.
struct PackedLift {
  int exponent;            // float16's field of the largest step so far (0 below 2^-14); the same in all lanes
  f16x2 by[2];             // of this lane's word
  __device__ __forceinline__ static PackedLift none(int lane) { return at(0, lane); }
  __device__ __forceinline__ static PackedLift at(int exponent, int lane) {
    // 2^(29 - exponent), -1 to 29, as 2^half and 2^(the rest): scalars, by their fields
    const int up = 29 - exponent, half = up >> 1;
    const unsigned a = (unsigned)(15 + half) * 0x04000400u, b = (unsigned)(15 + up - half) * 0x04000400u, one = 0x3c003c00u;
    const bool bias = lane % 4 >= 2;
    return PackedLift{exponent, {__builtin_bit_cast(f16x2, bias ? one : a), __builtin_bit_cast(f16x2, bias ? one : b)}};
  }
  // 2^n for -126 <= n <= 127, a scalar where n is.
  __device__ __forceinline__ static float power(int n) { return __uint_as_float((unsigned)(127 + n) << 23); }
  __device__ __forceinline__ float down() const { return power(exponent - 29); }
  __device__ __forceinline__ unsigned raised(unsigned word) const {
    return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, word) * by[0] * by[1]);
  }
};

template <int NB, bool WIDE>
struct PackedTile {
  static constexpr int NG = (NB + 1) / 2;        // groups that exist
  u32x4 q[WIDE ? 2 : 1][NB]; // bfloat16, or two parts in float16
  float qsum[NG];            // the row's sum over each group; WIDE: qsum[0] is what turns a product into q . k
  f32x4 o[2 * NB], oz[WIDE ? 2 * NB : NG];       // oz: the zeros' share; WIDE: sums of the second parts
  PackedLift lift;           // o and oz count so many times
  float m, l;
  int pos, lo, keep;
  int last, first;           // of all rows: the last key, and the first one that is not behind the window
};

// The parts of eight numbers: 11 bits, and 2^up times the next 11.
template <int UP>
__device__ __forceinline__ void two_parts(u32x4 (&part)[2], const float (&x)[8]) {
  f16x8 hi, lo;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi[j] = (_Float16)x[j];
    lo[j] = (_Float16)((x[j] - (float)hi[j]) * (float)(1 << UP));
  }
  part[0] = __builtin_bit_cast(u32x4, hi);
  part[1] = __builtin_bit_cast(u32x4, lo);
}

template <int NB, bool WIDE, typename T>
__device__ __forceinline__ void load_packed_query(PackedTile<NB, WIDE>& t, const T* row, bool row_ok, int hd, int g) {
  constexpr int NG = PackedTile<NB, WIDE>::NG;
  typedef T eight __attribute__((ext_vector_type(8)));
  eight y[NB];
#pragma unroll
  for (int s = 0; s < NB; ++s) {
    const int e = s * 32 + g * 8;
    y[s] = eight{};
    if (row_ok && e < hd) y[s] = *(const eight*)(row + e);
  }
  if constexpr (WIDE) {
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < NB; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(to_f32(y[s][j])));
    // the largest magnitude to 2^13 .. 2^14 (a row of zeros, or of what is no number, as it is)
    top = col4_max(top);
    const int up = top > 0.f && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
    t.qsum[0] = ldexpf(1.f, -max(up, -126));
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = ldexpf(to_f32(y[s][j]), max(up, -126));
      u32x4 part[2];
      two_parts<0>(part, x);
      t.q[0][s] = part[0], t.q[1][s] = part[1];
    }
  } else {
    float sum[NG] = {};
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      t.q[0][s] = __builtin_bit_cast(u32x4, y[s]);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[s / 2] += to_f32(y[s][j]);
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) t.qsum[i] = col4_sum(sum[i]);
  }
#pragma unroll
  for (int i = 0; i < (WIDE ? 2 * NB : NG); ++i) t.oz[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int db = 0; db < 2 * NB; ++db) t.o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  t.lift = PackedLift::none(threadIdx.x % kWave);
  t.m = -INFINITY;
  t.l = 0.f;
}

// Scores of 32 keys, masked softmax update, and O^T += V^T P^T.  `interior` (wave-uniform): every key is visible
// to every row.
template <int NB, bool WIDE, bool EXTRA>
__device__ __forceinline__ void packed_update(PackedTile<NB, WIDE>& t, const PackedBlock<NB>& b, int kb,
                                              float scale_log2, bool interior, int g, const ScoreExtraLog2* x) {
  constexpr int NG = PackedTile<NB, WIDE>::NG;
  f32x4 st[2];
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const u32x4 scale = packed_scale_of<PackedBlock<NB>::G>(b.ks[blk], i);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      if constexpr (!WIDE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = half_times(half_of(scale, 4 + j), t.qsum[i]);
      }
#pragma unroll
      for (int s = 2 * i; s < 2 * i + 2 && s < NB; ++s) {
        unsigned c[4];
        if constexpr (!WIDE) {
          packed_codes<false>(b.k[blk][s], c);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(c[0], c[1], c[2], c[3]),
                                                        __builtin_bit_cast(bf16x8, t.q[0][s]), acc, 0, 0, 0);
        } else {
          whole_keys(b.k[blk][s], __builtin_bit_cast(_Float16, (unsigned short)b.kz[blk][i]), c);
          const f16x8 k = as_f16x8(c[0], c[1], c[2], c[3]);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, __builtin_bit_cast(f16x8, t.q[1][s]), acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, __builtin_bit_cast(f16x8, t.q[0][s]), acc, 0, 0, 0);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        st[blk][j] = fmaf((float)half_of(scale, j), acc[j], i == 0 ? 0.f : st[blk][j]);
    }
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int j = 0; j < 4; ++j) st[blk][j] *= t.qsum[0];
  }
  if constexpr (EXTRA) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int j = 0; j < 4; ++j) st[blk][j] = extra_score_log2(*x, st[blk][j], kb + blk * 16 + g * 4 + j);
    scale_log2 = 1.f;
  }
  unsigned steps[2] = {b.vs[0], b.vs[1]};        // with their biases
  if (!interior || (b.page[0] | b.page[1]) < 0) {
    asm volatile("" ::: "memory");       // keeps this a branch
    // (steps that a page holds of nobody's keys are none: they have no say in the lift)
    const int word = threadIdx.x % 4;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int key = kb + blk * 16 + g * 4 + word * 2, last = b.page[blk] >= 0 ? t.last : -1;
      unsigned there = (key <= last ? 0xffffu : 0u) | (key < last ? 0xffff0000u : 0u);
      if (kb < t.first)
        there &= (key >= t.first || key < t.keep ? 0xffffu : 0u) | (key + 1 >= t.first || key + 1 < t.keep ? 0xffff0000u : 0u);
      steps[blk] &= word < 2 ? there : ~0u;
    }
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = kb + blk * 16 + g * 4 + j;
        st[blk][j] = (b.page[blk] >= 0 && key <= t.pos && (key >= t.lo || key < t.keep)) ? st[blk][j] : -INFINITY;
      }
  }
  const float mx = max2(max2(max2(max2(st[0][0], st[0][1]), st[0][2]), max2(max2(st[0][3], st[1][0]), st[1][1])),
                        max2(st[1][2], st[1][3]));
  const float m_new = max2(t.m, col4_max(mx) * scale_log2), m_use = max2(m_new, -1e30f);
  const float corr = __builtin_amdgcn_exp2f(t.m - m_use);
  float p[8], sum = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[j / 4][j % 4], scale_log2, -m_use));
    sum += p[j];
  }
  t.l = t.l * corr + sum;
  t.m = m_new;
  // the block's largest step (as whole numbers float16's order is theirs, and biases are below all)
  typedef __attribute__((ext_vector_type(2))) short i16x2;
  const i16x2 top2 = __builtin_elementwise_max(__builtin_bit_cast(i16x2, steps[0]), __builtin_bit_cast(i16x2, steps[1]));
  const int top = max((int)top2[0], (int)top2[1]);
  float change = corr;
  if (__builtin_amdgcn_ballot_w64(top >= (t.lift.exponent + 1) << 10) != 0) {
    // (the largest of sixteen lanes in each, then of the four sixteens as scalars)
    int most = top;
    auto with = [&](auto how) {
      most = max(most, __builtin_amdgcn_update_dpp(0, most, decltype(how)::value, 0xf, 0xf, true));
    };
    with(std::integral_constant<int, 0xB1>{});
    with(std::integral_constant<int, 0x4E>{});
    with(std::integral_constant<int, 0x141>{});
    with(std::integral_constant<int, 0x140>{});
    const int exponent = max(max(__builtin_amdgcn_readlane(most, 0), __builtin_amdgcn_readlane(most, 16)),
                             max(__builtin_amdgcn_readlane(most, 32), __builtin_amdgcn_readlane(most, 48))) >> 10;
    change *= PackedLift::power(t.lift.exponent - exponent);
    t.lift = PackedLift::at(exponent, threadIdx.x % kWave);
  }
  // (far into a context most blocks bring no new largest score)
  if (__builtin_amdgcn_ballot_w64(change != 1.f) != 0) {
#pragma unroll
    for (int db = 0; db < 2 * NB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) t.o[db][j] *= change;
#pragma unroll
    for (int i = 0; i < (WIDE ? 2 * NB : NG); ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) t.oz[i][j] *= change;
  }
  steps[0] = t.lift.raised(steps[0]), steps[1] = t.lift.raised(steps[1]);
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const u32x4 s0 = packed_scale_of<PackedBlock<NB>::G>(steps[0], i), s1 = packed_scale_of<PackedBlock<NB>::G>(steps[1], i);
    if constexpr (!WIDE) {
      // (a multiplication and its rounding to float16 are one instruction)
      f16x8 w;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = (_Float16)half_times(half_of(j < 4 ? s0 : s1, j % 4), p[j]);
      t.oz[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(s0[2], s0[3], s1[2], s1[3]), w, t.oz[i], 0, 0, 0);
#pragma unroll
      for (int s = 2 * i; s < 2 * i + 2 && s < NB; ++s) {
        unsigned c[4], d[4];
        packed_codes<true>(b.v[0][s], c);
        packed_codes<true>(b.v[1][s], d);
        t.o[2 * s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(c[0], c[1], d[0], d[1]), w, t.o[2 * s], 0, 0, 0);
        t.o[2 * s + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(c[2], c[3], d[2], d[3]), w, t.o[2 * s + 1], 0, 0, 0);
      }
    } else {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = half_times(half_of(j < 4 ? s0 : s1, j % 4), p[j]);
      u32x4 part[2];
      two_parts<11>(part, w);
      const f16x8 hi = __builtin_bit_cast(f16x8, part[0]), lo = __builtin_bit_cast(f16x8, part[1]);
#pragma unroll
      for (int s = 2 * i; s < 2 * i + 2 && s < NB; ++s) {
        unsigned c[4], d[4];
        whole_values(b.v[0][s], f16x2{half_of(s0, 4), half_of(s0, 5)}, f16x2{half_of(s0, 6), half_of(s0, 7)}, c);
        whole_values(b.v[1][s], f16x2{half_of(s1, 4), half_of(s1, 5)}, f16x2{half_of(s1, 6), half_of(s1, 7)}, d);
        const f16x8 even = as_f16x8(c[0], c[1], d[0], d[1]), odd = as_f16x8(c[2], c[3], d[2], d[3]);
        t.o[2 * s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, hi, t.o[2 * s], 0, 0, 0);
        t.oz[2 * s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, lo, t.oz[2 * s], 0, 0, 0);
        t.o[2 * s + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, hi, t.o[2 * s + 1], 0, 0, 0);
        t.oz[2 * s + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, lo, t.oz[2 * s + 1], 0, 0, 0);
      }
    }
  }
}

// The rows' sums with what the zeros take off, or with the second parts; o counts as often as the lift says still.
template <int NB, bool WIDE>
__device__ __forceinline__ void packed_finish(PackedTile<NB, WIDE>& t) {
#pragma unroll
  for (int db = 0; db < 2 * NB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) t.o[db][j] = WIDE ? fmaf(t.oz[db][j], 1.f / 2048.f, t.o[db][j]) : t.o[db][j] + t.oz[db / 4][j];
  t.l = col4_sum(t.l);
}

// Workgroups of four wavefronts that a compute unit holds, by the registers they take.
__host__ __device__ constexpr int packed_waves(int nb, bool wide) { return nb > 4 ? (wide ? 1 : 2) : wide ? 2 : 3; }

// One tile's query rows and how far they see.
struct PackedItem {
  int entry, tok0, ntok, pos_first, pos_last;
  KeyWalk walk;
  template <int TURN>
  __device__ __forceinline__ int chunks() const { return (pos_last - walk.origin) / TURN + 1; }
};
__device__ __forceinline__ PackedItem packed_item(const PackedArgs& args, int tile) {
  PackedItem it;
  it.entry = args.tiles ? args.tiles[tile * 3] : tile;
  it.tok0 = args.tiles ? args.tiles[tile * 3 + 1] : tile;
  it.ntok = args.tiles ? args.tiles[tile * 3 + 2] : 1;
  it.pos_first = args.base.positions[it.tok0];                // positions are consecutive
  it.pos_last = it.pos_first + it.ntok - 1;
  it.walk = key_walk<32>(args.base, first_visible(args.base, it.pos_first));
  return it;
}

// The same of a tile that is the same for the whole wavefront: its numbers by scalar loads.
__device__ __forceinline__ PackedItem packed_item_of(const PackedArgs& args, int tile) {
  PackedItem it{tile, tile, 1, 0, 0, KeyWalk{0, 0}};
  if (args.tiles) {
    const ConstTable row = (ConstTable)args.tiles + tile * 3;
    it.entry = row[0], it.tok0 = row[1], it.ntok = row[2];
  }
  it.pos_first = ((ConstTable)args.base.positions)[it.tok0];
  it.pos_last = it.pos_first + it.ntok - 1;
  it.walk = key_walk<32>(args.base, first_visible(args.base, it.pos_first));
  return it;
}

// The sum over the lanes up to this one.
__device__ __forceinline__ int lanes_before(int v, int lane) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int other = __shfl_up(v, o, kWave);
    if (lane >= o) v += other;
  }
  return v;
}

// What is a workgroup's of all items, by one of its wavefronts: turns `at` .. `end` of all, the tile in which they begin and
// its first turn, and how many turns a workgroup has where they are shared.
template <int TURN>
__device__ __forceinline__ void packed_plan(const PackedArgs& args, int heads, int lane, int (&plan)[5]) {
  const int last = kWave - 1, index = blockIdx.x, items = args.num_tiles * heads;
  int total = 0, most = 0, n = 0, upto = 0;
  for (int t0 = 0; t0 < args.num_tiles; t0 += kWave) {
    n = t0 + lane < args.num_tiles ? packed_item(args, t0 + lane).template chunks<TURN>() : 0;
    upto = lanes_before(n, lane);
    total += __builtin_amdgcn_readlane(upto, last);
    most = max(most, n);
  }
  most = uniform((int)wave_max((float)most));
  const int len = (total * heads + args.workgroups - 1) / args.workgroups;
  // in half turns (1.1 us): whole, the longest item, or, of more items than run at a time, all of them and half the
  // longest behind; shared, a workgroup's turns, the look, the parts and their merge, and the ends of items on the way
  const bool in_turns = items > args.workgroups;
  const int whole_cost = max(2 * most, in_turns ? 2 * len + most : 0);
  const int shared_cost = 2 * len + 7 + 12 * items / args.workgroups;
  int at = 0, end = 0, tile = 0, tile_at = 0;
  if (whole_cost <= shared_cost) {
    if (index < items) {
      tile = index / heads;
      const int head_of = index - tile * heads;
      if (in_turns && args.num_tiles <= kWave && most * args.num_tiles > total + total / 4) {
        // the longest first (64 requests of 128 to 4,096 tokens: 43 us in place of 47)
        const int mine = n * kWave + lane;
        int longer = 0;
        for (int j = 0; j < args.num_tiles; ++j) longer += __builtin_amdgcn_readlane(mine, j) > mine ? 1 : 0;
        tile = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < args.num_tiles && longer == tile));
      }
      const int turns = packed_item_of(args, tile).template chunks<TURN>();
      at = head_of * turns, end = at + turns;
    }
  } else if (index < args.workgroups && index * len < total * heads) {
    at = index * len;
    end = min(at + len, total * heads);
    for (int t0 = 0, sum = 0; t0 < args.num_tiles; t0 += kWave) {
      if (args.num_tiles > kWave) {
        n = t0 + lane < args.num_tiles ? packed_item(args, t0 + lane).template chunks<TURN>() : 0;
        upto = sum + lanes_before(n, lane);
      }
      const unsigned long long here = __builtin_amdgcn_ballot_w64(upto * heads > at);
      if (here != 0) {
        const int l = __builtin_ctzll(here);
        tile = t0 + l;
        tile_at = __builtin_amdgcn_readlane(upto - n, l) * heads;
        break;
      }
      sum = __builtin_amdgcn_readlane(upto, last);
    }
  }
  if (lane == 0) plan[0] = at, plan[1] = end, plan[2] = tile, plan[3] = tile_at, plan[4] = len;
}

// An item is a tile and a key/value head (and a block of 16 of its query heads).  A workgroup of as many wavefronts as a
// compute unit holds takes 32 keys a wavefront at a time, a turn of 384 with heads of up to 128, and merges its
// wavefronts in LDS.  (Workgroups of four wavefronts, three to a unit, have three times the items' starts and ends and parts:
// 64 requests of 4,000 tokens, 8 heads of 128, took 68 us, 5.0 TB/s and 60 us so.)
//
// SHARED: how far the items reach is on the device only (a captured step's), so every workgroup looks: either an item is
// one workgroup's, or the turns of all items, one behind the other, are shared out evenly, whatever the lengths, where the
// estimates below say that this is sooner (1 request of 8,000 tokens 46 us whole and 14 shared, 16 of 1,300 12 and 15).
// An item that ends in another workgroup than it began in leaves its parts in memory, two places a workgroup (the part
// that an earlier one began, the part that a later one goes on with), and whoever comes last merges them in their order, sixteen
// parts asked for at a time (four: 25 us in place of 18 for that request).
//
// Not SHARED: an item a workgroup, without that look (2 us).
template <int NB, bool WIDE>
struct PackedShape {
  static constexpr int WAVES = 4 * packed_waves(NB, WIDE), THREADS = WAVES * kWave;
  static constexpr int ROW = 32 * NB + 4;                     // floats: neighbouring rows start four banks apart
  static constexpr int LDS = WAVES * 16 * (ROW + 2) * 4;
  static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
};
template <int NB, bool WIDE, bool EXTRA, typename T, bool SHARED>
__global__ __launch_bounds__((PackedShape<NB, WIDE>::THREADS), packed_waves(NB, WIDE)) void packed_attention_kernel(
    PackedArgs args) {
  constexpr int HD = 32 * NB, DB = 2 * NB;
  typedef PackedShape<NB, WIDE> Shape;
  constexpr int WAVES = Shape::WAVES, TURN = 32 * WAVES;      // TURN: keys that the workgroup takes at a time
  extern __shared__ __attribute__((aligned(16))) float packed_lds[];
  typedef float Results[16][Shape::ROW];
  typedef float Stats[16][2];
  Results* s_o = (Results*)packed_lds;
  Stats* s_ml = (Stats*)(packed_lds + WAVES * 16 * Shape::ROW);
  __shared__ float s_down[WAVES];
  __shared__ unsigned s_before[2];
  __shared__ int s_plan[5];
  const AttentionArgs& a = args.base;
  const int wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16;
  const int group = a.nq / a.nkv, heads = a.nkv * args.head_blocks;
  const float scale_log2 = a.scale * 1.44269504088896341f;
  T* out = (T*)a.out;

  // this workgroup's chunks [at, end) of all, and the tile in which they begin
  int at = 0, end = 0, len = 0, tile = 0, tile_at = 0;                // tile_at: the tile's first chunk among all
  if constexpr (!SHARED) {
    tile = blockIdx.x / heads;
    const int chunks = packed_item_of(args, tile).template chunks<TURN>();
    at = (blockIdx.x - tile * heads) * chunks;
    end = at + chunks;
  } else {
    if (wave == 0) packed_plan<TURN>(args, heads, lane, s_plan);
    __syncthreads();
    at = uniform(s_plan[0]), end = uniform(s_plan[1]), tile = uniform(s_plan[2]), tile_at = uniform(s_plan[3]), len = uniform(s_plan[4]);
  }
  // the parts that this workgroup leaves in memory, one that an earlier one began and one that a later one goes on with
  struct Part {
    int item, first_wg, parts, rows, hb, kvh, tok0;
  } part[2];
  int left = 0;

  while (at < end) {
    const PackedItem it = packed_item_of(args, uniform(tile));
    const int chunks = it.template chunks<TURN>(), head_of = (at - tile_at) / chunks, first_chunk = at - tile_at - head_of * chunks;
    const int count = min(chunks - first_chunk, end - at);
    const int item_at = at - first_chunk, item = tile * heads + head_of;
    const int hb = head_of % args.head_blocks, kvh = head_of / args.head_blocks;
    at += count;
    if (at == tile_at + chunks * heads) { tile_at = at; ++tile; }

    const int* table = a.table + (int64_t)it.entry * a.table_width;
    const int ti = r / args.rows_per_token;
    const int hh = hb * 16 + r % args.rows_per_token;        // head inside the group
    const bool row_ok = ti < it.ntok && hh < group;
    const int token = it.tok0 + min(ti, it.ntok - 1), head = kvh * group + min(hh, group - 1);
    const int key_begin = it.walk.origin + first_chunk * TURN + wave * 32;
    const int key_end = min(it.walk.origin + (first_chunk + count) * TURN, it.pos_last + 1);
    PageCursor cur{(ConstTable)table, a.page_size, it.pos_last, it.walk, -1, -1};
    cur.start(key_begin);
    PackedBlock<NB> A, B;
    load_packed<NB, WIDE>(A, a, cur, kvh, key_begin, TURN, lane);
    PackedTile<NB, WIDE> t;
    t.pos = row_ok ? it.pos_first + ti : -1;
    t.lo = first_visible(a, t.pos);
    t.keep = a.keep;
    t.last = it.pos_last, t.first = first_visible(a, it.pos_first);
    load_packed_query<NB, WIDE, T>(t, (const T*)a.q + ((int64_t)token * a.nq + head) * a.hd, row_ok, a.hd, g);
    ScoreExtraLog2 x;
    if (EXTRA) x = in_log2(score_extra(a, head, t.pos));
    const int lo_last = first_visible(a, it.pos_last);
    auto update = [&](const PackedBlock<NB>& b, int v) {
      const int kb = it.walk.real(v);
      packed_update<NB, WIDE, EXTRA>(t, b, kb, scale_log2, kb + 31 <= it.pos_first && kb >= lo_last, g, &x);
    };
    for (int v = key_begin; v < key_end; v += TURN) {
      load_packed<NB, WIDE>(B, a, cur, kvh, v + TURN, TURN, lane);
      update(A, v);
      A = B;
    }
    packed_finish<NB, WIDE>(t);

    // the wavefronts' results through LDS, an element at a time to a thread (rows that exist only)
    if (g == 0) {
      s_ml[wave][r][0] = t.m;
      s_ml[wave][r][1] = t.l;
    }
    if (lane == 0) s_down[wave] = t.lift.down();
#pragma unroll
    for (int db = 0; db < DB; ++db) *(f32x4*)&s_o[wave][r][db * 16 + g * 4] = t.o[db];
    __syncthreads();
    const int rows = it.ntok * args.rows_per_token;
    const bool whole = !SHARED || count == chunks;
    const int64_t slot0 = ((int64_t)blockIdx.x * 2 + (first_chunk == 0 ? 1 : 0)) * 16;
    auto place = [&](int row) -> int64_t {                    // of a row's result, or -1: no such head
      const int rt = row / args.rows_per_token, rh = hb * 16 + row % args.rows_per_token;
      return rh < group ? ((int64_t)(it.tok0 + rt) * a.nq + kvh * group + rh) * a.hd : -1;
    };
    auto sink_of = [&](int row) { return kvh * group + hb * 16 + row % args.rows_per_token; };
    for (int e = threadIdx.x; e < rows * HD; e += Shape::THREADS) {
      const int row = e / HD, d = e % HD;
      const int64_t to = place(row);
      if (to < 0 || d >= a.hd) continue;
      float M = s_ml[0][row][0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) M = fmaxf(M, s_ml[w][row][0]);
      const float Mc = M == -INFINITY ? 0.f : M;              // (no key: all weights are 0)
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float ww = __builtin_amdgcn_exp2f(s_ml[w][row][0] - Mc);
        sum = fmaf(s_ml[w][row][1], ww, sum);
        acc = fmaf(s_o[w][row][d], ww * s_down[w], acc);
      }
      if (whole) {
        sum = sum_with_sink(sum, M, a.sink, sink_of(row));
        out[to + d] = from_f32<T>(acc * (sum > 0.f ? 1.f / sum : 0.f));
      } else {
        __hip_atomic_store(args.partial_o + (slot0 + row) * HD + d, acc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0)
          __hip_atomic_store((uint64_t*)(args.partial_ml + (slot0 + row) * 2),
                             (uint64_t)__float_as_uint(sum) << 32 | __float_as_uint(M), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (!whole) {
      const int first_wg = item_at / len;
      part[left > 0 ? 1 : 0] = Part{item, first_wg, (item_at + chunks - 1) / len - first_wg + 1, rows, hb, kvh, it.tok0};
      ++left;
    }
    if (at < end) __syncthreads();                            // everybody has read what stands in LDS
  }
  if (!SHARED || left == 0) return;

  // The parts' results pass the caches that another XCD does not share; each wave waits until its own have
  // been taken, the workgroup counts itself in for both, and the one that finds all others there merges.
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if ((int)threadIdx.x < left)
    s_before[threadIdx.x] = __hip_atomic_fetch_add(args.arrivals + (threadIdx.x == 0 ? part[0].item : part[1].item), 1u,
                                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  for (int which = 0; which < left; ++which) {
    const Part p = which == 0 ? part[0] : part[1];
    if ((int)s_before[which] + 1 != p.parts) continue;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    if (threadIdx.x == 0) __hip_atomic_store(args.arrivals + p.item, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int e = threadIdx.x; e < p.rows * HD; e += Shape::THREADS) {
      const int row = e / HD, d = e % HD;
      const int rt = row / args.rows_per_token, rh = p.hb * 16 + row % args.rows_per_token;
      if (rh >= group || d >= a.hd) continue;
      float M = -INFINITY, sum = 0.f, acc = 0.f;
      constexpr int AT_ONCE = 16;
      for (int s0 = 0; s0 < p.parts; s0 += AT_ONCE) {               // everything asked for before its use
        float ms[AT_ONCE], ls[AT_ONCE], po[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const int n = min(s0 + j, p.parts - 1);
          const int64_t slot = ((int64_t)(p.first_wg + n) * 2 + (n == 0 ? 1 : 0)) * 16 + row;
          const uint64_t ml = __hip_atomic_load((const uint64_t*)args.partial_ml + slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          ms[j] = s0 + j < p.parts ? __uint_as_float((unsigned)ml) : -INFINITY;
          ls[j] = __uint_as_float((unsigned)(ml >> 32));
          po[j] = __hip_atomic_load(args.partial_o + slot * HD + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        float Mg = M;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) Mg = fmaxf(Mg, ms[j]);
        const float Mc = Mg == -INFINITY ? 0.f : Mg, keep = __builtin_amdgcn_exp2f(M - Mc);
        sum *= keep;
        acc *= keep;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const float w = __builtin_amdgcn_exp2f(ms[j] - Mc);
          sum = fmaf(ls[j], w, sum);
          acc = fmaf(po[j], w, acc);
        }
        M = Mg;
      }
      sum = sum_with_sink(sum, M, a.sink, p.kvh * group + rh);
      out[((int64_t)(p.tok0 + rt) * a.nq + p.kvh * group + rh) * a.hd + d] = from_f32<T>(acc * (sum > 0.f ? 1.f / sum : 0.f));
    }
  }
}

// A wavefront per tile and head, which walks its keys alone: tiles enough to fill the chip (prompts).
template <int NB, bool WIDE, bool EXTRA, typename T>
__global__ __launch_bounds__(256, packed_waves(NB, WIDE)) void packed_walk_kernel(PackedArgs args) {
  constexpr int DB = 2 * NB;
  const AttentionArgs& a = args.base;
  const int wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16;
  const int group = a.nq / a.nkv, heads = a.nkv * args.head_blocks;
  const int item = blockIdx.x * 4 + wave;
  if (item >= args.num_tiles * heads) return;
  const int hb = item % args.head_blocks, kvh = item / args.head_blocks % a.nkv;
  const PackedItem it = packed_item_of(args, uniform(item / heads));
  const int ti = r / args.rows_per_token, hh = hb * 16 + r % args.rows_per_token;
  const bool row_ok = ti < it.ntok && hh < group;
  const int token = it.tok0 + min(ti, it.ntok - 1), head = kvh * group + min(hh, group - 1);
  const int key_begin = it.walk.origin, key_end = it.pos_last + 1;
  PageCursor cur{(ConstTable)(a.table + (int64_t)it.entry * a.table_width), a.page_size, it.pos_last, it.walk, -1, -1};
  cur.start(key_begin);
  PackedBlock<NB> A, B;
  load_packed<NB, WIDE>(A, a, cur, kvh, key_begin, 32, lane);
  PackedTile<NB, WIDE> t;
  t.pos = row_ok ? it.pos_first + ti : -1;
  t.lo = first_visible(a, t.pos);
  t.keep = a.keep;
  t.last = it.pos_last, t.first = first_visible(a, it.pos_first);
  load_packed_query<NB, WIDE, T>(t, (const T*)a.q + ((int64_t)token * a.nq + head) * a.hd, row_ok, a.hd, g);
  ScoreExtraLog2 x;
  if (EXTRA) x = in_log2(score_extra(a, head, t.pos));
  const int lo_last = first_visible(a, it.pos_last);
  auto update = [&](const PackedBlock<NB>& b, int v) {
    const int kb = it.walk.real(v);
    packed_update<NB, WIDE, EXTRA>(t, b, kb, a.scale * 1.44269504088896341f,
                                    kb + 31 <= it.pos_first && kb >= lo_last, g, &x);
  };
  for (int v = key_begin; v < key_end; v += 32) {
    load_packed<NB, WIDE>(B, a, cur, kvh, v + 32, 32, lane);
    update(A, v);
    A = B;
  }
  packed_finish<NB, WIDE>(t);
  if (!row_ok) return;
  const float sum = sum_with_sink(t.l, t.m, a.sink, head), inv = sum > 0.f ? t.lift.down() / sum : 0.f;
  typedef T four __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    if (db * 16 >= a.hd) break;
    four v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = from_f32<T>(t.o[db][j] * inv);
    *(four*)((T*)a.out + ((int64_t)token * a.nq + head) * a.hd + db * 16 + g * 4) = v;
  }
}

template <int NB, bool WIDE, bool EXTRA, typename T, bool SHARED>
static int launch_packed_shape(const PackedArgs& args, int workgroups, hipStream_t stream) {
  typedef PackedShape<NB, WIDE> Shape;
  auto kernel = packed_attention_kernel<NB, WIDE, EXTRA, T, SHARED>;
  if (Shape::LDS > 64 * 1024) {
    static bool raised[64] = {};               // per instantiation and device
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64)
      TS_FAIL("packed_attention: no current device below 64");
    if (!raised[device]) {
      if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, Shape::LDS) != hipSuccess)
        TS_FAIL("packed_attention: cannot raise the LDS limit to %d bytes", Shape::LDS);
      raised[device] = true;
    }
  }
  hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(Shape::THREADS), Shape::LDS, stream, args);
  TS_CHECK_LAUNCH("packed_attention");
  return 0;
}

template <int NB, bool WIDE, bool EXTRA, typename T>
static int launch_packed(const PackedArgs& args, bool coop, hipStream_t stream) {
  const int items = args.num_tiles * args.base.nkv * args.head_blocks;
  if (coop && args.workgroups)
    return launch_packed_shape<NB, WIDE, EXTRA, T, true>(args, items > args.workgroups ? items : args.workgroups, stream);
  else if (coop)
    return launch_packed_shape<NB, WIDE, EXTRA, T, false>(args, items, stream);
  else
    hipLaunchKernelGGL((packed_walk_kernel<NB, WIDE, EXTRA, T>), dim3((items + 3) / 4), dim3(256), 0, stream, args);
  TS_CHECK_LAUNCH("packed_attention");
  return 0;
}

// A translation unit's heads: of so many slices of 32 elements.
#define TS_PACKED_CASES(WIDE, EXTRA, T)                                      \
  switch (pack_slices(args.base.hd)) {                                        \
    case 1: return launch_packed<1, WIDE, EXTRA, T>(args, coop, stream);     \
    case 2: return launch_packed<2, WIDE, EXTRA, T>(args, coop, stream);     \
    case 3: return launch_packed<3, WIDE, EXTRA, T>(args, coop, stream);     \
    case 4: return launch_packed<4, WIDE, EXTRA, T>(args, coop, stream);     \
    case 5: return launch_packed<5, WIDE, EXTRA, T>(args, coop, stream);     \
    case 6: return launch_packed<6, WIDE, EXTRA, T>(args, coop, stream);     \
    case 7: return launch_packed<7, WIDE, EXTRA, T>(args, coop, stream);     \
    case 8: return launch_packed<8, WIDE, EXTRA, T>(args, coop, stream);     \
  }                                                                           \
  TS_FAIL("packed_attention: head_dim=%d not built", args.base.hd)

int launch_packed_bf16(const PackedArgs& args, bool coop, hipStream_t stream);
int launch_packed_bf16_scores(const PackedArgs& args, bool coop, hipStream_t stream);
int launch_packed_f32(const PackedArgs& args, bool coop, hipStream_t stream);
int launch_packed_f32_scores(const PackedArgs& args, bool coop, hipStream_t stream);
