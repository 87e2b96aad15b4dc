// Paged attention over keys and values of 4 bits (packed_kv.h) on the matrix cores, as a template whose forms
// compile in translation units of their own.
//
// As over a wider cache (attention_core.h) a wavefront owns 16 query rows and takes 32 keys at a time,
//     S^T = K Q^T,    O^T = V^T P^T         (v_mfma_f32_16x16x32_bf16),
// a lane's scores being in place its part of the second product's operand.  Here the operands of K and V are
// codes, turned into the bfloat16 numbers 16 + c, which are exact, and steps stand outside the products:
//     q . k  =  sum over groups of  step (q . (16 + c) - (16 + zero) sum(q))
//     o      =  sum over keys of    (p step) (16 + c) - (p step) (16 + zero)
// Sums of q over a group are float32 numbers of a query row, that is of a lane, and start the group's product as
// -(16 + zero) sum(q); p step is rounded to bfloat16 once and meets codes and -(16 + zero) (a product with the same number in
// every row) alike, so what its rounding costs is in proportion to the value.  PARTS = 3 (float32 activations): q and
// p step in three bfloat16 parts, which hold all their bits.
// A wavefront dequantises nothing: seven instructions make a word of eight codes operands, a score costs a
// multiplication a group and so does a weight.
#pragma once
#include "attention_core.h"
#include "packed_kv.h"

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

struct PackedArgs {
  AttentionArgs base;        // k_pages, v_pages: blocks
  const int* tiles;          // [num_tiles, 3]: batch entry, first flat token, tokens in tile; or null: tile = entry = token
  float* partial_o;          // [items, num_splits, 16, 32 NB]   (num_splits > 1)
  float* partial_ml;         // [items, num_splits, 16, 2]
  unsigned* arrivals;        // [items] zeros: the last workgroup of an item merges its splits and leaves a zero
  int num_tiles;
  int rows_per_token;        // query heads of a tile per token: min(group, 16)
  int head_blocks;           // ceil(group / 16)
  int num_splits;            // shares of an item's keys, of `span` keys each
  int span;                  // a multiple of 128
};

template <int NB>
struct PackedBlock {
  static constexpr int G = pack_groups(NB * 32);
  unsigned k[2][NB], v[2][NB];
  u32x4 ks[2][G], vs[2][G];        // steps and biases of tokens 4 g + i
};

// Eight codes as the bfloat16 numbers 16 + c: codes 0 and 4, 1 and 5, 2 and 6, 3 and 7.
__device__ __forceinline__ void packed_codes(unsigned word, unsigned (&out)[4]) {
  // (one of the two constants in a vector register, one in a scalar: `and` and `or` are one instruction then)
  unsigned bits = 0x00780078u, lead = 0x41804180u;
  asm("" : "+v"(bits));
  asm("" : "+s"(lead));
  out[0] = (word & bits) | lead;
  out[1] = (word >> 4 & bits) | lead;
  out[2] = (word >> 8 & bits) | lead;
  out[3] = (__builtin_amdgcn_alignbit(word, word, 12) & bits) | lead;
}

__device__ __forceinline__ bf16x8 as_bf16x8(unsigned a, unsigned b, unsigned c, unsigned d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(bf16x8, v);
}

// Number j of eight float16 in four words, and its product with a float32 in one instruction (of
// the form that adds a float32: a multiplication alone would convert first).
__device__ __forceinline__ _Float16 half_of(const u32x4& words, int j) {
  typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
  return __builtin_bit_cast(f16x8, words)[j];
}
__device__ __forceinline__ float half_times(_Float16 h, float x) { return __builtin_fmaf((float)h, x, 0.f); }

template <int N>
__device__ __forceinline__ void load_words(unsigned (&w)[N], const unsigned char* p) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = ((const unsigned*)p)[i];
}

// The 32 keys at walk coordinate `v`; calls come in steps of `stride` keys (the cursor holds this
// call's pages and then fetches those of v + stride).
template <int NB>
__device__ __forceinline__ void load_packed(PackedBlock<NB>& b, const AttentionArgs& a, PageCursor& cur, int kvh, int v,
                                            int stride, int lane) {
  constexpr int G = PackedBlock<NB>::G, BYTES = pack_block_bytes(NB * 32), CODES = pack_codes_bytes(NB * 32);
  const int r = lane % 16, g = lane / 16, kb = cur.walk.real(v), P = a.page_size;
  const int page[2] = {cur.next0, cur.next1};
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    const int64_t at = (((int64_t)max(page[blk], 0) * a.nkv + kvh) * P + ((kb + blk * 16) & (P - 1))) / 16 * BYTES;
    const unsigned char* kp = (const unsigned char*)a.k_pages + at;
    const unsigned char* vp = (const unsigned char*)a.v_pages + at;
    load_words<NB>(b.k[blk], kp + (r * 4 + g) * (NB * 4));
    load_words<NB>(b.v[blk], vp + lane * (NB * 4));
#pragma unroll
    for (int i = 0; i < G; ++i) {
      b.ks[blk][i] = *(const u32x4*)(kp + CODES + (g * G + i) * 16);
      b.vs[blk][i] = *(const u32x4*)(vp + CODES + (g * G + i) * 16);
    }
  }
  if (page[0] < 0 || page[1] < 0) {      // where the context ends or a window has let go: steps of zero
    const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int i = 0; i < G; ++i)
        if (page[blk] < 0) b.ks[blk][i] = b.vs[blk][i] = zero;
  }
  cur.start(v + stride);
}

template <int NB, int PARTS>
struct PackedTile {
  static constexpr int NG = (NB + 1) / 2;        // groups that exist
  bf16x8 q[PARTS][NB];
  float qsum[NG];            // the row's sum over each group
  f32x4 o[2 * NB], oz[NG];
  float m, l;
  int pos, lo, keep;
};

template <int PARTS, typename T>
__device__ __forceinline__ void split_parts(bf16x8 (&part)[PARTS], const T (&x)[8]) {
  float left[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) left[j] = to_f32(x[j]);
#pragma unroll
  for (int p = 0; p < PARTS; ++p)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      part[p][j] = (bf16_t)left[j];
      left[j] -= (float)part[p][j];
    }
}

template <int NB, int PARTS, typename T>
__device__ __forceinline__ void load_packed_query(PackedTile<NB, PARTS>& t, const T* row, bool row_ok, int hd, int g) {
  constexpr int NG = PackedTile<NB, PARTS>::NG;
  float sum[NG] = {};
#pragma unroll
  for (int s = 0; s < NB; ++s) {
    typedef T eight __attribute__((ext_vector_type(8)));
    const int e = s * 32 + g * 8;
    T x[8];
    eight y = {};
    if (row_ok && e < hd) y = *(const eight*)(row + e);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = y[j];
      sum[s / 2] += to_f32(x[j]);
    }
    bf16x8 part[PARTS];
    split_parts<PARTS, T>(part, x);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) t.q[p][s] = part[p];
  }
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    t.qsum[i] = col4_sum(sum[i]);
    t.oz[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int db = 0; db < 2 * NB; ++db) t.o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  t.m = -INFINITY;
  t.l = 0.f;
}

// Scores of 32 keys, masked softmax update, and O^T += V^T P^T.  `interior` (wave-uniform): every key is visible
// to every row.
template <int NB, int PARTS, bool EXTRA>
__device__ __forceinline__ void packed_update(PackedTile<NB, PARTS>& t, const PackedBlock<NB>& b, int kb,
                                              float scale_log2, bool interior, int g, const ScoreExtraLog2* x) {
  constexpr int NG = PackedTile<NB, PARTS>::NG;
  f32x4 st[2];
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      f32x4 acc;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = half_times(half_of(b.ks[blk][i], 4 + j), t.qsum[i]);
#pragma unroll
      for (int s = 2 * i; s < 2 * i + 2 && s < NB; ++s) {
        unsigned c[4];
        packed_codes(b.k[blk][s], c);
        const bf16x8 k = as_bf16x8(c[0], c[1], c[2], c[3]);
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, t.q[p][s], acc, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        st[blk][j] = fmaf((float)half_of(b.ks[blk][i], j), acc[j], i == 0 ? 0.f : st[blk][j]);
    }
  }
  if constexpr (EXTRA) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int j = 0; j < 4; ++j) st[blk][j] = extra_score_log2(*x, st[blk][j], kb + blk * 16 + g * 4 + j);
    scale_log2 = 1.f;
  }
  if (!interior) {
    asm volatile("" ::: "memory");       // keeps this a branch
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = kb + blk * 16 + g * 4 + j;
        st[blk][j] = (key <= t.pos && (key >= t.lo || key < t.keep)) ? st[blk][j] : -INFINITY;
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
  // (far into a context most blocks bring no new largest score)
  if (__builtin_amdgcn_ballot_w64(corr != 1.f) != 0) {
#pragma unroll
    for (int db = 0; db < 2 * NB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) t.o[db][j] *= corr;
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) t.oz[i][j] *= corr;
  }
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = half_times(half_of(b.vs[j / 4][i], j % 4), p[j]);
    bf16x8 part[PARTS];
    split_parts<PARTS, float>(part, w);
    const bf16x8 bias = as_bf16x8(b.vs[0][i][2], b.vs[0][i][3], b.vs[1][i][2], b.vs[1][i][3]);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) t.oz[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bias, part[q], t.oz[i], 0, 0, 0);
#pragma unroll
    for (int s = 2 * i; s < 2 * i + 2 && s < NB; ++s) {
      unsigned c[4], d[4];
      packed_codes(b.v[0][s], c);
      packed_codes(b.v[1][s], d);
      const bf16x8 even = as_bf16x8(c[0], c[1], d[0], d[1]), odd = as_bf16x8(c[2], c[3], d[2], d[3]);
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        t.o[2 * s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, part[q], t.o[2 * s], 0, 0, 0);
        t.o[2 * s + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, part[q], t.o[2 * s + 1], 0, 0, 0);
      }
    }
  }
}

// The rows' sums with what the zeros take off.
template <int NB, int PARTS>
__device__ __forceinline__ void packed_finish(PackedTile<NB, PARTS>& t) {
#pragma unroll
  for (int db = 0; db < 2 * NB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) t.o[db][j] += t.oz[db / 4][j];
  t.l = col4_sum(t.l);
}

// COOP: a workgroup of four wavefronts per item and share of its keys, each every fourth block of 32 keys, merged in
// LDS; else a wavefront per item, which walks its keys alone (prompts: tiles enough to fill the chip).
// Shares are of `span` keys at fixed places from the item's first key on, so that requests of unlike lengths
// give workgroups of like lengths; the last of an item's workgroups to finish merges its shares.
template <int NB, int PARTS, bool COOP, bool EXTRA, typename T>
__global__ __launch_bounds__(256, PARTS == 1 && NB <= 4 ? 2 : 1) void packed_attention_kernel(PackedArgs args) {
  constexpr int HD = 32 * NB, DB = 2 * NB;
  const AttentionArgs& a = args.base;
  const int wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int r = lane % 16, g = lane / 16;
  const int group = a.nq / a.nkv;
  const int items = args.num_tiles * a.nkv * args.head_blocks;
  const int item = COOP ? blockIdx.x : blockIdx.x * 4 + wave;
  if (item >= items) return;
  const int hb = item % args.head_blocks, kvh = item / args.head_blocks % a.nkv;
  const int tile = item / args.head_blocks / a.nkv;
  const int entry = args.tiles ? uniform(args.tiles[tile * 3]) : tile,
            tok0 = args.tiles ? uniform(args.tiles[tile * 3 + 1]) : tile,
            ntok = args.tiles ? uniform(args.tiles[tile * 3 + 2]) : 1;
  const int* table = a.table + (int64_t)entry * a.table_width;
  const int ti = r / args.rows_per_token;
  const int hh = hb * 16 + r % args.rows_per_token;          // head inside the group
  const bool row_ok = ti < ntok && hh < group;
  const int token = tok0 + min(ti, ntok - 1);
  const int head = kvh * group + min(hh, group - 1);

  const int pos_first = uniform(a.positions[tok0]);           // positions are consecutive
  const int pos_last = pos_first + ntok - 1;
  const KeyWalk walk = key_walk<32>(a, first_visible(a, pos_first));
  const int share = COOP ? blockIdx.y : 0;
  const int first = COOP ? walk.origin + share * args.span : walk.origin;
  const int used = COOP ? min(args.num_splits, (pos_last - walk.origin) / args.span + 1) : 1;
  if (share >= used) return;                                  // an item with fewer shares than others
  // (the last share takes what more there is: positions beyond what the host planned for)
  const int key_end = share == used - 1 ? pos_last + 1 : first + args.span;
  constexpr int kStride = COOP ? 128 : 32;
  const int key_begin = first + (COOP ? wave * 32 : 0);

  PageCursor cur{(ConstTable)table, a.page_size, pos_last, walk, -1, -1};
  cur.start(key_begin);
  PackedBlock<NB> A, B;
  if (key_begin < key_end) load_packed<NB>(A, a, cur, kvh, key_begin, kStride, lane);
  PackedTile<NB, PARTS> t;
  t.pos = row_ok ? pos_first + ti : -1;
  t.lo = first_visible(a, t.pos);
  t.keep = a.keep;
  load_packed_query<NB, PARTS, T>(t, (const T*)a.q + ((int64_t)token * a.nq + head) * a.hd, row_ok, a.hd, g);
  const float scale_log2 = a.scale * 1.44269504088896341f;
  ScoreExtraLog2 x;
  if (EXTRA) x = in_log2(score_extra(a, head, t.pos));
  const int lo_last = first_visible(a, pos_last);
  auto update = [&](const PackedBlock<NB>& b, int v) {
    const int kb = walk.real(v);
    packed_update<NB, PARTS, EXTRA>(t, b, kb, scale_log2, kb + 31 <= pos_first && kb >= lo_last, g, &x);
  };
  for (int v = key_begin; v < key_end; v += 2 * kStride) {
    if (v + kStride < key_end) load_packed<NB>(B, a, cur, kvh, v + kStride, kStride, lane);
    update(A, v);
    if (v + kStride >= key_end) break;
    if (v + 2 * kStride < key_end) load_packed<NB>(A, a, cur, kvh, v + 2 * kStride, kStride, lane);
    update(B, v + kStride);
  }
  packed_finish<NB, PARTS>(t);
  T* out = (T*)a.out;

  if constexpr (!COOP) {
    if (!row_ok) return;
    const float sum = sum_with_sink(t.l, t.m, a.sink, head), inv = sum > 0.f ? 1.f / sum : 0.f;
    typedef T four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      if (db * 16 >= a.hd) break;
      four v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = from_f32<T>(t.o[db][j] * inv);
      *(four*)(out + ((int64_t)token * a.nq + head) * a.hd + db * 16 + g * 4) = v;
    }
    return;
  } else {
    // the wavefronts' results through LDS, an element at a time to a thread (rows that exist only)
    constexpr int kRow = HD + 4;                              // neighbouring rows start four banks apart
    __shared__ float s_ml[4][16][2];
    __shared__ __attribute__((aligned(16))) float s_o[4][16][kRow];
    __shared__ unsigned s_before;
    if (g == 0) {
      s_ml[wave][r][0] = t.m;
      s_ml[wave][r][1] = t.l;
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) *(f32x4*)&s_o[wave][r][db * 16 + g * 4] = t.o[db];
    __syncthreads();
    const int rows = ntok * args.rows_per_token;              // the last row of a tile of several tokens; heads past
    const int64_t slot0 = ((int64_t)item * args.num_splits + share) * 16;      // the group's are not stored
    const bool alone = used == 1;
    auto place = [&](int row) -> int64_t {                    // of a row's result, or -1
      const int rt = row / args.rows_per_token, rh = hb * 16 + row % args.rows_per_token;
      return rh < group ? ((int64_t)(tok0 + rt) * a.nq + kvh * group + rh) * a.hd : -1;
    };
    for (int e = threadIdx.x; e < rows * HD; e += 256) {
      const int row = e / HD, d = e % HD;
      const int64_t at = place(row);
      if (at < 0 || d >= a.hd) continue;
      float M = s_ml[0][row][0];
#pragma unroll
      for (int w = 1; w < 4; ++w) M = fmaxf(M, s_ml[w][row][0]);
      const float Mc = M == -INFINITY ? 0.f : M;              // (no key: all weights are 0)
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float ww = __builtin_amdgcn_exp2f(s_ml[w][row][0] - Mc);
        sum = fmaf(s_ml[w][row][1], ww, sum);
        acc = fmaf(s_o[w][row][d], ww, acc);
      }
      if (alone) {
        sum = sum_with_sink(sum, M, a.sink, kvh * group + hb * 16 + row % args.rows_per_token);
        out[at + d] = from_f32<T>(acc * (sum > 0.f ? 1.f / sum : 0.f));
      } else {
        __hip_atomic_store(args.partial_o + (slot0 + row) * HD + d, acc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0)
          __hip_atomic_store((uint64_t*)(args.partial_ml + (slot0 + row) * 2),
                             (uint64_t)__float_as_uint(sum) << 32 | __float_as_uint(M), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (alone) return;
    // The shares' results pass the caches that another XCD does not share; each wave waits until its own have
    // been taken, the workgroup counts itself in, and the one that finds all others there merges.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
      s_before = __hip_atomic_fetch_add(args.arrivals + item, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if ((int)s_before + 1 != used) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    if (threadIdx.x == 0) __hip_atomic_store(args.arrivals + item, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int e = threadIdx.x; e < rows * HD; e += 256) {
      const int row = e / HD, d = e % HD;
      const int64_t at = place(row);
      if (at < 0 || d >= a.hd) continue;
      float M = -INFINITY, sum = 0.f, acc = 0.f;
      for (int s0 = 0; s0 < used; s0 += 4) {                  // four at a time: everything asked for before its use
        float ms[4], ls[4], part[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t slot = ((int64_t)item * args.num_splits + min(s0 + j, used - 1)) * 16 + row;
          const uint64_t ml = __hip_atomic_load((const uint64_t*)args.partial_ml + slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          ms[j] = s0 + j < used ? __uint_as_float((unsigned)ml) : -INFINITY;
          ls[j] = __uint_as_float((unsigned)(ml >> 32));
          part[j] = __hip_atomic_load(args.partial_o + slot * HD + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        float Mg = M;
#pragma unroll
        for (int j = 0; j < 4; ++j) Mg = fmaxf(Mg, ms[j]);
        const float Mc = Mg == -INFINITY ? 0.f : Mg, keep = __builtin_amdgcn_exp2f(M - Mc);
        sum *= keep;
        acc *= keep;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w = __builtin_amdgcn_exp2f(ms[j] - Mc);
          sum = fmaf(ls[j], w, sum);
          acc = fmaf(part[j], w, acc);
        }
        M = Mg;
      }
      sum = sum_with_sink(sum, M, a.sink, kvh * group + hb * 16 + row % args.rows_per_token);
      out[at + d] = from_f32<T>(acc * (sum > 0.f ? 1.f / sum : 0.f));
    }
  }
}

template <int NB, int PARTS, bool EXTRA, typename T>
static int launch_packed(const PackedArgs& args, bool coop, hipStream_t stream) {
  const int items = args.num_tiles * args.base.nkv * args.head_blocks;
  if (coop)
    hipLaunchKernelGGL((packed_attention_kernel<NB, PARTS, true, EXTRA, T>), dim3(items, args.num_splits), dim3(256), 0, stream, args);
  else
    hipLaunchKernelGGL((packed_attention_kernel<NB, PARTS, false, EXTRA, T>), dim3((items + 3) / 4), dim3(256), 0, stream, args);
  TS_CHECK_LAUNCH("packed_attention");
  return 0;
}

// A translation unit's heads: of so many slices of 32 elements.
#define TS_PACKED_CASES(PARTS, EXTRA, T)                                      \
  switch (pack_slices(args.base.hd)) {                                        \
    case 1: return launch_packed<1, PARTS, EXTRA, T>(args, coop, stream);     \
    case 2: return launch_packed<2, PARTS, EXTRA, T>(args, coop, stream);     \
    case 3: return launch_packed<3, PARTS, EXTRA, T>(args, coop, stream);     \
    case 4: return launch_packed<4, PARTS, EXTRA, T>(args, coop, stream);     \
    case 5: return launch_packed<5, PARTS, EXTRA, T>(args, coop, stream);     \
    case 6: return launch_packed<6, PARTS, EXTRA, T>(args, coop, stream);     \
    case 7: return launch_packed<7, PARTS, EXTRA, T>(args, coop, stream);     \
    case 8: return launch_packed<8, PARTS, EXTRA, T>(args, coop, stream);     \
  }                                                                           \
  TS_FAIL("packed_attention: head_dim=%d not built", args.base.hd)

int launch_packed_bf16(const PackedArgs& args, bool coop, hipStream_t stream);
int launch_packed_bf16_scores(const PackedArgs& args, bool coop, hipStream_t stream);
int launch_packed_f32(const PackedArgs& args, bool coop, hipStream_t stream);
int launch_packed_f32_scores(const PackedArgs& args, bool coop, hipStream_t stream);
