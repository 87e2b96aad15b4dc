// Keys and values into a cache of 4 bits (packed_kv.h), with everything that lies between their projection and
// attention, and back out of it.
//
// One launch norms and turns query and key heads (qk_prepare.hip's arithmetic), rounds keys to the
// activation type, as a wider cache would keep them, and quantises keys and values.  Eight elements a lane, so a
// group of 64 is eight lanes and a head 8 to 32.  A token's keys are words of their own.  Four tokens share a word
// of values, so the first of a run of up to four that share words writes for the run, with what it leaves of other
// tokens' bits read first; no other request has tokens in that page's block, and a step's tokens of one request are in order.
#include "packed_kv.h"
#include "qk_prepare.h"

struct PackStoreArgs {
  const void *q, *k, *v;     // rows of T: heads of a token side by side, rows `*_stride` elements apart (q: or null)
  void* q_out;               // [T, nq, hd]
  unsigned char *k_pages, *v_pages;      // [num_pages, nkv, P / 16, block bytes]
  const float *q_weight, *k_weight, *cos, *sin;
  const int *positions, *entry_of_token, *table;
  int64_t stride;            // elements from a token's row to the next, the same in q, k and v
  int table_width, num_tokens, nq, nkv, hd, page_size;
  float eps;
  unsigned heads, heads_inv;     // heads of a token's row (inverse32: common.h)
};

// LANES: of a head (8, 16, 32), eight elements each.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void pack_store_kernel(PackStoreArgs a) {
  constexpr int kHeads = kWave / LANES;
  const int lane = threadIdx.x % kWave, sub = lane % LANES;
  const unsigned item = (blockIdx.x * 4 + threadIdx.x / kWave) * kHeads + lane / LANES;
  const int t = (int)divided(item, a.heads, a.heads_inv), h = (int)(item - t * a.heads);
  if (t >= a.num_tokens) return;                               // whole heads: groups of LANES lanes
  const int hd = a.hd, pos = a.positions[t], entry = a.entry_of_token[t];
  const bool there = sub * 8 < hd;
  const int at = there ? sub * 8 : 0;
  const int bytes = pack_block_bytes(hd), G = pack_groups(hd), NB = pack_slices(hd);
  if (h < a.nq + a.nkv) {
    const bool key = h >= a.nq;
    const int head = key ? h - a.nq : h;
    Eight<T> x;
    x.load((const T*)(key ? a.k : a.q) + (int64_t)t * a.stride + (int64_t)head * hd + at);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = there ? x.get(j) : 0.f;
    const float* w = key ? a.k_weight : a.q_weight;
    if (w) {
      const float rstd = head_rstd(v, LANES, hd, a.eps);
      const f32x4_qk w0 = *(const f32x4_qk*)(w + at), w1 = *(const f32x4_qk*)(w + at + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] *= rstd * w0[j]; v[4 + j] *= rstd * w1[j]; }
    }
    if (a.cos) {
      const int half = hd / 16;                                // lanes of half a head
      const bool first = sub < half;
      const int i0 = (first ? sub : there ? sub - half : 0) * 8;
      const float* cp = a.cos + (int64_t)pos * (hd / 2) + i0;
      const float* sp = a.sin + (int64_t)pos * (hd / 2) + i0;
      const f32x4_qk c0 = *(const f32x4_qk*)cp, c1 = *(const f32x4_qk*)(cp + 4);
      const f32x4_qk s0 = *(const f32x4_qk*)sp, s1 = *(const f32x4_qk*)(sp + 4);
      const int other_lane = there ? lane - sub + (first ? sub + half : sub - half) : lane;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float other = __shfl(v[j], other_lane, kWave);
        v[j] = head_turned(v[j], other, j < 4 ? c0[j] : c1[j - 4], j < 4 ? s0[j] : s1[j - 4], first);
      }
    }
    if (!key) {
      if (there) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x.set(j, v[j]);
        x.store((T*)a.q_out + ((int64_t)t * a.nq + head) * hd + at);
      }
      return;
    }
    const int page = a.table[(int64_t)entry * a.table_width + (pos >> __builtin_ctz(a.page_size))];
    unsigned code[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = there ? to_f32(from_f32<T>(v[j])) : 0.f;
    const PackGroup p = pack_eight(v, code);
    if (page < 0) return;                                      // no page behind this position: nothing is written
    const int slot = pos & (a.page_size - 1), token = slot % kPackTokens;
    unsigned char* block = a.k_pages + pack_block(page, a.nkv, head, a.page_size, slot, bytes);
    unsigned word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) word |= code[j] << (4 * (j / 2 + 4 * (j % 2)));
    if (sub < NB * 4) ((unsigned*)block)[(sub % 4 * 16 + token) * NB + sub / 4] = pack_turned<kPackTurnK>(word);
    if (sub % 8 == 0 && there) {
      _Float16* scale = (_Float16*)(block + pack_codes_bytes(hd) + (token / 4 * G + sub / 8) * 16);
      scale[token % 4] = p.step;
      scale[4 + token % 4] = (_Float16)(-16.f - p.zero);
    }
    return;
  }
  // values: the first token of those of this step that share words with it
  const int head = h - a.nq - a.nkv, i0 = pos & 3;
  if (i0 != 0 && t > 0 && a.entry_of_token[t - 1] == entry && a.positions[t - 1] == pos - 1) return;
  int count = 1;
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    const int n = min(t + j, a.num_tokens - 1);
    if (count == j && i0 + j < 4 && t + j < a.num_tokens && a.entry_of_token[n] == entry && a.positions[n] == pos + j)
      count = j + 1;
  }
  const int page = a.table[(int64_t)entry * a.table_width + (pos >> __builtin_ctz(a.page_size))];
  const int slot = pos & (a.page_size - 1), quad = slot % kPackTokens / 4, second = sub / 2 % 2;
  Eight<T> x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    x[j].load((const T*)a.v + (int64_t)(t + min(j, count - 1)) * a.stride + (int64_t)head * hd + at);
  unsigned part[8] = {};
  _Float16 step[4];
  float zero[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float v[8];
    unsigned code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = there ? x[j].get(e) : 0.f;
    const PackGroup p = pack_eight(v, code);
    step[j] = p.step, zero[j] = p.zero;
    const int i = (i0 + j) & 3;                                // (of tokens past the run: not used)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j < count) part[e] |= code[e] << (4 * (2 * second + i / 2 + 4 * (i % 2)));
  }
  unsigned mask = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = (i0 + j) & 3;
    if (j < count) mask |= 0xfu << (4 * (i / 2 + 4 * (i % 2)));
  }
  mask |= mask << 8;                                           // both elements of a word
  unsigned word[4];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned both = part[e] | __shfl_xor(part[e], 2, kWave);
    if (e / 4 == second) word[e % 4] = both;
  }
  if (page < 0) return;
  unsigned char* block = a.v_pages + pack_block(page, a.nkv, head, a.page_size, slot, bytes);
  if (sub < NB * 4) {
    unsigned* words = (unsigned*)block + (quad * 16 + sub % 2 * 8 + second * 4) * NB + sub / 4;
    if (count < 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) word[e] |= pack_unturned<kPackTurnV>(words[e * NB]) & ~mask;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) words[e * NB] = pack_turned<kPackTurnV>(word[e]);
  }
  if (sub % 8 == 0 && there) {
    unsigned char* scale = block + pack_codes_bytes(hd) + (quad * G + sub / 8) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < count) {
        ((_Float16*)scale)[i0 + j] = step[j];
        ((_Float16*)scale)[4 + i0 + j] = (_Float16)(-16.f - zero[j]);
      }
  }
}

static int launch_pack_store(PackStoreArgs a, int type, hipStream_t stream) {
  const int lanes = a.hd <= 64 ? 8 : a.hd <= 128 ? 16 : 32;
  a.heads = a.nq + 2 * a.nkv, a.heads_inv = inverse32(a.heads);
  const int64_t items = (int64_t)a.num_tokens * a.heads;
  const int per_block = 4 * (kWave / lanes);
  const int64_t blocks = (items + per_block - 1) / per_block;
  if (items > 2147483647LL - per_block) TS_FAIL("pack_store: too many tokens");
#define TS_LAUNCH(L) hipLaunchKernelGGL((pack_store_kernel<T, L>), dim3((unsigned)blocks), dim3(256), 0, stream, a)
  TS_DISPATCH_TYPE(type, T, if (lanes == 8) TS_LAUNCH(8); else if (lanes == 16) TS_LAUNCH(16); else TS_LAUNCH(32));
#undef TS_LAUNCH
  TS_CHECK_LAUNCH("pack_store");
  return 0;
}

// 1 if a cache of 4 bits is built for these sizes, and the bytes of its blocks.
extern "C" int ts_pack_fits(int hd, int page_size) { return pack_fits(hd, page_size) ? 1 : 0; }
extern "C" int ts_pack_block_bytes(int hd) { return pack_block_bytes(hd); }

// qk_prepare's work with a cache of 4 bits behind it: normed and turned queries, keys and values in their pages.
extern "C" int ts_pack_prepare(const QkPrepareArgs* p, int type, hipStream_t stream) {
  const QkPrepareArgs& h = *p;
  if (h.num_tokens <= 0) return 0;
  if (!pack_fits(h.hd, h.page_size)) TS_FAIL("pack_prepare: head_dim=%d, page_size=%d not built", h.hd, h.page_size);
  if (h.nq <= 0 || h.nkv <= 0) TS_FAIL("pack_prepare: heads nq=%d nkv=%d", h.nq, h.nkv);
  if (h.row_extra < 0 || h.row_extra % 8) TS_FAIL("pack_prepare: row_extra=%d must be a multiple of 8", h.row_extra);
  if ((h.cos == nullptr) != (h.sin == nullptr)) TS_FAIL("pack_prepare: cos and sin go together");
  if (!h.table || h.table_width <= 0) TS_FAIL("pack_prepare: no block table");
  if (((uintptr_t)h.qkv | (uintptr_t)h.q_out | (uintptr_t)h.k_dst | (uintptr_t)h.v_dst | (uintptr_t)h.q_weight |
       (uintptr_t)h.k_weight | (uintptr_t)h.cos | (uintptr_t)h.sin) & 15)
    TS_FAIL("pack_prepare: tensors must be 16-byte aligned");
  const int size = type == TS_F32 ? 4 : 2;
  PackStoreArgs a{};
  a.q = h.qkv;
  a.k = (const char*)h.qkv + (int64_t)h.nq * h.hd * size;
  a.v = (const char*)h.qkv + (int64_t)(h.nq + h.nkv) * h.hd * size;
  a.q_out = h.q_out, a.k_pages = (unsigned char*)h.k_dst, a.v_pages = (unsigned char*)h.v_dst;
  a.q_weight = h.q_weight, a.k_weight = h.k_weight, a.cos = h.cos, a.sin = h.sin;
  a.positions = h.positions, a.entry_of_token = h.entry_of_token, a.table = h.table;
  a.stride = (int64_t)(h.nq + 2 * h.nkv) * h.hd + h.row_extra;
  a.table_width = h.table_width, a.num_tokens = h.num_tokens, a.nq = h.nq, a.nkv = h.nkv, a.hd = h.hd;
  a.page_size = h.page_size, a.eps = h.eps;
  return launch_pack_store(a, type, stream);
}

// Keys and values [T, nkv, hd] as they are into their pages.
extern "C" int ts_pack_store(const void* k, const void* v, int type, void* k_pages, void* v_pages, const int* positions,
                             const int* entry_of_token, const int* table, int table_width, int num_tokens, int nkv,
                             int hd, int page_size, hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (!pack_fits(hd, page_size)) TS_FAIL("pack_store: head_dim=%d, page_size=%d not built", hd, page_size);
  if (nkv <= 0 || !table || table_width <= 0) TS_FAIL("pack_store: nkv=%d, block table of width %d", nkv, table_width);
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15)
    TS_FAIL("pack_store: tensors must be 16-byte aligned");
  PackStoreArgs a{};
  a.k = k, a.v = v, a.k_pages = (unsigned char*)k_pages, a.v_pages = (unsigned char*)v_pages;
  a.positions = positions, a.entry_of_token = entry_of_token, a.table = table;
  a.stride = (int64_t)nkv * hd;
  a.table_width = table_width, a.num_tokens = num_tokens, a.nkv = nkv, a.hd = hd, a.page_size = page_size;
  return launch_pack_store(a, type, stream);
}

// ---------------------------------------------------------------- back out of the cache
// Eight elements a lane of a token's key or value head; the first of up to four tokens that share words of values reads
// for all of them.  Positions without a page read as zeros.
struct PackValuesArgs {
  const unsigned char *k_pages, *v_pages;
  void *k, *v;                   // [T, nkv, hd]
  const int *positions, *entry_of_token, *table;
  int table_width, num_tokens, nkv, hd, page_size;
  unsigned per, per_inv, heads_inv;      // pieces of a head; of 2 nkv
};

template <typename T>
__global__ __launch_bounds__(256) void pack_values_kernel(PackValuesArgs a) {
  const unsigned piece = blockIdx.x * 256 + threadIdx.x, row = divided(piece, a.per, a.per_inv);
  const int sub = (int)(piece - row * a.per);
  const int t = (int)divided(row, 2 * a.nkv, a.heads_inv), h = (int)(row - (unsigned)t * 2 * a.nkv);
  if (t >= a.num_tokens) return;
  const bool key = h < a.nkv;
  const int head = key ? h : h - a.nkv, pos = a.positions[t], entry = a.entry_of_token[t];
  int count = 1;
  if (!key) {
    const int i0 = pos & 3;
    if (i0 != 0 && t > 0 && a.entry_of_token[t - 1] == entry && a.positions[t - 1] == pos - 1) return;
#pragma unroll
    for (int j = 1; j < 4; ++j) {
      const int n = min(t + j, a.num_tokens - 1);
      if (count == j && i0 + j < 4 && t + j < a.num_tokens && a.entry_of_token[n] == entry && a.positions[n] == pos + j)
        count = j + 1;
    }
  }
  const int page = a.table[(int64_t)entry * a.table_width + (pos >> __builtin_ctz(a.page_size))];
  const int G = pack_groups(a.hd), NB = pack_slices(a.hd), slot = pos & (a.page_size - 1), token = slot % kPackTokens;
  const int quad = token / 4, i0 = token % 4;
  const unsigned char* block = (key ? a.k_pages : a.v_pages) +
                               pack_block(max(page, 0), a.nkv, head, a.page_size, slot, pack_block_bytes(a.hd));
  const unsigned* words = (const unsigned*)block;
  typedef _Float16 eight_h __attribute__((ext_vector_type(8)));
  const eight_h scale = *(const eight_h*)(block + pack_codes_bytes(a.hd) + (quad * G + sub / 8) * 16);
  T* dst = (T*)(key ? a.k : a.v) + ((int64_t)t * a.nkv + head) * a.hd + sub * 8;
  unsigned word[8];
  if (key) {
    word[0] = pack_unturned<kPackTurnK>(words[(sub % 4 * 16 + token) * NB + sub / 4]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) word[e] = pack_unturned<kPackTurnV>(words[(quad * 16 + sub % 2 * 8 + e) * NB + sub / 4]);
  }
  for (int j = 0; j < count; ++j) {
    const int i = i0 + j;
    const float step = page >= 0 ? (float)(i == 0 ? scale[0] : i == 1 ? scale[1] : i == 2 ? scale[2] : scale[3]) : 0.f;
    const float bias = (float)(i == 0 ? scale[4] : i == 1 ? scale[5] : i == 2 ? scale[6] : scale[7]);
    const int at = 4 * (2 * (sub / 2 % 2) + i / 2 + 4 * (i % 2));
    Eight<T> out;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned code = key ? word[0] >> (4 * (e / 2 + 4 * (e % 2))) & 15 : word[e] >> at & 15;
      out.set(e, page >= 0 ? step * ((float)code + 16.f + bias) : 0.f);
    }
    out.store(dst + (int64_t)j * a.nkv * a.hd);
  }
}

extern "C" int ts_pack_values(const void* k_pages, const void* v_pages, void* k, void* v, int type, const int* positions,
                              const int* entry_of_token, const int* table, int table_width, int num_tokens, int nkv,
                              int hd, int page_size, hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (!pack_fits(hd, page_size)) TS_FAIL("pack_values: head_dim=%d, page_size=%d not built", hd, page_size);
  if (nkv <= 0 || !table || table_width <= 0) TS_FAIL("pack_values: nkv=%d, block table of width %d", nkv, table_width);
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15)
    TS_FAIL("pack_values: tensors must be 16-byte aligned");
  const int64_t pieces = (int64_t)num_tokens * 2 * nkv * (hd / 8), blocks = (pieces + 255) / 256;
  if (pieces > 2147483647LL - 256) TS_FAIL("pack_values: too many tokens");
  const unsigned per = hd / 8, heads = 2 * nkv;
  const PackValuesArgs a{(const unsigned char*)k_pages, (const unsigned char*)v_pages, k, v, positions, entry_of_token,
                         table, table_width, num_tokens, nkv, hd, page_size, per, inverse32(per), inverse32(heads)};
  TS_DISPATCH_TYPE(type, T,
      hipLaunchKernelGGL(pack_values_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, a));
  TS_CHECK_LAUNCH("pack_values");
  return 0;
}
