// Keys and values into a cache of 4 bits (packed_kv.h), with everything that lies between their projection and
// attention, and back out of it.
//
// One launch norms and turns query and key heads (qk_prepare.hip's arithmetic), rounds keys to the
// activation type, as a wider cache would keep them, and quantises keys and values, eight elements a lane.  A wave
// takes a head of neighbouring tokens, for queries and keys (a token's keys are words of their own).  Four tokens share
// words of values, so there a wave takes those of a run of up to four that share words, sixteen lanes each, and makes
// the words between its lanes (pack_turned_round); of a run that is not whole, what the words hold of other tokens is read first; no
// other request has tokens in that page's block, and a step's tokens of one request are in order.  Prompts: four heads a wave,
// which its tokens' positions and pages are looked up for once.  Bound by the instructions, 200 for eight elements:
// 16,384 tokens with 8 heads of 128 take 30 us, their bytes would 18; back out of the cache 19.
#include "packed_kv.h"
#include "qk_prepare.h"

// How a step's tokens and heads go round the waves: first those that take a head of 64 / lanes tokens (`rows`), then those
// that take runs of tokens that share words of values, and units of sixteen lanes: two heads of up to 64
// elements, one of up to 128, half of a longer one.
constexpr int kPackHeads = 4;
struct PackWaves {
  unsigned rows, values;                     // waves
  unsigned head_parts, head_parts_inv;       // waves that share a window's heads
  unsigned unit_parts, unit_parts_inv;       // that share a window's units
  int units, window;                         // window: tokens whose runs (by their first token) a wave takes
};
static int pack_lanes(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }
// Steps that fill the card many times over: four heads and the runs of four tokens a wave; fewer: one, for the sake of
// the time of one.
static bool pack_waves(PackWaves& w, int& heads, unsigned& blocks, int64_t tokens, int row_heads, int nkv, int lanes) {
  w.units = (nkv * lanes + 15) / 16;
  const int64_t in_wave = kWave / lanes, windows = (tokens + in_wave - 1) / in_wave;
  const bool many = windows * row_heads > 16384;
  heads = many ? kPackHeads : 1, w.window = many ? 4 : 1;
  w.head_parts = (row_heads + heads - 1) / heads, w.unit_parts = (w.units + heads - 1) / heads;
  w.head_parts_inv = inverse32(w.head_parts), w.unit_parts_inv = inverse32(w.unit_parts);
  const int64_t rows = windows * w.head_parts, values = (tokens + w.window - 1) / w.window * w.unit_parts;
  if (rows + values > 2147483647LL) return false;
  w.rows = (unsigned)rows, w.values = (unsigned)values, blocks = (unsigned)((rows + values + 3) / 4);
  return true;
}

// The runs of a wave of the second kind, one after the other (all of it is the same in all lanes).
struct PackRuns {
  int token, count, entry, pos;              // the run: its first token, how many, whose, where
  int part;                                  // which of the waves that share the window's units
  int base, first_pos, first_entry;          // (of lane l: of token base + l)
  unsigned firsts, left;
  template <typename ARGS>
  __device__ __forceinline__ PackRuns(const ARGS& a, unsigned wave) {
    const unsigned at = divided(wave, a.waves.unit_parts, a.waves.unit_parts_inv);
    part = (int)(wave - at * a.waves.unit_parts);
    base = (int)at * a.waves.window;
    const int t = base + (int)(threadIdx.x % kWave % 8), here = min(t, a.num_tokens - 1), before = max(here - 1, 0);
    first_pos = a.positions[here], first_entry = a.entry_of_token[here];
    const bool goes_on = t > 0 && t < a.num_tokens && (first_pos & 3) != 0 && a.entry_of_token[before] == first_entry &&
                         a.positions[before] == first_pos - 1;
    firsts = (unsigned)__builtin_amdgcn_ballot_w64(!goes_on) & 0xffu;
    left = firsts & ((1u << min(a.waves.window, a.num_tokens - base)) - 1u);
  }
  __device__ __forceinline__ bool next() {
    if (left == 0) return false;
    const int c = __builtin_ctz(left);
    left &= left - 1;
    token = base + c;
    count = __builtin_ctz(firsts >> (c + 1) | 8u) + 1;
    pos = __builtin_amdgcn_readlane(first_pos, c), entry = __builtin_amdgcn_readlane(first_entry, c);
    return true;
  }
};

// What of a unit a lane has.
struct PackUnit {
  int head, sub;           // eight elements from 8 sub on
  bool held, there;        // the head, and elements of it
  __device__ __forceinline__ PackUnit(int u, int lanes, int lane, int hd, int nkv) {
    const int in = lane % 16;
    const int h = lanes == 8 ? 2 * u + in / 8 : lanes == 16 ? u : u / 2;
    sub = lanes == 8 ? in % 8 : lanes == 16 ? in : u % 2 * 16 + in;
    held = h < nkv, head = min(h, nkv - 1), there = held && sub * 8 < hd;
  }
  // The word of its block that is this lane's behind pack_turned_round; i: which of the four tokens is the lane's.
  __device__ __forceinline__ int word(int quad, int i, int slices) const {
    return (quad * 16 + sub % 2 * 8 + (i / 2 + sub / 2 % 2 * 2 + i % 2 * 4)) * slices + sub / 4;
  }
};

struct PackStoreArgs {
  const void *q, *k, *v;     // rows of T: heads of a token side by side, rows `*_stride` elements apart (q: or null)
  void* q_out;               // [T, nq, hd]
  unsigned char *k_pages, *v_pages;      // [num_pages, nkv, P / 16, block bytes]
  const float *q_weight, *k_weight, *cos, *sin;
  const int *positions, *entry_of_token, *table;
  int64_t stride;            // elements from a token's row to the next, the same in q, k and v
  int table_width, num_tokens, nq, nkv, hd, page_size;
  float eps;
  PackWaves waves;
};

// LANES: of a head (8, 16, 32), eight elements each; HEADS: that a wave takes one after the other.
template <typename T, int LANES, int HEADS>
__global__ __launch_bounds__(256) void pack_store_kernel(PackStoreArgs a) {
  const int lane = threadIdx.x % kWave;
  const int hd = a.hd, bytes = pack_block_bytes(hd), G = pack_groups(hd), NB = pack_slices(hd);
  unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / kWave);
  if (wave < a.waves.rows) {
    const int sub = lane % LANES;
    const unsigned window = divided(wave, a.waves.head_parts, a.waves.head_parts_inv);
    const int h0 = (int)(wave - window * a.waves.head_parts) * HEADS;
    const int token_at = (int)window * (kWave / LANES) + lane / LANES;
    const bool in_step = token_at < a.num_tokens, there = sub * 8 < hd;
    const int t = min(token_at, a.num_tokens - 1), at = there ? sub * 8 : 0;
    const int pos = a.positions[t], entry = a.entry_of_token[t], last = a.nq + a.nkv - 1;
    Eight<T> x[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = min(h0 + i, last);
      x[i].load((const T*)(h >= a.nq ? a.k : a.q) + (int64_t)t * a.stride + (int64_t)(h >= a.nq ? h - a.nq : h) * hd + at);
    }
    const int page = a.table[(int64_t)entry * a.table_width + (pos >> __builtin_ctz(a.page_size))];
    const int half = hd / 16;                                  // lanes of half a head
    const bool first = sub < half;
    const int other_lane = there ? lane - sub + (first ? sub + half : sub - half) : lane;
    f32x4_qk c0, c1, s0, s1;
    if (a.cos) {
      const int i0 = (first ? sub : there ? sub - half : 0) * 8;
      const float* cp = a.cos + (int64_t)pos * (hd / 2) + i0;
      const float* sp = a.sin + (int64_t)pos * (hd / 2) + i0;
      c0 = *(const f32x4_qk*)cp, c1 = *(const f32x4_qk*)(cp + 4);
      s0 = *(const f32x4_qk*)sp, s1 = *(const f32x4_qk*)(sp + 4);
    }
    const int slot = pos & (a.page_size - 1), token = slot % kPackTokens;
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = h0 + i;
      if (h > last) break;
      const bool key = h >= a.nq;
      const int head = key ? h - a.nq : h;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = there ? x[i].get(j) : 0.f;
      const float* w = key ? a.k_weight : a.q_weight;
      if (w) {
        const float rstd = head_rstd(v, LANES, hd, a.eps);
        const f32x4_qk w0 = *(const f32x4_qk*)(w + at), w1 = *(const f32x4_qk*)(w + at + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] *= rstd * w0[j]; v[4 + j] *= rstd * w1[j]; }
      }
      if (a.cos) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = __shfl(v[j], other_lane, kWave);
          v[j] = head_turned(v[j], other, j < 4 ? c0[j] : c1[j - 4], j < 4 ? s0[j] : s1[j - 4], first);
        }
      }
      if (!key) {
        if (there && in_step) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[i].set(j, v[j]);
          x[i].store((T*)a.q_out + ((int64_t)t * a.nq + head) * hd + at);
        }
        continue;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = there ? to_f32(from_f32<T>(v[j])) : 0.f;
      unsigned word;
      const PackGroup p = pack_eight(v, word, [](int j) { return j / 2 + 4 * (j % 2); });
      if (page < 0 || !in_step) continue;                      // no page behind this position: nothing is written
      unsigned char* block = a.k_pages + pack_block(page, a.nkv, head, a.page_size, slot, bytes);
      if (sub < NB * 4) ((unsigned*)block)[(sub % 4 * 16 + token) * NB + sub / 4] = pack_turned<kPackTurnK>(word);
      if (sub % 8 == 0 && there) {
        _Float16* scale = (_Float16*)(block + pack_codes_bytes(hd) + (token / 4 * G + sub / 8) * 16);
        scale[token % 4] = p.step;
        scale[4 + token % 4] = (_Float16)(-16.f - p.zero);
      }
    }
    return;
  }
  wave -= a.waves.rows;
  if (wave >= a.waves.values) return;
  PackRuns runs(a, wave);
  const int i = lane / 16, u0 = runs.part * HEADS;
  while (runs.next()) {
    const int j = i - (runs.pos & 3), t = runs.token + max(min(j, runs.count - 1), 0);
    const bool present = j >= 0 && j < runs.count;
    Eight<T> x[HEADS];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const PackUnit u(u0 + n, LANES, lane, hd, a.nkv);
      x[n].load((const T*)a.v + (int64_t)t * a.stride + (int64_t)u.head * hd + (u.there ? u.sub * 8 : 0));
    }
    const int page = a.table[(int64_t)runs.entry * a.table_width + (runs.pos >> __builtin_ctz(a.page_size))];
    const int slot = runs.pos & (a.page_size - 1), quad = slot % kPackTokens / 4;
    unsigned mask = 0;                                         // of the run's tokens in a word
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k >= (runs.pos & 3) && k < (runs.pos & 3) + runs.count) mask |= 0xf0fu << (4 * (k / 2 + 4 * (k % 2)));
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      if (u0 + n >= a.waves.units) break;
      const PackUnit u(u0 + n, LANES, lane, hd, a.nkv);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = u.there ? x[n].get(e) : 0.f;
      unsigned word;
      const PackGroup p = pack_eight(v, word, [](int e) { return e; });
      word = pack_turned_round(present ? word : 0u, lane);
      if (page < 0 || !u.held) continue;
      unsigned char* block = a.v_pages + pack_block(page, a.nkv, u.head, a.page_size, slot, bytes);
      if (u.sub < NB * 4) {
        unsigned* at = (unsigned*)block + u.word(quad, i, NB);
        if (runs.count < 4) word |= pack_unturned<kPackTurnV>(*at) & ~mask;
        *at = pack_turned<kPackTurnV>(word);
      }
      if (u.sub % 8 == 0 && u.there && present) {
        _Float16* scale = (_Float16*)(block + pack_codes_bytes(hd) + (quad * G + u.sub / 8) * 16);
        scale[i] = p.step;
        scale[4 + i] = (_Float16)(-16.f - p.zero);
      }
    }
  }
}

static int launch_pack_store(PackStoreArgs a, int type, hipStream_t stream) {
  const int lanes = pack_lanes(a.hd);
  int heads;
  unsigned blocks;
  if (!pack_waves(a.waves, heads, blocks, a.num_tokens, a.nq + a.nkv, a.nkv, lanes)) TS_FAIL("pack_store: too many tokens");
#define TS_LAUNCH(L) \
  if (heads == 1) hipLaunchKernelGGL((pack_store_kernel<T, L, 1>), dim3(blocks), dim3(256), 0, stream, a); \
  else hipLaunchKernelGGL((pack_store_kernel<T, L, kPackHeads>), dim3(blocks), dim3(256), 0, stream, a);
  TS_DISPATCH_TYPE(type, T, if (lanes == 8) { TS_LAUNCH(8) } else if (lanes == 16) { TS_LAUNCH(16) } else { TS_LAUNCH(32) });
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
// The same waves: a head of neighbouring tokens' keys, then runs that share words of values.  Positions without a page
// read as zeros.
struct PackValuesArgs {
  const unsigned char *k_pages, *v_pages;
  void *k, *v;                   // [T, nkv, hd]
  const int *positions, *entry_of_token, *table;
  int table_width, num_tokens, nkv, hd, page_size;
  PackWaves waves;
};

template <typename T, int LANES, int HEADS>
__global__ __launch_bounds__(256) void pack_values_kernel(PackValuesArgs a) {
  const int lane = threadIdx.x % kWave;
  const int hd = a.hd, bytes = pack_block_bytes(hd), G = pack_groups(hd), NB = pack_slices(hd);
  auto put = [&](T* dst, unsigned word, float step, float bias, auto place) {
    Eight<T> out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out.set(e, step * ((float)(word >> (4 * place(e)) & 15u) + 16.f + bias));
    out.store(dst);
  };
  unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / kWave);
  if (wave < a.waves.rows) {
    const int sub = lane % LANES;
    const unsigned window = divided(wave, a.waves.head_parts, a.waves.head_parts_inv);
    const int h0 = (int)(wave - window * a.waves.head_parts) * HEADS;
    const int t = (int)window * (kWave / LANES) + lane / LANES;
    if (t >= a.num_tokens || sub * 8 >= hd) return;
    const int pos = a.positions[t], entry = a.entry_of_token[t];
    const int page = a.table[(int64_t)entry * a.table_width + (pos >> __builtin_ctz(a.page_size))];
    const int slot = pos & (a.page_size - 1), token = slot % kPackTokens;
    unsigned word[HEADS];
    _Float16 step[HEADS], bias[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const unsigned char* block = a.k_pages + pack_block(max(page, 0), a.nkv, min(h0 + i, a.nkv - 1), a.page_size, slot, bytes);
      word[i] = ((const unsigned*)block)[(sub % 4 * 16 + token) * NB + sub / 4];
      const _Float16* scale = (const _Float16*)(block + pack_codes_bytes(hd) + (token / 4 * G + sub / 8) * 16) + token % 4;
      step[i] = scale[0], bias[i] = scale[4];
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      if (h0 + i < a.nkv)
        put((T*)a.k + ((int64_t)t * a.nkv + h0 + i) * hd + sub * 8, pack_unturned<kPackTurnK>(word[i]),
            page >= 0 ? (float)step[i] : 0.f, page >= 0 ? (float)bias[i] : 0.f, [](int j) { return j / 2 + 4 * (j % 2); });
    return;
  }
  wave -= a.waves.rows;
  if (wave >= a.waves.values) return;
  PackRuns runs(a, wave);
  const int i = lane / 16, u0 = runs.part * HEADS;
  while (runs.next()) {
    const int j = i - (runs.pos & 3), t = runs.token + max(min(j, runs.count - 1), 0);
    const bool present = j >= 0 && j < runs.count;
    const int page = a.table[(int64_t)runs.entry * a.table_width + (runs.pos >> __builtin_ctz(a.page_size))];
    const int slot = runs.pos & (a.page_size - 1), quad = slot % kPackTokens / 4;
    unsigned word[HEADS];
    _Float16 step[HEADS], bias[HEADS];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      const PackUnit u(min(u0 + n, a.waves.units - 1), LANES, lane, hd, a.nkv);
      const int sub = u.there ? u.sub : 0;                     // (a lane behind the head's end: of no consequence)
      const unsigned char* block = a.v_pages + pack_block(max(page, 0), a.nkv, u.head, a.page_size, slot, bytes);
      word[n] = u.sub < NB * 4 ? ((const unsigned*)block)[u.word(quad, i, NB)] : 0u;
      const _Float16* scale = (const _Float16*)(block + pack_codes_bytes(hd) + (quad * G + sub / 8) * 16) + i;
      step[n] = scale[0], bias[n] = scale[4];
    }
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      if (u0 + n >= a.waves.units) break;
      const PackUnit u(u0 + n, LANES, lane, hd, a.nkv);
      const unsigned own = pack_turned_round(pack_unturned<kPackTurnV>(word[n]), lane);
      if (present && u.there)
        put((T*)a.v + ((int64_t)t * a.nkv + u.head) * hd + u.sub * 8, own, page >= 0 ? (float)step[n] : 0.f,
            page >= 0 ? (float)bias[n] : 0.f, [](int e) { return e; });
    }
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
  const int lanes = pack_lanes(hd);
  PackValuesArgs a{(const unsigned char*)k_pages, (const unsigned char*)v_pages, k, v, positions, entry_of_token,
                   table, table_width, num_tokens, nkv, hd, page_size, {}};
  int heads;
  unsigned blocks;
  if (!pack_waves(a.waves, heads, blocks, num_tokens, nkv, nkv, lanes)) TS_FAIL("pack_values: too many tokens");
#define TS_LAUNCH(L) \
  if (heads == 1) hipLaunchKernelGGL((pack_values_kernel<T, L, 1>), dim3(blocks), dim3(256), 0, stream, a); \
  else hipLaunchKernelGGL((pack_values_kernel<T, L, kPackHeads>), dim3(blocks), dim3(256), 0, stream, a);
  TS_DISPATCH_TYPE(type, T, if (lanes == 8) { TS_LAUNCH(8) } else if (lanes == 16) { TS_LAUNCH(16) } else { TS_LAUNCH(32) });
#undef TS_LAUNCH
  TS_CHECK_LAUNCH("pack_values");
  return 0;
}
