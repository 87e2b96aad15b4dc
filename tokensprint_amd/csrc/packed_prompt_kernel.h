// Prompts' attention over keys and values of 4 bits: 32 query rows a wavefront, four wavefronts an item, as over a
// cache of bfloat16 (attention_prefill_tall_kernel.h), whose tiles in LDS are made here from a turn's codes: head sizes 64 and 128.
//
// A turn is 64 keys, four blocks of a page; a wavefront turns one block's codes into float16 numbers step (code - zero)
// and writes them where its operands are read, once for the 128 rows of an item.  Numbers count a power of two times, so
// that they stand high in float16's range (PromptScale); queries are float16 as well, scaled by a power of two a row
// (their bfloat16 bits are exact then), and so are weights, which count 2^15 times: as they are, 9 below the row's largest
// score they would have fewer than 11 bits, and 17 below none (4,000 keys 14 below one of no value: 0.6 % of the result;
// now bits go from 20 below on).  What is rounded is a key's or a value's number, to 11 bits (a score s that one element
// makes alone is off by 2^-11 s at the most).  (As
// step (16 + code) less a rounded step (16 + zero), in 4 instructions less, results were three times as far off.)
// The next turn's codes, asked for a turn ahead, become numbers between the scores' products, a word a step, and the second
// half of a turn's weights are made between the first half's products: a turn is one meeting of the workgroup.
// 4,096 tokens behind 4,096, 32 heads of 128 over 8: 475 to 495 us by card, 835 to 870 TFLOP/s (all codes of a turn first, then
// its products: 0.6 % longer; over a cache of bfloat16 a tenth shorter), vector instructions 59 % of a SIMD's cycles and
// matrix instructions 36 %.
#pragma once
#include "attention_prefill_tall_kernel.h"
#include "packed_attention_kernel.h"

// What a block's numbers count: values 2^11 times where its largest step is below 2, 2^(11 - n) times where it is below
// 2^(1 + n), n up to 15, keys 2^4 times below 256, else 2^-4: 15 steps stay below float16's largest number, and a step of
// float16's smallest has 11 bits in an ordinary block (in another, values are held to 2^(n - 36), large keys to 2^-21).
// Nearly every block is ordinary; another is told to the workgroup beside the tile, and the scores and weights of a turn with
// such a block make up for it: from there on the weights of ordinary blocks count 2^n times less, and have 11 bits down to
// 2^(n - 29) of the row's largest.
// (A sixteenth for all, the most that holds the largest step, took 1.7 % less time and left numbers below 2^-10 without all
// their bits: values of 1e-4 came out 0.3 % off, of 1e-5 3 %.)
struct PromptScale {
  static constexpr int kKeys = 4, kValues = 11;
  static constexpr int kLargeKeys = 1, kValuesDown = 2;                // a block's flags: of its keys, and n times the other
};

// Tiles and operands lie as there. SETS sets of four wavefronts split an item's turns and merge through LDS at the end.
template <int HD, int SETS, bool EXTRA>
__global__ __launch_bounds__(256 * SETS) __attribute__((amdgpu_waves_per_eu(2, 2))) void packed_prompt_kernel(PackedArgs args) {
  constexpr int TILES = 4, KEYS = 64, NB = HD / 32, PG = pack_groups(HD);
  constexpr int KS = HD / 16, DB = HD / 32, B = KEYS / 32, G = KEYS / 16;
  constexpr int SUB = HD / 32;                 // slots of 1 KB per sixteen keys
  constexpr int VALUES = KEYS * HD * 2;        // bytes of a turn's keys; its values lie behind them
  constexpr int BUF = 2 * VALUES;
  constexpr float kUp = 15.f;                  // weights and their sums count 2^kUp times
  static_assert((HD == 64 || HD == 128) && G == TILES, "rows of 128 or 256 bytes, a block a wavefront");
  extern __shared__ __attribute__((aligned(1024))) unsigned char prefill_lds[];
  __shared__ int s_flags[SETS][2][TILES], s_any[SETS];     // PromptScale's, of the rings' blocks; whether there are any
  __shared__ float s_down[SETS][TILES];
  const AttentionArgs& a = args.base;
  const int wave_all = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int wave = wave_all % TILES, set = SETS == 1 ? 0 : wave_all / TILES;
  const int c = lane % 32, h = lane / 32;
  const int group = a.nq / a.nkv;
  const int heads = a.nkv * args.head_blocks;
  const int head_slot = blockIdx.x % heads;                   // one head per XCD's L2
  const int rank = blockIdx.x / heads;
  const int kvh = head_slot / args.head_blocks;
  const int hb = head_slot % args.head_blocks;
  const int P = a.page_size, lp = __builtin_ctz(P);
  const int tq = 16 / args.rows_per_token;                    // tokens of sixteen rows
  float scale_log2 = a.scale * 1.44269504088896341f;

  unsigned char* ring = prefill_lds + set * 2 * BUF;
  const int key_c = (c & 0x13) | ((c & 4) << 1) | ((c & 8) >> 1);       // sigma(c)
  const int key_f = HD == 128 ? key_c % 16 : key_c % 16 / 2;
  const unsigned k_read = key_c * (HD * 2), k_piece = h ^ key_f;
  const unsigned v_read = VALUES + (2 * c + (h ^ (c / 8 % 2))) * 16;

  // Where this lane's codes lie in their block, and where the numbers that they become go: as the lane (r, g) of a
  // block it holds elements 32 b + 8 g .. + 7 of token r's keys and tokens 4 g .. + 3 of elements 16 n + r of the values.
  constexpr int BYTES = pack_block_bytes(HD), CODES = pack_codes_bytes(HD);
  const int r16 = lane % 16, g4 = lane / 16;
  const unsigned at_code = lane * (NB * 4), at_s = CODES + g4 * PG * 16 + r16 % (4 * PG) * 4;
  const unsigned at_z = CODES + r16 / 4 * PG * 16 + r16 % 4 * 2;
  const unsigned k_write = (wave * 16 + r16) * (HD * 2) + (g4 ^ (HD == 128 ? r16 : r16 / 2)) * 16;
  const unsigned v_write = VALUES + wave * SUB * 1024 + (2 * r16 + ((g4 / 2) ^ (r16 / 8))) * 16 + g4 % 2 * 8;

  // the item, and the lane's row of it
  const int entry = uniform(args.tiles[rank * 3]), tok0 = uniform(args.tiles[rank * 3 + 1]),
            ntok = uniform(args.tiles[rank * 3 + 2]);
  const int in16 = c % 16 / args.rows_per_token;
  const int ti = (wave * 2 + c / 16) * tq + in16;
  const int hh = hb * 16 + c % 16 % args.rows_per_token;
  const int head = kvh * group + min(hh, group - 1);
  const bool row_ok = in16 < tq && ti < ntok && hh < group;
  // the query row in float16, its largest magnitude brought to 2^13 .. 2^14; `back`: what takes that and the keys' 2^4
  // out of a product
  f16x8 q[KS];
  float back;
  {
    const bf16_t* qrow = (const bf16_t*)a.q + ((int64_t)(tok0 + min(ti, ntok - 1)) * a.nq + head) * HD;
    bf16x8 y[KS];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      y[s] = *(const bf16x8*)(qrow + 16 * s + 8 * h);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!row_ok) y[s][j] = (bf16_t)0.f;
        top = fmaxf(top, fabsf((float)y[s][j]));
      }
    }
    top = halves_max(top);
    const int up = top > 0.f && top < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(top), 120) : 0;
    back = ldexpf(1.f, -PromptScale::kKeys - up);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) q[s][j] = (_Float16)ldexpf((float)y[s][j], up);
  }
  scale_log2 *= back;
  const int pos_first = uniform(a.positions[tok0]);           // positions are consecutive
  const ConstTable table = (ConstTable)(a.table + (int64_t)entry * a.table_width);
  const int pos_last = pos_first + ntok - 1;
  const int lo_all = first_visible(a, pos_first);

  const int row_pos = row_ok ? pos_first + ti : -1;
  const int row_lo = first_visible(a, row_pos);
  ScoreExtraLog2 x;
  if (EXTRA) {
    x = in_log2(score_extra(a, head, row_pos));
    x.row *= back, x.in *= back;
  }
  // the wavefront's tokens (scalars)
  const int t0 = wave * 2 * tq, t1 = min(ntok, (wave + 1) * 2 * tq);
  const int tile_first = pos_first + t0;
  const int tile_last = t0 < ntok ? pos_first + t1 - 1 : -1;
  const int tile_lo = first_visible(a, tile_first);
  const int tile_lo_last = first_visible(a, tile_last);

  // The item's turns, numbered from its first; this set takes turns set, set + SETS, ...:
  // `mine` of them, numbered j here.  Every set passes the same number of barriers.
  const KeyWalk walk = key_walk<KEYS>(a, lo_all);
  const int key_begin = walk.origin;
  const int nturns = (pos_last - key_begin) / KEYS + 1;
  const int rounds = (nturns + SETS - 1) / SETS;
  const int mine = (nturns - set + SETS - 1) / SETS;
  const int kb_first = key_begin + KEYS * set;
  const int last_page = pos_last >> lp;              // the last page the item may name
  // the page of this wavefront's block of the turn that will be sent for next (a page beyond the item's last is the
  // last again, one that a window has let go reads page 0: their keys are masked, and what the cache holds is finite)
  int next_page;
  auto fetch_id = [&](int v) { next_page = table[min((walk.real(v) + 16 * wave) >> lp, last_page)]; };
  fetch_id(kb_first);
  unsigned kw[NB], vw[NB], vs;
  unsigned ks[PG], kz[PG];
  int held;                                          // the first key of the block that they are of
  auto issue = [&](int j) {
    const int v = kb_first + KEYS * SETS * j, at_key = walk.real(v) + 16 * wave, in = at_key & (P - 1);
    held = next_page < 0 ? 1 << 30 : at_key;
    const int64_t at = (((int64_t)max(next_page, 0) * a.nkv + kvh) * P + in) / 16 * BYTES;
    const unsigned char* kp = (const unsigned char*)a.k_pages + at;
    const unsigned char* vp = (const unsigned char*)a.v_pages + at;
    load_words<NB>(kw, kp + at_code);
    load_words<NB>(vw, vp + at_code);
    vs = *(const unsigned*)(vp + at_s);
#pragma unroll
    for (int i = 0; i < PG; ++i) {
      ks[i] = *(const unsigned short*)(kp + at_z + i * 16);
      kz[i] = *(const unsigned short*)(kp + at_z + i * 16 + 8);
    }
    fetch_id(v + KEYS * SETS);
  };
  // Of the item's last turn: steps that a page holds of nobody's keys are none, and have no say in scales.
  auto mask_steps = [&]() {
    const int key = held + g4 * 4 + lane % 4 * 2;
    const unsigned there = (key <= pos_last ? 0xffffu : 0u) | (key < pos_last ? 0xffff0000u : 0u);
    vs &= lane % 4 < 2 ? there : ~0u;
#pragma unroll
    for (int i = 0; i < PG; ++i) ks[i] = held + r16 <= pos_last ? ks[i] : 0u;
  };
  // The values' n, ahead of a turn, so that another than 0 is a branch's.
  const unsigned step_lanes = lane % 4 < 2 ? 0x40004000u : 0u;         // bit 14: 2 and more
  int down = 0;
  auto look = [&]() {
    down = 0;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64((vs & step_lanes) != 0) == 0, 1)) return;
    asm volatile("" ::: "memory");             // keeps this a branch
    const unsigned exponent = step_lanes != 0 ? max(vs >> 10 & 31u, vs >> 26 & 31u) : 0u;
    down = uniform((int)wave_max((float)exponent)) - 15;
  };
  // Steps as the numbers want them, keys', then values', and the block's flags.  (Without a branch, which would end the
  // stretch in which the compiler may order products and these.)
  int flags_now = 0, told = 0;
  // (of their own: in the registers that loads go to, they would make the next turn's be waited for)
  _Float16 key_step[PG];
  unsigned value_steps = 0;
  auto scale_keys = [&]() {
    unsigned top = ks[0];
#pragma unroll
    for (int i = 1; i < PG; ++i) top = max(top, ks[i]);
    const bool large = __builtin_amdgcn_ballot_w64(top >= 0x5c00u) != 0;          // 256
    const _Float16 up = __builtin_bit_cast(_Float16, (unsigned short)(large ? 0x2c00u : 0x4c00u));
    flags_now = large ? PromptScale::kLargeKeys : 0;
#pragma unroll
    for (int i = 0; i < PG; ++i)
      key_step[i] = __builtin_bit_cast(_Float16, (unsigned short)ks[i]) * up;
  };
  auto scale_values = [&]() {
    flags_now += PromptScale::kValuesDown * down;
    const unsigned by = (unsigned)(15 + PromptScale::kValues - down) * 0x04000400u;
    const unsigned up = step_lanes != 0 ? by : 0x3c003c00u;
    value_steps = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, vs) * __builtin_bit_cast(f16x2, up));
  };
  // (a wavefront that has told of a block once does so for all that follow, so that what stands there is this turn's)
  auto tell = [&](int* flags) {
    if ((flags_now | told) == 0) return;
    told = 1;
    flags[wave] = flags_now;
    s_any[set] = 1;
  };
  // Codes into the tile, a word of a lane's at a time (keys, then values): 16 + c, less 16 + zero (exact), times the step.
  auto unpack = [&](unsigned char* buf, int n) {
    if (n < NB) {
      const int b = n;
      unsigned w[4];
      whole_keys(kw[b], __builtin_bit_cast(_Float16, (unsigned short)kz[b / 2]), w);
      const f16x2 s = {key_step[b / 2], key_step[b / 2]};
      u32x4 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, w[i]) * s);
      unsigned piece = k_write;                    // (worked out here: a register for every word would not be left)
      asm volatile("" : "+v"(piece));
      *(u32x4*)(buf + (piece ^ (64 * b))) = out;
    } else {
      const int b = n - NB;
      const u32x4 scale = packed_scale_of<PG>(value_steps, b / 2);
      const f16x2 s01 = f16x2{half_of(scale, 0), half_of(scale, 1)};
      const f16x2 s23 = f16x2{half_of(scale, 2), half_of(scale, 3)};
      unsigned w[4];
      whole_values(vw[b], f16x2{half_of(scale, 4), half_of(scale, 5)}, f16x2{half_of(scale, 6), half_of(scale, 7)}, w);
      typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
#pragma unroll
      for (int i = 0; i < 2; ++i)                  // elements 32 b + r, 32 b + 16 + r
        *(u32x2*)(buf + v_write + b * 1024 + i * 512) =
            u32x2{__builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, w[2 * i]) * s01),
                  __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, w[2 * i + 1]) * s23)};
    }
  };
  auto unpack_all = [&](unsigned char* buf) {
    scale_keys();
    scale_values();
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n) unpack(buf, n);
  };

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = -INFINITY, l = 0.f;      // l: this lane's share of the row's sum
  int up_o = PromptScale::kValues;   // o counts 2^(kUp + up_o) times: as the least of the blocks' values so far

  static_assert(KS == 2 * NB, "a word to unpack for every step of the scores");
  auto work = [&](int j, int kb, const unsigned char* buf, unsigned char* next, const int* flags) {
    const int any = s_any[set];
    // a step's operands are asked for ahead of its products
    constexpr int AHEAD = 2;
    f16x8 kf[AHEAD][B];
    auto read_keys = [&](int s) {
      const unsigned char* at = buf + k_read + ((k_piece ^ (2 * s)) * 16);
#pragma unroll
      for (int b = 0; b < B; ++b) kf[s % AHEAD][b] = *(const f16x8*)(at + b * (32 * HD * 2));
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) read_keys(s);
    f32x16 st[B];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[b][i] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int b = 0; b < B; ++b)
        st[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[s % AHEAD][b], q[s], st[b], 0, 0, 0);
      if (s + AHEAD < KS) read_keys(s + AHEAD);
      if (s == 0) scale_keys();
      if (s == 1) scale_values();
      unpack(next, s);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (j + 2 < mine) issue(j + 2);
    f16x8 vf[G][DB];
    auto read_values = [&](int g) {
#pragma unroll
      for (int db = 0; db < DB; ++db) vf[g][db] = *(const f16x8*)(buf + v_read + (g * SUB + db) * 1024);
    };
    read_values(0), read_values(1);
    __builtin_amdgcn_sched_barrier(0);
    const bool other = uniform(any) != 0;
    // keys that count 2^-4 times: their products as the others'
    auto even_keys = [&]() {
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          st[b][i] *= uniform(flags[2 * b + i / 8]) & PromptScale::kLargeKeys ? 256.f : 1.f;
    };
    const int at = kb + 8 * h;       // register i of block b: key at + 32 b + 16 (i / 8) + i % 8
    if (EXTRA) {
      if (other) even_keys();
      if (x.capped) {
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[b][i] = capped_log2(x, st[b][i]);
      } else {
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[b][i] *= x.row;
      }
      if (x.sloped) {
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[b][i] = off_by_distance(x, st[b][i], at + 32 * b + 16 * (i / 8) + i % 8);
      }
      scale_log2 = 1.f;
    }
    if (!(kb + KEYS - 1 <= tile_first && kb >= tile_lo_last) || (!EXTRA && other)) {
      asm volatile("" ::: "memory");   // keeps this a branch
      if (!EXTRA && other) even_keys();
      // (a key's number is a constant beyond the lane's first: the row's bounds are brought
      // there once a turn, so no register holds a key's)
      const int last = row_pos - at, lowest = row_lo - at, kept = a.keep - at;
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int n = 32 * b + 16 * (i / 8) + i % 8;
          st[b][i] = (n <= last && (n >= lowest || n < kept)) ? st[b][i] : -INFINITY;
        }
    }
    float mx[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      mx[b] = st[b][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx[b] = max2(mx[b], st[b][i]);
    }
    const float top = halves_max(B == 2 ? max2(mx[0], mx[B - 1]) : mx[0]) * scale_log2;
    if (top > m) {
      const float corr = __builtin_amdgcn_exp2f(m - max2(top, -1e30f));
      m = top;
      l *= corr;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= corr;
    }
    const float rise = kUp - max2(m, -1e30f);
    float by = scale_log2;
    unsigned ones[G];                // what two weights count in the row's sum, which knows no scales
#pragma unroll
    for (int g = 0; g < G; ++g) ones[g] = 0x3c003c00u;
    if (other) {
      asm volatile("" ::: "memory");
      int up[G], least = up_o;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        up[g] = PromptScale::kValues - uniform(flags[g]) / PromptScale::kValuesDown;
        least = min(least, up[g]);
      }
      if (least != up_o) {
        const float change = PackedLift::power(least - up_o);
        up_o = least;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[db][i] *= change;
      }
      // (weights of 2^-n: scores less by n)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        ones[g] = (unsigned)(15 + up[g] - up_o) * 0x04000400u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          st[g / 2][g % 2 * 8 + i] = fmaf(st[g / 2][g % 2 * 8 + i], by, (float)(up_o - up[g]));
      }
      by = 1.f;
    }
    // the first block's weights, then its values' products between those of the second
    f16x8 pv[G];
    // (the row's sum is of the weights as they enter the products, two at a time)
    float before = 0.f;
    auto weight = [&](int b, int i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[b][i], by, rise));
      if (i % 2 == 0) {
        before = p;
        return;
      }
      const f16x2 two = {(_Float16)before, (_Float16)p};
      l = __builtin_amdgcn_fdot2(two, __builtin_bit_cast(f16x2, ones[2 * b + i / 8]), l, false);
      pv[2 * b + i / 8][i % 8 - 1] = two[0], pv[2 * b + i / 8][i % 8] = two[1];
    };
    auto product = [&](int g, int db) { o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[g][db], pv[g], o[db], 0, 0, 0); };
#pragma unroll
    for (int i = 0; i < 16; ++i) weight(0, i);
    read_values(2), read_values(3);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i < 2 * DB) product(i / DB, i % DB);
      weight(1, i);
      if (i % 2) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int n = 0; n < 2 * DB; ++n) product(2 + n / DB, n % DB);
  };

  auto meet = [&]() {                          // everyone's codes are in the tile, and everyone is through with this turn's
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (lane == 0) s_flags[set][0][wave] = s_flags[set][1][wave] = s_any[set] = 0;
  meet();
  if (mine > 0) {
    issue(0);
    if (held + 15 > pos_last) mask_steps();
    look();
    unpack_all(ring);
    tell(s_flags[set][0]);
    if (mine > 1) issue(1);
  }
  meet();
  for (int j = 0; j < rounds; ++j) {
    const int kb = walk.real(kb_first + KEYS * SETS * j);
    unsigned char *buf = ring + (j & 1) * BUF, *next = ring + (~j & 1) * BUF;
    if (j + 1 < mine && held + 15 > pos_last) mask_steps();
    look();
    // (behind the last turn what is left in the registers once more, into a tile that nobody reads)
    const bool seen = kb <= tile_last && (kb + KEYS - 1 >= tile_lo || kb < a.keep);
    if (j < mine && !seen) {
      unpack_all(next);
      if (j + 2 < mine) issue(j + 2);
    }
    asm volatile("" ::: "memory");             // (one branch and another: as the two ways of one, the sums would be moved)
    if (j < mine && seen) work(j, kb, buf, next, s_flags[set][j & 1]);
    tell(s_flags[set][~j & 1]);
    meet();
  }

  l = halves_sum(l) * 0x1p-15f;                // (by all lanes: it crosses lanes)
  bf16_t* out = (bf16_t*)a.out + ((int64_t)(tok0 + ti) * a.nq + head) * HD;
  // Unit u of the results: registers 8 (u % 2) .. + 7 of o[u / 2], elements 16 u + 4 h .. + 3 and
  // 16 u + 8 + 4 h .. + 3.  The lane's halves exchange four each, and a lane has eight in a row.
  auto store_unit = [&](int u, const float* v) {
    typedef unsigned U2 __attribute__((ext_vector_type(2)));
    typedef unsigned U4 __attribute__((ext_vector_type(4)));
    bf16x4 lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = (bf16_t)v[i], hi[i] = (bf16_t)v[4 + i];
    const U2 y = __builtin_bit_cast(U2, lo), z = __builtin_bit_cast(U2, hi);
    auto s0 = __builtin_amdgcn_permlane32_swap(y[0], z[0], false, false);
    auto s1 = __builtin_amdgcn_permlane32_swap(y[1], z[1], false, false);
    const U4 eight = {s0[0], s1[0], s0[1], s1[1]};
    if (row_ok) *(U4*)(out + 16 * u + 8 * h) = eight;
  };
  if constexpr (SETS == 1) {
    const float sum = sum_with_sink(l, m, a.sink, head);
    const float inv = sum > 0.f ? PackedLift::power(-15 - up_o) / sum : 0.f;
#pragma unroll
    for (int u = 0; u < 2 * DB; ++u) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = o[u / 2][8 * (u % 2) + i] * inv;
      store_unit(u, v);
    }
  } else {
    // The sets leave their results in LDS, in the rings' space: [set][tile][register][lane], the
    // row statistics behind them; each then adds up its share of the units, set by set.
    constexpr int REGS = DB * 16, UNITS = 2 * DB / SETS;
    static_assert(2 * DB % SETS == 0, "whole units");
    float* lds_o = (float*)prefill_lds;
    float* lds_ml = lds_o + SETS * TILES * REGS * kWave;
    __syncthreads();                             // the rings have been read for the last time
#pragma unroll
    for (int i = 0; i < REGS; ++i) lds_o[(wave_all * REGS + i) * kWave + lane] = o[i / 16][i % 16];
    lds_ml[wave_all * 2 * kWave + lane] = m;
    lds_ml[(wave_all * 2 + 1) * kWave + lane] = l;
    if (lane == 0) s_down[set][wave] = PackedLift::power(-15 - up_o);
    __syncthreads();
    float ms[SETS], w[SETS], m_use = -1e30f, sum = 0.f;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      ms[s] = lds_ml[(s * TILES + wave) * 2 * kWave + lane];
      m_use = max2(m_use, ms[s]);
    }
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      // (a set that saw no key of this row has m = -inf and weight 0)
      w[s] = __builtin_amdgcn_exp2f(ms[s] - m_use);
      sum += lds_ml[((s * TILES + wave) * 2 + 1) * kWave + lane] * w[s];
      w[s] *= s_down[s][wave];
    }
    sum = sum_with_sink(sum, m_use, a.sink, head);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
      const int u = set * UNITS + n;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int s = 0; s < SETS; ++s) v[i] += lds_o[((s * TILES + wave) * REGS + u * 8 + i) * kWave + lane] * w[s];
        v[i] *= inv;
      }
      store_unit(u, v);
    }
  }
}


template <int HD, int SETS, bool EXTRA>
static int launch_packed_prompt_of(const PackedArgs& args, hipStream_t stream) {
  constexpr int TILES = 4, KEYS = 64;
  const int heads = args.base.nkv * args.head_blocks;
  constexpr int rings = SETS * 2 * KEYS * HD * 4, merge = SETS == 1 ? 0 : SETS * TILES * (HD / 2 + 2) * kWave * 4;
  constexpr int lds = rings > merge ? rings : merge;
  static_assert(lds + 1024 <= 160 * 1024, "LDS of a compute unit, with the flags in front");
  auto kernel = packed_prompt_kernel<HD, SETS, EXTRA>;
  static bool raised[64] = {};                 // per instantiation and device
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) TS_FAIL("packed_prompt: no current device below 64");
  if (!raised[device]) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
      TS_FAIL("packed_prompt: cannot raise the LDS limit to %d bytes", lds);
    raised[device] = true;
  }
  hipLaunchKernelGGL(kernel, dim3(args.num_tiles * heads), dim3(256 * SETS), lds, stream, args);
  TS_CHECK_LAUNCH("packed_prompt");
  return 0;
}

template <bool EXTRA>
static int launch_packed_prompt_forms(const PackedArgs& args, int sets, hipStream_t stream) {
  if (args.base.hd == 128)
    return sets == 2 ? launch_packed_prompt_of<128, 2, EXTRA>(args, stream) : launch_packed_prompt_of<128, 1, EXTRA>(args, stream);
  return sets == 2 ? launch_packed_prompt_of<64, 2, EXTRA>(args, stream) : launch_packed_prompt_of<64, 1, EXTRA>(args, stream);
}

int launch_packed_prompt(const PackedArgs& args, int sets, hipStream_t stream);
int launch_packed_prompt_scores(const PackedArgs& args, int sets, hipStream_t stream);
