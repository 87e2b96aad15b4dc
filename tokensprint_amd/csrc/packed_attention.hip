// Attention over keys and values of 4 bits: the entry point, and the kernels for bfloat16 activations.
#include "packed_attention_kernel.h"

int launch_packed_bf16(const PackedArgs& args, bool coop, hipStream_t stream) {
  TS_PACKED_CASES(false, false, bf16_t);
}

int ts_check_attention_args(const AttentionArgs& a, const char* who);

int ts_check_packed_args(const PackedArgs& args, const char* who) {
  const AttentionArgs& a = args.base;
  if (ts_check_attention_args(a, who)) return -1;
  if (!pack_fits(a.hd, a.page_size)) TS_FAIL("%s: head_dim=%d, page_size=%d not built", who, a.hd, a.page_size);
  const int group = a.nq / a.nkv;
  if (args.rows_per_token != (group < 16 ? group : 16) || args.head_blocks != (group + 15) / 16)
    TS_FAIL("%s: rows_per_token/head_blocks do not fit a group of %d", who, group);
  if ((int64_t)args.num_tiles * a.nkv * args.head_blocks > 1 << 30) TS_FAIL("%s: too many tiles", who);
  if (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages | (uintptr_t)args.partial_ml) & 15)
    TS_FAIL("%s: tensors must be 16-byte aligned", who);
  return 0;
}

// Workgroups of the kernel that shares keys out which the card holds at a time.
extern "C" int ts_packed_resident() { return compute_units(); }

// `coop`: all items' keys shared out over `workgroups` workgroups, else a wavefront per item.
extern "C" int ts_packed_attention(const PackedArgs* p, int type, int coop, hipStream_t stream) {
  const PackedArgs& args = *p;
  const AttentionArgs& a = args.base;
  if (a.num_tokens <= 0 || args.num_tiles <= 0) return 0;
  if (type != TS_F32 && type != TS_BF16) TS_FAIL("packed_attention: element type code %d", type);
  if (ts_check_packed_args(args, "packed_attention")) return -1;
  if (!args.tiles && (args.num_tiles != a.num_entries || a.num_tokens != a.num_entries))
    TS_FAIL("packed_attention: without a tile list there is one token per entry");
  if (coop) {
    if (args.workgroups < 0 || args.workgroups > 1 << 20 || (args.workgroups && (!args.partial_o || !args.partial_ml || !args.arrivals)))
      TS_FAIL("packed_attention: %d workgroups need partial buffers and arrival counts", args.workgroups);
  }
  if (has_score_extras(a))
    return type == TS_BF16 ? launch_packed_bf16_scores(args, coop != 0, stream) : launch_packed_f32_scores(args, coop != 0, stream);
  return type == TS_BF16 ? launch_packed_bf16(args, coop != 0, stream) : launch_packed_f32(args, coop != 0, stream);
}
