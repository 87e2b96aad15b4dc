// Prompts' attention over keys and values of 4 bits: the entry point, and the kernels without score extras.
#include "packed_prompt_kernel.h"

int launch_packed_prompt(const PackedArgs& args, int sets, hipStream_t stream) {
  return launch_packed_prompt_forms<false>(args, sets, stream);
}

int ts_check_packed_args(const PackedArgs& args, const char* who);

// 1 if ts_packed_prompt takes this head size (bfloat16 activations).
extern "C" int ts_packed_prompt_fits(int hd) { return hd == 64 || hd == 128; }

// `tiles` lists items (entry, first flat token, tokens) of at most eight times 16 / rows_per_token consecutive tokens each;
// `sets`: of four wavefronts that split an item's keys, 1 or 2.
extern "C" int ts_packed_prompt(const PackedArgs* p, int sets, hipStream_t stream) {
  const PackedArgs& args = *p;
  const AttentionArgs& a = args.base;
  if (a.num_tokens <= 0 || args.num_tiles <= 0) return 0;
  if (ts_check_packed_args(args, "packed_prompt")) return -1;
  if (!ts_packed_prompt_fits(a.hd)) TS_FAIL("packed_prompt: head_dim=%d not built", a.hd);
  if (!args.tiles) TS_FAIL("packed_prompt: no tile list");
  if (sets != 1 && sets != 2) TS_FAIL("packed_prompt: %d sets", sets);
  return has_score_extras(a) ? launch_packed_prompt_scores(args, sets, stream) : launch_packed_prompt(args, sets, stream);
}
