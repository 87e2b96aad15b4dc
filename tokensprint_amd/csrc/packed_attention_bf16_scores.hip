// Attention over keys and values of 4 bits: bfloat16 activations, scores with a cap, a distance bias or a query temperature.
#include "packed_attention_kernel.h"

int launch_packed_bf16_scores(const PackedArgs& args, bool coop, hipStream_t stream) {
  TS_PACKED_CASES(false, true, bf16_t);
}
