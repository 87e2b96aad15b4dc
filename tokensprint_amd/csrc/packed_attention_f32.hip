// Attention over keys and values of 4 bits: float32 activations.
#include "packed_attention_kernel.h"

int launch_packed_f32(const PackedArgs& args, bool coop, hipStream_t stream) {
  TS_PACKED_CASES(true, false, float);
}
