// Prompts' attention over keys and values of 4 bits, scores with a cap, a distance bias or a query temperature.
#include "packed_prompt_kernel.h"

int launch_packed_prompt_scores(const PackedArgs& args, int sets, hipStream_t stream) {
  return launch_packed_prompt_forms<true>(args, sets, stream);
}
