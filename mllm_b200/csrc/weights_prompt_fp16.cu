// The attention weights of prompts: fp16 queries.  A type a file: there are many kernels.
#include "weights_prompt.cuh"

namespace mb200 {

int launch_weights_prompt_fp16(const WeightsPromptArgs& a, cudaStream_t s) { return launch_prompt<__half>(a, s); }

}  // namespace mb200
