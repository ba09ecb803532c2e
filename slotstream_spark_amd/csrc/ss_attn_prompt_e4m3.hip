// Attention of many rows over pages of e4m3 numbers, causal rows and trees (the kernel is in ss_attn_prompt.hpp).
#include "ss_attn_prompt.hpp"

namespace ss {

hipError_t launch_attn_prompt_e4m3(const AttnArgs& a, int dim, hipStream_t st) {
  return a.tree ? launch_prompt_of<Bf16, true, true>(a, dim, st) : launch_prompt_of<Bf16, true, false>(a, dim, st);
}

}  // namespace ss
