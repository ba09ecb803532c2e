// Attention of many rows, the rows of trees of drafts, over 16-bit pages (the kernel is in ss_attn_prompt.hpp).
#include "ss_attn_prompt.hpp"

namespace ss {

hipError_t launch_attn_prompt_tree(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  return fp16 ? launch_prompt_of<Fp16, false, true>(a, dim, st) : launch_prompt_of<Bf16, false, true>(a, dim, st);
}

}  // namespace ss
