// Attention of many rows: the kernels over 16-bit pages with causal rows (the kernel is in ss_attn_prompt.hpp).
#include "ss_attn_prompt.hpp"

namespace ss {

// Workgroups that share the output dimensions of a row tile (a quarter each where pages of 16 tokens of 16 bits take more registers).
int attn_prompt_parts(int dim, int page_shift, bool e4m3) { return dim < 256 ? 1 : page_shift >= 5 || e4m3 ? 2 : 4; }

hipError_t launch_attn_prompt(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  return fp16 ? launch_prompt_of<Fp16, false, false>(a, dim, st) : launch_prompt_of<Bf16, false, false>(a, dim, st);
}

}  // namespace ss
