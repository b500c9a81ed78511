// attn_prompt.cuh -- arguments shared by the prompt-attention kernels.
#pragma once
#include "llm_ops.cuh"

namespace simp {

struct AttnPromptArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* q_off;
  const int32_t* k_off;
  int64_t total_q, total_k, q_stride, kv_stride, out_stride;
  int n_seqs, H, G, rep, D;
  float scale_log2;   // scale * log2(e): weights are powers of two
  int* status;
};

bool attn_prompt_tc_takes(const AttnPromptArgs& a, int dtype);
int attn_prompt_tc(const AttnPromptArgs& a, int dtype);

}  // namespace simp
