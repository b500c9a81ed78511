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

// Tensor-core forms; 1: the call is not for them (nothing was launched).
int attn_prompt_tc(const AttnPromptArgs& a, int dtype);    // 16-bit types
int attn_prompt_f32_tc(const AttnPromptArgs& a);           // f32
// Scratch that is refused (inside a recording) or not to be had sends a call to the FFMA kernel, which needs none; the
// allocation's error must not be taken for that launch's.
inline int attn_no_scratch() {
  cudaGetLastError();
  return 1;
}
// Rows to padded rows (f32: three bf16 planes), see attn_prompt_tc.cu.
struct AttnPack {
  const void* src;
  void* dst;
  uint8_t* odd;   // f32: per row and head, whether something is not finite
  int64_t rows, stride;
  int heads;
};
int attn_pack(bool split, const AttnPack& q, const AttnPack& k, const AttnPack& v, int D, int DP, int* any);

}  // namespace simp
