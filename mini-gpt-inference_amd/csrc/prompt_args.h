// prompt_args.h -- the arguments of packed prompt attention (prompt_attention.h). Strides in
// elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mgi {

struct PromptArgs {
  void* out;
  int64_t o_st, o_sh, o_sd;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_st, q_sh, q_sd;
  int64_t k_st, k_sh, k_sd;
  int64_t v_st, v_sh, v_sd;
  const void* starts;   // [B + 1]
  int64_t cu_s;
  int cu_i64;
  int B, T, Hq, G, D;
  int heads;            // query heads of a workgroup: 1, 2 or 4, a divisor of G
  int zero_rest;        // rows of no sequence become 0
  int vec;              // 16-byte pieces of contiguous rows (else element by element)
  float scale_log2;     // |scale| * log2(e) (1 for a scale of 0)
  uint32_t q_flip;      // sign bits of a word of q, for a negative scale
  int q_zero;           // scale is 0
};
constexpr int kPromptMaxDim = 256;
constexpr int kPromptRows = 128;  // query rows of a workgroup, over its heads

hipError_t launch_prompt_f32(const PromptArgs& a, hipStream_t stream);
hipError_t launch_prompt_bf16(const PromptArgs& a, hipStream_t stream);
hipError_t launch_prompt_f16(const PromptArgs& a, hipStream_t stream);

}  // namespace mgi
