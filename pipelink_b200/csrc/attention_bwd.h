// Arguments of the attention backward kernels (attention_bwd.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace plb {

struct AttnBwdParams {
  const __nv_bfloat16* out;
  const __nv_bfloat16* d_out;
  const float* lse;          // [batch * q_heads, seq], natural log
  // Left by the first kernel for the second, per 128-row tile of a query head: -delta, and the log-sum-exp as it is
  // added to S, as tiles of constants (32 bytes a row); with a soft cap the latter as fp32 in base 2, negated.
  // -inf where a row has no probabilities.
  uint8_t* lse2;
  uint8_t* delta;
  __nv_bfloat16* dq;
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  int batch, seq, tiles, q_heads, kv_heads, group;
  int64_t seq_pad;           // tiles * 128
  int window;                // 0 = none
  float scale, scale_log2, inv_scale_log2;
  float cap_in, cap_out;     // soft cap: y = cap_out * tanh(score * cap_in) in base 2
  float4* partial;           // two slots of fp32 sums of dK and dV a run
  Status* status;
};

struct AttnBwdArgs {
  const void *q, *k, *v, *out, *d_out;
  const float* lse;
  void *dq, *dk, *dv;
  void* workspace;           // attention_bwd_workspace_bytes(), 16-byte aligned
  int batch, seq, q_heads, kv_heads;
  float scale, softcap;
  int window;
  int num_sms;
  Status* status;            // or null: failures go unreported
};

size_t attention_bwd_workspace_bytes(int batch, int seq, int q_heads, int kv_heads, int window);
cudaError_t launch_attention_bwd(const AttnBwdArgs& a, cudaStream_t stream);

}  // namespace plb
