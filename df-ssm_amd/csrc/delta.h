// Arguments and device helpers shared by the gated delta rule's kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "packed.h"

namespace dfssm {

struct DeltaArgs {
  const uint16_t *q, *k, *v;  // 16-bit rows, ld_* elements from token to token, heads contiguous
  const float *g, *beta;
  const float* state;         // (n_slots, Hv, Dv, Dk)
  float* state_out;           // the same tensor, or one of its shape
  const int32_t* slots;       // (n_seq), or null: sequence b has slot b
  const int32_t* cu;          // (n_seq + 1), or null: len tokens each
  uint16_t* out;
  int64_t ld_q, ld_k, ld_v, ld_g, ld_beta, ld_out;
  int64_t n_tokens, len;
  int n_seq, n_slots, Hk, Hv, Dk, Dv;
  int bf16, l2norm;
  float scale;
};

// Token by token (delta.hip), and over chunks with the workspace of delta_chunk_workspace (delta_chunk.hip).
hipError_t launch_delta_token(const DeltaArgs& a, hipStream_t s);
hipError_t launch_delta_chunked(const DeltaArgs& a, void* workspace, hipStream_t s);
size_t delta_chunk_workspace(const DeltaArgs& a);

__device__ __forceinline__ float l2_factor(float ss) { return __builtin_amdgcn_rsqf(ss + 1e-6f); }  // (1 ulp)

}  // namespace dfssm
