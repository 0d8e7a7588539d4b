// Arguments and device helpers shared by the gated delta rule's kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

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

constexpr int kSlotPad = -1;  // a negative slot: the sequence is padding
constexpr int kSlotBad = -2;  // past the state, or taken by an earlier sequence of the call

template <bool BF>
__device__ __forceinline__ float w2f(uint16_t x) {
  if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)x << 16);
  return h2f(x);
}
template <bool BF>
__device__ __forceinline__ uint16_t f2w(float x) {  // RNE
  if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)x);
  return f2h(x);
}

__device__ __forceinline__ float l2_factor(float ss) { return __builtin_amdgcn_rsqf(ss + 1e-6f); }  // (1 ulp)

// Tokens [t0, t1) of sequence b. Offsets read from device memory are held to [0, n_tokens] and an end
// before its start is an empty sequence, so no value of cu reaches past the tensors. (Offsets that fall may still make
// sequences overlap, or leave chunks that nothing prepared: the results are then not specified.)
__device__ __forceinline__ void seq_range(const DeltaArgs& a, int b, int64_t& t0, int64_t& t1) {
  if (!a.cu) {
    t0 = (int64_t)b * a.len;
    t1 = t0 + a.len;
    return;
  }
  const int64_t lo = a.cu[b], hi = a.cu[b + 1];
  t0 = lo < 0 ? 0 : (lo > a.n_tokens ? a.n_tokens : lo);
  t1 = hi < t0 ? t0 : (hi > a.n_tokens ? a.n_tokens : hi);
}

// The slot of sequence b, or kSlotPad / kSlotBad; the same in every lane of a wave. Two sequences with
// one slot would race on its state: the first has it, the others are refused.
__device__ __forceinline__ int slot_of(const DeltaArgs& a, int b) {
  if (!a.slots) return b < a.n_slots ? b : kSlotBad;
  const int s = a.slots[b];
  if (s < 0) return kSlotPad;
  bool taken = s >= a.n_slots;
  for (int i = threadIdx.x & 63; i < b; i += 64) taken |= a.slots[i] == s;
  return __any(taken) ? kSlotBad : s;
}

}  // namespace dfssm
