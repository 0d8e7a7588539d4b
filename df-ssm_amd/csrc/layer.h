// Arguments of the operators between a state space layer's projections, and what their kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "packed.h"

namespace dfssm {

struct PackedConvArgs {
  const uint16_t *x, *weight, *bias;  // (tokens, C) rows ld_x elements apart, (C, W), (C) or null
  const uint16_t* state;              // (n_slots, C, W - 1), the oldest first
  uint16_t* state_out;                // the same tensor, or one of its shape
  const int32_t *slots, *cu;
  uint16_t* out;
  int64_t ld_x, ld_out, n_tokens, len;
  int n_seq, n_slots, C, W;
  int bf16, silu;
};
hipError_t launch_conv_step(const PackedConvArgs& a, hipStream_t s);
hipError_t launch_conv_prefill(const PackedConvArgs& a, hipStream_t s);

struct PackedScanArgs {
  const uint16_t *x, *B, *C;            // (tokens, H, P), (tokens, G, N), 16-bit, heads contiguous
  const void* dt;                       // (tokens, H), of x's type or fp32
  const float *A_log, *D, *dt_bias;     // (H); D and dt_bias may be null
  const float* state;                   // (n_slots, H, P, N)
  float* state_out;
  const int32_t *slots, *cu;
  uint16_t* out;
  int64_t ld_x, ld_dt, ld_B, ld_C, ld_out, n_tokens, len;
  int n_seq, n_slots, H, G, P, N;
  int bf16, dt32, softplus;
};
// Token by token (scan.hip), and over chunks with the workspace of scan_chunk_workspace (scan_chunk.hip).
hipError_t launch_scan_token(const PackedScanArgs& a, hipStream_t s);
hipError_t launch_scan_chunked(const PackedScanArgs& a, void* workspace, hipStream_t s);
size_t scan_chunk_workspace(const PackedScanArgs& a);

struct GatedNormArgs {
  const uint16_t *x, *gate;  // rows ld_* elements apart; gate may be null
  const float* weight;       // (cols)
  uint16_t* out;
  int64_t ld_x, ld_gate, ld_out, rows;
  int cols, groups;
  int bf16, gate_first;
  float eps;
};
hipError_t launch_gated_norm(const GatedNormArgs& a, hipStream_t s);

struct ResidualNormArgs {
  const uint16_t* x;
  const void* residual;                         // of x's type, or fp32
  const float *post_weight, *scales, *weight;   // (cols); the first two may be null
  uint16_t* out;
  void* residual_out;
  int64_t ld_x, ld_res, ld_out, ld_res_out, rows;
  int cols;
  int bf16, res32;
  float scale, eps;
};
hipError_t launch_residual_norm(const ResidualNormArgs& a, hipStream_t s);

// x / (1 + e^-x). Relative error at most (3 + |x|) 2^-23: the rounding of x log2 e is |x| 2^-23 of e^-x, the hardware's exponential
// and reciprocal 2^-23 each (1 ulp), the sum and the last product 2^-24 each; outputs have 12 bits at most. Below x = -87 the
// reciprocal leaves the normal numbers: off by up to 2^-119.
__device__ __forceinline__ float silu_f32(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}

// V 16-bit values at once, from any address that is a multiple of 2.
template <int V>
struct Pack16 {
  typedef uint16_t type __attribute__((ext_vector_type(V)));
  typedef type loose __attribute__((aligned(2)));
};
template <>
struct Pack16<1> {
  typedef uint16_t type;
  typedef uint16_t loose;
};
template <int V>
struct Raw16 {
  typename Pack16<V>::type v;
};
template <int V>
__device__ __forceinline__ Raw16<V> load_raw(const uint16_t* p) {
  return Raw16<V>{*(const typename Pack16<V>::loose*)p};
}
template <int V, bool BF>
__device__ __forceinline__ void widen(const Raw16<V>& r, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = w2f<BF>(r.v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = w2f<BF>(r.v[i]);
  }
}
template <int V, bool BF>
__device__ __forceinline__ void load16(const uint16_t* p, float (&x)[V]) {
  widen<V, BF>(load_raw<V>(p), x);
}
template <int V, bool BF>
__device__ __forceinline__ void store16(uint16_t* p, const float (&x)[V]) {
  typename Pack16<V>::type v;
  if constexpr (V == 1) {
    v = f2w<BF>(x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = f2w<BF>(x[i]);
  }
  *(typename Pack16<V>::loose*)p = v;
}

}  // namespace dfssm
