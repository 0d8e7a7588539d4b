// What the selective scan's kernels share: a head's parameters and its time steps.
#pragma once
#include "layer.h"

namespace dfssm {

struct HeadParams {
  float A, D, bias;  // A = -e^{A_log}
};
__device__ __forceinline__ HeadParams head_params(const PackedScanArgs& a, int h) {
  return HeadParams{-dev_expf(a.A_log[h]), a.D ? a.D[h] : 0.0f, a.dt_bias ? a.dt_bias[h] : 0.0f};
}

template <bool BF>
__device__ __forceinline__ float load_dt(const PackedScanArgs& a, int64_t t, int h) {
  if (a.dt32) return ((const float*)a.dt)[t * a.ld_dt + h];
  return w2f<BF>(((const uint16_t*)a.dt)[t * a.ld_dt + h]);
}

// softplus as max(z, 0) + log1p(e^-|z|), which neither overflows nor loses a small result; a NaN stays one. About 25
// instructions, within 4 roundings: the exponential with the rounding of z log2 e put back; log1p(t) = 2 artanh(t / (2 + t)) by
// its series, whose next term is below 2^-29 of it.
__device__ __forceinline__ float softplus_f32(float z) {
  const float v = -__builtin_fminf(__builtin_fabsf(z), 128.0f), hi = v * 1.44269502f;
  const float lo = __builtin_fmaf(v, 1.92596299e-8f, __builtin_fmaf(v, 1.44269502f, -hi));
  const float e = __builtin_amdgcn_exp2f(hi), t = __builtin_fmaf(e * lo, 0.693147182f, e);
  const float u = 2.0f + t, r = __builtin_amdgcn_rcpf(u), s0 = t * r;
  const float s = __builtin_fmaf(__builtin_fmaf(-u, s0, t), r, s0), q = s * s;
  float p = 1.0f / 15;
  p = __builtin_fmaf(p, q, 1.0f / 13);
  p = __builtin_fmaf(p, q, 1.0f / 11);
  p = __builtin_fmaf(p, q, 1.0f / 9);
  p = __builtin_fmaf(p, q, 1.0f / 7);
  p = __builtin_fmaf(p, q, 1.0f / 5);
  p = __builtin_fmaf(p, q, 1.0f / 3);
  return (z < 0.0f ? 0.0f : z) + 2.0f * __builtin_fmaf(s * q, p, s);
}
__device__ __forceinline__ float time_step(float raw, const HeadParams& p, int softplus) {
  const float z = raw + p.bias;
  return softplus ? softplus_f32(z) : (z < 0.0f ? 0.0f : z);
}

}  // namespace dfssm
