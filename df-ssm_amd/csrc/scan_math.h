// What the selective scan's kernels share: a head's parameters and its time steps.
#pragma once
#include "layer.h"

namespace dfssm {

struct HeadParams {
  float A, D, bias;  // A = -e^{A_log}
};
__device__ __forceinline__ HeadParams head_params(const ScanArgs& a, int h) {
  return HeadParams{-dev_expf(a.A_log[h]), a.D ? a.D[h] : 0.0f, a.dt_bias ? a.dt_bias[h] : 0.0f};
}

template <bool BF>
__device__ __forceinline__ float load_dt(const ScanArgs& a, int64_t t, int h) {
  if (a.dt32) return ((const float*)a.dt)[t * a.ld_dt + h];
  return w2f<BF>(((const uint16_t*)a.dt)[t * a.ld_dt + h]);
}

// softplus as max(z, 0) + log1p(e^-|z|), which neither overflows nor loses a small result; a NaN stays one.
__device__ __forceinline__ float time_step(float raw, const HeadParams& p, int softplus) {
  const float z = raw + p.bias, top = z < 0.0f ? 0.0f : z;
  return softplus ? top + dev_log1pf(dev_expf(-__builtin_fabsf(z))) : top;
}

}  // namespace dfssm
