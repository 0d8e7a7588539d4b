// RMSNorms of a state space block, fused with what surrounds them (gfx950).
//   gated_norm     out = rmsnorm(x s(z)) w, or rmsnorm(x) w s(z);  s(z) = z / (1 + e^-z), per group of a row's columns
//   residual_norm  r' = r + scale (rmsnorm(x) pw, or x);  out = rmsnorm(r') w
// with rmsnorm(v) = v / sqrt(mean(v^2) + eps). Everything is fp32 up to one rounding of each output (out is made of r' before
// its own rounding). What bounds them: memory, each input read once and each output written once.
#include "common.h"
#include "layer.h"

namespace dfssm {

namespace {

// The sum over the workgroup, the same in every thread, in the same order for every row. slot alternates between
// calls, so that one barrier is enough.
template <int WAVES>
__device__ __forceinline__ float wg_sum(float v, float (*part)[WAVES], int slot) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, 64);
  if constexpr (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += part[slot][w];
  return s;
}

__device__ __forceinline__ float rms_factor(float ss, int n, float eps) {
  return __builtin_amdgcn_rsqf(ss / (float)n + eps);  // (1 ulp)
}

// A row, or a group of one, over a workgroup: thread i has columns V (i + 64 WAVES k) .., k < K.
template <int WAVES, int V, int K, bool BF>
__global__ __launch_bounds__(64 * WAVES) void gated_norm_kernel(GatedNormArgs a) {
  __shared__ float part[2][WAVES];
  const int n = a.cols / a.groups;
  const int64_t row = blockIdx.x / a.groups, c0 = (int64_t)(blockIdx.x % a.groups) * n;
  const uint16_t *x = a.x + row * a.ld_x + c0, *z = a.gate ? a.gate + row * a.ld_gate + c0 : nullptr;
  float v[K][V], g[K][V], ss = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = V * (threadIdx.x + 64 * WAVES * k);
    if (c < n) {
      load16<V, BF>(x + c, v[k]);
      if (z) load16<V, BF>(z + c, g[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (V * (int)(threadIdx.x + 64 * WAVES * k) >= n) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      g[k][i] = z ? silu_f32(g[k][i]) : 1.0f;
      if (a.gate_first) v[k][i] *= g[k][i], g[k][i] = 1.0f;
      ss = __builtin_fmaf(v[k][i], v[k][i], ss);
    }
  }
  const float f = rms_factor(wg_sum<WAVES>(ss, part, 0), n, a.eps);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = V * (threadIdx.x + 64 * WAVES * k);
    if (c >= n) continue;
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = v[k][i] * f * a.weight[c0 + c + i] * g[k][i];
    store16<V, BF>(a.out + row * a.ld_out + c0 + c, y);
  }
}

template <int WAVES, int V, int K, bool BF>
__global__ __launch_bounds__(64 * WAVES) void residual_norm_kernel(ResidualNormArgs a) {
  __shared__ float part[2][WAVES];
  const int n = a.cols;
  const int64_t row = blockIdx.x;
  float v[K][V], r[K][V], ss = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = V * (threadIdx.x + 64 * WAVES * k);
    if (c < n) {
      load16<V, BF>(a.x + row * a.ld_x + c, v[k]);
      if (a.res32) {
#pragma unroll
        for (int i = 0; i < V; ++i) r[k][i] = ((const float*)a.residual)[row * a.ld_res + c + i];
      } else {
        load16<V, BF>((const uint16_t*)a.residual + row * a.ld_res + c, r[k]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) ss = __builtin_fmaf(v[k][i], v[k][i], ss);
    }
  }
  const float f = a.post_weight ? rms_factor(wg_sum<WAVES>(ss, part, 0), n, a.eps) : 1.0f;
  ss = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = V * (threadIdx.x + 64 * WAVES * k);
    if (c >= n) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float p = a.post_weight ? v[k][i] * f * a.post_weight[c + i] : v[k][i];
      r[k][i] = __builtin_fmaf(a.scales ? a.scales[c + i] : a.scale, p, r[k][i]);
      ss = __builtin_fmaf(r[k][i], r[k][i], ss);
    }
  }
  const float f2 = rms_factor(wg_sum<WAVES>(ss, part, 1), n, a.eps);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = V * (threadIdx.x + 64 * WAVES * k);
    if (c >= n) continue;
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = r[k][i] * f2 * a.weight[c + i];
    store16<V, BF>(a.out + row * a.ld_out + c, y);
    if (a.res32) {
#pragma unroll
      for (int i = 0; i < V; ++i) ((float*)a.residual_out)[row * a.ld_res_out + c + i] = r[k][i];
    } else {
      store16<V, BF>((uint16_t*)a.residual_out + row * a.ld_res_out + c, r[k]);
    }
  }
}

// 16384 columns at most: 16 waves of 16 values a lane.
template <bool BF, class Launch>
hipError_t by_width(int n, Launch launch) {
  if (n % 8 == 0) {
    if (n <= 512) launch.template go<1, 8, 1, BF>();
    else if (n <= 2048) launch.template go<4, 8, 1, BF>();
    else if (n <= 8192) launch.template go<8, 8, 2, BF>();
    else launch.template go<16, 8, 2, BF>();
  } else {
    if (n <= 256) launch.template go<1, 1, 4, BF>();
    else if (n <= 4096) launch.template go<4, 1, 16, BF>();
    else launch.template go<16, 1, 16, BF>();
  }
  return hipGetLastError();
}

struct LaunchGated {
  const GatedNormArgs& a;
  hipStream_t s;
  template <int WAVES, int V, int K, bool BF>
  void go() const {
    hipLaunchKernelGGL((gated_norm_kernel<WAVES, V, K, BF>), dim3((unsigned)(a.rows * a.groups)), dim3(64 * WAVES), 0, s, a);
  }
};
struct LaunchResidual {
  const ResidualNormArgs& a;
  hipStream_t s;
  template <int WAVES, int V, int K, bool BF>
  void go() const {
    hipLaunchKernelGGL((residual_norm_kernel<WAVES, V, K, BF>), dim3((unsigned)a.rows), dim3(64 * WAVES), 0, s, a);
  }
};

}  // namespace

hipError_t launch_gated_norm(const GatedNormArgs& a, hipStream_t s) {
  if (a.rows * a.groups > 0x7fffffff) return hipErrorInvalidValue;
  const LaunchGated l{a, s};
  return a.bf16 ? by_width<true>(a.cols / a.groups, l) : by_width<false>(a.cols / a.groups, l);
}
hipError_t launch_residual_norm(const ResidualNormArgs& a, hipStream_t s) {
  if (a.rows > 0x7fffffff) return hipErrorInvalidValue;
  const LaunchResidual l{a, s};
  return a.bf16 ? by_width<true>(a.cols, l) : by_width<false>(a.cols, l);
}

}  // namespace dfssm
