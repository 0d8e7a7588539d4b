// RMSNorms of a state space block, fused with what surrounds them (gfx950).
//   gated_norm     out = rmsnorm(x s(z)) w, or rmsnorm(x) w s(z);  s(z) = z / (1 + e^-z), per group of a row's columns
//   residual_norm  r' = r + scale (rmsnorm(x) pw, or x);  out = rmsnorm(r') w
// with rmsnorm(v) = v / sqrt(mean(v^2) + eps). Everything is fp32 up to one rounding of each output (out is made of r' before
// its own rounding). What bounds them: memory, each input read once and each output written once.
//
// A row, or a group of one, lies in registers over 8, 16 or 64 lanes or a workgroup; a lane has eight columns at a time, loaded
// from any address. Where a width is no multiple of 8, the last lane's columns end with the row and overlap its neighbour's: it
// leaves those out of sums, and both store the same values. A workgroup goes over many rows with its columns' weights in
// registers, and the next row is on its way while it reduces this one. 32768 rows of 5120, eight groups (bf16, 1.01 GB), 0.206 ms;
// 32768 of 2560 with a residual in 32 bits (1.01 GB) 0.199 ms: 4.9 and 5.0 TB/s, what a copy reaches. (A row to a workgroup at a
// time, weights read for each: 0.366 and 0.399 ms.) Few rows: the launch; one of 4096 3.7 us, 32 of 2048 3.3 us in a replayed graph.
#include "common.h"
#include "layer.h"

namespace dfssm {

namespace {

// The sum over T lanes, or the workgroup's T threads, the same in every one of them, in the same order for every row. The slot
// alternates from sum to sum, so that one barrier is enough: a wave that writes a slot again has passed the barrier behind all
// reads of its former values.
template <int T>
constexpr int kWaves = T <= 64 ? 1 : T / 64;
template <int T>
__device__ __forceinline__ float row_sum(float v, float (*part)[kWaves<T>], int& slot) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  if constexpr (T == 8) return v + dpp_f32<0x141>(v);  // (the other four of eight lanes)
  v += dpp_f32<0x124>(v);
  v += dpp_f32<0x128>(v);
  if constexpr (T == 16) return v;
  const int x = __builtin_bit_cast(int, v);
  v = (__builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 0)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 16))) +
      (__builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 32)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 48)));
  if constexpr (T == 64) return v;
  if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6] = v;
  lds_barrier();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves<T>; ++w) s += part[slot][w];
  slot ^= 1;
  return s;
}

__device__ __forceinline__ float rms_factor(float ss, float inv_n, float eps) {
  return __builtin_amdgcn_rsqf(__builtin_fmaf(ss, inv_n, eps));  // (1 ulp)
}

template <int V>
struct Wide {
  typedef float type __attribute__((ext_vector_type(V)));
  typedef type loose __attribute__((aligned(4)));
};
template <>
struct Wide<1> {
  typedef float type, loose;
};
template <int V>
__device__ __forceinline__ void load32(const float* p, float (&x)[V]) {
  const typename Wide<V>::type v = *(const typename Wide<V>::loose*)p;
  if constexpr (V == 1) {
    x[0] = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = v[i];
  }
}
template <int V>
__device__ __forceinline__ void store32(float* p, const float (&x)[V]) {
  typename Wide<V>::type v;
  if constexpr (V == 1) {
    v = x[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = x[i];
  }
  *(typename Wide<V>::loose*)p = v;
}

// A lane's columns of a row of n: V from at[k] on, of which the first skip[k] are another's (V: it has none).
template <int T, int V, int K, bool TAIL>
struct Columns {
  int at[K], skip[K];
  __device__ __forceinline__ Columns(int i, int n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = V * (i + T * k);
      at[k] = first < n ? first : 0;
      skip[k] = first < n ? 0 : V;
      if (TAIL && first < n && first > n - V) {
        at[k] = n - V;
        skip[k] = first - at[k];
      }
    }
  }
  __device__ __forceinline__ bool any(int k) const { return skip[k] < V; }
  // x, or zero in another's column, before it is squared: an infinity times zero would be NaN.
  __device__ __forceinline__ float own(int k, int e, float x) const { return (TAIL ? e >= skip[k] : skip[k] == 0) ? x : 0.0f; }
};

// T threads to a row or group; workgroup: 256 threads, or the T.
template <int T>
constexpr int kThreads = T <= 64 ? 256 : T;
template <int T, int V, int K, bool TAIL, bool BF>
__global__ __launch_bounds__(kThreads<T>) void gated_norm_kernel(GatedNormArgs a, int64_t workers) {
  __shared__ float part[2][kWaves<T>];
  const int i = threadIdx.x % T, n = a.cols / a.groups;
  const int64_t worker = (int64_t)blockIdx.x * (kThreads<T> / T) + threadIdx.x / T;
  const int64_t c0 = worker % a.groups * n, step = workers / a.groups;
  int64_t row = worker / a.groups;
  if (worker >= workers || row >= a.rows) return;  // (workers is a multiple of the groups)
  const float inv_n = 1.0f / (float)n;
  const Columns<T, V, K, TAIL> cs(i, n);
  const int (&at)[K] = cs.at;
  float w[K][V];
  Raw16<V> x[K], z[K];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k] = load_raw<V>(a.x + r * a.ld_x + c0 + at[k]);
      if (a.gate) z[k] = load_raw<V>(a.gate + r * a.ld_gate + c0 + at[k]);
    }
  };
  load(row);
#pragma unroll
  for (int k = 0; k < K; ++k) load32<V>(a.weight + c0 + at[k], w[k]);
  int slot = 0;
  for (;;) {
    float v[K][V], g[K][V], ss = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      widen<V, BF>(x[k], v[k]);
      if (a.gate) widen<V, BF>(z[k], g[k]);
    }
    const int64_t next = row + step;
    const bool more = next < a.rows;
    if (more) load(next);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        g[k][e] = a.gate ? silu_f32(g[k][e]) : 1.0f;
        if (a.gate_first) v[k][e] *= g[k][e];
        const float o = cs.own(k, e, v[k][e]);
        ss = __builtin_fmaf(o, o, ss);
      }
    const float f = rms_factor(row_sum<T>(ss, part, slot), inv_n, a.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        y[e] = v[k][e] * f * w[k][e];
        if (!a.gate_first) y[e] *= g[k][e];
      }
      if (cs.any(k)) store16<V, BF>(a.out + row * a.ld_out + c0 + at[k], y);
    }
    if (!more) break;
    row = next;
  }
}

template <int T, int V, int K, bool TAIL, bool BF, bool R32>
__global__ __launch_bounds__(kThreads<T>) void residual_norm_kernel(ResidualNormArgs a, int64_t workers) {
  __shared__ float part[2][kWaves<T>];
  const int i = threadIdx.x % T, n = a.cols;
  int64_t row = (int64_t)blockIdx.x * (kThreads<T> / T) + threadIdx.x / T;
  if (row >= a.rows) return;
  const float inv_n = 1.0f / (float)n;
  const Columns<T, V, K, TAIL> cs(i, n);
  const int (&at)[K] = cs.at;
  Raw16<V> x[K], rh[R32 ? 1 : K];
  float r[K][V];
  auto load = [&](int64_t t) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k] = load_raw<V>(a.x + t * a.ld_x + at[k]);
      if constexpr (R32) load32<V>((const float*)a.residual + t * a.ld_res + at[k], r[k]);
      else rh[k] = load_raw<V>((const uint16_t*)a.residual + t * a.ld_res + at[k]);
    }
  };
  load(row);
  float w[K][V], m[K][V];  // the norm's weight; what rmsnorm(x), or x, is multiplied by
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load32<V>(a.weight + at[k], w[k]);
#pragma unroll
    for (int e = 0; e < V; ++e) m[k][e] = a.scale;
    if (a.scales) load32<V>(a.scales + at[k], m[k]);
  }
  int slot = 0;
  for (;;) {
    float v[K][V], s[K][V], ss = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      widen<V, BF>(x[k], v[k]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (R32) s[k][e] = r[k][e];
        const float o = cs.own(k, e, v[k][e]);
        ss = __builtin_fmaf(o, o, ss);
      }
      if constexpr (!R32) widen<V, BF>(rh[k], s[k]);
    }
    const int64_t next = row + workers;
    const bool more = next < a.rows;
    if (more) load(next);
    if (a.post_weight) {
      const float f = rms_factor(row_sum<T>(ss, part, slot), inv_n, a.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float pw[V];
        load32<V>(a.post_weight + at[k], pw);
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] = v[k][e] * f * pw[e];
      }
    }
    ss = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s[k][e] = __builtin_fmaf(m[k][e], v[k][e], s[k][e]);
        const float o = cs.own(k, e, s[k][e]);
        ss = __builtin_fmaf(o, o, ss);
      }
    const float f = rms_factor(row_sum<T>(ss, part, slot), inv_n, a.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!cs.any(k)) continue;
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = s[k][e] * f * w[k][e];
      store16<V, BF>(a.out + row * a.ld_out + at[k], y);
      if constexpr (R32) store32<V>((float*)a.residual_out + row * a.ld_res_out + at[k], s[k]);
      else store16<V, BF>((uint16_t*)a.residual_out + row * a.ld_res_out + at[k], s[k]);
    }
    if (!more) break;
    row = next;
  }
}

// Threads of a row: 16 columns each at most, up to 16384. (Fewer than eight columns: one each.) 8192 rows of 5119 59 us, of 5120 51,
// where one column at a time took 764; 8192 x 8 groups of 8 columns 6.3 us, a wave to each 23.
template <bool TAIL, class Launch>
void by_width(int n, Launch launch) {
  if (n <= 64) launch.template go<8, 8, 1, TAIL>();
  else if (n <= 128) launch.template go<16, 8, 1, TAIL>();
  else if (n <= 512) launch.template go<64, 8, 1, TAIL>();
  else if (n <= 1024) launch.template go<64, 8, 2, TAIL>();
  else if (n <= 2048) launch.template go<256, 8, 1, TAIL>();
  else if (n <= 4096) launch.template go<256, 8, 2, TAIL>();
  else if (n <= 8192) launch.template go<512, 8, 2, TAIL>();
  else launch.template go<1024, 8, 2, TAIL>();
}
template <class Launch>
void by_width(int n, Launch launch) {
  if (n < 8) launch.template go<8, 1, 1, false>();
  else if (n % 8) by_width<true>(n, launch);
  else by_width<false>(n, launch);
}
// Rows or groups at once: as many as are resident, so that each has several in turn.
template <int T>
constexpr int64_t kResident = 256 * 2048 / T;
template <int T>
dim3 grid_of(int64_t workers) {
  constexpr int per = kThreads<T> / T;
  return dim3((unsigned)((workers + per - 1) / per));
}

struct LaunchGated {
  const GatedNormArgs& a;
  hipStream_t s;
  template <int T, int V, int K, bool TAIL>
  void go() const {
    int64_t rows = kResident<T> / a.groups;  // of a row's groups each
    rows = rows < 1 ? 1 : (rows < a.rows ? rows : a.rows);
    const int64_t workers = rows * a.groups;
    const dim3 grid = grid_of<T>(workers), block(kThreads<T>);
    if (a.bf16) hipLaunchKernelGGL((gated_norm_kernel<T, V, K, TAIL, true>), grid, block, 0, s, a, workers);
    else hipLaunchKernelGGL((gated_norm_kernel<T, V, K, TAIL, false>), grid, block, 0, s, a, workers);
  }
};
struct LaunchResidual {
  const ResidualNormArgs& a;
  hipStream_t s;
  template <int T, int V, int K, bool TAIL>
  void go() const {
    constexpr int64_t per = kThreads<T> / T;
    const int64_t up = (a.rows + per - 1) / per * per, workers = kResident<T> < up ? kResident<T> : up;
    const dim3 grid = grid_of<T>(workers), block(kThreads<T>);
    if (a.bf16) type<T, V, K, TAIL, true>(grid, block, workers);
    else type<T, V, K, TAIL, false>(grid, block, workers);
  }
  template <int T, int V, int K, bool TAIL, bool BF>
  void type(dim3 grid, dim3 block, int64_t workers) const {
    if (a.res32) hipLaunchKernelGGL((residual_norm_kernel<T, V, K, TAIL, BF, true>), grid, block, 0, s, a, workers);
    else hipLaunchKernelGGL((residual_norm_kernel<T, V, K, TAIL, BF, false>), grid, block, 0, s, a, workers);
  }
};

}  // namespace

hipError_t launch_gated_norm(const GatedNormArgs& a, hipStream_t s) {
  by_width(a.cols / a.groups, LaunchGated{a, s});
  return hipGetLastError();
}
hipError_t launch_residual_norm(const ResidualNormArgs& a, hipStream_t s) {
  by_width(a.cols, LaunchResidual{a, s});
  return hipGetLastError();
}

}  // namespace dfssm
