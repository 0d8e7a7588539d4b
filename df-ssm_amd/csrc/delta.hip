// The gated delta rule (gfx950): one token per sequence (delta_token_kernel) and whole prompts.
//
// State S (Dv x Dk) fp32 per value head, a_t = exp(g_t):
//   S' = a_t S;  u_t = beta_t (v_t - S' k_t);  S = S' + u_t k_t^T;  o_t = scale S q_t
// with q and k divided by sqrt(sum x^2 + 1e-6) first if l2norm. All of it in fp32; o is rounded once.
#include "common.h"
#include "delta.h"
#include "dfssm_kernels.h"

namespace dfssm {

// ---------------------------------------------------------------------------------------------
// Token by token. A row of S (one value column, DK keys) lies over 16 lanes, DK / 16 columns each in
// two halves of 16-byte loads, so both dot products of a row are DPP sums over a row of lanes and no
// LDS or barrier is needed; a wave holds 4 NI rows. S k and S q are taken of the state as loaded, in
// one reduction: S' k = a (S k) and S q = a (S_old q) + u (k q).
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float row_sum_f32(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x124>(v);
  v += dpp_f32<0x128>(v);
  return v;
}

template <int DK>
struct Row16 {  // DK / 16 values of a row of 16-bit values: lane j has columns 4 j + 64 i + (0..3)
  uint2 w[DK / 64];
};
template <int DK>
__device__ __forceinline__ Row16<DK> load_row16(const uint16_t* p, int j) {
  Row16<DK> r;
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) r.w[i] = *(const uint2*)(p + 64 * i + 4 * j);
  return r;
}
template <int DK, bool BF>
__device__ __forceinline__ void widen(const Row16<DK>& r, float* x) {
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    x[4 * i] = w2f<BF>((uint16_t)r.w[i].x);
    x[4 * i + 1] = w2f<BF>((uint16_t)(r.w[i].x >> 16));
    x[4 * i + 2] = w2f<BF>((uint16_t)r.w[i].y);
    x[4 * i + 3] = w2f<BF>((uint16_t)(r.w[i].y >> 16));
  }
}

// Workgroup: one sequence, one value head, 16 NI value rows (4 waves of 4 NI).
template <int DK, bool BF, int NI>
__global__ __launch_bounds__(256) void delta_token_kernel(DeltaArgs a) {
  constexpr int NV = DK / 16;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, j = lane & 15, sub = lane >> 4;
  const int nrb = (a.Dv + 16 * NI - 1) / (16 * NI);
  int bx = blockIdx.x;
  const int rb = bx % nrb;
  bx /= nrb;
  const int h = bx % a.Hv, b = bx / a.Hv;
  const int hk = h / (a.Hv / a.Hk);
  int64_t t0, t1;
  seq_range(a, b, t0, t1);
  const int slot = slot_of(a, b);
  if (slot < 0) {  // padding: zeros; a bad slot: NaN. No state is read or written.
    const uint16_t fill = slot == kSlotPad ? 0 : 0x7fff;
    for (int64_t t = t0; t < t1; ++t)
      for (int i = tid; i < 16 * NI; i += 256)
        if (rb * 16 * NI + i < a.Dv) a.out[t * a.ld_out + (int64_t)h * a.Dv + rb * 16 * NI + i] = fill;
    return;
  }
  float S[NI][NV];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (rb * NI + i) * 16 + 4 * w + sub;  // (rows come in whole sixteens: uniform in a workgroup)
    if ((rb * NI + i) * 16 >= a.Dv) continue;
    const float* p = a.state + (((size_t)slot * a.Hv + h) * a.Dv + r) * DK;
#pragma unroll
    for (int c = 0; c < NV / 4; ++c) {
      const f32x4 x = ld_nt_f4(p + 64 * c + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][4 * c + e] = x[e];
    }
  }
  for (int64_t t = t0; t < t1; ++t) {
    float q[NV], k[NV];
    widen<DK, BF>(load_row16<DK>(a.k + t * a.ld_k + hk * DK, j), k);
    widen<DK, BF>(load_row16<DK>(a.q + t * a.ld_q + hk * DK, j), q);
    const float dec = dev_expf(a.g[t * a.ld_g + h]), be = a.beta[t * a.ld_beta + h];
    float kk = 0.0f, qq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      kk = __builtin_fmaf(k[c], k[c], kk);
      qq = __builtin_fmaf(q[c], q[c], qq);
      kq = __builtin_fmaf(k[c], q[c], kq);
    }
    kq = row_sum_f32(kq);
    float rk = 1.0f, rq = a.scale;
    if (a.l2norm) {
      rk = l2_factor(row_sum_f32(kk));
      rq *= l2_factor(row_sum_f32(qq));
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if ((rb * NI + i) * 16 >= a.Dv) continue;
      const int r = (rb * NI + i) * 16 + 4 * w + sub;
      const float v = w2f<BF>(a.v[t * a.ld_v + (int64_t)h * a.Dv + r]);
      float sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        sk = __builtin_fmaf(S[i][c], k[c], sk);
        sq = __builtin_fmaf(S[i][c], q[c], sq);
      }
      sk = row_sum_f32(sk);
      sq = row_sum_f32(sq);
      const float u = be * (v - dec * (rk * sk)) * rk;
#pragma unroll
      for (int c = 0; c < NV; ++c) S[i][c] = __builtin_fmaf(u, k[c], dec * S[i][c]);
      if (j == 0) a.out[t * a.ld_out + (int64_t)h * a.Dv + r] = f2w<BF>(rq * __builtin_fmaf(u, kq, dec * sq));
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if ((rb * NI + i) * 16 >= a.Dv) continue;
    const int r = (rb * NI + i) * 16 + 4 * w + sub;
    float* p = a.state_out + (((size_t)slot * a.Hv + h) * a.Dv + r) * DK;
#pragma unroll
    for (int c = 0; c < NV / 4; ++c)
      st_nt_f4(p + 64 * c + 4 * j, f32x4{S[i][4 * c], S[i][4 * c + 1], S[i][4 * c + 2], S[i][4 * c + 3]});
  }
}

template <int DK, bool BF, int NI>
static void launch_rows(const DeltaArgs& a, hipStream_t s) {
  const int64_t wgs = (int64_t)a.n_seq * a.Hv * ((a.Dv + 16 * NI - 1) / (16 * NI));
  hipLaunchKernelGGL((delta_token_kernel<DK, BF, NI>), dim3((unsigned)wgs), dim3(256), 0, s, a);
}
// 16 KiB of state to a workgroup where there are plenty of them, else 16 rows. One token, state streamed, with
// 4, 8, 16 and 32 KiB: Dk = 64, 37 x 24 heads of 208 rows 33.5, 24.0 and 23.8 us; Dk = 128, 32 x 64 heads of 64
// rows 29.7 (8), 28.5 and 27.4 us, 64 x 80 heads of 64 rows 63.0, 62.8 and 64.1 us. Few, the kernel in a replayed graph
// with 16 rows and with 16 KiB: 64 heads of 64 x 128, one sequence 3.4 and 3.7 us, two 4.0 and 4.1, four 5.3 and 4.9;
// one of 2 heads of 256 x 64 3.0 and 4.0, eight of 12 heads of 128 x 64 4.1 and 4.4.
template <int DK, bool BF>
static hipError_t launch_token(const DeltaArgs& a, hipStream_t s) {
  const int64_t tiles = (int64_t)a.n_seq * a.Hv * (a.Dv / 16);
  if (tiles > 0x7fffffff) return hipErrorInvalidValue;
  if (tiles >= 2048) launch_rows<DK, BF, 256 / DK>(a, s);
  else launch_rows<DK, BF, 1>(a, s);
  return hipGetLastError();
}

hipError_t launch_delta_token(const DeltaArgs& a, hipStream_t s) {
  if (a.n_seq == 0) return hipSuccess;
  if (a.Dk == 128) return a.bf16 ? launch_token<128, true>(a, s) : launch_token<128, false>(a, s);
  return a.bf16 ? launch_token<64, true>(a, s) : launch_token<64, false>(a, s);
}

}  // namespace dfssm
