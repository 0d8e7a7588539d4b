// The selective state space scan token by token (gfx950): single tokens, and prompts of a few.
//
// Per head, with the state h (P x N) fp32 and the head's group of B and C (N):
//   d_t = max(softplus(dt_t + dt_bias), 0);  h_t = e^{-d_t e^{A_log}} h_{t-1} + (d_t x_t) B_t^T;  y_t = h_t C_t + D x_t
// All of it in fp32; y is rounded once. What bounds it: the states, read and written once per call; 32 tokens x 64 heads of
// 64 x 128 (135 MB) 25 us, 5.4 TB/s. A prompt's tokens wait for each other, 0.75 us each.
#include "common.h"
#include "layer.h"
#include "scan_math.h"

namespace dfssm {

namespace {

// The sum over a row of 16 lanes, in each of them.
__device__ __forceinline__ float row_sum16(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x124>(v);
  v += dpp_f32<0x128>(v);
  return v;
}

// A workgroup: 16 NI rows p of a sequence's head. A row's N columns lie over 16 lanes, lane j with columns
// 64 i + 4 j .., so that a row is read in whole 256-byte pieces and its sum with C needs no LDS.
template <int N, bool BF, int NI>
__global__ __launch_bounds__(256) void scan_token_kernel(PackedScanArgs a) {
  constexpr int NV = N / 16;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, j = lane & 15, sub = lane >> 4;
  const int nrb = (a.P + 16 * NI - 1) / (16 * NI);
  int bx = blockIdx.x;
  const int rb = bx % nrb;
  bx /= nrb;
  const int h = bx % a.H, b = bx / a.H, gr = h / (a.H / a.G);
  int64_t t0, t1;
  seq_range(a, b, t0, t1);
  const int slot = slot_of(a, b);
  if (slot < 0) {  // padding: zeros; a bad slot: NaN. No state is read or written.
    const uint16_t fill = slot == kSlotPad ? 0 : 0x7fff;
    for (int64_t t = t0; t < t1; ++t)
      for (int i = tid; i < 16 * NI; i += 256)
        if (rb * 16 * NI + i < a.P) a.out[t * a.ld_out + (int64_t)h * a.P + rb * 16 * NI + i] = fill;
    return;
  }
  float S[NI][NV];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (rb * NI + i) * 16 + 4 * w + sub;  // (rows come in whole sixteens: uniform in a workgroup)
    if ((rb * NI + i) * 16 >= a.P) continue;
    const float* p = a.state + (((size_t)slot * a.H + h) * a.P + r) * N;
#pragma unroll
    for (int c = 0; c < NV / 4; ++c) {
      const f32x4 x = ld_nt_f4(p + 64 * c + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][4 * c + e] = x[e];
    }
  }
  const HeadParams hp = head_params(a, h);
  for (int64_t t = t0; t < t1; ++t) {
    float B[NV], C[NV];
#pragma unroll
    for (int c = 0; c < NV / 4; ++c) {
      float b4[4], c4[4];
      load16<4, BF>(a.B + t * a.ld_B + gr * N + 64 * c + 4 * j, b4);
      load16<4, BF>(a.C + t * a.ld_C + gr * N + 64 * c + 4 * j, c4);
#pragma unroll
      for (int e = 0; e < 4; ++e) B[4 * c + e] = b4[e], C[4 * c + e] = c4[e];
    }
    const float d = time_step(load_dt<BF>(a, t, h), hp, a.softplus);
    const float dec = dev_expf(d * hp.A);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if ((rb * NI + i) * 16 >= a.P) continue;
      const int r = (rb * NI + i) * 16 + 4 * w + sub;
      const float x = w2f<BF>(a.x[t * a.ld_x + (int64_t)h * a.P + r]), u = x * d;
      float y = 0.0f;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        S[i][c] = __builtin_fmaf(u, B[c], dec * S[i][c]);
        y = __builtin_fmaf(S[i][c], C[c], y);
      }
      y = row_sum16(y);
      if (j == 0) a.out[t * a.ld_out + (int64_t)h * a.P + r] = f2w<BF>(__builtin_fmaf(hp.D, x, y));
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if ((rb * NI + i) * 16 >= a.P) continue;
    const int r = (rb * NI + i) * 16 + 4 * w + sub;
    float* p = a.state_out + (((size_t)slot * a.H + h) * a.P + r) * N;
#pragma unroll
    for (int c = 0; c < NV / 4; ++c)
      st_nt_f4(p + 64 * c + 4 * j, f32x4{S[i][4 * c], S[i][4 * c + 1], S[i][4 * c + 2], S[i][4 * c + 3]});
  }
}

template <int N, bool BF, int NI>
void launch_rows(const PackedScanArgs& a, hipStream_t s) {
  const int64_t wgs = (int64_t)a.n_seq * a.H * ((a.P + 16 * NI - 1) / (16 * NI));
  hipLaunchKernelGGL((scan_token_kernel<N, BF, NI>), dim3((unsigned)wgs), dim3(256), 0, s, a);
}
// 16 KiB of state to a workgroup where there are plenty of them, else 16 rows. One token, with 16 rows, 32 and 64: 64 heads of
// 64 x 128, one sequence 3.7, 4.1 and 4.9 us in a replayed graph, four 5.8, 5.1 and 5.6, 32 26.5, 25.4 and 24.2; 64 x 80 heads
// 60.7, 59.8 and 61.8; 30 x 8 heads of 208 x 64 10.6, 8.2 and 7.0.
template <int N, bool BF>
hipError_t launch_token(const PackedScanArgs& a, hipStream_t s) {
  const int64_t tiles = (int64_t)a.n_seq * a.H * (a.P / 16);
  if (tiles > 0x7fffffff) return hipErrorInvalidValue;
  if (tiles >= 1024) launch_rows<N, BF, 256 / N>(a, s);
  else launch_rows<N, BF, 1>(a, s);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_scan_token(const PackedScanArgs& a, hipStream_t s) {
  if (a.N == 128) return a.bf16 ? launch_token<128, true>(a, s) : launch_token<128, false>(a, s);
  return a.bf16 ? launch_token<64, true>(a, s) : launch_token<64, false>(a, s);
}

}  // namespace dfssm
