// The gated delta rule over chunks of 64 tokens (gfx950 matrix cores).
//
// Per value head and chunk, with G_i = g_1 + .. + g_i, S0 the state before it (S^T stored as Dk x Dv tiles) and
// row factors r_i that undo a normalisation or a power-of-two scaling of k_i or q_i:
//   A_ij = beta_i k_i.k_j e^{G_i - G_j} (i > j),  T = (I + A)^-1 diag(beta),  P_ij = scale q_i.k_j e^{G_i - G_j} (i >= j)
//   U = T (V - diag(e^G) K S0^T);  O = diag(scale e^G) Q S0^T + P U;  S1 = e^{G_C} S0 + (diag(e^{G_C - G}) U)^T K
// Two launches: delta_prep_kernel makes T and P of all chunks in parallel, delta_chain_kernel walks the chunks
// of a sequence and head with its state in registers.
//
// Numbers. States, sums and everything between products are fp32. The products run on the fp16 matrix cores
// with fp32 accumulation: q and k are exact there (16-bit inputs; bf16 rows are scaled by a power of two into
// fp16's range), every other operand is a pair of halves, x 2^s = hi + lo, which holds 22 bits, with s per row
// of T and P and per value column of S, V - .. and U chosen so that the largest magnitude lies in [2^14, 2^15).
// A product of two pairs leaves out lo lo, 2^-24 of it. So an fp32 state comes out as from fp32 arithmetic
// (2e-7 of its norm), at 2 or 3 matrix instructions per product instead of the 8 times as slow fp32 ones.
// G is summed in fp64, so that differences survive a decay of any size in the same chunk; -inf is held to -1e5.
#include "common.h"
#include "delta.h"
#include "dfssm_kernels.h"

namespace dfssm {

namespace {

typedef f16 h4 __attribute__((ext_vector_type(4)));
typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr int kC = 64;        // tokens of a chunk
constexpr int kGroup = 4;     // value heads of one preparing workgroup (a wave each for the inverse)

// What the preparation leaves per chunk and value head. T and P are in the order in which a lane of the matrix
// cores takes them: fragments of 16 rows x 32 columns, lane (g, r) row r, columns 4 g .. 4 g + 3 and 16 + 4 g ..,
// the order in which 16 x 16 results lie in registers, so results are operands without moving between lanes.
// Six fragments cover a lower triangle.
struct ChunkRec {
  f16 T[6][2][64][8];   // [fragment][hi, lo][lane]
  f16 P[6][2][64][8];
  float c1[kC];         // e^{G_i} times k's row factor
  float c2[kC];         // scale e^{G_i} times q's
  float tr[kC], pr[kC]; // row factors of T and P
  float w[kC];          // e^{G_C - G_i} times k's row factor
  float ks[kC], qs[kC]; // the powers of two that k and q are scaled by (bf16)
  float dec;            // e^{G_C}
  float pad[63];
};
static_assert(sizeof(ChunkRec) == 26624, "whole KiB");

__device__ __forceinline__ int frag_of(int t, int j) { return t + (t > 2 ? 1 : 0) + j; }  // row tile, column block

// LDS written by other lanes of the same wave is read after this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 2^s with m 2^s in [2^14, 2^15) for m > 0 (s at most 126: smaller m stay small), and 2^-s.
__device__ __forceinline__ float pow2_scale(float m, float& inv) {
  uint32_t e = __builtin_bit_cast(uint32_t, m) & 0x7f800000u;
  e = e < (15u << 23) ? (15u << 23) : e;
  inv = __builtin_bit_cast(float, e - (14u << 23));
  return __builtin_bit_cast(float, (268u << 23) - e);
}

__device__ __forceinline__ void split(float x, f16& hi, f16& lo) {
  hi = (f16)x;
  lo = (f16)(x - (float)hi);
}

// The largest of v >= 0 over the four lanes of a column (16 apart). As whole numbers, which order as the floats
// do: the compiler drops a float maximum of the two results of one lane swap.
__device__ __forceinline__ float max_rows4(float v) {
  uint32_t x = __builtin_bit_cast(uint32_t, v);
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max((uint32_t)p[0], (uint32_t)p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __builtin_bit_cast(float, max((uint32_t)q[0], (uint32_t)q[1]));
}

// The sequence and chunk of slot s of the launch's chunk numbering: sequence b starts at slot
// floor(t0 / 64) + b, which needs no sums over the lengths and leaves room for every chunk.
__device__ __forceinline__ int64_t first_slot(const DeltaArgs& a, int b) {
  int64_t t0, t1;
  seq_range(a, b, t0, t1);
  return t0 / kC + b;
}
__device__ bool chunk_of(const DeltaArgs& a, int64_t s, int64_t& tok, int& len) {
  int lo = 0, hi = a.n_seq;  // the last sequence that starts at or before s
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_slot(a, mid) <= s) lo = mid;
    else hi = mid;
  }
  int64_t t0, t1;
  seq_range(a, lo, t0, t1);
  const int64_t c = s - (t0 / kC + lo);
  if (c < 0 || c * kC >= t1 - t0) return false;
  tok = t0 + c * kC;
  len = (int)(t1 - tok < kC ? t1 - tok : kC);
  return true;
}

// ---------------------------------------------------------------------------------------------
// Preparation: one chunk, one key head, up to four of its value heads.
// ---------------------------------------------------------------------------------------------
constexpr int kMS = kC + 4;   // row stride of a matrix in LDS (floats): rows of 16-byte reads start 4 banks apart

template <int DK>
struct PrepLds {
  union {
    struct {
      f16 k[kC][DK + 8], q[kC][DK + 8];
    } in;
    float M[kGroup][kC][kMS];
  };
  double G[kGroup][kC];       // in units of log 2
  float be[kGroup][kC];
  float rk[kC], rq[kC];
};

// 8 values of a 16-bit row as halves times sc (1 for fp16), their squares added to ss.
template <bool BF>
__device__ __forceinline__ h8 to_halves(u32x4 x, float sc) {
  if constexpr (!BF) return __builtin_bit_cast(h8, x);
  h8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = (f16)(__builtin_bit_cast(float, x[i] << 16) * sc);
    r[2 * i + 1] = (f16)(__builtin_bit_cast(float, x[i] & 0xffff0000u) * sc);
  }
  return r;
}

// A row's quarter (thread t of the four of a row) into LDS; returns the row's power-of-two scale in sc and
// its factor (normalisation over that scale).
template <int DK, bool BF>
__device__ __forceinline__ float prep_row(const uint16_t* p, f16* dst, int t, bool real, bool l2norm, float& sc) {
  constexpr int NV = DK / 32;
  u32x4 x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i] = real ? *(const u32x4*)(p + (t * NV + i) * 8) : u32x4{0, 0, 0, 0};
  float ss = 0.0f, inv = 1.0f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const float a = w2f<BF>((uint16_t)x[i][d]), b = w2f<BF>((uint16_t)(x[i][d] >> 16));
      ss = __builtin_fmaf(a, a, ss);
      ss = __builtin_fmaf(b, b, ss);
      const uint32_t u = x[i][d] & 0x7fff7fffu;
      top = max(top, max(u >> 16, u & 0xffffu));
    }
  ss += dpp_f32<0xB1>(ss);
  ss += dpp_f32<0x4E>(ss);
  sc = 1.0f;
  if constexpr (BF) {
    top = max(top, (uint32_t)dpp_i32<0xB1>((int)top));
    top = max(top, (uint32_t)dpp_i32<0x4E>((int)top));
    sc = pow2_scale(__builtin_bit_cast(float, top << 16), inv);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) *(h8*)(dst + (t * NV + i) * 8) = to_halves<BF>(x[i], sc);
  return l2norm ? l2_factor(ss) * inv : inv;
}

// Rows of M (LDS) to a fragment row's pair of halves with the row's own scale; returns the row factor.
__device__ __forceinline__ float store_frags(const float (*M)[kMS], int t, int lane, f16 (*out)[2][64][8]) {
  const int g = lane >> 4, r = 16 * t + (lane & 15);
  f32x4 x[4];
  float m = 0.0f;
  const int nj = t / 2 + 1;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (j >= nj) continue;
    x[2 * j] = *(const f32x4*)&M[r][32 * j + 4 * g];
    x[2 * j + 1] = *(const f32x4*)&M[r][32 * j + 16 + 4 * g];
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(__builtin_fabsf(x[2 * j][i]), __builtin_fabsf(x[2 * j + 1][i])));
  }
  float inv;
  const float sc = pow2_scale(max_rows4(m), inv);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (j >= nj) continue;
    h8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f16 a, b;
      split(x[2 * j + i / 4][i % 4] * sc, a, b);
      hi[i] = a;
      lo[i] = b;
    }
    const int f = frag_of(t, j);
    *(h8*)out[f][0][lane] = hi;
    *(h8*)out[f][1][lane] = lo;
  }
  return inv;
}

template <int DK, bool BF>
__global__ __launch_bounds__(256) void delta_prep_kernel(DeltaArgs a, ChunkRec* recs, int64_t slot0) {
  __shared__ __align__(16) PrepLds<DK> L;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
  const int rep = a.Hv / a.Hk, ng = (rep + kGroup - 1) / kGroup;
  const int64_t bx = blockIdx.x;
  const int hg = (int)(bx % (a.Hk * ng));
  const int64_t slot = bx / (a.Hk * ng);
  const int hk = hg / ng, h0 = hk * rep + (hg % ng) * kGroup;
  const int nh = min(kGroup, (hk + 1) * rep - h0);
  int64_t tok;
  int len;
  if (!chunk_of(a, slot0 + slot, tok, len)) return;
  ChunkRec* rec = recs + slot * a.Hv + h0;

  float ks, qs;
  {
    const int row = tid >> 2, t = tid & 3;
    const bool real = row < len;
    const float rk = prep_row<DK, BF>(a.k + (tok + row) * a.ld_k + hk * DK, L.in.k[row], t, real, a.l2norm, ks);
    const float rq = prep_row<DK, BF>(a.q + (tok + row) * a.ld_q + hk * DK, L.in.q[row], t, real, a.l2norm, qs) * a.scale;
    if (t == 0) {
      L.rk[row] = rk;
      L.rq[row] = rq;
    }
    for (int h = t; h < nh; h += 4) {
      rec[h].ks[row] = ks;
      rec[h].qs[row] = qs;
    }
  }
  if (w < nh) {  // wave w: the decays of head w
    const bool real = lane < len;
    float gv = real ? a.g[(tok + lane) * a.ld_g + h0 + w] : 0.0f;
    gv = gv < -1e5f ? -1e5f : gv;
    double G = (double)gv * 1.4426950408889634;
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t u = __builtin_bit_cast(uint64_t, G);
      const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)u, o, 64), hi = (uint32_t)__shfl_up((int)(uint32_t)(u >> 32), o, 64);
      if (lane >= o) G += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
    }
    L.G[w][lane] = G;
    L.be[w][lane] = real ? a.beta[(tok + lane) * a.ld_beta + h0 + w] : 0.0f;
  }
  __syncthreads();

  // k_i.k_j and q_i.k_j: wave w has the rows of tile w
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    kk[t] = f32x4{0, 0, 0, 0};
    qk[t] = f32x4{0, 0, 0, 0};
  }
#pragma unroll
  for (int s = 0; s < DK / 32; ++s) {
    const h8 ka = *(const h8*)&L.in.k[16 * w + c][32 * s + 8 * g];
    const h8 qa = *(const h8*)&L.in.q[16 * w + c][32 * s + 8 * g];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t > w) continue;
      const h8 b = *(const h8*)&L.in.k[16 * t + c][32 * s + 8 * g];
      kk[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, b, kk[t], 0, 0, 0);
      qk[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa, b, qk[t], 0, 0, 0);
    }
  }
  __syncthreads();  // the rows are read: M takes their place

  if (w < nh) {     // wave w: the row factors of head w
    const double G = L.G[w][lane], GC = L.G[w][kC - 1];
    const float eG = __builtin_amdgcn_exp2f((float)G), rk = L.rk[lane];
    rec[w].c1[lane] = eG * rk;
    rec[w].c2[lane] = eG * L.rq[lane];
    rec[w].w[lane] = __builtin_amdgcn_exp2f((float)(GC - G)) * rk;
    if (lane == 0) rec[w].dec = __builtin_amdgcn_exp2f((float)GC);
  }
  for (int h = 0; h < nh; ++h) {
    float (*M)[kMS] = L.M[h];
    f32x4 d[4];
    float rkj[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t > w) continue;
      const double Gj = L.G[h][16 * t + c];
      rkj[t] = L.rk[16 * t + c];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * w + 4 * g + i;
        // (above the diagonal the difference may be of any size: it is not exponentiated)
        d[t][i] = 16 * t + c <= row ? __builtin_amdgcn_exp2f((float)(L.G[h][row] - Gj)) : 0.0f;
        M[row][16 * t + c] = 16 * t + c <= row ? ((qk[t][i] * L.rq[row]) * rkj[t]) * d[t][i] : 0.0f;
      }
    }
    if (!(w & 1))
#pragma unroll
      for (int i = 0; i < 4; ++i) M[16 * w + 4 * g + i][16 * w + 16 + c] = 0.0f;  // the rest of the column block
    wave_sync();
    const float pr = store_frags(M, w, lane, rec[h].P);
    if (g == 0) rec[h].pr[16 * w + c] = pr;
    wave_sync();
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t > w) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * w + 4 * g + i;
        M[row][16 * t + c] = 16 * t + c < row ? (((kk[t][i] * L.rk[row]) * rkj[t]) * d[t][i]) * L.be[h][row] : 0.0f;
      }
    }
  }
  __syncthreads();
  if (w >= nh) return;

  // (I + A)^-1 of head w by 16 x 16 blocks. The diagonal blocks first: lane (b, c) solves column c of block b.
  float (*M)[kMS] = L.M[w];
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.0f : 0.0f;
#pragma unroll
      for (int q = 0; q < i; q += 4) {
        const f32x4 m = *(const f32x4*)&M[16 * g + i][16 * g + q];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (q + e < i) s = __builtin_fmaf(-m[e], x[q + e], s);
      }
      x[i] = s;
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < 16; ++i) M[16 * g + i][16 * g + c] = x[i];
    wave_sync();
  }
  // Then X_ij = -X_ii sum_{j <= k < i} A_ik X_kj down each block column, in fp32 on the matrix cores. With the
  // contraction taken in the order 4 g + s (s the step), a result is the next product's operand as it lies.
  f32x4 X[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) X[j][j][i] = M[16 * j + 4 * g + i][16 * j + c];
#pragma unroll
  for (int dist = 1; dist < 4; ++dist)
#pragma unroll
    for (int j = 0; j + dist < 4; ++j) {
      const int i = j + dist;
      f32x4 y = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k < j || k >= i) continue;
        const f32x4 m = *(const f32x4*)&M[16 * i + c][16 * k + 4 * g];
#pragma unroll
        for (int s = 0; s < 4; ++s) y = __builtin_amdgcn_mfma_f32_16x16x4f32(m[s], X[k][j][s], y, 0, 0, 0);
      }
      const f32x4 m = *(const f32x4*)&M[16 * i + c][16 * i + 4 * g];
      f32x4 z = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 4; ++s) z = __builtin_amdgcn_mfma_f32_16x16x4f32(m[s], -y[s], z, 0, 0, 0);
      X[i][j] = z;
    }
  wave_sync();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float be = L.be[w][16 * j + c];
#pragma unroll
    for (int i = j; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) M[16 * i + 4 * g + e][16 * j + c] = X[i][j][e] * be;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    M[4 * g + e][16 + c] = 0.0f;
    M[32 + 4 * g + e][48 + c] = 0.0f;
  }
  wave_sync();
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float tr = store_frags(M, t, lane, rec[w].T);
    if (g == 0) rec[w].tr[16 * t + c] = tr;
  }
}

// ---------------------------------------------------------------------------------------------
// The chain: one sequence, one value head, 64 value columns, 16 per wave. The state lies in a wave's registers
// as 16 x 16 results (rows dk, columns dv); each wave needs nothing of the others, they share the operands
// in LDS. The next chunk's operands are in flight in registers meanwhile.
// ---------------------------------------------------------------------------------------------
template <int DK>
struct ChainLds {
  f16 k[kC][DK + 8], q[kC][DK + 8];  // columns in the order 32 j + 8 g + 4 h + i for dk = 32 j + 16 h + 4 g + i
  f16 T[6][2][64][8], P[6][2][64][8];
  float vec[448];                    // c1, c2, tr, pr, w, ks, qs of the record
  float dec;
};

template <int DK>
struct Stage {  // a thread's part of a chunk's operands
  u32x4 k[DK / 32], q[DK / 32];
  u32x4 tp[6];
  float v0, v1;
  float dec;
};

template <int DK>
__device__ __forceinline__ void stage_load(const DeltaArgs& a, const ChunkRec* rec, int64_t tok, int len, int hk, Stage<DK>& s) {
  const int tid = threadIdx.x, row = tid >> 2, t = tid & 3;
  const bool real = row < len;
  const uint16_t* kp = a.k + (tok + row) * a.ld_k + hk * DK;
  const uint16_t* qp = a.q + (tok + row) * a.ld_q + hk * DK;
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) {
    s.k[i] = real ? *(const u32x4*)(kp + (i * 4 + t) * 8) : u32x4{0, 0, 0, 0};
    s.q[i] = real ? *(const u32x4*)(qp + (i * 4 + t) * 8) : u32x4{0, 0, 0, 0};
  }
  const u32x4* r = (const u32x4*)rec;
#pragma unroll
  for (int i = 0; i < 6; ++i) s.tp[i] = r[i * 256 + tid];
  const float* v = rec->c1;
  s.v0 = v[tid];
  s.v1 = tid < 192 ? v[256 + tid] : 0.0f;
  s.dec = rec->dec;
}

template <int DK, bool BF>
__device__ __forceinline__ void stage_store(const Stage<DK>& s, ChainLds<DK>& L, float ks, float qs) {
  const int tid = threadIdx.x, row = tid >> 2, t = tid & 3;
  // 8 columns 32 i + 8 t ..: halves h = t / 2, groups 2 (t % 2) and the next
  const int at = 16 * (t & 1) + 4 * (t >> 1);
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) {
    const h8 k = to_halves<BF>(s.k[i], ks), q = to_halves<BF>(s.q[i], qs);
    *(h4*)&L.k[row][32 * i + at] = __builtin_shufflevector(k, k, 0, 1, 2, 3);
    *(h4*)&L.k[row][32 * i + at + 8] = __builtin_shufflevector(k, k, 4, 5, 6, 7);
    *(h4*)&L.q[row][32 * i + at] = __builtin_shufflevector(q, q, 0, 1, 2, 3);
    *(h4*)&L.q[row][32 * i + at + 8] = __builtin_shufflevector(q, q, 4, 5, 6, 7);
  }
  u32x4* d = (u32x4*)&L.T[0][0][0][0];  // T and P are adjacent here as in the record
#pragma unroll
  for (int i = 0; i < 6; ++i) d[i * 256 + tid] = s.tp[i];
  L.vec[tid] = s.v0;
  if (tid < 192) L.vec[256 + tid] = s.v1;
  if (tid == 0) L.dec = s.dec;
}

// The pair of halves of a 32-deep operand from two results' registers, scaled.
__device__ __forceinline__ void split8(const f32x4& x, const f32x4& y, float sc, h8& hi, h8& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f16 a, b;
    split(x[i] * sc, a, b);
    hi[i] = a;
    lo[i] = b;
    split(y[i] * sc, a, b);
    hi[4 + i] = a;
    lo[4 + i] = b;
  }
}
__device__ __forceinline__ float max4(const f32x4& x, float m) {
  return fmaxf(fmaxf(m, fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1]))), fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3])));
}

template <int N>
__device__ __forceinline__ void split_col(const f32x4 (&x)[N], h8 (&hi)[N / 2], h8 (&lo)[N / 2], float& inv) {
  float m = 0.0f;
#pragma unroll
  for (int t = 0; t < N; ++t) m = max4(x[t], m);
  const float sc = pow2_scale(max_rows4(m), inv);
#pragma unroll
  for (int j = 0; j < N / 2; ++j) split8(x[2 * j], x[2 * j + 1], sc, hi[j], lo[j]);
}

#define DELTA_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

// y = M x for a lower triangle M of fragments and a column operand x (both pairs).
__device__ __forceinline__ void tri_product(const f16 (*F)[2][64][8], int lane, const h8 (&xh)[2], const h8 (&xl)[2], f32x4 (&y)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    f32x4 s = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j <= t / 2; ++j) {
      const int f = t + (t > 2 ? 1 : 0) + j;
      const h8 hi = *(const h8*)F[f][0][lane], lo = *(const h8*)F[f][1][lane];
      s = DELTA_MFMA(lo, xh[j], s);
      s = DELTA_MFMA(hi, xl[j], s);
      s = DELTA_MFMA(hi, xh[j], s);
    }
    y[t] = s;
  }
}

template <int DK, bool BF>
__global__ __launch_bounds__(256) void delta_chain_kernel(DeltaArgs a, const ChunkRec* recs, int64_t slot0, int64_t slot1) {
  __shared__ __align__(16) ChainLds<DK> L;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
  const int nb = (a.Dv + 63) / 64;
  int bx = blockIdx.x;
  const int vb = bx % nb;
  bx /= nb;
  const int h = bx % a.Hv, b = bx / a.Hv, hk = h / (a.Hv / a.Hk);
  const int dv = 64 * vb + 16 * w + c;
  const bool active = 64 * vb + 16 * w < a.Dv;  // (whole waves)
  int64_t t0, t1;
  seq_range(a, b, t0, t1);
  const int64_t key = t0 / kC + b, nch = (t1 - t0 + kC - 1) / kC;
  int64_t cb = slot0 - key, ce = slot1 - key;  // this launch's chunks of the sequence
  cb = cb < 0 ? 0 : cb;
  ce = ce > nch ? nch : ce;
  if (cb >= ce && !(nch == 0 && slot0 == 0)) return;
  const int slot = slot_of(a, b);
  if (slot < 0) {
    const uint16_t fill = slot == kSlotPad ? 0 : 0x7fff;
    if (active)
      for (int64_t t = t0 + cb * kC + g; t < t1 && t < t0 + ce * kC; t += 4) a.out[t * a.ld_out + (int64_t)h * a.Dv + dv] = fill;
    return;
  }
  constexpr int NM = DK / 16;
  f32x4 S[NM];
  const size_t so = (((size_t)slot * a.Hv + h) * a.Dv + (active ? dv : 0)) * DK + 4 * g;
  const float* sp = (cb == 0 ? a.state : a.state_out) + so;
#pragma unroll
  for (int m = 0; m < NM; ++m) S[m] = *(const f32x4*)(sp + 16 * m);

  Stage<DK> st;
  const ChunkRec* rec = recs + (key + cb - slot0) * a.Hv + h;
  uint16_t vv[16];
  int64_t tok = t0 + cb * kC;
  int len = (int)(t1 - tok < kC ? t1 - tok : kC);
  const int64_t vcol = (int64_t)h * a.Dv + (active ? dv : 0);
  auto load_v = [&](int64_t tk, int ln) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 16 * (i / 4) + 4 * g + (i & 3);
      vv[i] = r < ln ? a.v[(tk + r) * a.ld_v + vcol] : (uint16_t)0;
    }
  };
  if (cb < ce) {
    stage_load<DK>(a, rec, tok, len, hk, st);
    load_v(tok, len);
  }
  for (int64_t ch = cb; ch < ce; ++ch) {
    lds_barrier();  // every wave is done with the last chunk's operands
    float ks = 1.0f, qs = 1.0f;
    if constexpr (BF) {
      ks = rec->ks[tid >> 2];
      qs = rec->qs[tid >> 2];
    }
    stage_store<DK, BF>(st, L, ks, qs);
    lds_barrier();
    f32x4 v[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i / 4][i & 3] = w2f<BF>(vv[i]);
    const int64_t tk = tok;
    const int ln = len;
    if (ch + 1 < ce) {
      rec += a.Hv;
      tok += kC;
      len = (int)(t1 - tok < kC ? t1 - tok : kC);
      stage_load<DK>(a, rec, tok, len, hk, st);
      load_v(tok, len);
    }
    // K S^T and Q S^T
    h8 sh[NM / 2], sl[NM / 2];
    float sinv;
    split_col<NM>(S, sh, sl, sinv);
    f32x4 ks4[4], qs4[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 x = f32x4{0, 0, 0, 0}, y = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NM / 2; ++j) {
        const h8 ka = *(const h8*)&L.k[16 * t + c][32 * j + 8 * g], qa = *(const h8*)&L.q[16 * t + c][32 * j + 8 * g];
        x = DELTA_MFMA(ka, sl[j], x);
        x = DELTA_MFMA(ka, sh[j], x);
        y = DELTA_MFMA(qa, sl[j], y);
        y = DELTA_MFMA(qa, sh[j], y);
      }
      ks4[t] = x;
      qs4[t] = y;
    }
    const f32x4* vec = (const f32x4*)L.vec;
    f32x4 u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 c1 = vec[4 * t + g];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[t][i] = __builtin_fmaf(-(c1[i] * sinv), ks4[t][i], v[t][i]);
    }
    h8 xh[2], xl[2];
    float xinv;
    split_col<4>(v, xh, xl, xinv);
    tri_product(L.T, lane, xh, xl, u);
    f32x4 uw[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 tr = vec[2 * 16 + 4 * t + g], ww = vec[4 * 16 + 4 * t + g];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[t][i] = u[t][i] * (tr[i] * xinv);
        uw[t][i] = u[t][i] * ww[i];
      }
    }
    // the state
    h8 wh[2], wl[2];
    float winv;
    split_col<4>(uw, wh, wl, winv);
    const float dec = L.dec;
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      f32x4 x = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // rows dk 16 m + 4 q + e of k^T: the lane's address is token 32 j + 4 g + c / 4 (then 16 more), chunk q = c % 4
        const f16* p = &L.k[32 * j + 4 * g + (c >> 2)][32 * (m >> 1) + 8 * (c & 3) + 4 * (m & 1)];
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 16 * (DK + 8)));
        const h8 ka = __builtin_bit_cast(h8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        x = DELTA_MFMA(ka, wl[j], x);
        x = DELTA_MFMA(ka, wh[j], x);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) S[m][i] = __builtin_fmaf(x[i], winv, dec * S[m][i]);
    }
    // the outputs
    h8 uh[2], ul[2];
    float uinv;
    split_col<4>(u, uh, ul, uinv);
    f32x4 o[4];
    tri_product(L.P, lane, uh, ul, o);
    if (active) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 c2 = vec[16 + 4 * t + g], pr = vec[3 * 16 + 4 * t + g];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * t + 4 * g + i;
          const float x = __builtin_fmaf(qs4[t][i], c2[i] * sinv, o[t][i] * (pr[i] * uinv));
          if (r < ln) a.out[(tk + r) * a.ld_out + vcol] = f2w<BF>(x);
        }
      }
    }
  }
  if (active) {
    float* op = a.state_out + so;
#pragma unroll
    for (int m = 0; m < NM; ++m) *(f32x4*)(op + 16 * m) = S[m];
  }
}

template <int DK, bool BF>
hipError_t launch_chunked(const DeltaArgs& a, void* ws, int64_t per, hipStream_t s) {
  const int rep = a.Hv / a.Hk;
  const int64_t ng = (int64_t)a.Hk * ((rep + kGroup - 1) / kGroup), slots = delta_chunk_slots(a.n_tokens, a.n_seq);
  const int64_t chains = (int64_t)a.n_seq * a.Hv * ((a.Dv + 63) / 64);
  if (chains > 0x7fffffff || per * ng > 0x7fffffff) return hipErrorInvalidValue;
  ChunkRec* recs = (ChunkRec*)ws;
  for (int64_t s0 = 0; s0 < slots; s0 += per) {
    const int64_t n = s0 + per < slots ? per : slots - s0;
    hipLaunchKernelGGL((delta_prep_kernel<DK, BF>), dim3((unsigned)(n * ng)), dim3(256), 0, s, a, recs, s0);
    hipLaunchKernelGGL((delta_chain_kernel<DK, BF>), dim3((unsigned)chains), dim3(256), 0, s, a, recs, s0, s0 + n);
  }
  return hipGetLastError();
}

}  // namespace

int64_t delta_chunk_slots(int64_t n_tokens, int n_seq) { return n_tokens / kC + n_seq; }

// Chunks whose records are held at once: all, or as many as fit 1 GiB.
static int64_t slots_per_pass(const DeltaArgs& a) {
  const int64_t all = delta_chunk_slots(a.n_tokens, a.n_seq), fit = ((int64_t)1 << 30) / ((int64_t)a.Hv * sizeof(ChunkRec));
  return fit < 1 ? 1 : (fit < all ? fit : all);
}
size_t delta_chunk_workspace(const DeltaArgs& a) { return (size_t)(slots_per_pass(a) * a.Hv) * sizeof(ChunkRec); }

hipError_t launch_delta_chunked(const DeltaArgs& a, void* ws, hipStream_t s) {
  const int64_t per = slots_per_pass(a);
  if (a.Dk == 128) return a.bf16 ? launch_chunked<128, true>(a, ws, per, s) : launch_chunked<128, false>(a, ws, per, s);
  return a.bf16 ? launch_chunked<64, true>(a, ws, per, s) : launch_chunked<64, false>(a, ws, per, s);
}

}  // namespace dfssm
