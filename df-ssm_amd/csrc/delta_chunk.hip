// The gated delta rule over chunks of 64 tokens (gfx950 matrix cores).
//
// Per value head and chunk, with G_i = g_1 + .. + g_i, S0 the state before it (S^T stored as Dk x Dv tiles) and
// row factors r_i that undo a normalisation or a power-of-two scaling of k_i or q_i:
//   A_ij = beta_i k_i.k_j e^{G_i - G_j} (i > j),  T = (I + A)^-1 diag(beta),  P_ij = scale q_i.k_j e^{G_i - G_j} (i >= j)
//   U = T (V - diag(e^G) K S0^T);  O = diag(scale e^G) Q S0^T + P U;  S1 = e^{G_C} S0 + (diag(e^{G_C - G}) U)^T K
// Two launches: delta_prep_kernel makes T and the row factors of all chunks in parallel, delta_chain_kernel walks the
// chunks of a sequence and head with its state in registers and makes P, which is less work than reading it, beside
// them.
//
// What bounds it. One long sequence: the path from chunk to chunk (K S^T, T (V - ..), the new state: three dependent
// products with a split into 16-bit parts before each, all of a chunk's on one wave), 4700 clocks a chunk; 16411 tokens x
// 64 heads of 64 x 128 take 0.59 ms, 0.09 of it the preparation (fp16; 416 MB, 0.085 ms of copying; the matrix cores are
// busy 16% of the chain). Ragged ones: that path of the longest at 64 value columns to a workgroup (NW = 4), 8200 clocks.
// Many sequences: memory. 64 x 512 tokens x 80 heads move 2.4 GB that they cannot do without, 0.57 GB of T's records once
// out and once in, and k twice, 4.2 GB in 1.00 ms, 0.27 of it the preparation (bf16; 4.9 TB/s is what a copy reaches; of
// the chain the matrix cores are busy 32%). Records in passes small enough for the last-level cache were slower: each
// pass reads and writes the states.
//
// Numbers. States, sums and everything between products are fp32. Products run on the 16-bit matrix cores with
// fp32 accumulation. q and k are exact operands there, in their own type. A factor of fp32 values is a sum of
// 16-bit parts: beside fp16 rows, and where both factors are fp32 (T (V - ..), P U), pairs of halves,
// x 2^s = hi + lo, which hold 22 bits, with s per row of T and P and per value column of S, V - .. and U chosen so
// that the largest magnitude lies in [2^14, 2^15); beside bf16 rows three bf16 parts, which hold 24 bits and need
// no scale. (Q S^T is no exception, though its sum with P U is rounded to 16 bits: where a token overwrites what the
// state has for its key, the two nearly cancel.) A product of two pairs leaves out lo lo, 2^-24 of it. So an fp32 state
// comes out as from fp32 arithmetic (2e-7 of its norm), at 2 or 3 matrix instructions per product instead of the 8 times
// as slow fp32 ones. A pair's value far below the largest M of its scale keeps fewer bits than 22: below 2^-17 M it is off
// by up to 2^-39 M, the last of a subnormal half. That shows where a large v - .. is forgotten again in the same 64
// tokens and small ones follow (three bf16 parts of T, P, V - .. and U would need six products for three, and 18 KiB more
// LDS, which 32 columns to a workgroup do not have). And the chunk's equations have as many factors A_ij as pairs of
// tokens, each rounded by itself: where neighbouring keys are alike and beta |k|^2 is close to 2, so that each token undoes
// the one before and nothing dies out, a state is off by 2^-15 of its largest value after a few chunks, in fp32
// throughout too.
// G is summed in fp64, so that differences survive a decay of any size in the same chunk; -inf is held to -1e5.
#include "common.h"
#include "delta.h"
#include "delta_plan.h"
#include "dfssm_kernels.h"
#include "parts.h"

namespace dfssm {

namespace {

constexpr int kC = 64;        // tokens of a chunk

// What the preparation leaves per chunk and value head: T in the order in which a lane of the matrix cores takes
// it, fragments of 16 rows x 32 columns, lane (g, r) row r, columns 4 g .. 4 g + 3 and 16 + 4 g ..: the order in
// which 16 x 16 results lie in registers, so results are operands without moving between lanes. Six fragments
// cover a lower triangle.
struct ChunkRec {
  f16 T[6][2][64][8];   // [fragment][hi, lo][lane]
  float c1[kC];         // e^{G_i} times k's row factor
  float tr[kC];         // row factor of T
  float w[kC];          // e^{G_C - G_i} times k's row factor
  float rk[kC];         // k's row factor, its normalisation
  float Gh[kC], Gl[kC]; // G_i over log 2, the float nearest and the rest
};
static_assert(sizeof(ChunkRec) == 13824, "T, 1.5 KiB of factors");

// Rows of q and k in LDS: the 16-byte pieces of a row are exchanged so that the same piece of 16 rows, an operand,
// lies in all 64 banks.
template <int DK>
__device__ __forceinline__ int piece_at(int row, int p) {
  return p ^ (DK == 128 ? row & 15 : (row >> 1) & 7);
}

__device__ __forceinline__ int frag_of(int t, int j) { return t + (t > 2 ? 1 : 0) + j; }  // row tile, column block

// ---------------------------------------------------------------------------------------------
// Preparation: a chunk and value head per wave, which needs no barrier. The four waves of a workgroup take four
// heads, which find a key head's rows in the L1 cache; a workgroup goes over several chunks, and the rows of the
// next are on their way while it inverts.
// Products are taken with the operands exchanged, (K Q^T)^T: a lane then holds a row's four neighbouring columns,
// which is how the next product wants a left operand, so neither P nor A passes through LDS (but the diagonal
// blocks of A, whose elements every lane of a block reads).
// ---------------------------------------------------------------------------------------------
constexpr int kBS = 20, kBlock = 16 * kBS + 16;  // a 16 x 16 block in LDS: row and block stride, in floats

struct PrepLds {              // of a wave
  float B[6 * kBlock];        // the diagonal blocks, then their inverses, then the blocks below the diagonal
  double G[kC];               // in units of log 2
  float F[3][kC];             // e^{G_16w - G_j} rk_j for the row tiles w = 1 .. 3
  float rk[kC], kb[kC], ke[kC], be[kC];
  float ss[kC];
};
// Element c of the diagonal of a 16 x 16 result, in its lane (g = c / 4).
__device__ __forceinline__ float diagonal(const f32x4& x, int c) {
  return (c & 2) ? ((c & 1) ? x[3] : x[2]) : ((c & 1) ? x[1] : x[0]);
}

// 16 rows, lane (g, r): row r, columns 32 j + 8 g ..
template <int DK>
__device__ __forceinline__ void load_rows(Rsrc rows, int64_t ld, int t, int lane, u32x4 (&x)[DK / 32]) {
  const int off = (16 * t + (lane & 15)) * (int)ld * 2 + (lane >> 4) * 16;
#pragma unroll
  for (int j = 0; j < DK / 32; ++j) x[j] = row_load16(rows, off, j * 64);
}
// Row tile W of a triangle, x[t] a lane's four columns of column tile t <= W, as pairs of halves with the row's
// own scale; returns the row factor.
template <int W>
__device__ __forceinline__ float store_frags(const f32x4 (&x)[W + 1], int lane, f16 (*out)[2][64][8]) {
  float m = 0.0f;
#pragma unroll
  for (int t = 0; t <= W; ++t) m = max4(x[t], m);
  float inv;
  const float sc = pow2_scale(max_rows4(m), inv);
#pragma unroll
  for (int j = 0; 2 * j <= W; ++j) {
    h8 part[2];
    split8(x[2 * j], 2 * j + 1 <= W ? x[2 * j + 1 <= W ? 2 * j + 1 : W] : f32x4{0, 0, 0, 0}, sc, part);
    const int f = frag_of(W, j);
    *(h8*)out[f][0][lane] = part[0];
    *(h8*)out[f][1][lane] = part[1];
  }
  return inv;
}

template <int DK>
struct PrepRows {  // what is loaded ahead for a task
  u32x4 k[4][DK / 32];
  float g, be;
};

// The sequences from the longest to the shortest, the first one first among equals, into order; by 256 threads.
constexpr int kOrdered = 256;
__device__ __forceinline__ void order_by_length(const DeltaArgs& a, int* len, int* order) {
  const int i = threadIdx.x;
  int mine = 0, rank = 0;
  if (i < a.n_seq) {
    int64_t t0, t1;
    seq_range(a, i, t0, t1);
    len[i] = mine = (int)(t1 - t0);
  }
  __syncthreads();
  if (i < a.n_seq) {
    for (int q = 0; q < a.n_seq; ++q) rank += len[q] > mine || (len[q] == mine && q < i) ? 1 : 0;
    order[rank] = i;
  }
  __syncthreads();
}

template <int DK, bool BF>
__global__ __attribute__((amdgpu_waves_per_eu(2))) __launch_bounds__(256) void
delta_prep_kernel(DeltaArgs a, ChunkRec* recs, int* order, int64_t slot0, int64_t n_tasks) {
  constexpr int NJ = DK / 32;
  __shared__ __align__(16) PrepLds lds[4];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  PrepLds& L = lds[wave];
  if (order && blockIdx.x == 0) order_by_length(a, (int*)lds, order);
  const int rep = a.Hv / a.Hk, nw = (a.Hv + 3) / 4;

  Where seq{0, 0, 0, 0};
  PrepRows<DK> in;
  int64_t task = blockIdx.x, slot = 0;
  int h = 0, len = 0;
  auto load = [&]() {
    slot = task / nw;
    h = (int)(task % nw) * 4 + wave;
    int64_t tok;
    len = (int)tile_of<kC>(a, slot0 + slot, seq, tok);
    if (h >= a.Hv) {  // (a head there is, rows there are none)
      len = 0;
      h = 0;
    }
    const int hk = h / rep;
    const Rsrc kr = rows_of(a.k + tok * a.ld_k + hk * DK, a.ld_k, len, DK);
#pragma unroll
    for (int t = 0; t < 4; ++t) load_rows<DK>(kr, a.ld_k, t, lane, in.k[t]);
    const int64_t at = tok + (lane < len ? lane : 0);
    in.g = a.g[at * a.ld_g + h];
    in.be = a.beta[at * a.ld_beta + h];
  };
  load();
  for (;;) {
    ChunkRec* rec = recs + slot * a.Hv + h;
    const bool some = len > 0;
    f32x4 A[4][4];
    if (some) {
      double G;
      {
        const bool real = lane < len;
        float gv = real ? in.g : 0.0f;
        gv = gv < -1e5f ? -1e5f : gv;
        G = (double)gv * 1.4426950408889634;
        G += moved<0x111, 0xf>(G);  // running sums: from 1, 2, 4 and 8 lanes before, in the row of 16
        G += moved<0x112, 0xf>(G);
        G += moved<0x114, 0xf>(G);
        G += moved<0x118, 0xf>(G);
        G += moved<0x142, 0xa>(G);  // row 0's last to row 1, 2's to 3; then lane 31's to rows 2 and 3
        G += moved<0x143, 0xc>(G);
      }
      const float be = lane < len ? in.be : 0.0f;
      h8 k[4][NJ];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < NJ; ++j) k[t][j] = __builtin_bit_cast(h8, in.k[t][j]);
      f32x4 kd[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        kd[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NJ; ++j) kd[t] = mm<BF>(k[t][j], k[t][j], kd[t]);
      }
      // a row's squares are on the diagonal of k k^T: in the lane of that row that has its column
      if (a.l2norm)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (g == (c >> 2)) L.ss[16 * t + c] = diagonal(kd[t], c);
      L.G[lane] = G;
      L.be[lane] = be;
      wave_sync();
      {  // lane: a token
        const float rk = a.l2norm ? l2_factor(L.ss[lane]) : 1.0f;
        const double GC = L.G[kC - 1], Gt = L.G[lane & 48];
        const float eG = __builtin_amdgcn_exp2f((float)G), et = __builtin_amdgcn_exp2f((float)(G - Gt));
        rec->c1[lane] = eG * rk;
        rec->w[lane] = __builtin_amdgcn_exp2f((float)(GC - G)) * rk;
        rec->rk[lane] = rk;
        rec->Gh[lane] = (float)G;
        rec->Gl[lane] = (float)(G - (double)(float)G);
        // e^{G_i - G_j} is taken apart at the first row of i's tile where j lies before it: with g <= 0 neither
        // factor exceeds 1, so the product of two is as good as one exponential
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float x = (float)(L.G[16 * w] - G);
          L.F[w - 1][lane] = __builtin_amdgcn_exp2f(lane < 16 * w ? x : 0.0f) * rk;
        }
        L.rk[lane] = rk;
        L.kb[lane] = be * rk;
        L.ke[lane] = (be * rk) * et;
      }
      wave_sync();
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 16 * w + c;  // the lane's row
#pragma unroll
        for (int t = 0; t < w; ++t) {
          A[w][t] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < NJ; ++j) A[w][t] = mm<BF>(k[t][j], k[w][j], A[w][t]);
        }
        const float ke = L.ke[i], kb = L.kb[i];
#pragma unroll
        for (int t = 0; t < w; ++t) {
          const f32x4 F = *(const f32x4*)&L.F[w - 1][16 * t + 4 * g];
#pragma unroll
          for (int e = 0; e < 4; ++e) A[w][t][e] = (A[w][t][e] * ke) * F[e];
        }
        const double Gi = L.G[i];
        const f32x4 rkj = *(const f32x4*)&L.rk[16 * w + 4 * g];
        f32x4 D;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (beyond the diagonal the difference may be of any size: not exponentiated)
          const int j = 4 * g + e;
          const float d = __builtin_amdgcn_exp2f(j < c ? (float)(Gi - L.G[16 * w + j]) : 0.0f) * rkj[e];
          D[e] = j < c ? (kd[w][e] * kb) * d : 0.0f;
        }
        *(f32x4*)&L.B[w * kBlock + c * kBS + 4 * g] = D;
      }
      wave_sync();
    }
    task += gridDim.x;
    const bool more = task < n_tasks;
    if (more) load();  // the registers of this task's rows are free
    if (some) {
      // (I + A)^-1 by 16 x 16 blocks. The diagonal blocks first: lane (b, c) solves column c of block b.
      {
        const float* B = &L.B[g * kBlock];
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == c ? 1.0f : 0.0f;
        f32x4 m[2][4];  // a row's elements, the next row's on their way
        m[1][0] = *(const f32x4*)&B[kBS];
#pragma unroll
        for (int i = 1; i < 16; ++i) {
          if (i < 15)
#pragma unroll
            for (int q = 0; q <= i; q += 4) m[(i + 1) & 1][q / 4] = *(const f32x4*)&B[(i + 1) * kBS + q];
          float s[4] = {x[i], 0.0f, 0.0f, 0.0f};  // four partial sums, so that no addition waits for the one before
#pragma unroll
          for (int j = 0; j < i; ++j) s[j & 3] = __builtin_fmaf(-m[i & 1][j / 4][j % 4], x[j], s[j & 3]);
          x[i] = (s[0] + s[1]) + (s[2] + s[3]);
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < 16; ++i) L.B[g * kBlock + i * kBS + c] = x[i];
        wave_sync();
      }
      // Then X_ij = -X_ii sum_{j <= k < i} A_ik X_kj, one block diagonal after another, in fp32 on the matrix
      // cores. With the contraction taken in the order 4 g + s (s the step) a result is a right operand as it lies.
      f32x4 X[4][4], D[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        D[j] = *(const f32x4*)&L.B[j * kBlock + c * kBS + 4 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) X[j][j][e] = L.B[j * kBlock + (4 * g + e) * kBS + c];
      }
      wave_sync();
#pragma unroll
      for (int dist = 1; dist < 4; ++dist) {
        f32x4 y[3];
#pragma unroll
        for (int j = 0; j + dist < 4; ++j) y[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < dist; ++k)
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j + dist < 4; ++j)
              y[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(A[j + dist][j + k][s], X[j + k][j][s], y[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j + dist < 4; ++j) X[j + dist][j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int j = 0; j + dist < 4; ++j)
            X[j + dist][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(D[j + dist][s], -y[j][s], X[j + dist][j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j + dist < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) L.B[((j + dist) * (j + dist - 1) / 2 + j) * kBlock + (4 * g + e) * kBS + c] = X[j + dist][j][e];
      }
      wave_sync();
      auto store_t = [&](auto tile) {
        constexpr int W = decltype(tile)::value;
        f32x4 T[W + 1];
#pragma unroll
        for (int t = 0; t <= W; ++t) {
          T[t] = t == W ? D[W] : *(const f32x4*)&L.B[(W * (W - 1) / 2 + t) * kBlock + c * kBS + 4 * g];
          const f32x4 bej = *(const f32x4*)&L.be[16 * t + 4 * g];
#pragma unroll
          for (int e = 0; e < 4; ++e) T[t][e] *= bej[e];
        }
        const float tr = store_frags<W>(T, lane, rec->T);
        if (g == 0) rec->tr[16 * W + c] = tr;
      };
      store_t(Int<0>{});
      store_t(Int<1>{});
      store_t(Int<2>{});
      store_t(Int<3>{});
      wave_sync();
    }
    if (!more) break;
  }
}

// ---------------------------------------------------------------------------------------------
// The chain: one sequence, one value head, 16 NW value columns. The state lies in registers as 16 x 16 results
// (rows of k's columns, 16 value columns per wave), and the waves that carry it need nothing of each other.
//   NW waves, the chain proper: K S^T, U and the new state; with NW = 4, where it is not what a chunk waits for, Q S^T too
//   NW waves, the outputs: Q S^T, P U
//   the fetchers: this chunk's P = tril(Q K^T ..), a fragment or two each, and the next one's operands, straight
//   into LDS. Waves of their own, as many as make eight in all; with NW = 4 the output waves do it beside their work
//   (12 waves would be three to a SIMD and have 168 registers each, and the chain needs 224).
// So waves of different kinds share a SIMD, products of one fill the gaps of the other, and only what the state
// needs is on the path from chunk to chunk.
// Result row 4 g + i of tile 2 j + h is k's column 32 j + 8 g + 4 h + i, so that a lane's part of a 32-deep
// operand is 16 contiguous bytes of a row of k.
// ---------------------------------------------------------------------------------------------
template <int DK>
struct Operands {
  f16 k[kC][DK], q[kC][DK];
  f16 T[6][2][64][8];             // the record: T
  float vec[384];                 // c1, tr, w, rk, Gh, Gl
};
template <int DK, int NW, int NT>
struct ChainLds {
  Operands<DK> op[2];
  uint16_t v[NW == 4 ? 1 : 2][NW == 4 ? 8 : kC * 16 * NW];  // NW < 4: rows of v, two chunks; else in registers
  f16 S[NW == 4 ? 1 : NW][NW == 4 ? 1 : DK / 32][NT][64][8];  // NW < 4: the state before the chunk, as operands
  f32x4 qs[NW == 4 ? NW : 1][NW == 4 ? 4 : 1][64];           // NW = 4: Q S^T
  f32x4 u[NW][4][64];
  f16 P[6][2][64][8];
  float F[6][32];                 // of P's fragments, see make_p
  float c2[kC], pr[2][kC];        // scale e^{G_i} times q's row factor; the row factors of P, by column block
  float sfac[2][NW][16], ufac[NW][16];  // per value column: what undoes the scaling of S and of U
};

template <int N>
__device__ __forceinline__ float col_max(const f32x4 (&x)[N], float m = 0.0f) {
#pragma unroll
  for (int t = 0; t < N; ++t) m = max4(x[t], m);
  return max_rows4(m);
}
template <int N, int NT>
__device__ __forceinline__ void split_all(const f32x4 (&x)[N], float sc, h8 (&part)[NT][N / 2]) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    h8 p[NT];
    split8(x[2 * j], x[2 * j + 1], sc, p);
#pragma unroll
    for (int i = 0; i < NT; ++i) part[i][j] = p[i];
  }
}

// Fragments of a triangle in LDS or global memory.
struct Tri {
  h8 hi[6], lo[6];
};
__device__ __forceinline__ void load_tri(Tri& f, const f16 (*F)[2][64][8], int lane) {
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    f.hi[i] = *(const h8*)F[i][0][lane];
    f.lo[i] = *(const h8*)F[i][1][lane];
  }
}
// y[j] = M_j x_j for the 32-column blocks M_j of a triangle (both pairs; with FLIP the transpose), the row tiles in
// turn so that no product waits for the one before. With SUM the blocks have one scale and y[0] takes both.
template <bool FLIP, bool SUM>
__device__ __forceinline__ void tri_product(const Tri& f, const h8 (&x)[2][2], f32x4 (&y)[2][4]) {
  const int at[4] = {0, 1, 2, 4};
  auto add = [&](const h8& u, const h8& v, f32x4& w) { w = FLIP ? mm<false>(v, u, w) : mm<false>(u, v, w); };
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int t = 2 * j; t < 4; ++t) y[j][t] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    f32x4 (&z)[4] = y[SUM ? 0 : j];
#pragma unroll
    for (int t = 2 * j; t < 4; ++t) add(f.lo[at[t] + j], x[0][j], z[t]);
#pragma unroll
    for (int t = 2 * j; t < 4; ++t) add(f.hi[at[t] + j], x[1][j], z[t]);
#pragma unroll
    for (int t = 2 * j; t < 4; ++t) add(f.hi[at[t] + j], x[0][j], z[t]);
  }
}

// y = X S^T for 64 rows X in LDS (two row tiles at a time, the next two in flight) and S in NT parts; with FLIP
// its transpose, a lane then has four neighbouring value columns of a token.
template <int DK, bool BF, bool FLIP, int NT>
__device__ __forceinline__ void rows_product(const f16 (*X)[DK], int lane, const h8 (&s)[NT][DK / 32], f32x4 (&y)[4]) {
  constexpr int NJ = DK / 32;
  const int g = lane >> 4, c = lane & 15;
  h8 x[2][2][NJ];
  auto load = [&](int p) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * (2 * p + t) + c;
        x[p][t][j] = *(const h8*)&X[row][piece_at<DK>(row, 4 * j + g) * 8];
      }
  };
  auto add = [&](const h8& u, const h8& v, f32x4& w) { w = FLIP ? mm<BF>(v, u, w) : mm<BF>(u, v, w); };
  load(0);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (p == 0) load(1);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 a = f32x4{0, 0, 0, 0}, b = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = NT - 1; i >= 0; --i) {
        add(x[p][0][j], s[i][j], a);
        add(x[p][1][j], s[i][j], b);
      }
    y[2 * p] = a;
    y[2 * p + 1] = b;
  }
}


// 64 rows into LDS, KiB i, i + 4, .. of it, i < 4: 1 KiB per wave and instruction, the lanes reading the pieces that
// belong there. Every fourth KiB has the same exchange of pieces, so a lane's offset (rows_off) serves them all.
template <int DK>
__device__ __forceinline__ int rows_off(int64_t ld, int i, int lane) {
  constexpr int per = 512 / DK, pieces = DK / 8;  // rows of a KiB, pieces of a row
  const int row = per * i + lane / pieces;
  return row * (int)ld * 2 + piece_at<DK>(row, lane % pieces) * 16;
}
template <int DK>
__device__ __forceinline__ void fetch_rows(f16 (*to)[DK], const uint16_t* p, int64_t ld, int len, int i, int off) {
  constexpr int per = 512 / DK;
  const Rsrc r = rows_of(p, ld, len, DK);
  const int step = per * 8 * (int)ld;
#pragma unroll
  for (int n = 0; n < kC / per / 4; ++n)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)((char*)to + (4 * n + i) * 1024), 16, off, n * step, 0, 0);
}
// KiB i, i + NP, .. of a chunk's record.
template <int NP>
__device__ __forceinline__ void fetch_record(void* to, const ChunkRec* rec, int i, int lane) {
  constexpr int size = sizeof(ChunkRec);
  const Rsrc r = __builtin_amdgcn_make_buffer_rsrc((void*)rec, 0, size, 0x00027000);
#pragma unroll
  for (int n = 0; n < size / 1024; n += NP)
    if (n + i < size / 1024)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)((char*)to + (n + i) * 1024), 16, lane * 16, (n + i) * 1024, 0, 0);
  if (i == NP - 1)  // the last half, 8 bytes a lane: two instructions of 4
#pragma unroll
    for (int n = 0; n < 2; ++n)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)((char*)to + size / 1024 * 1024 + n * 256), 4, lane * 4,
                                               size / 1024 * 1024 + n * 256, 0, 0);
}

// Fragment (W, J) of P = tril(q_i.k_j e^{G_i - G_j}), rows 16 W .., columns 32 J .., with a scale of its own per row,
// so that no fragment waits for another; the one on the diagonal also leaves q's factors.
template <int W, int J, int DK, bool BF, int NW>
__device__ __forceinline__ void make_p(ChainLds<DK, NW, kParts<BF>>& L, const Operands<DK>& op, int lane, bool l2norm, float scale) {
  constexpr int NJ = DK / 32, F = W + (W > 2 ? 1 : 0) + J, T0 = 2 * J, NT = W > T0 ? 2 : 1;  // column tiles T0 .. T0 + NT - 1
  constexpr bool diag = T0 + NT - 1 == W;
  const int g = lane >> 4, c = lane & 15, i = 16 * W + c;
  const float *rk = op.vec + 192, *Gh = op.vec + 256, *Gl = op.vec + 320;
  const float bh = Gh[16 * W], bl = Gl[16 * W];
  // e^{G_i - G_j} for a j before the row tile is taken apart at the tile's first row, as in the preparation
  if constexpr (NT == 2 || !diag) {
    const int j = 32 * J + (lane & 31);
    const float x = (bh - Gh[j]) + (bl - Gl[j]);
    if (lane < 32) L.F[F][lane] = __builtin_amdgcn_exp2f(j < 16 * W ? x : 0.0f) * rk[j];
  }
  h8 q[NJ], k[NT][NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) q[j] = *(const h8*)&op.q[i][piece_at<DK>(i, 4 * j + g) * 8];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int row = 16 * (T0 + t) + c;
      k[t][j] = *(const h8*)&op.k[row][piece_at<DK>(row, 4 * j + g) * 8];
    }
  f32x4 x[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}, qq = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (l2norm) qq = mm<BF>(q[j], q[j], qq);
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = mm<BF>(k[t][j], q[j], x[t]);
  }
  const float gh = Gh[i], gl = Gl[i];
  const float pe = __builtin_amdgcn_exp2f((gh - bh) + (gl - bl));
  wave_sync();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (T0 + t < W) {
      const f32x4 f = *(const f32x4*)&L.F[F][16 * t + 4 * g];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = (x[t][e] * pe) * f[e];
    } else {
      const f32x4 jh = *(const f32x4*)&Gh[16 * W + 4 * g], jl = *(const f32x4*)&Gl[16 * W + 4 * g];
      const f32x4 rj = *(const f32x4*)&rk[16 * W + 4 * g];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = 4 * g + e <= c;
        const float d = __builtin_amdgcn_exp2f(in ? (gh - jh[e]) + (gl - jl[e]) : 0.0f) * rj[e];
        x[t][e] = in ? x[t][e] * d : 0.0f;
      }
    }
  }
  float inv;
  const float sc = pow2_scale(max_rows4(max4(x[1], max4(x[0], 0.0f))), inv);
  h8 part[2];
  split8(x[0], x[1], sc, part);
  *(h8*)L.P[F][0][lane] = part[0];
  *(h8*)L.P[F][1][lane] = part[1];
  // (the row has a scale of its own, so q's factor goes there, off the way to the operand)
  float rq = scale;  // the squares are the diagonal of q q^T; lane (c / 4, c) has it for row c
  if (l2norm) rq *= l2_factor(__shfl(diagonal(qq, c), 16 * (c >> 2) + c, 64));
  if (g == 0) {
    L.pr[J][i] = inv * rq;
    if (diag) L.c2[i] = rq * __builtin_amdgcn_exp2f(gh + gl);
  }
}

template <int NW>
constexpr int kFetchers = NW == 4 ? 0 : (NW == 2 ? 4 : 6);  // waves of their own

template <int DK, bool BF, int NW>
__global__ __attribute__((amdgpu_waves_per_eu(2))) __launch_bounds__(64 * (2 * NW + kFetchers<NW>)) void
delta_chain_kernel(DeltaArgs a, const ChunkRec* recs, const int* order, int64_t slot0, int64_t slot1) {
  constexpr int NM = DK / 16, NJ = DK / 32, NT = kParts<BF>, NF = kFetchers<NW>, NP = NF ? NF : NW;
  __shared__ __align__(16) ChainLds<DK, NW, NT> L;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % NW;
  // Workgroups go to the eight dies in turn: all that share a key head run on one, next to its L2.
  const int rep = a.Hv / a.Hk, nb = (a.Dv + 16 * NW - 1) / (16 * NW);
  const int64_t bx = blockIdx.x, die = bx & 7, in = bx >> 3;
  const int64_t unit = in / (rep * nb) * 8 + die;
  if (unit >= (int64_t)a.n_seq * a.Hk) return;
  const int vb = (int)(in % nb), hk = (int)(unit % a.Hk), h = hk * rep + (int)(in / nb % rep);
  int b = (int)(unit / a.Hk);
  if (order) b = order[b];
  const int dv0 = 16 * (NW * vb + w), dv = dv0 + c;
  const bool active = dv0 < a.Dv;
  int64_t t0, t1;
  seq_range(a, b, t0, t1);
  const int64_t first = t0 / kC + b, nch = (t1 - t0 + kC - 1) / kC;
  const PassChunks pass = pass_chunks(first, nch, slot0, slot1);  // this launch's chunks of the sequence
  const int64_t cb = pass.begin;
  const int n = (int)pass.count;
  if (n == 0 && !(nch == 0 && slot0 == 0)) return;  // (an empty sequence's state is passed on by the first launch)
  const int slot = slot_of(a, b);
  if (slot < 0) {
    const uint16_t fill = slot == kSlotPad ? 0 : 0x7fff;
    if (active && wave < NW)
      for (int64_t t = t0 + cb * kC + g; t < t1 && t < t0 + (cb + n) * kC; t += 4) a.out[t * a.ld_out + (int64_t)h * a.Dv + dv] = fill;
    return;
  }
  int64_t tok = t0 + cb * kC;
  auto len_at = [&](int64_t t) { return (int)(t1 - t < kC ? t1 - t : kC); };

  if (wave < NW) {  // ------------------------------------------------------------ the state
    f32x4 S[NM];
    float sfac = 1.0f;  // S holds the state over sfac, a power of two per value column
    const size_t so = (((size_t)slot * a.Hv + h) * a.Dv + (active ? dv : 0)) * DK + 8 * g;
    const float* sp = (cb == 0 ? a.state : a.state_out) + so;
#pragma unroll
    for (int m = 0; m < NM; ++m) S[m] = *(const f32x4*)(sp + 32 * (m >> 1) + 4 * (m & 1));
    const int ldv = (int)a.ld_v * 2, vo = 4 * g * ldv + (active ? dv : c) * 2;
    uint32_t vv[16], vn[16];  // (NW = 4) this chunk's and the next one's
    auto load_v = [&](int64_t tk) {
      const Rsrc r = rows_of(a.v + tk * a.ld_v + (int64_t)h * a.Dv, a.ld_v, len_at(tk), a.Dv);
#pragma unroll
      for (int i = 0; i < 16; ++i) vn[i] = __builtin_amdgcn_raw_buffer_load_b16(r, vo, (16 * (i / 4) + (i & 3)) * ldv, 0);
    };
    __builtin_amdgcn_s_waitcnt(0);  // the state is here: within the loop only v is waited for
    if (NW == 4 && n > 0) load_v(tok);
    for (int i = 0; i < n; ++i, tok += kC) {
      const Operands<DK>& op = L.op[i & 1];
      const f32x4* vec = (const f32x4*)op.vec;
      if constexpr (NW == 4) {
#pragma unroll
        for (int q = 0; q < 16; ++q) vv[q] = vn[q];
        load_v(i + 1 < n ? tok + kC : tok);  // (the last time for nothing)
      }
      h8 s[NT][NJ];
      float smax = 0.0f, ssc = 1.0f, sinv = 1.0f;
      if constexpr (!BF) {
        smax = col_max<NM>(S);
        ssc = pow2_scale(smax, sinv);
      }
      split_all<NM>(S, ssc, s);
      if constexpr (NW < 4)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int q = 0; q < NT; ++q) *(h8*)L.S[w][j][q][lane] = s[q][j];
      if constexpr (!BF) {
        sinv *= sfac;
        if (g == 0) L.sfac[i & 1][w][c] = sinv;
      }
      step_barrier();  // the operands of this chunk and the state are in LDS
      f32x4 v[4], ks[4];
      rows_product<DK, BF, false>(op.k, lane, s, ks);
      if constexpr (NW == 4) {
        f32x4 qs[4];
        rows_product<DK, BF, true>(op.q, lane, s, qs);
#pragma unroll
        for (int t = 0; t < 4; ++t) L.qs[w][t][lane] = qs[t];
      }
      Tri T;
      load_tri(T, op.T, lane);
      s4 vx[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (NW == 4)
#pragma unroll
          for (int e = 0; e < 4; ++e) vx[t][e] = (short)vv[4 * t + e];
        else  // four rows of the lane's column: the lane's address is row c / 4 of them, columns 4 (c % 4) ..
          vx[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)
              &L.v[i & 1][(16 * t + 4 * g + (c >> 2)) * 16 * NW + 16 * w + 4 * (c & 3)]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 c1 = vec[4 * t + g];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[t][e] = __builtin_fmaf(-(BF ? c1[e] : c1[e] * sinv), ks[t][e], w2f<BF>((uint16_t)vx[t][e]));
      }
      h8 x[2][2];
      float xinv;
      const float xsc = pow2_scale(col_max<4>(v), xinv);
      split_all<4>(v, xsc, x);
      f32x4 y[2][4];
      tri_product<false, true>(T, x, y);
      f32x4 (&u)[4] = y[0];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 tr = vec[16 + 4 * t + g], ww = vec[2 * 16 + 4 * t + g];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[t][e] = u[t][e] * (tr[e] * xinv);
        L.u[w][t][lane] = u[t];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[t][e] *= ww[e];
      }
      step_barrier();  // U is in LDS
      // S1 = e^{G_C} S + U'^T K, summed on the matrix cores onto S (fp16: in a scale that fits both)
      const float dec = __builtin_amdgcn_exp2f(op.vec[256 + kC - 1] + op.vec[320 + kC - 1]);
      float keep = dec, wsc = 1.0f;
      if constexpr (!BF) {
        float winv;
        wsc = pow2_scale(fmaxf(col_max<4>(u), dec * (smax * sfac)), winv);
        keep = dec * sfac * wsc;
        sfac = winv;
      }
      h8 uw[NT][2];
      split_all<4>(u, wsc, uw);
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[m][e] *= keep;
#pragma unroll
      for (int p = 0; p < NM; p += 4) {
        h8 ka[4][2];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // rows of k^T: the lane's address is token 32 j + 4 g + c / 4 (and 16 more), the four columns that
            // result rows 4 q .. 4 q + 3 stand for, q = c % 4
            s4 x[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int row = 32 * j + 16 * y + 4 * g + (c >> 2);
              const f16* at = &op.k[row][piece_at<DK>(row, 4 * ((p + m) >> 1) + (c & 3)) * 8 + 4 * ((p + m) & 1)];
              x[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)at);
            }
            ka[m][j] = __builtin_bit_cast(h8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
          }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int q = NT - 1; q >= 0; --q)
#pragma unroll
            for (int m = 0; m < 4; ++m) S[p + m] = mm<BF>(ka[m][j], uw[q][j], S[p + m]);
        }
      }
    }
    if (active) {
      float* o = a.state_out + so;
#pragma unroll
      for (int m = 0; m < NM; ++m) *(f32x4*)(o + 32 * (m >> 1) + 4 * (m & 1)) = BF ? S[m] : S[m] * sfac;
    }
    return;
  }

  // -------------------------------------------------------------------- the fetchers and the outputs
  const ChunkRec* rec = recs + (first + cb - slot0) * a.Hv + h;
  const bool outputs = wave < 2 * NW, fetches = !NF || !outputs;
  const int fi = NF ? wave - 2 * NW : w;  // which fetcher
  // Chunk i's rows of k, of q, and the rest: four fetchers have the rows, the others (or the same) the rest. Of the
  // four output waves that fetch where NW = 4, the two with one fragment of P have all of it, one k and one q.
  int off[4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
    off[m] = NF ? rows_off<DK>(m == 0 ? a.ld_k : a.ld_q, fi & 3, lane) : rows_off<DK>(fi ? a.ld_q : a.ld_k, m, lane);
  auto fetch_k = [&](int i) {
    const int64_t tk = t0 + (cb + i) * kC;
    const uint16_t* p = a.k + tk * a.ld_k + hk * DK;
    if (NF) {
      if (fi < 4) fetch_rows<DK>(L.op[i & 1].k, p, a.ld_k, len_at(tk), fi, off[0]);
    } else if (fi == 0) {
#pragma unroll
      for (int m = 0; m < 4; ++m) fetch_rows<DK>(L.op[i & 1].k, p, a.ld_k, len_at(tk), m, off[m]);
    }
  };
  auto fetch_q = [&](int i) {
    const int64_t tk = t0 + (cb + i) * kC;
    const uint16_t* p = a.q + tk * a.ld_q + hk * DK;
    if (NF) {
      if (fi < 4) fetch_rows<DK>(L.op[i & 1].q, p, a.ld_q, len_at(tk), fi, off[1]);
    } else if (fi == 1) {
#pragma unroll
      for (int m = 0; m < 4; ++m) fetch_rows<DK>(L.op[i & 1].q, p, a.ld_q, len_at(tk), m, off[m]);
    }
  };
  auto fetch_rest = [&](int i, int part) {  // part of 4
    const int64_t tk = t0 + (cb + i) * kC;
    fetch_record<4>(L.op[i & 1].T, rec + (int64_t)i * a.Hv, part, lane);
    if constexpr (NW < 4) {  // v in KiB of 32 / NW rows, by the last parts
      const Rsrc r = rows_of(a.v + tk * a.ld_v + (int64_t)h * a.Dv + 16 * NW * vb, a.ld_v, len_at(tk), a.Dv - 16 * NW * vb);
      const int per = 32 / NW, row = lane / (2 * NW), ldb = (int)a.ld_v * 2, m = part - (4 - 2 * NW);
      if (m >= 0)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)((char*)L.v[i & 1] + m * 1024), 16, row * ldb + lane % (2 * NW) * 16,
                                                 per * m * ldb, 0, 0);
    }
  };
  const int ldo = (int)a.ld_out * 2, oo = c * ldo + (dv0 + 4 * g) * 2;
  if (fetches && n > 0) {
    fetch_k(0);
    fetch_q(0);
    if (NF < 6) fetch_rest(0, fi);
    else if (fi < 4) fetch_rest(0, fi);
    __builtin_amdgcn_s_waitcnt(0);
  }
  for (int i = 0; i < n; ++i, tok += kC) {
    const Operands<DK>& op = L.op[i & 1];
    step_barrier();
    if (fetches) {
      const bool next = i + 1 < n;
      if (next) {
        fetch_k(i + 1);
        fetch_q(i + 1);
      }
      auto p = [&](auto w, auto j) {
        make_p<decltype(w)::value, decltype(j)::value, DK, BF>(L, op, lane, a.l2norm, a.scale);
      };
      if constexpr (NP == 6) {
        switch (fi) {
          case 0: p(Int<2>{}, Int<0>{}); break;
          case 1: p(Int<1>{}, Int<0>{}); break;
          case 2: p(Int<0>{}, Int<0>{}); break;  // (one tile: it shares its SIMD with the chain)
          case 3: p(Int<2>{}, Int<1>{}); break;
          case 4: p(Int<3>{}, Int<0>{}); break;
          default: p(Int<3>{}, Int<1>{});
        }
      } else {  // by fours: three of the ten tiles at most
        switch (fi) {
          case 0: p(Int<3>{}, Int<1>{}); break;
          case 1: p(Int<3>{}, Int<0>{}); break;
          case 2: p(Int<2>{}, Int<0>{}), p(Int<0>{}, Int<0>{}); break;
          default: p(Int<1>{}, Int<0>{}), p(Int<2>{}, Int<1>{});
        }
      }
    }
    f32x4 qs[4];
    f32x4 sinv;
    if (NW < 4 && outputs) {
      h8 s[NT][NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < NT; ++q) s[q][j] = *(const h8*)L.S[w][j][q][lane];
      rows_product<DK, BF, true>(op.q, lane, s, qs);
    }
    if (outputs) sinv = BF ? f32x4{1.0f, 1.0f, 1.0f, 1.0f} : *(const f32x4*)&L.sfac[i & 1][w][4 * g];
    if (i + 1 < n) {  // with six fetchers the output wave, which has less to do, helps
      if (!NF && fi < 2) fetch_rest(i + 1, 2 * fi), fetch_rest(i + 1, 2 * fi + 1);
      if (NF == 6 && outputs) fetch_rest(i + 1, 0), fetch_rest(i + 1, 1);
    }
    step_barrier();
    if (i + 1 < n && fetches) {
      if (NF == 4) fetch_rest(i + 1, fi);
      if (NF == 6 && fi >= 4) fetch_rest(i + 1, fi - 2);
    }
    f32x4 o[2][4];
    f32x4 uinv;
    if (outputs) {
      Tri P;
      load_tri(P, L.P, lane);
      f32x4 u[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) u[t] = L.u[w][t][lane];
      h8 x[2][2];
      float inv;
      const float usc = pow2_scale(col_max<4>(u), inv);
      if (g == 0) L.ufac[w][c] = inv;
      split_all<4>(u, usc, x);
      tri_product<true, false>(P, x, o);
      wave_sync();
      uinv = *(const f32x4*)&L.ufac[w][4 * g];
      if constexpr (NW == 4)
#pragma unroll
        for (int t = 0; t < 4; ++t) qs[t] = L.qs[w][t][lane];
    }
    // what this wave loads for the next chunk is in before it stores, so that the wait is not for the stores
    if (fetches || NF == 6) __builtin_amdgcn_s_waitcnt(0);
    if (outputs && active) {
      const Rsrc orow = rows_of(a.out + tok * a.ld_out + (int64_t)h * a.Dv, a.ld_out, len_at(tok), a.Dv);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float c2 = L.c2[16 * t + c], p0 = L.pr[0][16 * t + c], p1 = t >= 2 ? L.pr[1][16 * t + c] : 0.0f;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pu = t >= 2 ? __builtin_fmaf(o[1][t][e], p1, o[0][t][e] * p0) : o[0][t][e] * p0;
          x[e] = __builtin_fmaf(qs[t][e], BF ? c2 : c2 * sinv[e], pu * uinv[e]);
        }
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3])}, orow, oo, 16 * t * ldo, 0);
      }
    }
  }
}

int64_t chunk_slots(const DeltaArgs& a) { return a.n_tokens / kC + a.n_seq; }

// Chunks whose records are held at once: all, or as many as fit 1 GiB.
int64_t slots_per_pass(const DeltaArgs& a) {
  const int64_t all = chunk_slots(a), fit = ((int64_t)1 << 30) / ((int64_t)a.Hv * sizeof(ChunkRec));
  return fit < 1 ? 1 : (fit < all ? fit : all);
}

template <int DK, bool BF, int NW>
void launch_chain(const DeltaArgs& a, const ChunkRec* r, const int* order, int64_t s0, int64_t s1, hipStream_t s) {
  const int64_t units = (int64_t)a.n_seq * a.Hk, per = (int64_t)(a.Hv / a.Hk) * ((a.Dv + 16 * NW - 1) / (16 * NW));
  const dim3 grid((unsigned)((units + 7) / 8 * 8 * per)), block(64 * (2 * NW + kFetchers<NW>));
  hipLaunchKernelGGL((delta_chain_kernel<DK, BF, NW>), grid, block, 0, s, a, r, order, s0, s1);
}

template <int DK, bool BF>
hipError_t launch_chunked(const DeltaArgs& a, void* ws, hipStream_t s) {
  const int rep = a.Hv / a.Hk;
  const int64_t ng = (a.Hv + 3) / 4, slots = chunk_slots(a), per = slots_per_pass(a);
  const int64_t heads = (int64_t)a.n_seq * a.Hv, tiles = a.Dv / 16;
  if ((heads + 8 * rep) * tiles > 0x7fffffff || per * ng > 0x7fffffff) return hipErrorInvalidValue;
  ChunkRec* r = (ChunkRec*)ws;
  // Workgroups begin in order, and one that begins late with the longest chain ends late: twelve sequences of 0 to 3001
  // tokens, 64 heads, 235 us in the order they come and 211 by length (bf16); 32 of 50 to 2200 tokens 837 and 815; 64
  // of one length 1006 and 1005. (More than kOrdered even out by themselves.)
  int* order = a.cu && a.n_seq > 1 && a.n_seq <= kOrdered ? (int*)(r + slots_per_pass(a) * a.Hv) : nullptr;
  for (int64_t s0 = 0; s0 < slots; s0 += per) {
    const int64_t n = s0 + per < slots ? per : slots - s0;
    // Two workgroups to a CU: 16411 tokens x 64 heads 592 us (with 256 workgroups 605, with 1024 591), twelve ragged
    // sequences 211 (218, 214).
    const int64_t tasks = n * ng, resident = 512;
    const dim3 grid((unsigned)(tasks < resident ? tasks : resident));
    hipLaunchKernelGGL((delta_prep_kernel<DK, BF>), grid, dim3(256), 0, s, a, r, order, s0, tasks);
    switch (chain_tiles(heads, tiles)) {
      case 1: launch_chain<DK, BF, 1>(a, r, order, s0, s0 + n, s); break;
      case 2: launch_chain<DK, BF, 2>(a, r, order, s0, s0 + n, s); break;
      default: launch_chain<DK, BF, 4>(a, r, order, s0, s0 + n, s);
    }
  }
  return hipGetLastError();
}

}  // namespace

size_t delta_chunk_workspace(const DeltaArgs& a) {
  return (size_t)(slots_per_pass(a) * a.Hv) * sizeof(ChunkRec) + kOrdered * sizeof(int);
}

hipError_t launch_delta_chunked(const DeltaArgs& a, void* ws, hipStream_t s) {
  if (a.Dk == 128) return a.bf16 ? launch_chunked<128, true>(a, ws, s) : launch_chunked<128, false>(a, ws, s);
  return a.bf16 ? launch_chunked<64, true>(a, ws, s) : launch_chunked<64, false>(a, ws, s);
}

}  // namespace dfssm
