// The selective state space scan over chunks of 64 tokens (gfx950 matrix cores).
//
// Per head and chunk, with a_t = -d_t e^{A_log}, G_i = a_1 + .. + a_i, h0 (P x N) the state before it and w_j = e^{G_64 - G_j} d_j:
//   M_ij = C_i.B_j e^{G_i - G_j} d_j (i >= j) + D (i = j);  y_i = e^{G_i} h0 C_i + sum_j M_ij x_j
//   h1 = e^{G_64} h0 + sum_j (w_j x_j) B_j^T
// A workgroup walks the chunks of a sequence, or of a segment of one, with four waves that share B and C in LDS; each has
// 32 columns p of a head, their state in registers and their x to itself. Products are taken so that results lie in
// registers as the next product wants its operand: the state as rows n of 32 x 32 results (a lane has a column p), the
// scores transposed (a lane has a row i of M), y transposed (a lane has a token, and 32 bytes of its row to store). What a step of
// a product needs is loaded from LDS and split beside the step before; B, C, x and dt of the next chunk are on their way.
// Sequences longer than a segment take three launches: states of the segments from zero, their chain, everything.
//
// What bounds it. Per chunk and 32 columns (N = 128, bf16) 138 matrix instructions of 32 clocks and about 1400 others: the
// scores and M are made by each wave anew, the state is split into parts for C h0, U for the new state. 64 x 512 tokens x 80 heads
// take 0.45 ms (1.03 GB, 0.21 ms of copying); two waves to a SIMD overlap the matrix cores and the other pipe little. One sequence
// of 16411 tokens x 64 heads: 0.07 ms for the segments' states, 0.02 for their chain, 0.16 for the rest (fp16; 0.06 ms of copying).
// One chunk: 12 us, most of it the code's way into the instruction cache and the loads before the first product. Measured with two
// bf16 parts of h0 and M (0.40 ms) and not kept: M shared between the two waves of a head (10% fewer matrix instructions, 20% fewer
// others, a barrier more and 24 KiB), three waves to a SIMD (168 registers, B not held twice); both came out the same.
//
// Numbers. States, sums and everything between products are fp32; G is summed in fp64, and its differences taken of float pairs,
// so that they survive a decay of any size in the same chunk (a_t is held to -1e5). x, B and C are exact operands of the 16-bit
// matrix cores in their own type. An fp32 factor beside them (h0, M, w_j x_j) is a sum of 16-bit parts. Beside bf16 three of them,
// which hold its 24 bits (two of h0 and M, 16 bits, took 0.40 ms instead of 0.45, but an output that is small beside its terms
// was off by more than its rounding). Beside fp16 pairs of halves, x 2^s = hi + lo, 22 bits, with s per column of h0 and w x
// and per row of M so that the largest magnitude lies in [2^14, 2^15); a value below 2^-16 of the largest M of its scale is off
// by up to 2^-39 M, whatever it is multiplied by. The state's own values are kept and added to in fp32. D is on M's diagonal.
#include "common.h"
#include "layer.h"
#include "parts.h"
#include "scan_math.h"
#include "scan_plan.h"

namespace dfssm {

namespace {

constexpr int kC = kScanChunk, kW = kScanWaves;
// Fewer groups of B and C than this, over all places, are spread over all dies. One prompt of 45 tokens, 64 heads in one group, 15.0
// us on one die and 12.4 on eight; with 25 and 37 places (16411 tokens, and the ragged batch) 242 and 175 us by dies, 247 and 164
// spread.
constexpr int kSpread = 16;
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool BF>
__device__ __forceinline__ f32x16 mm32(h8 a, h8 b, f32x16 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Eight values as NT parts: pairs of halves of x sc, or NT parts of bf16 (sc is 1). What a bf16 part leaves of two values
// comes from a dot product each, x + (-1, 0) (p0, p1) and x + (0, -1) (p0, p1), which is exact. (The factors are in registers: the
// compiler writes the first as the constant -1.0, which the instruction takes as the second.)
template <bool BF, int NT, bool DIES = true>
__device__ __forceinline__ void parts8(const float (&x)[8], float sc, h8 (&part)[NT]) {
  uint32_t p[NT][4], k0 = 0x0000bf80u, k1 = 0xbf800000u;
  asm("" : "+s"(k0), "+s"(k1));
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (!BF) {
      uint32_t t[2];
      split2(x[2 * q], x[2 * q + 1], sc, t);
      p[0][q] = t[0];
      p[1][q] = t[1];
    } else {
      float x0 = x[2 * q], x1 = x[2 * q + 1];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const b2 t = __builtin_convertvector(f32x2{x0, x1}, b2);
        p[i][q] = __builtin_bit_cast(uint32_t, t);
        if (i + 1 < NT && !DIES) {
          x0 -= __builtin_bit_cast(float, p[i][q] << 16);
          x1 -= __builtin_bit_cast(float, p[i][q] & 0xffff0000u);
        } else if (i + 1 < NT) {
          x0 = __builtin_amdgcn_fdot2_f32_bf16(t, __builtin_bit_cast(b2, k0), x0, false);
          x1 = __builtin_amdgcn_fdot2_f32_bf16(t, __builtin_bit_cast(b2, k1), x1, false);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) part[i] = __builtin_bit_cast(h8, u32x4{p[i][0], p[i][1], p[i][2], p[i][3]});
}

// The larger of v >= 0 in the two lanes of a column (32 apart).
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __builtin_bit_cast(float, max((uint32_t)q[0], (uint32_t)q[1]));
}
template <int N>
__device__ __forceinline__ float max_abs(const float (&x)[N], float m) {
#pragma unroll
  for (int e = 0; e < N; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(x[e]));
  return m;
}

// Rows of B and C in LDS: their 16-byte pieces are exchanged so that one piece of 8 rows, and two neighbouring ones of
// four rows, lie in different banks.
template <int N>
__device__ __forceinline__ int swap_of(int row) {
  return N == 128 ? ((row & 7) << 1) | ((row >> 3) & 1) : (row & 2) | (row & 4) | ((row >> 3) & 1);
}

typedef __attribute__((address_space(3))) s4* tptr;

// Row 8 m + 4 h + e of a 32 x 32 result is column 16 h + 4 m + e, so that a lane has 16 neighbouring columns of a token. The
// column of a lane that has a column of the state:
__device__ __forceinline__ int scan_col(int lane) { return 16 * ((lane >> 2) & 1) + 4 * ((lane & 31) >> 3) + (lane & 3); }

// The lane, as a value that the compiler derives offsets from anew where it is asked for: held over the whole loop they are more
// registers than there are.
__device__ __forceinline__ int lane_again() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

template <int N, bool STATE>
struct ScanLds {
  f16 B[2][kC][N];
  f16 C[STATE ? 1 : kC][STATE ? 8 : N];
  f16 x[kW][kC][kScanCols];
  struct {
    float Gh[kC], Gl[kC], d[kC], w[kC];  // by tokens: G over log 2, the float nearest and the rest; d; w
    float F[32], F16[32];                // d e^{G_32 - G_j}, j < 32; d e^{G_16 - G_j}, j < 16, and of tokens 32 .. 47
    float s[kScanCols];                  // by columns: what undoes the scaling of the state
  } v[kW];
};

// `len` rows, ld bytes apart, of `bytes` bytes: loads behind the last one give zero, stores are dropped.
__device__ __forceinline__ Rsrc bytes_of(const void* p, int ld, int len, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (len - 1) * ld + bytes, 0x00027000);
}

// A wave's quarter of 64 rows of B or C, into LDS.
template <int N>
__device__ __forceinline__ void fetch_shared(f16 (*to)[N], const char* p, int ld, int len, int wave, int off) {
  constexpr int per = 512 / N;  // rows of a KiB
  const Rsrc r = bytes_of(p, ld, len, 2 * N);
#pragma unroll
  for (int n = 0; n < kC / per / kW; ++n)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)((char*)to + (kW * n + wave) * 1024), 16, off + n * kW * per * ld, 0, 0, 0);
}

// Places of the launch's numbering of segments (of `seg` tokens; one for an empty sequence). Up to kCounted sequences the
// segments are counted, so that places are taken without gaps and the dies have equally many: with the numbering of tile_of 64
// sequences of 512 tokens gave one die nine and another seven. Beyond, they even out by themselves.
constexpr int kCounted = 512;
// The segments of 64 sequences from `from` on, a lane's and those before it; all of them returned.
__device__ __forceinline__ int count_segments(const PackedScanArgs& a, int from, int seg, int& own, int& before) {
  const int lane = threadIdx.x & 63, i = from + lane;
  own = 0;
  if (i < a.n_seq) {
    int64_t t0, t1;
    seq_range(a, i, t0, t1);
    own = scan_segments(t1 - t0, seg);
  }
  int sum = own;
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xf, 0xf, true);  // from 1, 2, 4 and 8 lanes before, in the row of 16
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xf, 0xf, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xf, 0xf, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xf, 0xf, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x142, 0xa, 0xf, true);  // row 0's last to row 1, 2's to 3; lane 31's to rows 2 and 3
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x143, 0xc, 0xf, true);
  before = sum - own;
  return __builtin_amdgcn_readlane(sum, 63);
}
// The sequence of a place; false where there is none.
__device__ __forceinline__ bool sequence_at(const PackedScanArgs& a, int place, int seg, Where& q) {
  if (!a.cu) {
    const int per = scan_segments(a.len, seg);
    q.seq = (int)((uint32_t)place / (uint32_t)per);
    q.first = (int64_t)q.seq * per;
    if (q.seq >= a.n_seq) return false;
    seq_range(a, q.seq, q.t0, q.t1);
    return true;
  }
  if (a.n_seq > kCounted) {
    find_seq<0>(a, place, q, seg);
    return scan_holds(place, q.first, q.t1 - q.t0, seg);
  }
  int base = 0;
  for (int from = 0; from < a.n_seq; from += 64) {
    int own, before;
    const int all = count_segments(a, from, seg, own, before);
    if (place < base + all) {
      const int at = __ffsll((unsigned long long)__ballot(place < base + before + own)) - 1;
      q.seq = from + at;
      q.first = base + __builtin_amdgcn_readlane(before, at);
      seq_range(a, q.seq, q.t0, q.t1);
      return true;
    }
    base += all;
  }
  return false;
}
// The first place of a sequence.
__device__ __forceinline__ int64_t first_place(const PackedScanArgs& a, int b, int seg, int64_t t0) {
  if (!a.cu) return (int64_t)b * scan_segments(a.len, seg);
  if (a.n_seq > kCounted) return (int64_t)((uint32_t)t0 / (uint32_t)seg) + b;
  int base = 0;
  for (int from = 0;; from += 64) {
    int own, before;
    const int all = count_segments(a, from, seg, own, before);
    if (b < from + 64) return base + __builtin_amdgcn_readlane(before, b - from);
    base += all;
  }
}

// STATE: the states that a segment leaves from zero, and its decay, of all segments but the last of a sequence.
template <int N, bool BF, bool STATE>
__global__ __attribute__((amdgpu_waves_per_eu(2))) __launch_bounds__(64 * kW) void
scan_chunk_kernel(PackedScanArgs a, int seg, int places, float* seg_state, float* seg_decay) {
  constexpr int NB = N / 16, NN = N / 32, NU = kParts<BF>, pieces = N / 8;
  __shared__ __align__(16) ScanLds<N, STATE> L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the eight dies in turn: all that share a group's B and C run on one, next to its L2, unless there are so few
  // that dies would be idle.
  const int rep = a.H / a.G, ncb = (a.P + kScanCols - 1) / kScanCols, nwg = (rep * ncb + kW - 1) / kW;
  const bool spread = (int64_t)places * a.G < kSpread;
  const uint32_t in = spread ? blockIdx.x : blockIdx.x >> 3, turn = in / (uint32_t)nwg;
  const uint32_t unit = spread ? turn : turn * 8 + (blockIdx.x & 7), place = unit / (uint32_t)a.G;
  if (place >= (uint32_t)places) return;
  const int gr = (int)(unit % (uint32_t)a.G), blk = (int)(in % (uint32_t)nwg) * kW + wave;
  Where q;
  if (!sequence_at(a, (int)place, seg, q)) return;
  const int64_t tok = q.t0 + (place - q.first) * seg;
  const bool last = q.t1 - tok <= seg;
  const int len = (int)(last ? q.t1 - tok : seg);  // (of an empty sequence 0: its state is passed on)
  if (STATE && last) return;
  const bool active = blk < rep * ncb;
  const int h = gr * rep + (active ? blk / ncb : 0), p0 = active ? blk % ncb * kScanCols : 0;
  const bool wide = p0 + 16 < a.P;
  const int slot = slot_of(a, q.seq);
  if (slot < 0) {
    const uint16_t fill = slot == kSlotPad ? 0 : 0x7fff;
    const int c = threadIdx.x & 31;
    if (!STATE && active && (c < 16 || wide))
      for (int64_t t = threadIdx.x >> 5 & 1; t < len; t += 2) a.out[(tok + t) * a.ld_out + (int64_t)h * a.P + p0 + c] = fill;
    return;
  }
  const bool whole = place == q.first && last;  // the sequence is one segment

  // S[t][8 b + e] is the state of row n = 32 t + 16 b + 8 hi + e and column p0 + scan_col, over sfac.
  f32x16 S[NN];
  float sfac = 1.0f, decay = 1.0f;
  const int64_t size = (int64_t)a.H * a.P * N, so = ((int64_t)h * a.P + p0) * N;
  auto state_at = [&](int lane) {  // (columns that are not there do their neighbours' work)
    const int col = scan_col(lane);
    return (uint32_t)((col < 16 || wide ? col : col - 16) * N + 8 * (lane >> 5));
  };
  if constexpr (STATE) {
#pragma unroll
    for (int t = 0; t < NN; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] = 0.0f;
  } else {
    const float* sp = (whole || len == 0 ? a.state + slot * size : seg_state + place * size) + so;
    const uint32_t at = state_at(threadIdx.x & 63);
#pragma unroll
    for (int t = 0; t < NN; ++t)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const f32x4 v = *(const f32x4*)(sp + at + 32 * t + 16 * (m >> 1) + 4 * (m & 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) S[t][4 * m + e] = v[e];
      }
  }
  HeadParams hp = head_params(a, h);
  hp.A = uniform(hp.A), hp.D = uniform(hp.D), hp.bias = uniform(hp.bias);
  auto& V = L.v[wave];
  f16 (&X)[kC][kScanCols] = L.x[wave];
  const int xw = 2 * (a.P - p0 < kScanCols ? a.P - p0 : kScanCols);  // bytes of a row
  // (in bytes from here on; 64 rows are 2^30 at most)
  const int ld_b = (int)a.ld_B * 2, ld_c = (int)a.ld_C * 2, ld_x = (int)a.ld_x * 2, ld_o = (int)a.ld_out * 2;
  const int dt_size = a.dt32 ? 4 : 2, ld_t = (int)a.ld_dt * dt_size;
  const char *pb = (const char*)(a.B + tok * a.ld_B + gr * N), *pc = (const char*)(a.C + tok * a.ld_C + gr * N);
  const char *px = (const char*)(a.x + tok * a.ld_x + (int64_t)h * a.P + p0), *pt = (const char*)a.dt + tok * ld_t + h * dt_size;
  char* po = (char*)(a.out + tok * a.ld_out + (int64_t)h * a.P + p0);
  // x as an operand: column p0 + scan_col, tokens 16 k + 4 hi + 0 .. 3 and 8 more
  auto x_frag = [&](int lane, int k) {
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), at = 16 * (lane & 1) + 8 * ((lane >> 4) & 1) + 4 * ((lane >> 1) & 1);
    s4 t[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) t[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tptr)&X[16 * k + 8 * y + row][at]);
    return __builtin_bit_cast(h8, __builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  int raw = 0;
  auto fetch_dt = [&](int left) {  // (zero behind the last token)
    const Rsrc r = bytes_of(pt, ld_t, left < kC ? left : kC, dt_size);
    const int at = lane_again() * ld_t;
    raw = a.dt32 ? (int)__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0) : (int)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
    pt += (int64_t)kC * ld_t;
  };
  const int xo = 16 * ld_x;
  auto fetch_b = [&](int i, int n) {
    const int lane = lane_again(), row = 512 / N * wave + lane / pieces, piece = ((lane % pieces) ^ swap_of<N>(row)) * 16;
    fetch_shared<N>(L.B[i], pb, ld_b, n, wave, row * ld_b + piece);
    pb += kC * ld_b;
  };
  auto fetch_c = [&](int n) {
    if constexpr (!STATE) {
      const int lane = lane_again(), row = 512 / N * wave + lane / pieces, piece = ((lane % pieces) ^ swap_of<N>(row)) * 16;
      fetch_shared<N>(L.C, pc, ld_c, n, wave, row * ld_c + piece);
      pc += kC * ld_c;
    }
  };
  auto fetch_x = [&](int n) {
    const Rsrc r = bytes_of(px, ld_x, n, xw);
    const int lane = lane_again(), off = (lane >> 2) * ld_x + (lane & 3) * 16;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)((char*)X + m * 1024), 16, off + m * xo, 0, 0, 0);
    px += kC * ld_x;
  };
  // The time steps; a lane has a token. Returns e^{G_64}.
  auto times = [&](int n) {
    const int lane = lane_again();
    const float dt = a.dt32 ? __builtin_bit_cast(float, raw) : w2f<BF>((uint16_t)raw);
    const float d = lane < n ? time_step(dt, hp, a.softplus) : 0.0f;
    float al = d * hp.A;
    al = al < -1e5f ? -1e5f : al;
    double G = (double)al * 1.4426950408889634;
    G += moved<0x111, 0xf>(G);  // running sums: from 1, 2, 4 and 8 lanes before, in the row of 16
    G += moved<0x112, 0xf>(G);
    G += moved<0x114, 0xf>(G);
    G += moved<0x118, 0xf>(G);
    G += moved<0x142, 0xa>(G);  // row 0's last to row 1, 2's to 3; then lane 31's to rows 2 and 3
    G += moved<0x143, 0xc>(G);
    const double GC = readlane_f64(G, 63);
    V.w[lane] = __builtin_amdgcn_exp2f((float)(GC - G)) * d;
    if constexpr (!STATE) {
      V.Gh[lane] = (float)G;
      V.Gl[lane] = (float)(G - (double)(float)G);
      V.d[lane] = d;
      const float f = __builtin_amdgcn_exp2f((float)(readlane_f64(G, 32) - G)) * d;
      const double G16 = readlane_f64(G, 16), G48 = readlane_f64(G, 48);
      const float near = __builtin_amdgcn_exp2f((float)((lane < 32 ? G16 : G48) - G)) * d;
      if (lane < 32) V.F[lane] = f;
      if (!(lane & 16)) V.F16[(lane & 15) + (lane >> 5) * 16] = near;
    }
    return __builtin_amdgcn_exp2f((float)GC);
  };
  if (len) {
    const int n = len < kC ? len : kC;
    fetch_b(0, n);
    fetch_c(n);
    fetch_x(n);
    fetch_dt(len);
  }
  __builtin_amdgcn_s_waitcnt(0);

  // B, x and the time steps of the next chunk are loaded from the start of this one on, C once all waves have their scores; they
  // are in before a wave stores y, so that no wait is for the stores.
  int cur = 0;
  for (int left = len; left > 0; left -= kC, cur ^= 1) {
    const int n = left < kC ? left : kC, next = left - kC < kC ? left - kC : kC;
    step_barrier();  // this chunk's B, C and x are in LDS, and the next one's place for B is free
    const f16 (*LB)[N] = L.B[cur];
    h8 xf[4];
    {
      const int lane = lane_again();
#pragma unroll
      for (int k = 0; k < 4; ++k) xf[k] = x_frag(lane, k);
    }
    const float dec = times(n);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): x is in registers, its place free
    asm volatile("" ::: "memory");
    if (next > 0) {
      fetch_b(cur ^ 1, next);
      fetch_x(next);
      fetch_dt(next);
    }
    float smax = 0.0f, ssc = 1.0f;
    if constexpr (!BF) {
#pragma unroll
      for (int t = 0; t < NN; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) smax = __builtin_elementwise_maximum(smax, __builtin_fabsf(S[t][r]));
      smax = max_halves(smax);
      float sinv;
      ssc = pow2_scale(smax, sinv);
      if (!(threadIdx.x & 32)) V.s[scan_col(lane_again())] = sinv * sfac;
    }
    if constexpr (!STATE) {
      f32x16 y[2], sc[3];  // y by tokens; scores: columns 0 .. 31 of rows 0 .. 31; of rows 32 .. 63; columns 32 .. of those
#pragma unroll
      for (int r = 0; r < 16; ++r) y[0][r] = y[1][r] = sc[0][r] = sc[1][r] = sc[2][r] = 0.0f;
      const int lane = lane_again(), hi = lane >> 5, c = lane & 31;
      auto row_frag = [&](const f16 (*rows)[N], int t, int b) {
        return *(const h8*)&rows[32 * t + c][((2 * b + hi) ^ swap_of<N>(c)) * 8];
      };
      // What the products of a step need is loaded and split beside those of the step before.
      {
        h8 cf[2][2], sp[2][NU];
        auto load = [&](int b) { cf[b & 1][0] = row_frag(L.C, 0, b), cf[b & 1][1] = row_frag(L.C, 1, b); };
        auto split = [&](int b) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = S[b >> 1][8 * (b & 1) + e];
          parts8<BF, NU, false>(v, ssc, sp[b & 1]);
        };
        load(0);
        split(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          __builtin_amdgcn_sched_barrier(0);
          if (b + 1 < NB) load(b + 1);
#pragma unroll
          for (int p = NU - 1; p >= 0; --p)
#pragma unroll
            for (int t = 0; t < 2; ++t) y[t] = mm32<BF>(sp[b & 1][p], cf[b & 1][t], y[t]);
          if (b + 1 < NB) split(b + 1);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      {
        h8 cf[2][2], bf[2][2];
        auto load = [&](int b) {
#pragma unroll
          for (int t = 0; t < 2; ++t) cf[b & 1][t] = row_frag(L.C, t, b), bf[b & 1][t] = row_frag(LB, t, b);
        };
        load(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          __builtin_amdgcn_sched_barrier(0);
          if (b + 1 < NB) load(b + 1);
          sc[0] = mm32<BF>(bf[b & 1][0], cf[b & 1][0], sc[0]);
          sc[1] = mm32<BF>(bf[b & 1][0], cf[b & 1][1], sc[1]);
          sc[2] = mm32<BF>(bf[b & 1][1], cf[b & 1][1], sc[2]);
        }
      }
      step_barrier();  // C is free
      if (next > 0) fetch_c(next);
      // M: a lane has row 32 t + c, columns 8 q + 4 hi + e of each block of 32. Of a block on the diagonal it has 8 exponentials, of
      // its own 16 columns; the other 16 are before its row, and e^{G_i - G_j} is taken apart at column 16, or behind it.
      const bool own = c & 16;
      const int lim = (c & 15) - 4 * hi;
      float pinv[2] = {1.0f, 1.0f};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16& D = sc[2 * t];
        const float Gi = V.Gh[32 * t + c], gi = V.Gl[32 * t + c];
        if (t) {
          const float ei = __builtin_amdgcn_exp2f((Gi - V.Gh[32]) + (gi - V.Gl[32]));
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 F = *(const f32x4*)&V.F[8 * q4 + 4 * hi];
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[1][4 * q4 + e] = (sc[1][4 * q4 + e] * ei) * F[e];
          }
        }
        const float ei = __builtin_amdgcn_exp2f((Gi - V.Gh[32 * t + 16]) + (gi - V.Gl[32 * t + 16]));
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int j0 = 8 * z + 4 * hi;
          const f32x4 jh = *(const f32x4*)&V.Gh[32 * t + (c & 16) + j0], jl = *(const f32x4*)&V.Gl[32 * t + (c & 16) + j0];
          const f32x4 dj = *(const f32x4*)&V.d[32 * t + (c & 16) + j0], F = *(const f32x4*)&V.F16[16 * t + j0];
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // (right of the diagonal the exponential may be infinite: not used)
            const int k = 4 * z + e;
            const float ex = __builtin_amdgcn_exp2f((Gi - jh[e]) + (gi - jl[e])) * dj[e];
            const float near = D[k], far = D[8 + k];
            float v = __builtin_fmaf(own ? far : near, ex, 8 * z + e == lim ? hp.D : 0.0f);
            v = 8 * z + e <= lim ? v : 0.0f;
            D[k] = own ? near * (ei * F[e]) : v;
            D[8 + k] = own ? v : 0.0f;
          }
        }
        // y of the state comes into M's scale (at most 2^40: what is lost of smaller M is below 2^-60), by a finite factor: where it
        // would not be, y is infinite, unless C leaves the state out
        float ys = __builtin_amdgcn_exp2f(Gi + gi), msc = 1.0f;
        if constexpr (!BF) {
          float top = 0x1p-26f;
#pragma unroll
          for (int u = 2 * t; u >= t; --u)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = __builtin_elementwise_maximum(top, __builtin_fabsf(sc[u][r]));
          msc = pow2_scale(max_halves(top), pinv[t]);
          ys *= msc;
        }
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const f32x4 sv = BF ? f32x4{1.0f, 1.0f, 1.0f, 1.0f} : *(const f32x4*)&V.s[16 * hi + r];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[t][r + e] *= BF ? ys : __builtin_fminf(ys * sv[e], 0x1.fffffep127f);
        }
#pragma unroll
        for (int k = 0; k < 2 * (t + 1); ++k) {
          float v[8];
          h8 m[NU];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = sc[(k >> 1) + t][8 * (k & 1) + e];
          parts8<BF, NU>(v, msc, m);
#pragma unroll
          for (int p = NU - 1; p >= 0; --p) y[t] = mm32<BF>(xf[k], m[p], y[t]);
        }
      }
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      if (active && (hi == 0 || wide)) {
        const Rsrc orow = bytes_of(po, ld_o, n, xw);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; r += 8) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[e] = BF ? pack2<BF>(y[t][r + 2 * e], y[t][r + 2 * e + 1])
                        : pack2<BF>(y[t][r + 2 * e] * pinv[t], y[t][r + 2 * e + 1] * pinv[t]);
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{o[0], o[1], o[2], o[3]}, orow, (32 * t + c) * ld_o + 32 * hi + 2 * r, 0, 0);
          }
      }
      po += kC * ld_o;
    } else {
      decay *= dec;
    }
    __builtin_amdgcn_sched_barrier(0);
    // the new state
    const int lane = lane_again(), hi = lane >> 5, l = lane & 15;
    float keep = dec, usc = 1.0f;
    auto weighted = [&](int k, float (&u)[8]) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const f32x4 w = *(const f32x4*)&V.w[16 * k + 8 * y + 4 * hi];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f16 v = xf[k][4 * y + e];  // (a bit cast of the element itself takes the vector's first one)
          u[4 * y + e] = w2f<BF>(__builtin_bit_cast(uint16_t, v)) * w[e];
        }
      }
    };
    float u[4][8];
    if constexpr (!BF) {
      float top = 0.0f, uinv;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        weighted(k, u[k]);
        top = max_abs(u[k], top);
      }
      // The state is only added to, in fp32: it may be 2^60 times what it gets, which is split by its own size. (The last term keeps
      // sfac usc finite.)
      top = __builtin_elementwise_maximum(max_halves(top), dec * (smax * sfac) * 0x1p-60f);
      usc = pow2_scale(__builtin_elementwise_maximum(top, sfac * 0x1p-100f), uinv);
      keep = dec * sfac * usc;
      sfac = uinv;
    }
#pragma unroll
    for (int t = 0; t < NN; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] *= keep;
    {
      h8 up[2][NU], bt[2][NN];
      auto load = [&](int k) {
#pragma unroll
        for (int t = 0; t < NN; ++t) {
          // rows of B^T: result row 4 m + e of 16 is n = 4 m' + e, m' being m with its two bits exchanged
          s4 b[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int row = 16 * k + 8 * y + 4 * hi + (l >> 2), m = (l & 3) >> 1 | (l & 1) << 1;
            const int piece = (4 * t + 2 * ((lane >> 4) & 1) + (m >> 1)) ^ swap_of<N>(row & 15);
            b[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tptr)&LB[row][piece * 8 + 4 * (m & 1)]);
          }
          bt[k & 1][t] = __builtin_bit_cast(h8, __builtin_shufflevector(b[0], b[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
      };
      auto split = [&](int k) {
        if constexpr (BF) weighted(k, u[k]);
        parts8<BF, NU>(u[k], usc, up[k & 1]);
      };
      load(0);
      split(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k < 3) load(k + 1);
#pragma unroll
        for (int p = NU - 1; p >= 0; --p)
#pragma unroll
          for (int t = 0; t < NN; ++t) S[t] = mm32<BF>(bt[k & 1][t], up[k & 1][p], S[t]);
        if (k < 3) split(k + 1);
      }
    }
    if constexpr (STATE) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  }

  const int lane = lane_again();
  if (!active || !(scan_col(lane) < 16 || wide) || !(STATE || last)) return;
  float* o = (STATE ? seg_state + place * size : a.state_out + slot * size) + so + state_at(lane);
#pragma unroll
  for (int t = 0; t < NN; ++t)
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = BF ? S[t][4 * m + e] : S[t][4 * m + e] * sfac;
      *(f32x4*)(o + 32 * t + 16 * (m >> 1) + 4 * (m & 1)) = v;
    }
  if (STATE && p0 == 0 && lane == 0) seg_decay[place * a.H + h] = decay;
}

// The states before each segment of a sequence of several, in place of those that its segments leave from zero. A thread
// has four values of a head at a time, and those of eight segments on their way together (one by one, 16 segments of 64 heads
// took 13 us); `per` workgroups to a sequence.
__global__ __launch_bounds__(256) void scan_states_kernel(PackedScanArgs a, int seg, int places, int64_t per, float* seg_state,
                                                          const float* seg_decay) {
  constexpr int kAhead = 8;
  const int64_t size = (int64_t)a.H * a.P * a.N;
  const int b = (int)(blockIdx.x / per);
  int64_t t0, t1;
  seq_range(a, b, t0, t1);
  const int n = scan_segments(t1 - t0, seg);
  if (n < 2) return;
  const int64_t first = first_place(a, b, seg, t0);
  if (first + n > places) return;  // (only where offsets fall)
  const int slot = slot_of(a, b);
  if (slot < 0) return;
  for (int64_t at = (blockIdx.x % per * 256 + threadIdx.x) * 4; at < size; at += per * 1024) {
    const float* dec = seg_decay + first * a.H + at / ((int64_t)a.P * a.N);
    float* p = seg_state + first * size + at;
    f32x4 S = *(const f32x4*)(a.state + slot * size + at);
    for (int k = 0; k < n; k += kAhead, p += kAhead * size, dec += (int64_t)kAhead * a.H) {
      f32x4 own[kAhead];
      float d[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (k + i + 1 < n) {  // (the last segment leaves its state itself)
          own[i] = *(const f32x4*)(p + i * size);
          d[i] = dec[(int64_t)i * a.H];
        }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (k + i < n) {
          *(f32x4*)(p + i * size) = S;
          if (k + i + 1 < n)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[e] = __builtin_fmaf(d[i], S[e], own[i][e]);
        }
    }
  }
}

int64_t segment(const PackedScanArgs& a) {
  const int64_t longest = a.cu ? a.n_tokens : a.len, seg = scan_segment(a.n_tokens, a.n_seq, scan_wgs(a.H, a.G, a.P));
  return seg >= longest ? (longest + kC) / kC * kC : seg;
}
bool split(const PackedScanArgs& a) { return segment(a) < (a.cu ? a.n_tokens : a.len); }

template <int N, bool BF>
hipError_t launch(const PackedScanArgs& a, void* ws, hipStream_t s) {
  const int64_t seg = segment(a), places = scan_places(a.n_tokens, a.n_seq, seg), wgs = scan_wgs(a.H, a.G, a.P) / a.G;
  const int64_t units = places * a.G, grid = (units + 7) / 8 * 8 * wgs, size = (int64_t)a.H * a.P * N;
  if (grid > 0x7fffffff || seg > 0x7fffffff) return hipErrorInvalidValue;
  float *st = (float*)ws, *de = st + (ws ? places * size : 0);
  if (split(a)) {
    hipLaunchKernelGGL((scan_chunk_kernel<N, BF, true>), dim3((unsigned)grid), dim3(64 * kW), 0, s, a, (int)seg, (int)places, st, de);
    // (sequences of one segment end at once: 64 of them with 640 workgroups each took 33 us)
    const int64_t most = (size / 4 + 255) / 256, few = 2048 / a.n_seq, per = few < 1 ? 1 : (few < most ? few : most);
    hipLaunchKernelGGL(scan_states_kernel, dim3((unsigned)(a.n_seq * per)), dim3(256), 0, s, a, (int)seg, (int)places, per, st,
                       (const float*)de);
  }
  hipLaunchKernelGGL((scan_chunk_kernel<N, BF, false>), dim3((unsigned)grid), dim3(64 * kW), 0, s, a, (int)seg, (int)places, st, de);
  return hipGetLastError();
}

}  // namespace

size_t scan_chunk_workspace(const PackedScanArgs& a) {
  if (!split(a)) return 0;
  const int64_t places = scan_places(a.n_tokens, a.n_seq, segment(a));
  return (size_t)places * ((size_t)a.H * a.P * a.N + a.H) * sizeof(float);
}

hipError_t launch_scan_chunked(const PackedScanArgs& a, void* ws, hipStream_t s) {
  if (a.N == 128) return a.bf16 ? launch<128, true>(a, ws, s) : launch<128, false>(a, ws, s);
  return a.bf16 ? launch<64, true>(a, ws, s) : launch<64, false>(a, ws, s);
}

}  // namespace dfssm
