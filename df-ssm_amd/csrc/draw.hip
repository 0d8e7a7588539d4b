// Token draw with temperature, top-k, top-p and min-p from given random numbers (gfx950).
//
// Per row, ranked by (logit descending, index ascending), with m the largest logit:
//   e_r = exp((l_r - m) / T) in rank order; n_k = top_k (all if 0); Z = sum of e over the first n_k;
//   n_p = ranks r < n_k with (mass ranked above r) <= top_p Z; n_m = ranks with e_r >= min_p;
//   n = max(1, min(n_k, n_p, n_m)); S = mass of the first n; token = the last rank whose mass above is
//   <= u S, i.e. the first whose inclusive mass exceeds it.
// All three filters keep a prefix of the ranking, so no row is sorted: every question ("the last rank
// with fewer than n_k above it", "... with mass at most x above it") is one search over the cumulative
// counts and masses. e is computed in fp64 and its masses are held as integers, E = rint(e 2^44), so
// sums are exact and the same in any order (V <= 2^18, so they stay below 2^62).
//
// One workgroup per row. The row is spread over 2048 bins of falling logit (a monotone map, so bins are ranges of
// the ranking) whose counts, and masses where all tokens' matter, are summed by LDS atomics.
//   Few kept: with a top_k, or only a min_p, the first bins hold all that can be kept. They are gathered into LDS
//   and sorted, if they are at most 2046 tokens, and nothing but they needs an exponential.
//   Else every token's mass goes into its bin, and a search takes its bin from the prefix sums and resolves it
//   there: the bin's tokens gathered and sorted, or, where they are more than 2046, found by the exact 32-bit
//   order key and the index, a byte at a time over the row.
//
// What bounds it. Few kept: two passes over the logits, 256 rows of 131072 fp16, top_k 50, 27 us (67 MB, 5 TB/s of the
// passes' bytes); one row of 50288 takes 11 to 13 us, two reads of its logits and a dozen barriers one after the
// other. Else the arithmetic of the masses, about 30 instructions a token of which 11 are fp64, and the LDS atomics beside them: one
// row of 50288 takes 29 us, 12 of them that pass, as it has the arithmetic of one compute unit. 256 rows of 131072 fp32
// with settings of all kinds: 87 us. Spreading a row over up to 24 workgroups (three launches, bins summed in global
// memory) took 28 us for that one row and 19 for one with top_k 20, which takes 11 this way.
#include "common.h"
#include "dfssm.h"
#include "dfssm_kernels.h"

namespace dfssm {

namespace {

constexpr int kDT = 1024;      // threads of a row's workgroup
constexpr int kBins = 2048;
constexpr int kFine = 1024;    // bins of 1/64 in (m - l) / T; the others share what lies below
constexpr int kList = 2046;    // tokens that are sorted in LDS (and their masses, one more)
constexpr double kOne = 17592186044416.0;  // 2^44
constexpr int kTab = 1024;     // entries of the exponential's table

typedef unsigned long long u64;

template <int TYPE>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  if constexpr (TYPE == DFSSM_TYPE_F32) return ((const float*)row)[i];
  if constexpr (TYPE == DFSSM_TYPE_BF16) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[i] << 16);
  return h2f(((const uint16_t*)row)[i]);
}
// A NaN ranks as -inf; -0 as +0 (they are equal, so their order is that of the indexes).
__device__ __forceinline__ float clean(float l) { return l != l ? -__builtin_inff() : l + 0.0f; }

// f(index, logit, first of its load) for every token of the row, by all threads: 16 bytes a load between the row's
// aligned ends, two loads ahead.
template <int TYPE, class F>
__device__ __forceinline__ void each_token(const void* row, int V, F f) {
  constexpr int ES = TYPE == DFSSM_TYPE_F32 ? 4 : 2, N = 16 / ES;
  const int tid = threadIdx.x;
  const int head = min(V, (int)((16 - ((uintptr_t)row & 15)) & 15) / ES), nb = (V - head) / N, tail = head + nb * N;
  if (tid < head) f(tid, logit_at<TYPE>(row, tid), true);
  if (tail + tid < V) f(tail + tid, logit_at<TYPE>(row, tail + tid), true);
  const u32x4* p = (const u32x4*)((const char*)row + head * ES);
  auto piece = [&](const u32x4 x, int c) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t word = x[e * ES / 4];  // (a copy: a bit_cast of a vector's element takes the first one)
      float l;
      if constexpr (TYPE == DFSSM_TYPE_F32) l = __builtin_bit_cast(float, word);
      else if constexpr (TYPE == DFSSM_TYPE_BF16) l = __builtin_bit_cast(float, (e & 1) ? word & 0xffff0000u : word << 16);
      else l = h2f((uint16_t)(word >> (16 * (e & 1))));
      f(head + c * N + e, l, e == 0);
    }
  };
  // (the loop is not unrolled: a body is passed over a few times only, and its fetching from memory would cost more)
  if (nb > 0) {
    u32x4 x0 = p[min(tid, nb - 1)], x1 = p[min(tid + kDT, nb - 1)];
#pragma unroll 1
    for (int c = tid; c < nb; c += kDT) {
      const u32x4 x2 = p[min(c + 2 * kDT, nb - 1)];
      piece(x0, c);
      x0 = x1;
      x1 = x2;
    }
  }
}

// Ascending in falling logit.
__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return (b >> 31) ? b : 0x7fffffffu - b;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __builtin_bit_cast(float, (k >> 31) ? k : 0x7fffffffu - k);
}

struct RowScale {
  float m;           // the largest logit, finite here (rows with a +inf go their own way)
  float s1, s2, c2;  // bins: x = (m - l) s1 below kFine, then s2 x + c2, a line that is less steep
  float reach;       // tokens further than this below m have no mass (31.5 T: e < 2^-45)
  double y1;         // kTab log2(e) / T: e = 2^((l - m) y1 / kTab)
  const double* tab; // 2^(44 + j / kTab)
};
// -inf takes no part, nor does a NaN: both fail this (l <= m).
__device__ __forceinline__ bool taken(const RowScale r, float l) { return r.m - l < __builtin_inff(); }
// The bin of a token that takes part: the lower of the two lines (they cross at kFine).
__device__ __forceinline__ int bin_of(const RowScale r, float l) {
  const float x = (r.m - l) * r.s1;
  return (int)fminf(fminf(x, __builtin_fmaf(x, r.s2, r.c2)), (float)(kBins - 1));
}
// How far below m the upper end of bin b lies, `off` bins of tolerance for the roundings of bin_of (2^-13 of a bin).
__device__ __forceinline__ float bin_start(const RowScale r, int b, float off) {
  const float y = (float)b + off;
  return (y < (float)kFine ? y : (y - r.c2) / r.s2) / r.s1;
}
// e 2^44 = 2^44 exp((l - m) / T) for (m - l) <= reach, else 0: 2^((n + t) / kTab), n whole, |t| <= 1/2, from a table,
// an exponent added to it (44 + j / kTab + n / kTab > -2: it stays a normal number) and the Taylor polynomial of degree 3,
// whose rest is below 2^-50. n comes by adding 3 2^51, whose sum has it in its low bits. (exp() takes four times as
// many instructions, and this is most of the work.)
__device__ __forceinline__ double e44(const RowScale r, float l) {
  constexpr double c = 0.693147180559945309417 / kTab, big = 6755399441055744.0;
  if (!(r.m - l <= r.reach)) return 0.0;
  const double y = ((double)l - (double)r.m) * r.y1;
  const double z = y + big, t = y - (z - big);
  double p = __builtin_fma(c * c * c / 6.0, t, c * c / 2.0);
  p = __builtin_fma(p, t, c);
  p = __builtin_fma(p, t, 1.0);
  const int n = (int)(uint32_t)__builtin_bit_cast(u64, z);
  const u64 v = __builtin_bit_cast(u64, r.tab[n & (kTab - 1)] * p);
  const uint32_t hi = (uint32_t)(v >> 32) + ((uint32_t)(n >> 10) << 20);
  static_assert(kTab == 1 << 10, "n = kTab times the exponent and j");
  return __builtin_bit_cast(double, ((u64)hi << 32) | (uint32_t)v);
}
// The mass E = rint(e 2^44): added to 2^52 it is the low bits of the sum.
__device__ __forceinline__ u64 mass_of(double e44) {
  return __builtin_bit_cast(u64, e44 + 4503599627370496.0) & 0xfffffffffffffull;
}
constexpr u64 kUnit = 1ull << 44;  // the mass of the most probable token

struct DrawLds {
  double tab[kTab], ends[64];
  uint32_t cnt[kBins + 2];  // per bin, then tokens in earlier bins
  u64 mass[kBins + 2];      // the same for masses
  u64 comp[kList + 2];   // (order key << 24) | index of the listed tokens, sorted
  u64 lmass[kList + 2];  // mass ranked above each, of those listed; at the end that of all
  int rank[kDT / 2];
  uint32_t dcnt[256];
  u64 dmass[256];
  uint32_t wc[kDT / 64];
  u64 wm[kDT / 64];
  float wf[kDT / 64], wg[kDT / 64];
  int found, nlist, at[2];
  uint32_t rcnt;
  u64 rmass;
};

// v plus the values of the lanes before (inclusive prefix over the wave), moved within rows of 16 lanes and from row to
// row by the register file's own paths. (By lane shuffles through LDS a block's prefix took three times as long.)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(uint32_t& v) { v += moved<CTRL, ROWS>(v); }
template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(u64& v) {
  v += ((u64)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | moved<CTRL, ROWS>((uint32_t)v);
}
template <class X>
__device__ __forceinline__ X wave_scan(X v) {
  scan_step<0x111, 0xf>(v);  // from 1, 2, 4 and 8 lanes before, in the row
  scan_step<0x112, 0xf>(v);
  scan_step<0x114, 0xf>(v);
  scan_step<0x118, 0xf>(v);
  scan_step<0x142, 0xa>(v);  // row 0's last to row 1, 2's to 3; then lane 31's to rows 2 and 3
  scan_step<0x143, 0xc>(v);
  return v;
}

// Exclusive prefix over the block's threads, of which the first NT hold values; all call. total: of all.
template <int NT, class X>
__device__ __forceinline__ X block_excl(X v, X* waves, X& total) {
  const int tid = threadIdx.x, w = tid >> 6;
  const X in = wave_scan(v);
  if ((tid & 63) == 63 && w < NT / 64) waves[w] = in;
  __syncthreads();
  X before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i == w) before = all;
    all += waves[i];
  }
  __syncthreads();
  total = all;
  return (NT == kDT || w < NT / 64 ? before : all) + in - v;
}

// The tokens of bins lo .. hi and of bin far > hi (or -1) into L.comp, in any order. Returns how many they are; what
// exceeds kList is not listed.
template <int TYPE>
__device__ __forceinline__ int gather(const void* row, int V, const RowScale rs, int lo, int hi, int far, DrawLds& L) {
  const int tid = threadIdx.x;
  if (tid == 0) L.nlist = 0;
  __syncthreads();
  // Logits that may lie in the bins, by two compares; what passes is looked at closely.
  const float inf = __builtin_inff();
  auto upper = [&](int b) {  // of bin b's logits (a start out of fp32's reach bounds nothing)
    const float d = bin_start(rs, b, -0.01f);
    return b > 0 && d < 1e38f ? rs.m - d * 0.99999f : inf;
  };
  auto lower = [&](int b) { return b < kBins - 1 ? rs.m - bin_start(rs, b + 1, 0.01f) * 1.00001f : -inf; };
  const float near0 = upper(lo), near1 = lower(hi);
  const float far0 = far >= 0 ? upper(far) : -inf, far1 = far >= 0 ? lower(far) : inf;
  each_token<TYPE>(row, V, [&](int i, float l, bool) {
    if ((l <= near0 && l >= near1) || (l <= far0 && l >= far1)) {
      const int b = bin_of(rs, l);
      if (taken(rs, l) && ((b >= lo && b <= hi) || b == far)) {
        const int p = atomicAdd(&L.nlist, 1);
        if (p < kList) L.comp[p] = ((u64)order_key(clean(l)) << 24) | (uint32_t)i;
      }
    }
  });
  __syncthreads();
  return L.nlist;
}

// Sorts L.comp's first n <= kList entries and puts the masses ranked above each within the list into L.lmass.
__device__ __forceinline__ void sort_list(int n, const RowScale rs, DrawLds& L) {
  const int tid = threadIdx.x;
  if (n <= 64) {  // by one wave, with no barrier until the end
    if (tid < 64) {
      const u64 own = tid < n ? L.comp[tid] : ~0ull;
      int r = 0;
      for (int q = 0; q < n; ++q) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)own, q);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(own >> 32), q);
        r += (((u64)hi << 32) | lo) < own ? 1 : 0;
      }
      const u64 E = tid < n ? mass_of(e44(rs, key_logit((uint32_t)(own >> 24)))) : 0;
      if (tid < n) {
        L.comp[r] = own;
        L.lmass[r] = E;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      const u64 mine = tid < n ? L.lmass[tid] : 0, upto = wave_scan(mine);
      if (tid < n) L.lmass[tid] = upto - mine;
      if (tid == 63) L.lmass[n] = upto;
    }
    __syncthreads();
    return;
  }
  if (n <= kDT / 2) {
    // A token's rank is the number of smaller entries: kDT / n threads count for each, over parts of the list. No
    // barriers between, as the stages of a sorting network have, but its work grows with the square: a whole draw from
    // a row of 50288 with a list of 20 tokens takes 13.2 us this way, 21.5 by the network and 10.9 by one wave; 220: 17.7
    // and 24.4, 490: 26.2 and 26.5.
    int parts = kDT / max(n, 1);
    parts = parts > 16 ? 16 : parts;
    const int i = tid % max(n, 1), part = tid / max(n, 1);
    for (int q = tid; q < n; q += kDT) L.rank[q] = 0;
    __syncthreads();
    u64 own = 0;
    if (n && part < parts) {
      own = L.comp[i];
      const int per = (n + parts - 1) / parts, from = part * per, to = min(n, from + per);
      int r = 0;
      int q = from;
      for (; q + 8 <= to; q += 8) {
        u64 x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = L.comp[q + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) r += x[e] < own ? 1 : 0;
      }
      for (; q < to; ++q) r += L.comp[q] < own ? 1 : 0;
      if (r) atomicAdd(&L.rank[i], r);
    }
    __syncthreads();
    const int at = tid < n ? L.rank[tid] : 0;  // (thread tid < n has entry tid)
    if (tid < n) L.comp[at] = own;
    __syncthreads();
  } else {
    int n2 = kDT;  // a power of two, filled up with what sorts last
    while (n2 < n) n2 *= 2;
    for (int i = n + tid; i < n2; i += kDT) L.comp[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= n2; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {  // bitonic
        if (tid < n2 / 2) {
          const int a = (tid / j) * 2 * j + tid % j, b = a + j;
          const u64 x = L.comp[a], y = L.comp[b];
          if ((x > y) == ((a & k) == 0)) {
            L.comp[a] = y;
            L.comp[b] = x;
          }
        }
        __syncthreads();
      }
  }
  u64 m[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = 2 * tid + q;
    m[q] = i < n ? mass_of(e44(rs, key_logit((uint32_t)(L.comp[i] >> 24)))) : 0;
  }
  u64 all;
  const u64 s = block_excl<kDT>(m[0] + m[1], L.wm, all);
  if (2 * tid <= n) {  // (one entry more: the list's mass)
    L.lmass[2 * tid] = s;
    L.lmass[2 * tid + 1] = s + m[0];
  }
  __syncthreads();
}
template <int TYPE>
__device__ __forceinline__ int sort_bins(const void* row, int V, const RowScale rs, int lo, int hi, int far, DrawLds& L) {
  const int n = gather<TYPE>(row, V, rs, lo, hi, far, L);
  if (n <= kList) sort_list(n, rs, L);
  return n;
}

// L.cnt: from tokens per bin to tokens in earlier bins, and in all behind the last one.
__device__ __forceinline__ void count_prefix(DrawLds& L) {
  const int tid = threadIdx.x;
  __syncthreads();
  const uint32_t c0 = L.cnt[2 * tid], c1 = L.cnt[2 * tid + 1];
  uint32_t all;
  const uint32_t c = block_excl<kDT>(c0 + c1, L.wc, all);
  L.cnt[2 * tid] = c;
  L.cnt[2 * tid + 1] = c + c0;
  if (tid == 0) L.cnt[kBins] = all;
  __syncthreads();
}

// L.mass: the same for masses.
__device__ __forceinline__ void mass_prefix(DrawLds& L) {
  const int tid = threadIdx.x;
  __syncthreads();
  const u64 m0 = L.mass[2 * tid], m1 = L.mass[2 * tid + 1];
  u64 all;
  const u64 m = block_excl<kDT>(m0 + m1, L.wm, all);
  L.mass[2 * tid] = m;
  L.mass[2 * tid + 1] = m + m0;
  if (tid == 0) L.mass[kBins] = all;
  __syncthreads();
}

// A question to the ranking: by count (the last rank with fewer than n above it) or by mass (the last
// rank with mass at most x above it). Rank 0 always qualifies.
struct Ask {
  bool by_mass;
  uint32_t n;
  double x;
  __device__ __forceinline__ bool holds(uint32_t above, u64 mass) const { return by_mass ? (double)mass <= x : above < n; }
};
struct Found {
  u64 above, mine;  // mass ranked above it, and its own
  uint32_t key, idx;
};
__device__ __forceinline__ Found found(u64 above, u64 comp, const RowScale rs) {
  const uint32_t key = (uint32_t)(comp >> 24);
  return Found{above, mass_of(e44(rs, key_logit(key))), key, (uint32_t)(comp & 0xffffffu)};
}

// The last bin in use whose first token qualifies. By mass, a bin without mass is not in use: what lies there comes
// after all that a mass can ask for. Bins qualify up to a last one, which sees it by itself: the next one in use begins
// where it ends. (x >= 0 and n >= 1: the first in use qualifies.) L.at[slot] has it after a barrier.
__device__ __forceinline__ void mark_bin(const Ask q, int slot, DrawLds& L) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int b = 2 * threadIdx.x + j;
    bool it;
    if (q.by_mass) {
      const u64 m0 = L.mass[b], m1 = L.mass[b + 1];
      it = m1 != m0 && q.holds(0, m0) && (!q.holds(0, m1) || m1 == L.mass[kBins]);
    } else {
      const uint32_t c0 = L.cnt[b], c1 = L.cnt[b + 1];
      it = c1 != c0 && q.holds(c0, 0) && (!q.holds(c1, 0) || c1 == L.cnt[kBins]);
    }
    if (it) L.at[slot] = b;
  }
}
__device__ __forceinline__ int last_bin(const Ask q, DrawLds& L) {
  mark_bin(q, 0, L);
  __syncthreads();
  const int bin = L.at[0];
  __syncthreads();
  return bin;
}
// The last i of [from, to) with f(i), true up to a last one; f(from) counts as true. All threads call; i into L.at[0].
template <class F>
__device__ __forceinline__ int last_true(int from, int to, DrawLds& L, F f) {
  if (threadIdx.x == 0 && to <= from) L.at[0] = from;
  for (int i = from + threadIdx.x; i < to; i += kDT)
    if ((i == from || f(i)) && (i + 1 == to || !f(i + 1))) L.at[0] = i;
  __syncthreads();
  const int i = L.at[0];
  __syncthreads();
  return i;
}
// The last of entries [from, to) of the list that qualifies; its masses are off by `base` (and its counts by above).
__device__ __forceinline__ int last_entry(const Ask q, int from, int to, uint32_t above, u64 base, DrawLds& L) {
  return last_true(from, to, L, [&](int i) { return q.holds(above + (uint32_t)(i - from), base + L.lmass[i]); });
}

// One question resolved by the exact order key and the index, a byte at a time over the row (more tokens in the bin
// than the list takes).
template <int TYPE>
__device__ __forceinline__ Found search_row(const Ask q, int bin, const void* row, int V, const RowScale rs, DrawLds& L) {
  const int tid = threadIdx.x;
  uint32_t above = q.by_mass ? 0 : L.cnt[bin];
  u64 mass = L.mass[bin];
  u64 prefix = 0;
  for (int sh = 48; sh >= 0; sh -= 8) {
    if (tid < 256) {
      L.dcnt[tid] = 0;
      L.dmass[tid] = 0;
    }
    if (tid == 0) L.found = -1;
    __syncthreads();
    each_token<TYPE>(row, V, [&](int i, float l, bool) {
      if (!taken(rs, l) || bin_of(rs, l) != bin) return;
      const u64 c = ((u64)order_key(clean(l)) << 24) | (uint32_t)i;
      if ((c >> (sh + 8)) == prefix) {
        atomicAdd(&L.dcnt[(c >> sh) & 255], 1u);
        atomicAdd(&L.dmass[(c >> sh) & 255], mass_of(e44(rs, l)));
      }
    });
    __syncthreads();
    const uint32_t c0 = tid < 256 ? L.dcnt[tid] : 0;
    const u64 m0 = tid < 256 ? L.dmass[tid] : 0;
    uint32_t call;
    u64 mall;
    const uint32_t c = block_excl<256>(c0, L.wc, call) + above;
    const u64 m = block_excl<256>(m0, L.wm, mall) + mass;
    // the first digit in use qualifies always: its prefix was found to (by mass, the first with any)
    const bool first = q.by_mass ? m == mass : c == above;
    if (tid < 256 && (q.by_mass ? m0 != 0 : c0 != 0) && (q.holds(c, m) || first)) atomicMax(&L.found, tid);
    __syncthreads();
    const int d = L.found;
    if (tid == d) {
      L.rcnt = c;
      L.rmass = m;
    }
    __syncthreads();
    above = L.rcnt;
    mass = L.rmass;
    prefix = (prefix << 8) | (u64)d;
  }
  return found(mass, prefix, rs);
}
template <int TYPE>
__device__ __forceinline__ Found search(const Ask q, const void* row, int V, const RowScale rs, DrawLds& L) {
  const int bin = last_bin(q, L);
  const int n = sort_bins<TYPE>(row, V, rs, bin, bin, -1, L);
  if (n > kList) return search_row<TYPE>(q, bin, row, V, rs, L);
  const int i = last_entry(q, 0, n, q.by_mass ? 0 : L.cnt[bin], L.mass[bin], L);
  return found(L.mass[bin] + L.lmass[i], L.comp[i], rs);
}

__device__ __forceinline__ u64 wave_add64(u64 v) {
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, o, 64), hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), o, 64);
    v += ((u64)hi << 32) | lo;
  }
  return v;
}

// A row and its settings.
template <int TYPE>
struct Row {
  const void* at;
  int b, V, k;
  float T, tp, mp, u;
  bool limit;     // a top_k that leaves something out
  bool by_k, by_m; // what can be kept lies in the first bins: a top_k, or a min_p and no top_p (whose mass is that of all)
  double mp44, share;  // min_p and top_p, the latter as a factor
  __device__ __forceinline__ Row(const DrawArgs& a, int row) : b(row), V(a.V) {
    at = (const char*)a.logits + (size_t)b * a.ld * (TYPE == DFSSM_TYPE_F32 ? 4 : 2);
    T = a.temperatures ? a.temperatures[b] : a.temperature;
    k = a.top_ks ? a.top_ks[b] : a.top_k;
    tp = a.top_ps ? a.top_ps[b] : a.top_p;
    mp = a.min_ps ? a.min_ps[b] : a.min_p;
    u = a.u[b];
    u = u >= 0.0f ? (u < 1.0f ? u : 0.99999994f) : 0.0f;
    limit = k > 0 && k < V;
    by_k = limit && k <= kList;
    by_m = !limit && mp > 0.0f && mp <= 1.0f && !(tp < 1.0f);
    mp44 = (double)mp * kOne;
    share = (double)(tp > 0.0f ? tp : 0.0f);
  }
  // The last bin that min_p can keep of (the bins are monotone).
  __device__ __forceinline__ int min_bin(const RowScale rs) const {
    return bin_of(rs, rs.m + T * (__builtin_logf(mp) * 1.0001f - 1e-6f));
  }
};

// A row with +inf logits: each has mass 1 and nothing else any, ranked by index. Which of them is drawn comes from
// their number; every thread counts those of a stretch of the row, and the one whose stretch holds it walks along.
template <int TYPE>
__device__ __forceinline__ void draw_inf(const DrawArgs& a, const Row<TYPE>& r, DrawLds& L) {
  const int tid = threadIdx.x, per = (r.V + kDT - 1) / kDT, from = min(r.V, tid * per), to = min(r.V, from + per);
  uint32_t mine = 0;
  for (int i = from; i < to; ++i) mine += logit_at<TYPE>(r.at, i) == __builtin_inff() ? 1 : 0;
  uint32_t all;
  uint32_t c = block_excl<kDT>(mine, L.wc, all);
  int n = (int)all;
  if (r.k > 0) n = min(n, r.k);
  if (r.tp < 1.0f) n = min(n, (int)(r.share * (double)n) + 1);
  if (!(r.mp <= 1.0f)) n = 1;
  const uint32_t at = (uint32_t)min(n - 1, (int)((double)r.u * (double)n));
  if (at < c || at >= c + mine) return;
  for (int i = from; i < to; ++i)
    if (logit_at<TYPE>(r.at, i) == __builtin_inff() && c++ == at) {
      a.next[r.b] = i;
      if (a.logprob) a.logprob[r.b] = (float)-log((double)n);
    }
}

// The largest logit of the block's tokens, and nearly the least finite one (of one in each load: only the bins' width
// comes from it). L.wf and L.wg are written; a barrier later block_range has the two.
template <int TYPE>
__device__ __forceinline__ float scan_range(const void* row, int V, DrawLds& L) {
  const int tid = threadIdx.x;
  float m = -__builtin_inff(), lo = __builtin_inff();
  each_token<TYPE>(row, V, [&](int, float l, bool first) {
    m = fmaxf(m, l);  // (of a NaN and a number, the number)
    if (first && l < lo && l > -__builtin_inff()) lo = l;
  });
  const float own = m;  // of this thread's tokens
  for (int o = 32; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor(m, o, 64));
    lo = fminf(lo, __shfl_xor(lo, o, 64));
  }
  if ((tid & 63) == 0) {
    L.wf[tid >> 6] = m;
    L.wg[tid >> 6] = lo;
  }
  return own;
}
__device__ __forceinline__ void block_range(float& m, float& lo, const DrawLds& L) {
  m = L.wf[0];
  lo = L.wg[0];
  for (int i = 1; i < kDT / 64; ++i) {
    m = fmaxf(m, L.wf[i]);
    lo = fminf(lo, L.wg[i]);
  }
}

// Clears the bins and begins the exponential's table, whose entries are products of two; a barrier later table_finish.
__device__ __forceinline__ void start(DrawLds& L) {
  const int tid = threadIdx.x;
  for (int i = tid; i < kBins; i += kDT) {
    L.cnt[i] = 0;
    L.mass[i] = 0;
  }
  if (tid < 64) L.ends[tid] = tid < 32 ? exp2((double)tid * (1.0 / 32)) * kOne : exp2((double)(tid - 32) * (1.0 / kTab));
  if (tid == 0) {
    L.rcnt = 0;
    L.rmass = 0;
    L.cnt[kBins] = 0;
    L.mass[kBins] = 0;
  }
}
__device__ __forceinline__ void table_finish(DrawLds& L) {
  L.tab[threadIdx.x] = L.ends[threadIdx.x >> 5] * L.ends[32 + (threadIdx.x & 31)];
  static_assert(kTab == kDT && kTab == 32 * 32, "an entry per thread");
}

__device__ __forceinline__ RowScale scale_of(float m, float lo, float T, const DrawLds& L) {
  RowScale rs;
  rs.m = m;
  rs.y1 = kTab * 1.4426950408889634074 / (double)T;
  rs.tab = L.tab;
  rs.reach = fminf(31.5f * T, 3.4028234e38f);
  rs.s1 = 64.0f / T;
  rs.s2 = 1.0f;
  if (lo < m) {
    const float span = m - lo, x = span * rs.s1;
    if (!(x >= (float)kBins)) rs.s1 = (float)(kBins - 1) / span;  // a narrow row spreads over all bins
    else rs.s2 = (float)(kBins - kFine - 1) / (x - (float)kFine);
  }
  rs.s1 = fminf(rs.s1, 1e38f);  // (so that 0 stays bin 0)
  rs.c2 = (float)kFine - (float)kFine * rs.s2;
  return rs;
}

// Counts or masses of the block's tokens into its bins (and L.rmass: the mass of the tokens with e >= min_p).
template <int TYPE>
__device__ __forceinline__ void count_tokens(const void* row, int V, const RowScale rs, DrawLds& L) {
  each_token<TYPE>(row, V, [&](int, float l, bool) {
    if (taken(rs, l)) atomicAdd(&L.cnt[bin_of(rs, l)], 1u);
  });
}
template <int TYPE>
__device__ __forceinline__ void add_masses(const void* row, int V, const Row<TYPE>& r, const RowScale rs, DrawLds& L) {
  u64 mm = 0;
  const double border = r.mp <= 0.0f ? __builtin_inf() : r.mp44;
  each_token<TYPE>(row, V, [&](int, float l, bool) {
    if (!(rs.m - l <= rs.reach)) return;
    const double e = e44(rs, l);
    const u64 E = mass_of(e);
    atomicAdd(&L.mass[bin_of(rs, l)], E);
    if (e >= border) mm += E;
  });
  mm = wave_add64(mm);
  if ((threadIdx.x & 63) == 0) atomicAdd(&L.rmass, mm);
}
// Of min_p's tokens (rank 0 is kept in any case).
__device__ __forceinline__ u64 min_mass(float mp, u64 mm) { return mp <= 0.0f ? ~0ull : mm > kUnit ? mm : kUnit; }

template <int TYPE>
__device__ __forceinline__ void answer(const DrawArgs& a, const Row<TYPE>& r, const RowScale rs, u64 comp, u64 S) {
  if (threadIdx.x == 0) {
    a.next[r.b] = (int64_t)(comp & 0xffffffu);
    if (a.logprob) a.logprob[r.b] = (float)log(e44(rs, key_logit((uint32_t)(comp >> 24))) / (double)S);
  }
}

// The draw where the sorted list holds all that can be kept.
template <int TYPE>
__device__ __forceinline__ void pick_few(const DrawArgs& a, const Row<TYPE>& r, const RowScale rs, int n, DrawLds& L) {
  const int nk = r.by_k ? min(r.k, n) : n;
  const u64 Z = L.lmass[nk];
  const int kept = 1 + last_true(0, nk, L, [&](int i) {
    return (!(r.tp < 1.0f) || (double)L.lmass[i] <= r.share * (double)Z) &&
           e44(rs, key_logit((uint32_t)(L.comp[i] >> 24))) >= r.mp44;
  });
  const u64 S = L.lmass[kept];
  const int i = last_entry(Ask{true, 0u, (double)r.u * (double)S}, 0, kept, 0, 0, L);
  answer(a, r, rs, L.comp[i], S);
}

// The draw by masses from one list, S the mass before top_p: top_p's border lies in one bin, `far`, which bounds the kept
// mass, and so the bins that the drawn token may lie in, d0 .. d1.
struct Plan {
  int d0, d1, far;
};
template <int TYPE>
__device__ __forceinline__ Plan plan(const Row<TYPE>& r, u64 S, u64 M_m, DrawLds& L) {
  Plan p{0, 0, -1};
  u64 s0 = S < M_m ? S : M_m, s1 = s0;
  if (r.tp < 1.0f) {
    p.far = last_bin(Ask{true, 0u, r.share * (double)S}, L);
    s0 = max(min(s0, L.mass[p.far]), (u64)1);
    s1 = min(s1, L.mass[p.far + 1]);
  }
  mark_bin(Ask{true, 0u, (double)r.u * (double)s0}, 0, L);
  mark_bin(Ask{true, 0u, (double)r.u * (double)s1}, 1, L);
  __syncthreads();
  p.d0 = L.at[0];
  p.d1 = L.at[1];
  __syncthreads();
  return p;
}
template <int TYPE>
__device__ __forceinline__ void pick_planned(const DrawArgs& a, const Row<TYPE>& r, const RowScale rs, const Plan p, int n,
                                             u64 S, u64 M_m, DrawLds& L) {
  int split = n;  // entries before it are of d0 .. d1; those of far follow, their masses counted from far's own start
  if (r.tp < 1.0f) {
    const Ask border{true, 0u, r.share * (double)S};
    u64 base = L.mass[p.d0];
    int from = 0;
    if (p.far > p.d1) {
      auto near = [&](int i) { return bin_of(rs, key_logit((uint32_t)(L.comp[i] >> 24))) <= p.d1; };
      from = split = 1 + last_true(0, n, L, near);
      base = L.mass[p.far] - (L.mass[p.d1 + 1] - L.mass[p.d0]);
    }
    const int last = last_entry(border, from, n, 0, base, L);
    S = min(S, base + L.lmass[last + 1]);
  }
  S = min(S, M_m);
  const int i = last_entry(Ask{true, 0u, (double)r.u * (double)S}, 0, split, 0, L.mass[p.d0], L);
  answer(a, r, rs, L.comp[i], S);
}

// A whole row by one workgroup.
template <int TYPE>
__device__ __forceinline__ void draw_row(const DrawArgs& a, int row, DrawLds& L) {
  const int tid = threadIdx.x;
  const Row<TYPE> r(a, row);
  const int V = r.V;
  const float own = scan_range<TYPE>(r.at, V, L);
  start(L);
  if (tid == 0) L.found = 0x7fffffff;
  __syncthreads();
  float m, lo;
  block_range(m, lo, L);
  table_finish(L);
  if (m == -__builtin_inff() || !(r.T > 0.0f)) {  // nothing to draw from; greedy
    const bool none = m == -__builtin_inff();
    if (!none) each_token<TYPE>(r.at, V, [&](int i, float l, bool) {
      if (l == m) atomicMin(&L.found, i);
    });
    __syncthreads();
    if (tid == 0) {
      a.next[r.b] = none ? -1 : L.found;
      if (a.logprob) a.logprob[r.b] = none ? -__builtin_inff() : 0.0f;
    }
    return;
  }
  if (m == __builtin_inff()) {
    draw_inf(a, r, L);
    return;
  }
  const RowScale rs = scale_of(m, lo, r.T, L);

  // A bin that has k threads' largest tokens in it or before it has the first k ranks too. That is nearly the bin of
  // rank k while k is small beside the threads (k = 512: 0.7 tokens a thread, 710 in all), and needs no pass to
  // count. 256 rows of 131072, with and without: k = 20 27 and 37 us, 200: 31 and 40, 512: 43 and 53; at 700 and more
  // both count (54 us; the list is then more often too long than not).
  const bool by_own = r.limit && r.k <= kDT / 2;
  int hi = kBins - 1, n = kList + 1;
  if (r.by_m) hi = r.min_bin(rs);
  if (by_own) {
    if (taken(rs, own)) atomicAdd(&L.cnt[bin_of(rs, own)], 1u);
    count_prefix(L);
    if (L.cnt[kBins] >= (uint32_t)r.k) hi = last_bin(Ask{false, (uint32_t)r.k, 0.0}, L);
  }
  if (by_own || r.by_m) {
    __syncthreads();
    n = sort_bins<TYPE>(r.at, V, rs, 0, hi, -1, L);
  }
  if (r.limit && n > kList) {
    for (int i = tid; i < kBins; i += kDT) L.cnt[i] = 0;
    __syncthreads();
    count_tokens<TYPE>(r.at, V, rs, L);
    count_prefix(L);
    hi = last_bin(Ask{false, (uint32_t)r.k, 0.0}, L);
    if (r.by_k && L.cnt[hi + 1] <= kList) n = sort_bins<TYPE>(r.at, V, rs, 0, hi, -1, L);
  }
  if ((r.by_k || r.by_m) && n <= kList) {
    pick_few(a, r, rs, n, L);
    return;
  }

  __syncthreads();
  add_masses<TYPE>(r.at, V, r, rs, L);
  mass_prefix(L);
  const u64 M_m = min_mass(r.mp, L.rmass);
  u64 S = L.mass[kBins];  // of what is kept: the shortest of three prefixes has the least
  if (r.limit) {
    const Found f = search<TYPE>(Ask{false, (uint32_t)r.k, 0.0}, r.at, V, rs, L);
    S = f.above + f.mine;
  }
  const Plan p = plan(r, S, M_m, L);
  n = sort_bins<TYPE>(r.at, V, rs, p.d0, p.d1, p.far > p.d1 ? p.far : -1, L);
  if (n <= kList) {
    pick_planned(a, r, rs, p, n, S, M_m, L);
    return;
  }
  if (r.tp < 1.0f) {
    const Found f = search<TYPE>(Ask{true, 0u, r.share * (double)S}, r.at, V, rs, L);
    S = min(S, f.above + f.mine);
  }
  S = min(S, M_m);
  const Found f = search<TYPE>(Ask{true, 0u, (double)r.u * (double)S}, r.at, V, rs, L);
  answer(a, r, rs, ((u64)f.key << 24) | f.idx, S);
}

template <int TYPE>
__global__ __launch_bounds__(kDT) void draw_row_kernel(DrawArgs a) {
  __shared__ DrawLds L;
  draw_row<TYPE>(a, blockIdx.x, L);
}

}  // namespace

hipError_t launch_draw(const DrawArgs& a, int type, int batch, hipStream_t s) {
  if (type == DFSSM_TYPE_F32) hipLaunchKernelGGL(draw_row_kernel<DFSSM_TYPE_F32>, dim3(batch), dim3(kDT), 0, s, a);
  else if (type == DFSSM_TYPE_BF16) hipLaunchKernelGGL(draw_row_kernel<DFSSM_TYPE_BF16>, dim3(batch), dim3(kDT), 0, s, a);
  else hipLaunchKernelGGL(draw_row_kernel<DFSSM_TYPE_F16>, dim3(batch), dim3(kDT), 0, s, a);
  return hipGetLastError();
}

}  // namespace dfssm
