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
// One workgroup per row. The row is spread over 2048 bins of falling logit (a monotone map, so bins are
// ranges of the ranking): counts and masses by LDS atomics, then their prefix sums. A search takes its
// bin from the prefix sums and resolves it by the exact 32-bit order key and the index, a byte at a
// time: over the bin's tokens gathered into LDS, or over the row where they are too many.
#include "common.h"
#include "dfssm.h"
#include "dfssm_kernels.h"

namespace dfssm {

namespace {

constexpr int kDT = 1024;      // threads of a row's workgroup
constexpr int kBins = 2048;
constexpr int kFine = 1024;    // bins of 1/64 in (m - l) / T; the others share what lies below
constexpr int kList = 2048;    // tokens of a bin held in LDS
constexpr double kOne = 17592186044416.0;  // 2^44

typedef unsigned long long u64;

template <int TYPE>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  if constexpr (TYPE == DFSSM_TYPE_F32) return ((const float*)row)[i];
  if constexpr (TYPE == DFSSM_TYPE_BF16) return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[i] << 16);
  return h2f(((const uint16_t*)row)[i]);
}
// A NaN ranks as -inf; -0 as +0 (they are equal, so their order is that of the indexes).
__device__ __forceinline__ float clean(float l) { return l != l ? -__builtin_inff() : l + 0.0f; }
// Ascending in falling logit.
__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return (b >> 31) ? b : 0x7fffffffu - b;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __builtin_bit_cast(float, (k >> 31) ? k : 0x7fffffffu - k);
}

struct RowScale {
  float m, s1, s2;   // bins: x = (m - l) s1 below kFine, then kFine + (x - kFine) s2
  double it;         // 1 / T
};
__device__ __forceinline__ int bin_of(const RowScale& r, float l) {
  if (l == r.m) return 0;  // (also where both are +inf)
  const float x = (r.m - l) * r.s1;
  if (x < (float)kFine) return (int)x;
  const float y = (x - (float)kFine) * r.s2;
  return kFine + (y < (float)(kBins - kFine - 1) ? (int)y : kBins - kFine - 1);
}
__device__ __forceinline__ double e_of(const RowScale& r, float l) {
  return l == r.m ? 1.0 : exp(((double)l - (double)r.m) * r.it);
}
__device__ __forceinline__ u64 mass_of(double e) { return (u64)__builtin_rint(e * kOne); }

struct DrawLds {
  uint32_t cnt[kBins];   // per bin, then tokens in earlier bins
  u64 mass[kBins];       // the same for masses
  u64 comp[kList];       // (order key << 24) | index of the listed bin's tokens
  u64 lmass[kList];
  uint32_t dcnt[256];
  u64 dmass[256];
  uint32_t wc[kDT / 64];
  u64 wm[kDT / 64];
  float wf[kDT / 64], wg[kDT / 64];
  int found, nlist, listbin;
  uint32_t rcnt;
  u64 rmass;
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int o) {
  const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, o, 64), hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), o, 64);
  return ((u64)hi << 32) | lo;
}

// Exclusive prefix over the block's threads of (c, m); NT threads take part, all call.
template <int NT>
__device__ __forceinline__ void block_excl(uint32_t& c, u64& m, DrawLds& L) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  uint32_t ci = c;
  u64 mi = m;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = (uint32_t)__shfl_up((int)ci, o, 64);
    const u64 y = shfl_up64(mi, o);
    if (lane >= o) {
      ci += x;
      mi += y;
    }
  }
  if (lane == 63 && w < NT / 64) {
    L.wc[w] = ci;
    L.wm[w] = mi;
  }
  __syncthreads();
  c = ci - c;
  m = mi - m;
  for (int i = 0; i < NT / 64; ++i)
    if (i < w) {
      c += L.wc[i];
      m += L.wm[i];
    }
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
  uint32_t rank;
  u64 above, mine;  // mass ranked above it, and its own
  uint32_t key, idx;
};

template <int TYPE>
__device__ Found search(const Ask q, const void* row, int V, const RowScale& rs, DrawLds& L) {
  const int tid = threadIdx.x;
  if (tid == 0) L.found = 0;
  __syncthreads();
  int best = -1;
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // bin 0 is never empty; a bin is empty where the next one's prefix is the same
    const int b = 2 * tid + j;
    const uint32_t next = b + 1 < kBins ? L.cnt[b + 1] : (uint32_t)V;
    if (next != L.cnt[b] && q.holds(L.cnt[b], L.mass[b])) best = b;
  }
  if (best >= 0) atomicMax(&L.found, best);
  __syncthreads();
  const int bin = L.found;
  uint32_t above = L.cnt[bin];
  u64 mass = L.mass[bin];
  const int n = (int)((bin + 1 < kBins ? L.cnt[bin + 1] : (uint32_t)V) - above);
  const bool list = n <= kList;
  if (list && L.listbin != bin) {  // (uniform)
    __syncthreads();
    if (tid == 0) {
      L.nlist = 0;
      L.listbin = bin;
    }
    __syncthreads();
    for (int i = tid; i < V; i += kDT) {
      const float l = clean(logit_at<TYPE>(row, i));
      if (bin_of(rs, l) == bin) {
        const int p = atomicAdd(&L.nlist, 1);
        if (p < kList) {
          L.comp[p] = ((u64)order_key(l) << 24) | (uint32_t)i;
          L.lmass[p] = mass_of(e_of(rs, l));
        }
      }
    }
    __syncthreads();
  }
  u64 prefix = 0;
  for (int sh = 48; sh >= 0; sh -= 8) {
    if (tid < 256) {
      L.dcnt[tid] = 0;
      L.dmass[tid] = 0;
    }
    if (tid == 0) L.found = -1;
    __syncthreads();
    if (list) {
      for (int i = tid; i < n; i += kDT) {
        const u64 c = L.comp[i];
        if ((c >> (sh + 8)) == prefix) {
          atomicAdd(&L.dcnt[(c >> sh) & 255], 1u);
          atomicAdd(&L.dmass[(c >> sh) & 255], L.lmass[i]);
        }
      }
    } else {
      for (int i = tid; i < V; i += kDT) {
        const float l = clean(logit_at<TYPE>(row, i));
        if (bin_of(rs, l) != bin) continue;
        const u64 c = ((u64)order_key(l) << 24) | (uint32_t)i;
        if ((c >> (sh + 8)) == prefix) {
          atomicAdd(&L.dcnt[(c >> sh) & 255], 1u);
          atomicAdd(&L.dmass[(c >> sh) & 255], mass_of(e_of(rs, l)));
        }
      }
    }
    __syncthreads();
    const uint32_t c0 = tid < 256 ? L.dcnt[tid] : 0;
    uint32_t c = c0;
    u64 m = tid < 256 ? L.dmass[tid] : 0;
    block_excl<256>(c, m, L);
    c += above;
    m += mass;
    // the first digit in use qualifies always: its prefix was found to
    if (tid < 256 && c0 && (q.holds(c, m) || c == above)) atomicMax(&L.found, tid);
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
  Found f;
  f.rank = above;
  f.above = mass;
  f.key = (uint32_t)(prefix >> 24);
  f.idx = (uint32_t)(prefix & 0xffffffu);
  f.mine = mass_of(e_of(rs, key_logit(f.key)));
  return f;
}

template <int TYPE>
__global__ __launch_bounds__(kDT) void draw_row_kernel(DrawArgs a) {
  __shared__ DrawLds L;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.x, V = a.V;
  const void* row = (const char*)a.logits + (size_t)b * a.ld * (TYPE == DFSSM_TYPE_F32 ? 4 : 2);
  const float T = a.temperatures ? a.temperatures[b] : a.temperature;
  int k = a.top_ks ? a.top_ks[b] : a.top_k;
  const float tp = a.top_ps ? a.top_ps[b] : a.top_p;
  const float mp = a.min_ps ? a.min_ps[b] : a.min_p;
  float u = a.u[b];
  u = u >= 0.0f ? (u < 1.0f ? u : 0.99999994f) : 0.0f;

  // the largest logit, the lowest index that has it, and the least finite one
  float m = -__builtin_inff(), lo = __builtin_inff();
  int im = 0x7fffffff;
  for (int i = tid; i < V; i += kDT) {
    const float l = clean(logit_at<TYPE>(row, i));
    if (l > m || (l == m && i < im)) {
      m = l;
      im = i;
    }
    if (l > -__builtin_inff()) lo = fminf(lo, l);
  }
  for (int i = tid; i < kBins; i += kDT) {
    L.cnt[i] = 0;
    L.mass[i] = 0;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(m, o, 64);
    const int oi = __shfl_xor(im, o, 64);
    if (om > m || (om == m && oi < im)) {
      m = om;
      im = oi;
    }
    lo = fminf(lo, __shfl_xor(lo, o, 64));
  }
  if (lane == 0) {
    L.wf[w] = m;
    L.wg[w] = lo;
    L.wc[w] = (uint32_t)im;
  }
  __syncthreads();
  m = L.wf[0];
  lo = L.wg[0];
  im = (int)L.wc[0];
  for (int i = 1; i < kDT / 64; ++i) {
    const float om = L.wf[i];
    const int oi = (int)L.wc[i];
    if (om > m || (om == m && oi < im)) {
      m = om;
      im = oi;
    }
    lo = fminf(lo, L.wg[i]);
  }
  __syncthreads();
  if (m == -__builtin_inff() || !(T > 0.0f)) {  // nothing to draw from; greedy
    if (tid == 0) {
      const bool none = m == -__builtin_inff();
      a.next[b] = none ? -1 : im;
      if (a.logprob) a.logprob[b] = none ? -__builtin_inff() : 0.0f;
    }
    return;
  }
  RowScale rs;
  rs.m = m;
  rs.it = 1.0 / (double)T;
  {
    const float span = m - lo;  // finite or +inf (m = +inf), never NaN: lo <= m, and both +inf give NaN
    const float s = 64.0f / T;
    rs.s1 = s;
    rs.s2 = 1.0f;
    if (span > 0.0f && span < __builtin_inff()) {
      const float x = span * s;
      if (!(x >= (float)kFine)) rs.s1 = (float)(kFine - 1) / span;  // a narrow row spreads over the fine bins
      else if (x > (float)kBins) rs.s2 = (float)(kBins - kFine - 1) / (x - (float)kFine);
    }
  }

  uint32_t nm = 0;
  u64 mm = 0;
  for (int i = tid; i < V; i += kDT) {
    const float l = clean(logit_at<TYPE>(row, i));
    const double e = e_of(rs, l);
    const u64 E = mass_of(e);
    const int bin = bin_of(rs, l);
    atomicAdd(&L.cnt[bin], 1u);
    if (E) atomicAdd(&L.mass[bin], E);
    if (e >= (double)mp) {
      ++nm;
      mm += E;
    }
  }
  __syncthreads();
  uint32_t c0 = L.cnt[2 * tid], c = c0 + L.cnt[2 * tid + 1];
  u64 m0 = L.mass[2 * tid], ms = m0 + L.mass[2 * tid + 1];
  block_excl<kDT>(c, ms, L);
  L.cnt[2 * tid] = c;
  L.cnt[2 * tid + 1] = c + c0;
  L.mass[2 * tid] = ms;
  L.mass[2 * tid + 1] = ms + m0;
  u64 S = 0;  // the mass of the whole row
  for (int i = 0; i < kDT / 64; ++i) S += L.wm[i];
  if (tid == kDT - 1) L.listbin = -1;
  // the tokens with e >= min_p
  if (tid == 0) {
    L.rcnt = 0;
    L.rmass = 0;
  }
  __syncthreads();
  if (nm) {
    atomicAdd(&L.rcnt, nm);
    atomicAdd(&L.rmass, mm);
  }
  __syncthreads();
  const uint32_t n_m = L.rcnt;
  const u64 M_m = L.rmass;
  __syncthreads();
  uint32_t n = (uint32_t)V;
  if (k > 0 && k < V) {
    const Found f = search<TYPE>(Ask{false, (uint32_t)k, 0.0}, row, V, rs, L);
    n = f.rank + 1;
    S = f.above + f.mine;
  }
  if (tp < 1.0f) {
    const Found f = search<TYPE>(Ask{true, 0u, (double)(tp > 0.0f ? tp : 0.0f) * (double)S}, row, V, rs, L);
    if (f.rank + 1 < n) {
      n = f.rank + 1;
      S = f.above + f.mine;
    }
  }
  if (n_m < n) {
    n = n_m > 1 ? n_m : 1;
    S = n > 1 ? M_m : mass_of(1.0);
  }
  const Found f = search<TYPE>(Ask{true, 0u, (double)u * (double)S}, row, V, rs, L);
  if (tid == 0) {
    a.next[b] = (int64_t)f.idx;
    if (a.logprob) a.logprob[b] = (float)log(e_of(rs, key_logit(f.key)) * kOne / (double)S);
  }
}

}  // namespace

hipError_t launch_draw(const DrawArgs& a, int type, int batch, hipStream_t s) {
  if (type == DFSSM_TYPE_F32) hipLaunchKernelGGL(draw_row_kernel<DFSSM_TYPE_F32>, dim3(batch), dim3(kDT), 0, s, a);
  else if (type == DFSSM_TYPE_BF16) hipLaunchKernelGGL(draw_row_kernel<DFSSM_TYPE_BF16>, dim3(batch), dim3(kDT), 0, s, a);
  else hipLaunchKernelGGL(draw_row_kernel<DFSSM_TYPE_F16>, dim3(batch), dim3(kDT), 0, s, a);
  return hipGetLastError();
}

}  // namespace dfssm
