// The short causal convolution of a state space layer's channels (gfx950), for packed prompts and single tokens:
//   y_t = f(b + sum_{k < W} w_k x_{t - W + 1 + k}),  f(y) = y or y / (1 + e^-y),  W = 2 .. 4 taps per channel
// where the x before a sequence are its state's, which is left as the last W - 1 of state and sequence together.
// Sums are fp32, in the order b, w_0 x, .. w_{W-1} x; y is rounded once. States are copied, never rounded.
// What bounds it: memory. 64 x 512 tokens of 5376 channels (bf16, 709 MB) 0.136 ms, 5.2 TB/s, where a copy of 1 GiB reaches 5.3; twelve
// ragged sequences of 4352 channels (fp16, 134 MB) 29 us. A wave reads 1 KiB of a row at a time, eight rows on their way
// together (one by one, a load waits for the store before it); a tile's three rows before it come out of L2. States and weights
// go in the same wide pieces: by 2 bytes each, 0.150 ms, and 700 sequences of 9 tokens of 2048 channels 34 us instead of 19 (14 at a
// copy's rate). Few rows: the launch; one of 4352 channels 3.5 us in a replayed graph.
#include "common.h"
#include "layer.h"

namespace dfssm {

namespace {

constexpr int kRows = 16;  // tokens of a tile, which reads W - 1 rows more

template <int V>
__device__ __forceinline__ uint16_t value(const Raw16<V>& r, int i) {
  if constexpr (V == 1) return r.v;
  else return r.v[i];
}
// M values of each of a lane's V channels, as they lie in memory: V M of them in a row.
template <int V, int M>
struct Channels {
  uint16_t v[V * M];
  __device__ __forceinline__ void load(const uint16_t* p) {
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const Raw16<V> r = load_raw<V>(p + j * V);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j * V + i] = value<V>(r, i);
    }
  }
  __device__ __forceinline__ void store(uint16_t* p) const {
#pragma unroll
    for (int j = 0; j < M; ++j) {
      Raw16<V> r;
      if constexpr (V == 1) {
        r.v = v[j];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = v[j * V + i];
      }
      *(typename Pack16<V>::loose*)(p + j * V) = r.v;
    }
  }
  __device__ __forceinline__ uint16_t& at(int i, int k) { return v[i * M + k]; }
};

// A lane's V channels from c on: their weights, and rows of x and of the state.
template <int V, int W, bool BF>
struct Lane {
  float w[W][V], b[V];
  __device__ __forceinline__ void weights(const PackedConvArgs& a, int c) {
    Channels<V, W> m;
    m.load(a.weight + (int64_t)c * W);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < W; ++k) w[k][i] = w2f<BF>(m.at(i, k));
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = 0.0f;
    if (a.bias) load16<V, BF>(a.bias + c, b);
  }
  __device__ __forceinline__ void apply(const float (&x)[W][V], bool silu, uint16_t* out) const {
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = b[i];
#pragma unroll
      for (int k = 0; k < W; ++k) s = __builtin_fmaf(w[k][i], x[k][i], s);
      y[i] = silu ? silu_f32(s) : s;
    }
    store16<V, BF>(out, y);
  }
};

template <int V>
__device__ __forceinline__ void fill_rows(uint16_t* out, int64_t ld, int64_t n, uint16_t v) {
  for (int64_t t = 0; t < n; ++t)
#pragma unroll
    for (int i = 0; i < V; ++i) out[t * ld + i] = v;
}

// One wave: 64 V channels of a tile of kRows tokens of one sequence; the first tile also leaves the state, which it alone
// reads (so that it may be the same memory).
template <int V, int W, bool BF>
__global__ __launch_bounds__(256) void conv_prefill_kernel(PackedConvArgs a, int64_t tasks) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nc = (a.C + 64 * V - 1) / (64 * V);
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  if (task >= tasks) return;
  const int64_t place = task / nc;
  const int c = ((int)(task % nc) * 64 + lane) * V;
  Where q{0, 0, 0, 0};
  int64_t tok;
  const int len = (int)tile_of<kRows>(a, place, q, tok);
  const bool first = place == q.first;
  if (!len && !first) return;
  const int slot = slot_of(a, q.seq);
  if (c >= a.C) return;
  if (!len) tok = q.t0;
  if (slot < 0) {
    fill_rows<V>(a.out + tok * a.ld_out + c, a.ld_out, len, slot == kSlotPad ? 0 : 0x7fff);
    return;
  }
  const uint16_t* x = a.x + c;
  Lane<V, W, BF> l;
  l.weights(a, c);
  float win[W][V];  // the window, moved on by a token at a time
  if (first) {
    const int64_t at = ((int64_t)slot * a.C + c) * (W - 1), n = q.t1 - q.t0;
    Channels<V, W - 1> h, left;
    h.load(a.state + at);
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) win[k][i] = w2f<BF>(h.at(i, k));
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {  // element k from the end of state and sequence
      const int64_t p = n - (W - 1) + k;
      if (p >= 0) {
        const Raw16<V> r = load_raw<V>(x + (q.t0 + p) * a.ld_x);
#pragma unroll
        for (int i = 0; i < V; ++i) left.at(i, k) = value<V>(r, i);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          uint16_t v = h.at(i, k);
#pragma unroll
          for (int j = 1; j < W - 1; ++j)
            if (n == j && k + j < W - 1) v = h.at(i, k + j < W - 1 ? k + j : 0);
          left.at(i, k) = v;
        }
      }
    }
    left.store(a.state_out + at);
  } else {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load16<V, BF>(x + (tok - (W - 1) + k) * a.ld_x, win[k]);
  }
  // Eight rows on their way together (one by one, a load waits for the store before it).
  for (int t0 = 0; t0 < len; t0 += 8) {
    Raw16<V> row[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) row[t] = load_raw<V>(x + (tok + (t0 + t < len ? t0 + t : len - 1)) * a.ld_x);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if (t0 + t >= len) break;
      widen<V, BF>(row[t], win[W - 1]);
      l.apply(win, a.silu, a.out + (tok + t0 + t) * a.ld_out + c);
#pragma unroll
      for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
    }
  }
}

// One token of each sequence: a wave per 64 V channels of a row.
template <int V, int W, bool BF>
__global__ __launch_bounds__(256) void conv_step_kernel(PackedConvArgs a, int64_t tasks) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nc = (a.C + 64 * V - 1) / (64 * V);
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  if (task >= tasks) return;
  const int64_t t = task / nc;
  const int c = ((int)(task % nc) * 64 + lane) * V;
  const int slot = slot_of(a, (int)t);
  if (c >= a.C) return;
  uint16_t* out = a.out + t * a.ld_out + c;
  if (slot < 0) {
    fill_rows<V>(out, 0, 1, slot == kSlotPad ? 0 : 0x7fff);
    return;
  }
  Lane<V, W, BF> l;
  l.weights(a, c);
  const int64_t at = ((int64_t)slot * a.C + c) * (W - 1);
  float win[W][V];
  Channels<V, W - 1> h, left;
  h.load(a.state + at);
  const Raw16<V> x = load_raw<V>(a.x + t * a.ld_x + c);
  widen<V, BF>(x, win[W - 1]);
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      win[k][i] = w2f<BF>(h.at(i, k));
      left.at(i, k) = k < W - 2 ? h.at(i, k + 1 < W - 1 ? k + 1 : 0) : value<V>(x, i);
    }
  left.store(a.state_out + at);
  l.apply(win, a.silu, out);
}

template <int V, int W, bool BF>
hipError_t launch(const PackedConvArgs& a, bool step, hipStream_t s) {
  const int64_t nc = (a.C + 64 * V - 1) / (64 * V), places = step ? a.n_seq : a.n_tokens / kRows + a.n_seq;
  const int64_t tasks = places * nc, wgs = (tasks + 3) / 4;
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  if (step) hipLaunchKernelGGL((conv_step_kernel<V, W, BF>), dim3((unsigned)wgs), dim3(256), 0, s, a, tasks);
  else hipLaunchKernelGGL((conv_prefill_kernel<V, W, BF>), dim3((unsigned)wgs), dim3(256), 0, s, a, tasks);
  return hipGetLastError();
}
template <int V, int W>
hipError_t launch(const PackedConvArgs& a, bool step, hipStream_t s) {
  return a.bf16 ? launch<V, W, true>(a, step, s) : launch<V, W, false>(a, step, s);
}
template <int V>
hipError_t launch(const PackedConvArgs& a, bool step, hipStream_t s) {
  return a.W == 2 ? launch<V, 2>(a, step, s) : (a.W == 3 ? launch<V, 3>(a, step, s) : launch<V, 4>(a, step, s));
}
// Channels to a lane: 16 bytes of them (at any address) where a row has whole ones and fills a wave, else a pair, else one. 8096 tokens
// of 64 channels 4.9 us by one, 19 by eight; of 4350 channels 29 by pairs, of 4351 38 by one (29 at a copy's rate).
hipError_t launch(const PackedConvArgs& a, bool step, hipStream_t s) {
  if (a.C % 8 == 0 && a.C >= 512) return launch<8>(a, step, s);
  return a.C % 2 == 0 && a.C >= 128 ? launch<2>(a, step, s) : launch<1>(a, step, s);
}

}  // namespace

hipError_t launch_conv_step(const PackedConvArgs& a, hipStream_t s) { return launch(a, true, s); }
hipError_t launch_conv_prefill(const PackedConvArgs& a, hipStream_t s) { return launch(a, false, s); }

}  // namespace dfssm
