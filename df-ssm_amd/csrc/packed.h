// Packed sequences, their slots, and 16-bit rows, for the operators over prompts. Args has n_tokens, n_seq, cu (n_seq + 1
// first tokens, or null: len tokens each), slots (n_seq, or null) and n_slots.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "places.h"

namespace dfssm {

constexpr int kSlotPad = -1;  // a negative slot: the sequence is padding
constexpr int kSlotBad = -2;  // past the state, or taken by an earlier sequence of the call

template <bool BF>
__device__ __forceinline__ float w2f(uint16_t x) {
  if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)x << 16);
  return h2f(x);
}
template <bool BF>
__device__ __forceinline__ uint16_t f2w(float x) {  // RNE
  if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)x);
  return f2h(x);
}

// Tokens [t0, t1) of sequence b. Offsets read from device memory are held to [0, n_tokens] and an end
// before its start is an empty sequence, so no value of cu reaches past the tensors. (Offsets that fall may still make
// sequences overlap, or leave chunks that nothing prepared: the results are then not specified.)
template <class Args>
__device__ __forceinline__ void seq_range(const Args& a, int b, int64_t& t0, int64_t& t1) {
  if (!a.cu) {
    t0 = (int64_t)b * a.len;
    t1 = t0 + a.len;
    return;
  }
  const int64_t lo = a.cu[b], hi = a.cu[b + 1];
  t0 = lo < 0 ? 0 : (lo > a.n_tokens ? a.n_tokens : lo);
  t1 = hi < t0 ? t0 : (hi > a.n_tokens ? a.n_tokens : hi);
}

// The slot of sequence b, or kSlotPad / kSlotBad; the same in every lane of a wave. Two sequences with
// one slot would race on its state: the first has it, the others are refused.
template <class Args>
__device__ __forceinline__ int slot_of(const Args& a, int b) {
  if (!a.slots) return b < a.n_slots ? b : kSlotBad;
  const int s = a.slots[b];
  if (s < 0) return kSlotPad;
  bool taken = s >= a.n_slots;
  for (int i = threadIdx.x & 63; i < b; i += 64) taken |= a.slots[i] == s;
  return __any(taken) ? kSlotBad : s;
}

// The sequence and tile of place s of a launch's numbering of tiles of C tokens: sequence b starts at place
// floor(t0 / C) + b, which needs no sums over the lengths and leaves room for every tile (and one for an empty
// sequence). The lanes of a wave look at 64 sequences at once, and the sequence found is kept for the places that follow.
struct Where {
  int64_t first, t0, t1;  // place, tokens of a sequence
  int seq;
};
// (C = 0: c tokens, and tokens that fit 31 bits.) The sequence found may start behind the place, if it is the first.
template <int64_t C, class Args>
__device__ __forceinline__ void find_seq(const Args& a, int64_t s, Where& q, int64_t c = C) {
  const int lane = threadIdx.x & 63;
  auto start = [&](int64_t t0, int b) {
    return C ? place_of(t0, b, C ? C : 1) : (int64_t)((uint32_t)t0 / (uint32_t)c) + b;
  };
  q.seq = last_started(a.n_seq, [&](int lo, int step, int end) {
    const int i = lo + lane * step;
    bool before = false;
    if (i < end) {
      int64_t t0, t1;
      seq_range(a, i, t0, t1);
      before = start(t0, i) <= s;
    }
    return (int)__popcll(__ballot(before));
  });
  seq_range(a, q.seq, q.t0, q.t1);
  q.first = start(q.t0, q.seq);
}
// Tokens [tok, tok + the result) of place s; 0 where it holds none.
template <int64_t C, class Args>
__device__ __forceinline__ int64_t tile_of(const Args& a, int64_t s, Where& q, int64_t& tok) {
  if (s < q.first || (s - q.first) * C >= q.t1 - q.t0) find_seq<C>(a, s, q);
  const int64_t i = s - q.first;
  tok = 0;
  if (i < 0 || i * C >= q.t1 - q.t0) return 0;
  tok = q.t0 + i * C;
  return q.t1 - tok < C ? q.t1 - tok : C;
}

}  // namespace dfssm
