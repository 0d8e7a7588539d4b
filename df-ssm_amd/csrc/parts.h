// Operands of the 16-bit matrix cores for the chunked operators: fp32 factors as sums of 16-bit parts, rows as buffers, sums
// and waits within a wave.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace dfssm {

typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

template <int N>
struct Int {
  static constexpr int value = N;
};

// LDS written by other lanes of the same wave is read after this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 2^s with m 2^s in [2^14, 2^15) for m > 0 (s at most 126: smaller m stay small), and 2^-s. Of a maximum that is not
// finite 2^-s is infinite, so that what was too small beside it does not come back as zero.
__device__ __forceinline__ float pow2_scale(float m, float& inv) {
  uint32_t e = __builtin_bit_cast(uint32_t, m) & 0x7f800000u;
  e = e < (15u << 23) ? (15u << 23) : e;
  inv = __builtin_bit_cast(float, e) * 0x1p-14f;
  return __builtin_bit_cast(float, (268u << 23) - e);
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

// A chunk's rows as a buffer of just that many bytes: loads past its last row return zero and stores there are
// dropped, with no branch (a predicated load cost its own round trip to memory: the compiler joins the loaded
// value with the zero, and waits for it there), and offsets are 32-bit.
typedef __amdgpu_buffer_rsrc_t Rsrc;
__device__ __forceinline__ Rsrc rows_of(const uint16_t* p, int64_t ld, int len, int dim) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, len > 0 ? ((len - 1) * (int)ld + dim) * 2 : 0, 0x00027000);
}
__device__ __forceinline__ u32x4 row_load16(Rsrc r, int voff, int soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}

// max(m, |x0|, .. |x3|), a NaN if one is: two instructions. (Left to the compiler, which knows what has to pass between a
// matrix instruction and the first reading of its result; for inline assembly it keeps no such distance.)
__device__ __forceinline__ float max4(const f32x4& x, float m) {
#pragma unroll
  for (int e = 0; e < 4; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(x[e]));
  return m;
}
typedef f16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// x0, x1 times sc as pairs of halves, in 5 instructions: the empty asm keeps the compiler from rounding the high
// part a second time on the way to the low one.
__device__ __forceinline__ void split2(float x0, float x1, float sc, uint32_t (&part)[2]) {
  h2 hi = __builtin_convertvector(f32x2{x0 * sc, x1 * sc}, h2);
  asm("" : "+v"(hi));
  const h2 lo = h2{(f16)__builtin_fmaf(x0, sc, -(float)hi[0]), (f16)__builtin_fmaf(x1, sc, -(float)hi[1])};
  part[0] = __builtin_bit_cast(uint32_t, hi);
  part[1] = __builtin_bit_cast(uint32_t, lo);
}
// x0, x1 in bf16 parts.
__device__ __forceinline__ void split2(float x0, float x1, float, uint32_t (&part)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint32_t p = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x0, x1}, b2));
    asm("" : "+v"(p));
    part[i] = p;
    x0 -= __builtin_bit_cast(float, p << 16);
    x1 -= __builtin_bit_cast(float, p & 0xffff0000u);
  }
}
// The parts of a 32-deep operand from two results' registers, scaled.
template <int NT>
__device__ __forceinline__ void split8(const f32x4& x, const f32x4& y, float sc, h8 (&part)[NT]) {
  uint32_t p[4][NT];
  split2(x[0], x[1], sc, p[0]);
  split2(x[2], x[3], sc, p[1]);
  split2(y[0], y[1], sc, p[2]);
  split2(y[2], y[3], sc, p[3]);
#pragma unroll
  for (int i = 0; i < NT; ++i) part[i] = __builtin_bit_cast(h8, u32x4{p[0][i], p[1][i], p[2][i], p[3][i]});
}

// The product of two operands of the rows' type (16 bits of either kind are carried as h8).
template <bool BF>
__device__ __forceinline__ f32x4 mm(h8 a, h8 b, f32x4 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, b2));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, h2));
}
template <bool BF>
constexpr int kParts = BF ? 3 : 2;  // of an fp32 factor beside rows of the type

// v as another lane has it, moved by the register file; 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, true);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// A barrier that waits for this wave's LDS accesses alone. lds_barrier() also waits for its loads into LDS, which
// here are for the next chunk.
__device__ __forceinline__ void step_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef __attribute__((address_space(3))) void* lptr;

}  // namespace dfssm
