// Products of queries and cached keys on the matrix cores, 16 queries by 16 keys at a time, shared by the attention of a
// tree of drafted tokens and the sums of attention weights.
//
// C = A B of a 16 x 16 tile: lane l holds column l % 16, rows 4 (l / 16) .. + 3.  Rows of A and columns of B are given by
// lane l % 16, and lane group l / 16 (a "quad") gives part of what is summed over.  What is summed over may come in any
// order, as long as both sides have the same: here a quad takes 16 bytes of every 64 of a row, so that one load of a wave
// covers 64 contiguous bytes of 16 rows, of bf16 (8 elements, one 16x16x32 product) and of fp32 (4 elements, four 16x16x4
// products, exact fp32) alike.
#pragma once
#include "common.hpp"

namespace lrqk {

typedef float ar_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 ar_bf8 __attribute__((ext_vector_type(8)));
typedef uint32_t ar_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t ar_u2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// One 64-byte step of the sum over a row: c += a b.
template <typename T>
__device__ __forceinline__ ar_f4 ar_step(ar_u4 a, ar_u4 b, ar_f4 c);
template <>
__device__ __forceinline__ ar_f4 ar_step<bf16_t>(ar_u4 a, ar_u4 b, ar_f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ar_bf8, a), __builtin_bit_cast(ar_bf8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ ar_f4 ar_step<float>(ar_u4 a, ar_u4 b, ar_f4 c) {
  const ar_f4 x = __builtin_bit_cast(ar_f4, a), y = __builtin_bit_cast(ar_f4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
  return c;
}

// A row as the operand of those steps: STEPS pieces of 16 bytes, piece 4 s + quad in step s.  `pieces`: of the row; what is
// beyond them (heads of a width between two of the kernels') is zero.
template <int STEPS>
__device__ __forceinline__ void ar_row(const void* row, int quad, int pieces, ar_u4 (&x)[STEPS]) {
  const ar_u4* p = (const ar_u4*)row;
  if (pieces == 4 * STEPS) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) x[s] = p[4 * s + quad];
  } else {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const ar_u4 v = p[min(4 * s + quad, pieces - 1)];
      x[s] = 4 * s + quad < pieces ? v : ar_u4{0, 0, 0, 0};
    }
  }
}

// Rows on their way from memory to those operands.  Read as operands they would be 64 accesses of 16 bytes per load (the
// cache joins what adjacent lanes read, and those have different rows: a whole prompt's weights were bound by that, at a
// third of the speed), so a wave reads whole rows, passes them through LDS and takes the operands from there.  Pieces
// change places within their row so that the 16 rows of an operand come from 16 different banks.
template <int CH>   // 16-byte pieces of a row: a power of two from 4 to 64
__device__ __forceinline__ int ar_place(int row, int piece) {
  constexpr int SH = CH >= 16 ? 0 : CH == 8 ? 1 : 2, MASK = CH >= 16 ? 15 : CH - 1;
  return row * CH + (piece ^ ((row >> SH) & MASK));
}

__device__ __forceinline__ void ar_wave_sync() {  // orders one wave's LDS writes and reads
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Over the four quads of a wave (lanes l, l + 16, l + 32, l + 48), result in all of them.
__device__ __forceinline__ float ar_quad_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float ar_quad_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

__device__ __forceinline__ float ar_exp2(float x) { return __builtin_amdgcn_exp2f(x); }  // (what is below 2^-126 counts as 0)

}  // namespace lrqk
