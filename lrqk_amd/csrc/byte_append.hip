// Tokens written into a cache held in 8 bits (byte_cache.hpp): of every sequence `count` rows, those that `path` names, go
// behind its `length` tokens.  A block is coded once, when its last token arrives, from all of its rows:
//
//   int8  s = amax / 127 (fp32), c = x / s rounded to the nearest whole number, half to even
//   fp8   s = 2^e, the smallest with amax / s <= 448, c = x / s rounded to the nearest e4m3 number, half to even
//
// s at least 2^-100, amax over the finite elements; an infinity gets the largest code, a NaN 0.  c is x / s rounded once:
// by a power of two the quotient is exact; the int8 one is formed with 1 / s and corrected where it lies next to a border.
#include <algorithm>

#include "byte_cache.hpp"

namespace lrqk {

constexpr int kBaThreads = 256;

struct AppendArgs {
  const void *k_new, *v_new;
  int64_t kb, kh, kr, vb, vh, vr;   // elements between sequences, heads and rows of the new tokens
  const int32_t *lengths, *counts, *path;   // counts, path: or null
  int64_t path_b;
  int32_t* new_lengths;
  void *k, *v;
  float *ks, *vs;
  void *k_tail, *v_tail;
  int blocks, h, t, most, d;
};

// The largest magnitude among sixteen bytes of elements, as bits of an fp32 number: of all, and of the finite ones.
typedef uint16_t ap_u16x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ uint32_t ap_top(const Vec16<T>& v) {
  const uint32_t* w = (const uint32_t*)&v.raw;
  if constexpr (sizeof(T) == 4) {
    return max(max(w[0] & 0x7fffffffu, w[1] & 0x7fffffffu), max(w[2] & 0x7fffffffu, w[3] & 0x7fffffffu));
  } else {   // (of bf16 numbers two at a time)
    ap_u16x2 top = __builtin_bit_cast(ap_u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(ap_u16x2, w[i] & 0x7fff7fffu));
    return (uint32_t)max(top[0], top[1]) << 16;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t ap_finite_top(const Vec16<T>& v) {
  float x[Vec16<T>::N];
  v.unpack(x);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
    top = max(top, u < 0x7f800000u ? u : 0u);
  }
  return top;
}

// Four codes in a word.  odd: there may be infinities and NaN among them.
template <bool FP8>
__device__ __forceinline__ uint32_t ap_codes(float a, float b, float c, float d, float s, float inv, bool odd) {
  float x[4] = {a, b, c, d};
  constexpr float MOST = FP8 ? 448.0f : 127.0f;
  if constexpr (FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= inv;   // exact (or far below the smallest code)
    if (odd) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -MOST), MOST) : 0.0f;
    }
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  } else {
    // added to 1.5 2^23 a number is rounded to a whole one, which is then in the lowest bits
    constexpr float ROUND = 12582912.0f;
    float r[4], near = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = fmaf(x[i], inv, ROUND);
      near = fmaxf(near, fabsf(fmaf(x[i], inv, ROUND - r[i])));
    }
    // x / s and x * inv differ by less than 2^-15, so that a code may be another one next to a half alone
    if (__builtin_expect(near > 0.4999f || odd, 0)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = x[i] == x[i] ? x[i] : 0.0f;
        float q = rintf(y * inv);
        // what is left is exact where it is near half of s (a multiple of half a unit of s, and at most s): so is the decision
        const float left = fmaf(-q, s, y), half = 0.5f * s;
        const bool uneven = (q - 2.0f * floorf(0.5f * q)) != 0.0f;
        if (fabsf(left) > half || (fabsf(left) == half && uneven)) q += copysignf(1.0f, left);
        r[i] = fminf(fmaxf(q, -MOST), MOST) + ROUND;
      }
    }
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(r[3]), __float_as_uint(r[2]), 0x04000c0cu);
    return lo | hi;
  }
}

template <bool FP8>
__device__ __forceinline__ float ap_scale(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  if constexpr (FP8) {
    // top = f 2^e, 1 <= f < 2; 448 = 1.75 2^8.  (A subnormal's e is far below the least scale's.)
    const int e = (int)(top_bits >> 23) - 127 - ((top_bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
    return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
  } else {
    return fmaxf(top / 127.0f, 0x1p-100f);
  }
}

// A workgroup: the keys or the values (blockIdx.z) of a block of a head that the call reaches, and in the first of them what
// goes into the tail.  (That one reads the rows that the tail has of the block before it writes there.)  Bound by memory: a
// prompt of 32K tokens, 8 heads of 128 bf16 elements, 201 MB in 42 us, 4.8 TB/s, what a large copy takes (4.7); a prompt of 4K
// by its launch and by one wave of workgroups that read, wait for their scale and write, 22 MB in 12; few tokens by the chain
// of lengths, rows, scale and codes, 4.3.
template <typename T, bool FP8, int U>
__global__ __launch_bounds__(kBaThreads) void byte_append_kernel(AppendArgs a, int dp) {
  constexpr int N = Vec16<T>::N;
  const int b = (int)blockIdx.y / a.h, h = (int)blockIdx.y % a.h, tid = threadIdx.x;
  const bool values = blockIdx.z != 0;
  const int len = min(max(a.lengths[b], 0), a.blocks * kByBlock);
  const int count = min(a.counts ? min(max(a.counts[b], 0), a.most) : a.most, a.blocks * kByBlock - len), end = len + count;
  if (blockIdx.x == 0 && h == 0 && !values && tid == 0) a.new_lengths[b] = end;
  const int block = len / kByBlock + (int)blockIdx.x;
  const bool whole = (block + 1) * kByBlock <= end;   // (blocks * 64 <= 2^30)
  if (!whole && blockIdx.x != 0) return;
  const int64_t head = (int64_t)b * a.h + h, row_stride = values ? a.vr : a.kr;
  const T* rows_new = values ? (const T*)a.v_new + b * a.vb + h * a.vh : (const T*)a.k_new + b * a.kb + h * a.kh;
  T* tail = (T*)(values ? a.v_tail : a.k_tail) + head * kByTail * a.d;
  const int32_t* path = a.path ? a.path + b * a.path_b : nullptr;
  auto fresh = [&](int token) {   // the new row that a token is
    const int i = token - len;
    return path ? min(max(path[i], 0), a.t - 1) : i;
  };
  const int pieces = a.d / N;
  __shared__ uint32_t turned[256 * 17];   // codes of V: [element][row / 4], a word of four rows
  __shared__ uint32_t tops[kBaThreads / kWave];
  if (whole) {
    Vec16<T> x[U][4];   // sixteen bytes of four successive rows
    int rows[U], piece[U];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int unit = tid + u * kBaThreads;
      rows[u] = unit / pieces;
      piece[u] = unit % pieces;
      if (rows[u] >= kByBlock / 4) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int token = block * kByBlock + 4 * rows[u] + r;
        x[u][r].load((token < len ? tail + (int64_t)(token % kByTail) * a.d : rows_new + fresh(token) * row_stride) + N * piece[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (rows[u] < kByBlock / 4)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = max(top, ap_top(x[u][r]));
    auto all = [&](uint32_t v) {   // over the workgroup; holds barriers
      v = wave_reduce_u32(v, [](uint32_t a, uint32_t b) { return max(a, b); });
      __syncthreads();
      if (lane_id() == 0) tops[wave_id()] = v;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBaThreads / kWave; ++w) v = max(v, tops[w]);
      return v;
    };
    top = all(top);
    const bool odd = top >= 0x7f800000u;
    if (odd) {
      top = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (rows[u] < kByBlock / 4)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = max(top, ap_finite_top(x[u][r]));
      top = all(top);
    }
    const float s = ap_scale<FP8>(top), inv = 1.0f / s;
    const int64_t at = head * a.blocks + block;
    if (tid == 0) (values ? a.vs : a.ks)[at] = s;
    char* codes = (char*)(values ? a.v : a.k) + at * kByBlock * dp;
    if (!values) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (rows[u] >= kByBlock / 4) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float y[N];
          x[u][r].unpack(y);
          uint32_t w[N / 4];
#pragma unroll
          for (int e = 0; e < N / 4; ++e) w[e] = ap_codes<FP8>(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3], s, inv, odd);
          char* to = codes + (4 * rows[u] + r) * dp + N * piece[u];
          if constexpr (N == 8)
            *(uint2*)to = make_uint2(w[0], w[1]);
          else
            *(uint32_t*)to = w[0];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (rows[u] >= kByBlock / 4) continue;
        float y[4][N];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[u][r].unpack(y[r]);
#pragma unroll
        for (int e = 0; e < N; ++e) turned[(N * piece[u] + e) * 17 + rows[u]] = ap_codes<FP8>(y[0][e], y[1][e], y[2][e], y[3][e], s, inv, odd);
      }
      __syncthreads();
      for (int i = tid; i < a.d * 4; i += kBaThreads) {
        const uint32_t* from = turned + (i / 4) * 17 + 4 * (i % 4);
        *(uint4*)(codes + 16 * i) = make_uint4(from[0], from[1], from[2], from[3]);
      }
    }
  }
  if (blockIdx.x == 0) {
    // (every row of the tail that the block wanted has been read: the barriers above)
    const int first = max(len, end - kByTail);
    for (int i = tid; i < (end - first) * pieces; i += kBaThreads) {
      const int token = first + i / pieces;
      Vec16<T> y;
      y.load(rows_new + fresh(token) * row_stride + N * (i % pieces));
      y.store(tail + (int64_t)(token % kByTail) * a.d + N * (i % pieces));
    }
  }
}

template <typename T, bool FP8>
static int append_launch(const AppendArgs& a, int b, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(((int64_t)a.most + kByBlock - 1) / kByBlock + 1, a.blocks), (unsigned)(b * a.h), 2);
  LRQK_REQUIRE((int64_t)grid.x * kBaThreads <= kMaxThreads, LRQK_ELIMIT, "%d tokens are more than a launch has places for", a.most);
  const int units = a.d / Vec16<T>::N * (kByBlock / 4), dp = by_width(a.d);
  if (units <= kBaThreads) hipLaunchKernelGGL((byte_append_kernel<T, FP8, 1>), grid, dim3(kBaThreads), 0, st, a, dp);
  else if (units <= 2 * kBaThreads) hipLaunchKernelGGL((byte_append_kernel<T, FP8, 2>), grid, dim3(kBaThreads), 0, st, a, dp);
  else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((byte_append_kernel<T, FP8, 4>), grid, dim3(kBaThreads), 0, st, a, dp);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}

}  // namespace lrqk

using namespace lrqk;

extern "C" int lrqk_byte_append(const void* k_new, const void* v_new, const int64_t* strides, int t, int most, const int32_t* lengths,
                                const int32_t* counts, const int32_t* path, int64_t path_stride, int32_t* new_lengths, void* k,
                                void* v, float* k_scale, float* v_scale, void* k_tail, void* v_tail, int64_t blocks, int b, int h,
                                int d, int kind, int dtype, void* stream) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(kind == LRQK_CODE_INT8 || kind == LRQK_CODE_FP8, LRQK_EINVAL, "kind=%d", kind);
  LRQK_REQUIRE(b > 0 && h > 0 && t > 0 && most > 0 && blocks > 0 && d > 0, LRQK_EINVAL, "bad sizes b=%d h=%d t=%d most=%d blocks=%lld d=%d",
               b, h, t, most, (long long)blocks, d);
  LRQK_REQUIRE(path || most <= t, LRQK_EINVAL, "%d of %d rows", most, t);
  LRQK_REQUIRE(d * (int)elem_size(dtype) % 16 == 0 && d <= 256, LRQK_ELIMIT,
               "head_dim %d unsupported (rows of whole 16-byte pieces, at most 256 elements)", d);
  LRQK_REQUIRE(blocks <= (1 << 24) && (int64_t)b * h <= 65535, LRQK_ELIMIT, "blocks=%lld (at most 2^24), b * h=%lld (65535)",
               (long long)blocks, (long long)b * h);
  LRQK_REQUIRE(k_new && v_new && strides && lengths && new_lengths && k && v && k_scale && v_scale && k_tail && v_tail, LRQK_EINVAL, "null pointer");
  const int vec = 16 / (int)elem_size(dtype);
  bool aligned = (uintptr_t)k_new % 16 == 0 && (uintptr_t)v_new % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 &&
                 (uintptr_t)k_tail % 16 == 0 && (uintptr_t)v_tail % 16 == 0;
  for (int i = 0; i < 6; ++i) aligned = aligned && strides[i] % vec == 0;
  LRQK_REQUIRE(aligned, LRQK_EINVAL, "pointers and rows must be 16-byte aligned");
  const AppendArgs a{k_new, v_new, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], lengths, counts, path, path_stride,
                     new_lengths, k, v, k_scale, v_scale, k_tail, v_tail, (int)blocks, h, t, most, d};
  hipStream_t st = (hipStream_t)stream;
  const bool fp8 = kind == LRQK_CODE_FP8;
  if (dtype == LRQK_F32) return fp8 ? append_launch<float, true>(a, b, st) : append_launch<float, false>(a, b, st);
  return fp8 ? append_launch<bf16_t, true>(a, b, st) : append_launch<bf16_t, false>(a, b, st);
}
