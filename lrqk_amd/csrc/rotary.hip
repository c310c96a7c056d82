// Rotary positions: every pair (a, b) of a head's first rotary_dim elements turned by the angle position * frequency,
//
//   a' = f (a cos - b sin),  b' = f (b cos + a sin)
//
// with f the factor of the results.  Pairs are elements i and i + rotary_dim / 2, or 2 i and 2 i + 1 (interleaved); the
// rest of the head is copied.  The transpose turns back (times f): the gradient of the turn.
//
// The angle's turns are formed and reduced in fp64 (at position 131071 an fp32 angle is 4e-3 off), its sine and cosine in
// fp32; the turn is fp32, rounded once.  Bound by HBM: every element is read and written once.  A workgroup forms the
// sines and cosines of a tile of tokens once, into LDS, and turns all heads of those tokens with them: one sine per 40
// pairs of a prompt with 32 + 8 heads.
//
// 32768 tokens of 32 + 8 heads of 128 bf16 elements, from the projections' layout into the heads': 671 MB in 133 to 136 us,
// 4.9 TB/s, what a large copy reaches.  One token: 4 us, a launch.
#include <math.h>

#include <algorithm>

#include "common.hpp"

namespace lrqk {

constexpr int kRotThreads = 256;
constexpr int kRotMaxHalf = 128;     // pairs of a head
constexpr double kTwoPi = 6.283185307179586476925286766559;

struct RotTensor {
  const void* in;
  void* out;
  int64_t ib, ih, is, ob, oh, os;  // elements between sequences, heads, tokens
  int heads;
};
struct RotArgs {
  RotTensor t[2];
  const int32_t* pos;   // or null: first + token
  int64_t pos_stride;   // between sequences (0: all have the same)
  int32_t first;
  const double* freq;
  float factor;
  int64_t s;
  int half, rest;       // pairs, elements behind them
  int groups;           // of heads
  int tokens;           // of a workgroup
  bool interleaved, transpose;
};

// V elements (V = 1: one, or a pair side by side) that a thread moves at a time
template <typename T, int V>
struct RotVec {
  float f[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      f[0] = ld_f32(p, 0);
    } else {
      Vec16<T> v;
      v.load(p);
      v.unpack(f);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      st_f32(p, 0, f[0]);
    } else {
      Vec16<T> v;
      v.pack(f);
      v.store(p);
    }
  }
};

template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a, int sub_log2) {
  extern __shared__ float2 cs[];  // [tokens][half]
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.s - t0);
  const int64_t b = blockIdx.z;
  for (int e = threadIdx.x; e < tokens * a.half; e += kRotThreads) {
    const int t = e / a.half, i = e - t * a.half;
    const int64_t p = a.pos ? (int64_t)a.pos[b * a.pos_stride + t0 + t] : (int64_t)a.first + t0 + t;
    const double turns = (double)p * a.freq[i] * (1.0 / kTwoPi);
    float sn, cn;
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cn);
    cs[e] = make_float2(cn * a.factor, (a.transpose ? -sn : sn) * a.factor);
  }
  __syncthreads();
  // A row (one head of one token) is the work of 2^sub_log2 adjacent threads, a piece each; the workgroup's rows are its
  // heads, token by token, kept apart over its row groups.
  const int all = a.t[0].heads + a.t[1].heads;
  const int per = (all + a.groups - 1) / a.groups;
  const int h0 = (int)blockIdx.y * per, nh = min(per, all - h0);
  if (nh <= 0) return;
  const int turn = INTERLEAVED && V > 1 ? 2 * a.half / V : a.half / V;  // pieces that turn
  const int pieces = turn + a.rest / V;
  const int rpp = kRotThreads >> sub_log2, sub = threadIdx.x & ((1 << sub_log2) - 1);
  const int rows = tokens * nh;
  constexpr int U = 4;
  for (int piece = sub; piece < pieces; piece += 1 << sub_log2) {
    const bool turns = piece < turn;
    // elements of the piece, and of its partner
    const int e0 = !turns ? 2 * a.half + (piece - turn) * V : INTERLEAVED && V == 1 ? 2 * piece : piece * V;
    const int e1 = !turns ? e0 : INTERLEAVED ? e0 + (V == 1 ? 1 : 0) : e0 + a.half;
    constexpr bool TWO = !INTERLEAVED || V == 1;
    for (int r0 = threadIdx.x >> sub_log2; r0 < rows; r0 += U * rpp) {
      RotVec<T, V> x[U], y[U];
      T* out[U];
      int tok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = min(r0 + u * rpp, rows - 1);
        tok[u] = row / nh;
        const int h = h0 + row - tok[u] * nh;
        const bool second = h >= a.t[0].heads;
        const RotTensor& w = second ? a.t[1] : a.t[0];
        const int64_t head = second ? h - a.t[0].heads : h;
        const T* in = (const T*)w.in + b * w.ib + head * w.ih + (t0 + tok[u]) * w.is;
        out[u] = (T*)w.out + b * w.ob + head * w.oh + (t0 + tok[u]) * w.os;
        x[u].load(in + e0);
        if (TWO) y[u].load(in + e1);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * rpp >= rows) break;
        if (turns) {
          if constexpr (TWO) {
            const float2* c = cs + tok[u] * a.half + (INTERLEAVED ? piece : piece * V);
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const float p = x[u].f[v], q = y[u].f[v];
              x[u].f[v] = p * c[v].x - q * c[v].y;
              y[u].f[v] = q * c[v].x + p * c[v].y;
            }
          } else {
            const float2* c = cs + tok[u] * a.half + piece * (V / 2);
#pragma unroll
            for (int v = 0; v < V; v += 2) {
              const float p = x[u].f[v], q = x[u].f[v + 1];
              x[u].f[v] = p * c[v / 2].x - q * c[v / 2].y;
              x[u].f[v + 1] = q * c[v / 2].x + p * c[v / 2].y;
            }
          }
        }
        x[u].store(out[u] + e0);
        if (TWO && turns) y[u].store(out[u] + e1);
      }
    }
  }
}

template <typename T>
static int rotary_launch(const RotArgs& a, int b, bool vec, hipStream_t st) {
  constexpr int VEC = Vec16<T>::N;
  const int V = vec ? VEC : 1;
  const int pieces = (a.interleaved && vec ? 2 * a.half / V : a.half / V) + a.rest / V;
  int lg = 0;
  while ((1 << lg) < pieces && (1 << lg) < kRotThreads) ++lg;
  const int64_t tiles = (a.s + a.tokens - 1) / a.tokens;
  const dim3 grid((unsigned)tiles, (unsigned)a.groups, (unsigned)b);
  const size_t lds = sizeof(float2) * a.tokens * (size_t)std::max(a.half, 1);
  if (a.interleaved) {
    if (vec)
      hipLaunchKernelGGL((rotary_kernel<T, VEC, true>), grid, dim3(kRotThreads), lds, st, a, lg);
    else
      hipLaunchKernelGGL((rotary_kernel<T, 1, true>), grid, dim3(kRotThreads), lds, st, a, lg);
  } else {
    if (vec)
      hipLaunchKernelGGL((rotary_kernel<T, VEC, false>), grid, dim3(kRotThreads), lds, st, a, lg);
    else
      hipLaunchKernelGGL((rotary_kernel<T, 1, false>), grid, dim3(kRotThreads), lds, st, a, lg);
  }
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}

}  // namespace lrqk

using namespace lrqk;

extern "C" int lrqk_rotary_frequencies(int rotary_dim, double theta, int scaling, double factor, double p0, double p1,
                                       double original_context, double* freq, double* result_factor) {
  LRQK_REQUIRE(freq && result_factor, LRQK_EINVAL, "null pointer");
  LRQK_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= 2 * kRotMaxHalf, LRQK_EINVAL,
               "rotary_dim=%d: an even number of elements from 2 to %d", rotary_dim, 2 * kRotMaxHalf);
  LRQK_REQUIRE(theta > 1.0 && isfinite(theta), LRQK_EINVAL, "theta=%g has to be finite and above 1", theta);
  LRQK_REQUIRE(scaling >= LRQK_ROPE_PLAIN && scaling <= LRQK_ROPE_YARN, LRQK_EINVAL, "scaling=%d", scaling);
  LRQK_REQUIRE(scaling == LRQK_ROPE_PLAIN || (factor >= 1.0 && isfinite(factor)), LRQK_EINVAL,
               "factor=%g has to be finite and at least 1", factor);
  const int half = rotary_dim / 2;
  *result_factor = 1.0;
  double low = 0.0, high = 0.0;
  if (scaling == LRQK_ROPE_NTK) {
    LRQK_REQUIRE(rotary_dim > 2, LRQK_EINVAL, "rotary_dim=2 has no base to stretch");
    theta *= pow(factor, (double)rotary_dim / (rotary_dim - 2));
  } else if (scaling == LRQK_ROPE_LLAMA3) {
    LRQK_REQUIRE(original_context > 0.0 && isfinite(original_context) && p0 > 0.0 && p1 > p0 && isfinite(p1), LRQK_EINVAL,
                 "needs 0 < low_freq_factor=%g < high_freq_factor=%g and original_context=%g > 0", p0, p1, original_context);
  } else if (scaling == LRQK_ROPE_YARN) {
    LRQK_REQUIRE(original_context > 0.0 && isfinite(original_context) && p1 > 0.0 && p0 > p1 && isfinite(p0), LRQK_EINVAL,
                 "needs beta_fast=%g > beta_slow=%g > 0 and original_context=%g > 0", p0, p1, original_context);
    // the pairs that make beta_fast and beta_slow turns over the original context: theta^(-2 i / dim) L = 2 pi beta
    const double scale = rotary_dim / (2.0 * log(theta));
    low = fmax(floor(scale * log(original_context / (kTwoPi * p0))), 0.0);
    high = fmin(ceil(scale * log(original_context / (kTwoPi * p1))), rotary_dim - 1.0);
    *result_factor = 0.1 * log(factor) + 1.0;
  }
  for (int i = 0; i < half; ++i) {
    double f = pow(theta, -2.0 * i / rotary_dim);
    if (scaling == LRQK_ROPE_LINEAR) {
      f /= factor;
    } else if (scaling == LRQK_ROPE_LLAMA3) {
      const double turns = original_context * f / kTwoPi;  // over the original context
      const double keep = fmin(fmax((turns - p0) / (p1 - p0), 0.0), 1.0);
      f *= keep + (1.0 - keep) / factor;
    } else if (scaling == LRQK_ROPE_YARN) {
      const double ramp = fmin(fmax((i - low) / fmax(high - low, 1e-3), 0.0), 1.0);
      f *= 1.0 - ramp + ramp / factor;
    }
    freq[i] = f;
  }
  return LRQK_OK;
}

extern "C" int lrqk_rotary(const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides,
                           const int32_t* positions, int64_t pos_stride, int32_t first, const double* freq, double factor,
                           int b, int hq, int hk, int64_t s, int d, int rotary_dim, int interleaved, int transpose, int dtype,
                           void* stream) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(b > 0 && b <= 65535 && hq > 0 && hk >= 0 && s >= 0 && d > 0, LRQK_EINVAL, "bad sizes b=%d hq=%d hk=%d s=%lld d=%d",
               b, hq, hk, (long long)s, d);
  LRQK_REQUIRE(hq <= 65535 && hk <= 65535 && s <= INT32_MAX, LRQK_ELIMIT, "hq=%d hk=%d s=%lld", hq, hk, (long long)s);
  LRQK_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= d && rotary_dim <= 2 * kRotMaxHalf, LRQK_EINVAL,
               "rotary_dim=%d: an even number of elements up to the head's %d and %d", rotary_dim, d, 2 * kRotMaxHalf);
  LRQK_REQUIRE(q && q_out && strides && freq && (hk == 0 || (k && k_out)), LRQK_EINVAL, "null pointer");
  if (s == 0) return LRQK_OK;
  RotArgs a{};
  const int vec = 16 / (int)elem_size(dtype);
  bool vok = d % vec == 0 && rotary_dim % vec == 0 && (interleaved || (rotary_dim / 2) % vec == 0);
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  for (int i = 0; i < (hk > 0 ? 2 : 1); ++i) {
    const int64_t* w = strides + 6 * i;
    a.t[i] = RotTensor{in[i], out[i], w[0], w[1], w[2], w[3], w[4], w[5], i ? hk : hq};
    vok = vok && (uintptr_t)in[i] % 16 == 0 && (uintptr_t)out[i] % 16 == 0;
    for (int j = 0; j < 6; ++j) vok = vok && w[j] % vec == 0;
  }
  a.pos = positions;
  a.pos_stride = pos_stride;
  a.first = first;
  a.freq = freq;
  a.factor = (float)factor;
  a.s = s;
  a.half = rotary_dim / 2;
  a.rest = d - rotary_dim;
  a.interleaved = interleaved != 0;
  a.transpose = transpose != 0;
  // as many groups of heads as give the launch a thousand workgroups, four heads each at least
  // Tiles of up to 40 KB, 64 tokens and 32 KB of sines and cosines.  (32K tokens of 32 + 8 heads of 128 bf16 elements: 2 tokens
  // 129 us, 4 133, 16 158; 128K of 8 heads: 4 tokens 179, 16 109, 64 134; 256K of one: 4 tokens 124, 64 52; 8K of 28 + 4 fp32:
  // 2 tokens 41, 4 47; 8K of 128 heads: 1 token 103, 4 114.)
  const int64_t bytes = (int64_t)(hq + hk) * d * elem_size(dtype);
  a.tokens = 64;
  while (a.tokens > 1 && (a.tokens * bytes > 40 * 1024 || a.tokens * a.half > 4096)) a.tokens /= 2;
  const int64_t tiles = (s + a.tokens - 1) / a.tokens;
  LRQK_REQUIRE(tiles <= kMaxThreads / kRotThreads, LRQK_ELIMIT, "%lld tokens are more than a launch has places for", (long long)s);
  a.groups = (int)std::max<int64_t>(1, std::min<int64_t>((hq + hk + 3) / 4, 1024 / (tiles * b)));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LRQK_F32) return rotary_launch<float>(a, b, vok, st);
  return rotary_launch<bf16_t>(a, b, vok, st);
}
