// The attention that every cached token got from the last t tokens of its sequence,
//
//   out_j = weights_j + sum over the query heads that read j's head, sum over the queries i that see j, exp(scale q_i.k_j - lse_i),
//
// query i being token length - t + i, which sees the tokens up to itself.  The attention itself leaves lse (lse_i = log of
// the sum of exp(scale q_i.k_j)); where the caller does not have it, a first pass over the keys forms it.
//
//   rows     lse: a wave has 16 MT queries and walks over the keys they see; S^T = K Q^T, so that a lane has a maximum and
//            a sum of its own for its query and meets the other lanes at the end only.  Few queries: the keys are split
//            and `merge` joins the parts.
//   columns  sums: a wave has 16 NT keys in registers and walks over the queries that see them, S = Q K^T, so that a
//            lane's sums are those of its keys.  Every sum is one workgroup's: no atomics, the same bits every time.
//
// A prompt is bound by the products and, as much, by the exponentials of both passes; a few queries over a long cache by
// the reading of the keys.
#include <algorithm>

#include "attn_rows.hpp"

namespace lrqk {

constexpr int kAwWaves = 4, kAwThreads = kAwWaves * kWave;
constexpr float kAwNone = -3.0e38f;    // maximum of no scores
constexpr float kAwSlack = 8.0f;        // a maximum may be exceeded by 2^8 before a sum is rescaled to the new one

struct WeightArgs {
  const void *q, *k;
  const int32_t* lengths;
  const float* lse;        // natural logarithms of the caller's, or those of base 2 of the first pass
  float lse_scale;         // what makes them base 2
  float* lse2;             // first pass: [b][hq][t]
  float* part;             // first pass: [b][hq][t][parts][2]; second pass: [chunks][b][hc][n]
  const float* weights;    // or null
  float* out;
  int64_t kv_b, kv_h, kv_r;
  int n, hq, hc, t, d, parts, groups, chunks;
  uint32_t heads;           // of the cache, of all sequences
  float scale_log2e;
};

__device__ __forceinline__ int weights_len(const WeightArgs& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.n) : a.n; }

// Item (head, part, group of 16 MT rows) of a wave: its queries' maximum and sum over its part of the keys.
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kAwThreads) void weights_rows_kernel(WeightArgs a) {
  constexpr int STEPS = DP * (int)sizeof(T) / 64, NU = 2, KT = 16 * NU;
  const int lane = lane_id(), col = lane & 15, quad = lane >> 4;
  // (the heads of a place follow each other: with 8 of them, or a divisor, a head's workgroups are on one XCD, whose L2 holds
  // its keys)
  const int item = (int)(blockIdx.x / a.heads) * kAwWaves + __builtin_amdgcn_readfirstlane(wave_id());
  const int head = (int)(blockIdx.x % a.heads), b = head / a.hc, hc = head % a.hc;
  if (item >= a.groups * a.parts) return;
  const int part = item % a.parts, group = a.groups - 1 - item / a.parts;   // (the longest walks first)
  const int gc = a.hq / a.hc, M = gc * a.t, row0 = group * 16 * MT;
  const int len = weights_len(a, b), behind = len - a.t;   // query i sees the keys up to behind + i
  const T* q = (const T*)a.q + ((int64_t)b * a.hq + (int64_t)hc * gc) * a.t * a.d;
  const T* k = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
  const int pieces = a.d * (int)sizeof(T) / 16;
  ar_u4 qf[MT][STEPS];
  int last[MT];   // last key that the lane's query sees
  int most = -1, least = a.n;
  float top[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(row0 + 16 * m + col, M - 1);
    last[m] = behind + row % a.t;
    most = max(most, last[m]);
    least = min(least, last[m]);
    ar_row(q + (int64_t)row * a.d, quad, pieces, qf[m]);
    top[m] = kAwNone;
    sum[m] = 0.0f;
  }
  most = (int)wave_reduce_u32((uint32_t)(most + 1), [](uint32_t x, uint32_t y) { return max(x, y); });   // keys to walk over
  least = (int)(wave_reduce_u32((uint32_t)least ^ 0x80000000u, [](uint32_t x, uint32_t y) { return min(x, y); }) ^ 0x80000000u);
  const int tiles = (most + KT - 1) / KT, per = (tiles + a.parts - 1) / a.parts;
  const int end = min(tiles, (part + 1) * per);
  ar_u4 kf[NU][STEPS];
  auto load = [&](int tile) {
#pragma unroll
    for (int u = 0; u < NU; ++u) ar_row(k + (int64_t)min(tile * KT + 16 * u + col, most - 1) * a.kv_r, quad, pieces, kf[u]);
  };
  if (part * per < end) load(part * per);
  for (int tile = part * per; tile < end; ++tile) {
    const int first = tile * KT;
    const bool whole = first + KT - 1 <= least;
    float x[MT][4 * NU];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        ar_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) s = ar_step<T>(kf[u][c], qf[m][c], s);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[m][4 * u + r] = s[r];
      }
    load(min(tile + 1, end - 1));   // (while the exponentials of this one are formed)
    if (!whole) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4 * NU; ++e) x[m][e] = first + 16 * (e >> 2) + 4 * quad + (e & 3) <= last[m] ? x[m][e] : -INFINITY;
    }
    float high[MT];
    bool more = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      high[m] = x[m][0];
#pragma unroll
      for (int e = 1; e < 4 * NU; ++e) high[m] = fmaxf(high[m], x[m][e]);
      high[m] *= a.scale_log2e;
      more = more | (high[m] > top[m] + kAwSlack);
    }
    if (__ballot(more)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float now = fmaxf(top[m], high[m]);
        sum[m] *= ar_exp2(top[m] - now);
        top[m] = now;
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 4 * NU; ++e) sum[m] += ar_exp2(fmaf(x[m][e], a.scale_log2e, -top[m]));
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const float all = ar_quad_max(top[m]);
    const float total = ar_quad_sum(sum[m] * ar_exp2(top[m] - all));
    const int row = row0 + 16 * m + col;
    if (quad != 0 || row >= M) continue;
    const int64_t at = (int64_t)head * M + row;
    if (a.parts == 1) {
      a.lse2[at] = total == 0.0f ? -INFINITY : all + log2f(total);
    } else {
      a.part[(at * a.parts + part) * 2] = all;
      a.part[(at * a.parts + part) * 2 + 1] = total;
    }
  }
}

// One wave a row.
__global__ __launch_bounds__(kAwThreads) void weights_merge_kernel(WeightArgs a, int64_t rows) {
  const int64_t row = (int64_t)blockIdx.x * kAwWaves + wave_id();
  if (row >= rows) return;
  const float* p = a.part + row * a.parts * 2;
  float top = kAwNone;
  for (int i = lane_id(); i < a.parts; i += kWave) top = fmaxf(top, p[2 * i]);
  top = wave_max(top);
  float sum = 0.0f;
  for (int i = lane_id(); i < a.parts; i += kWave) sum += p[2 * i + 1] * ar_exp2(p[2 * i] - top);
  sum = wave_sum(sum);
  if (lane_id() == 0) a.lse2[row] = sum == 0.0f ? -INFINITY : top + log2f(sum);
}

// 16 NT keys a wave; the waves of a workgroup walk over the same queries, a chunk of them, so that the L1 has what the
// others read.
template <typename T, int DP, int NT>
__global__ __launch_bounds__(kAwThreads) void weights_columns_kernel(WeightArgs a) {
  constexpr int STEPS = DP * (int)sizeof(T) / 64, KEYS = 16 * NT;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  const int head = (int)(blockIdx.x % a.heads), b = head / a.hc, hc = head % a.hc, place = (int)(blockIdx.x / a.heads);
  const int chunk = place % a.chunks, first = (place / a.chunks * kAwWaves + wave) * KEYS;   // (the most queries first)
  if (first >= a.n) return;
  const int gc = a.hq / a.hc, M = gc * a.t;
  const int len = weights_len(a, b), behind = len - a.t;
  const T* q = (const T*)a.q + ((int64_t)b * a.hq + (int64_t)hc * gc) * a.t * a.d;
  const T* k = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
  const float* lse = a.lse + (int64_t)head * M;
  const int pieces = a.d * (int)sizeof(T) / 16;
  const int64_t row = (int64_t)head * a.n + first;
  float had[NT], sum[NT], part[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    sum[j] = part[j] = 0.0f;
    had[j] = a.weights && a.chunks == 1 ? a.weights[row + min(16 * j + col, a.n - 1 - first)] : 0.0f;
  }
  if (first < len) {
    ar_u4 kf[NT][STEPS];
#pragma unroll
    for (int j = 0; j < NT; ++j) ar_row(k + (int64_t)min(first + 16 * j + col, len - 1) * a.kv_r, quad, pieces, kf[j]);
    // tiles of 16 queries: of one query head each, from the first that sees a key of the wave; or, of few queries, of all
    const bool packed = a.t < 16;
    const int t0 = packed ? 0 : max(0, first - behind) / 16;
    const int per = packed ? 1 : (a.t + 15) / 16 - t0;
    const int items = packed ? (M + 15) / 16 : gc * per;
    const int begin = (int)((int64_t)items * chunk / a.chunks), end = (int)((int64_t)items * (chunk + 1) / a.chunks);
    ar_u4 qf[STEPS];
    float l2[4];
    auto load = [&](int g, int tt) {   // rows of the tile: base .. min(base + 16, stop) - 1
      const int base = g * a.t + 16 * tt, stop = packed ? M : (g + 1) * a.t;
      ar_row(q + (int64_t)min(base + col, stop - 1) * a.d, quad, pieces, qf);
#pragma unroll
      for (int r = 0; r < 4; ++r) l2[r] = lse[min(base + 4 * quad + r, stop - 1)];
    };
    int g = packed ? 0 : begin / per, tt = packed ? begin : t0 + begin % per, held = 0;
    if (begin < end) load(g, tt);
    for (int item = begin; item < end; ++item) {
      const int base = g * a.t + 16 * tt, stop = packed ? M : (g + 1) * a.t, at = packed ? 0 : 16 * tt;
      ar_f4 s[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        s[j] = ar_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) s[j] = ar_step<T>(qf[c], kf[j][c], s[j]);
      }
      float l[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        l[r] = l2[r] * a.lse_scale;
        l[r] = l[r] == -INFINITY ? INFINITY : l[r];   // (a query that saw nothing gives nothing)
      }
      if (item + 1 < end) {   // (the next queries, while the exponentials of these are formed)
        if (!packed && tt + 1 == t0 + per) {
          ++g;
          tt = t0;
        } else {
          ++tt;
        }
        load(g, tt);
      }
      const bool whole = base + 16 <= stop && first + KEYS - 1 <= behind + at;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = ar_exp2(fmaf(s[j][r], a.scale_log2e, -l[r]));
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = base + 4 * quad + r, last = behind + (packed ? row % a.t : at + 4 * quad + r);
            const bool sees = (row < stop) & (first + 16 * j + col <= last);
            p[r] = sees ? p[r] : 0.0f;
          }
        }
        part[j] += (p[0] + p[1]) + (p[2] + p[3]);
      }
      if (++held == 32) {   // (sums of sums: thousands of addends to one fp32 number would lose its last bits)
        held = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          sum[j] += part[j];
          part[j] = 0.0f;
        }
      }
    }
  }
  float* out = a.chunks == 1 ? a.out + row : a.part + (int64_t)chunk * a.heads * a.n + row;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    sum[j] = ar_quad_sum(sum[j] + part[j]);
    if (quad == 0 && first + 16 * j + col < a.n) out[16 * j + col] = had[j] + sum[j];
  }
}

// out = weights + the chunks' sums, in their order.
__global__ __launch_bounds__(kAwThreads) void weights_sum_kernel(WeightArgs a, int64_t count) {
  const int64_t i = (int64_t)blockIdx.x * kAwThreads + threadIdx.x;
  if (i >= count) return;
  float v = 0.0f;
#pragma unroll 8
  for (int c = 0; c < a.chunks; ++c) v += a.part[c * count + i];
  a.out[i] = a.weights ? a.weights[i] + v : v;
}

struct WeightPlan {
  int dp, mt, groups, parts, nt, chunks;
  int64_t lse2, part;   // floats
};
static WeightPlan weights_plan(int b, int hq, int hc, int t, int64_t n, int d, int dtype, bool have_lse) {
  WeightPlan p{};
  p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t M = (int64_t)(hq / hc) * t, heads = (int64_t)b * hc;
  const int row = p.dp * (int)elem_size(dtype);
  p.nt = row <= 256 ? 4 : row <= 512 ? 2 : 1;
  // two thousand workgroups of keys and chunks of queries (half of a prompt's have little to do), sixteen tiles of queries
  // for each
  const int64_t blocks = (n + 16 * p.nt * kAwWaves - 1) / (16 * p.nt * kAwWaves), items = (M + 15) / 16;
  p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(2048 / (blocks * heads), items / 16));
  if (p.chunks > 1) p.part = heads * n * p.chunks;
  if (have_lse) return p;
  p.mt = M <= 16 || (p.dp == 256 && dtype == LRQK_F32) ? 1 : M <= 32 || p.dp == 256 || (p.dp == 128 && dtype == LRQK_F32) ? 2 : 4;
  p.groups = (int)((M + 16 * p.mt - 1) / (16 * p.mt));
  // two waves per SIMD, each with eight tiles of 32 keys at least
  int64_t parts = std::max<int64_t>(1, 2048 / (heads * p.groups));
  parts = std::min<int64_t>(parts, (n + 255) / 256);
  p.parts = (int)std::max<int64_t>(1, parts);
  p.lse2 = heads * M;
  if (p.parts > 1) p.part = std::max(p.part, heads * M * p.parts * 2);   // (the passes follow each other)
  return p;
}

template <typename T, int DP>
static int weights_rows_launch(const WeightArgs& a, const WeightPlan& p, int heads, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)p.groups * p.parts + kAwWaves - 1) / kAwWaves * heads));
  constexpr int MOST = DP * (int)sizeof(T) <= 256 ? 4 : DP * (int)sizeof(T) <= 512 ? 2 : 1;
  if constexpr (MOST >= 4)
    if (p.mt == 4) hipLaunchKernelGGL((weights_rows_kernel<T, DP, 4>), grid, dim3(kAwThreads), 0, st, a);
  if constexpr (MOST >= 2)
    if (p.mt == 2) hipLaunchKernelGGL((weights_rows_kernel<T, DP, 2>), grid, dim3(kAwThreads), 0, st, a);
  if (p.mt == 1) hipLaunchKernelGGL((weights_rows_kernel<T, DP, 1>), grid, dim3(kAwThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  if (p.parts > 1) {
    const int64_t rows = p.lse2;
    hipLaunchKernelGGL(weights_merge_kernel, dim3((unsigned)((rows + kAwWaves - 1) / kAwWaves)), dim3(kAwThreads), 0, st, a, rows);
    LRQK_HIP_CHECK(hipGetLastError());
  }
  return LRQK_OK;
}
template <typename T, int DP>
static int weights_launch(WeightArgs a, const WeightPlan& p, int heads, hipStream_t st) {
  if (a.lse == nullptr) {
    const int rc = weights_rows_launch<T, DP>(a, p, heads, st);
    if (rc) return rc;
    a.lse = a.lse2;
    a.lse_scale = 1.0f;
  }
  constexpr int NT = DP * (int)sizeof(T) <= 256 ? 4 : DP * (int)sizeof(T) <= 512 ? 2 : 1, KEYS = 16 * NT * kAwWaves;
  hipLaunchKernelGGL((weights_columns_kernel<T, DP, NT>), dim3((unsigned)((int64_t)(a.n + KEYS - 1) / KEYS * p.chunks * heads)),
                     dim3(kAwThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  if (p.chunks == 1) return LRQK_OK;
  const int64_t count = (int64_t)heads * a.n;
  hipLaunchKernelGGL(weights_sum_kernel, dim3((unsigned)((count + kAwThreads - 1) / kAwThreads)), dim3(kAwThreads), 0, st, a, count);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
template <typename T>
static int weights_launch_dp(const WeightArgs& a, const WeightPlan& p, int heads, hipStream_t st) {
  if (p.dp == 32) return weights_launch<T, 32>(a, p, heads, st);
  if (p.dp == 64) return weights_launch<T, 64>(a, p, heads, st);
  if (p.dp == 128) return weights_launch<T, 128>(a, p, heads, st);
  return weights_launch<T, 256>(a, p, heads, st);
}

static int weights_check(int b, int hq, int hc, int t, int64_t n, int d, int dtype) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(b > 0 && hq > 0 && hc > 0 && t > 0 && n > 0 && d > 0, LRQK_EINVAL, "bad sizes b=%d hq=%d hc=%d t=%d n=%lld d=%d", b, hq,
               hc, t, (long long)n, d);
  LRQK_REQUIRE(hq % hc == 0, LRQK_EINVAL, "%d query heads over %d cache heads", hq, hc);
  LRQK_REQUIRE(d * (int)elem_size(dtype) % 16 == 0 && d <= 256, LRQK_ELIMIT,
               "head_dim %d unsupported (rows of whole 16-byte pieces, at most 256 elements)", d);
  LRQK_REQUIRE(n <= (1 << 30) && (int64_t)b * hq <= 65535 && (int64_t)(hq / hc) * t <= (1 << 30), LRQK_ELIMIT,
               "n=%lld (at most 2^30), b * hq=%lld (65535), t=%d", (long long)n, (long long)b * hq, t);
  return LRQK_OK;
}

}  // namespace lrqk

using namespace lrqk;

extern "C" int64_t lrqk_attention_weights_workspace(int b, int hq, int hc, int t, int64_t n, int d, int have_lse, int dtype) {
  const int rc = weights_check(b, hq, hc, t, n, d, dtype);
  if (rc) return rc;
  const WeightPlan p = weights_plan(b, hq, hc, t, n, d, dtype, have_lse != 0);
  return (p.lse2 + p.part) * (int64_t)sizeof(float);
}

extern "C" int lrqk_attention_weights(const void* q, const void* k, int64_t k_batch_stride, int64_t k_head_stride, int64_t k_row_stride,
                                      int64_t n, const int32_t* lengths, const float* lse, const float* weights, float* out, int b,
                                      int hq, int hc, int t, int d, float scale, void* workspace, int64_t workspace_bytes, int dtype,
                                      void* stream) {
  int rc = weights_check(b, hq, hc, t, n, d, dtype);
  if (rc) return rc;
  LRQK_REQUIRE(q && k && out, LRQK_EINVAL, "null pointer");
  LRQK_REQUIRE(scale > 0.0f && scale < INFINITY, LRQK_EINVAL, "scale=%g has to be positive and finite", (double)scale);
  const int vec = 16 / (int)elem_size(dtype);
  LRQK_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)workspace % 16 == 0 && k_batch_stride % vec == 0 &&
                   k_head_stride % vec == 0 && k_row_stride % vec == 0,
               LRQK_EINVAL, "pointers and rows must be 16-byte aligned");
  const WeightPlan p = weights_plan(b, hq, hc, t, n, d, dtype, lse != nullptr);
  const int64_t need = (p.lse2 + p.part) * (int64_t)sizeof(float);
  LRQK_REQUIRE(workspace_bytes >= need && (workspace || need == 0), LRQK_EINVAL, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes,
               (long long)need);
  // (a launch's workgroups are counted in 31 bits; no memory holds what would need more)
  const int64_t places = std::max((int64_t)p.groups * std::max(p.parts, 1), (n + 63) / 64 * p.chunks);
  LRQK_REQUIRE(places * b * hc <= INT32_MAX, LRQK_ELIMIT, "%lld keys of %d heads and %d queries are more than a launch has places for",
               (long long)n, b * hc, t);
  WeightArgs a{q, k, lengths, lse, kLog2e, (float*)workspace, (float*)workspace + p.lse2, weights, out, k_batch_stride, k_head_stride,
               k_row_stride, (int)n, hq, hc, t, d, p.parts, p.groups, p.chunks, (uint32_t)(b * hc), scale * kLog2e};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LRQK_F32) return weights_launch_dp<float>(a, p, b * hc, st);
  return weights_launch_dp<bf16_t>(a, p, b * hc, st);
}
