// The attention that every cached token got from the last t tokens of its sequence,
//
//   out_j = weights_j + sum over the query heads that read j's head, sum over the queries i that see j, exp(scale q_i.k_j - lse_i),
//
// query i being token length - t + i, which sees the tokens up to itself.  The attention itself leaves lse (lse_i = log of
// the sum of exp(scale q_i.k_j)); where the caller does not have it, a first pass over the keys forms it.
//
//   rows     lse: a wave has 16 NT queries and walks over the keys they see; S^T = K Q^T, so that a lane has a maximum and
//            a sum of its own for its query and meets the other lanes at the end only.  Few queries: the keys are split
//            and `merge` joins the parts.
//   columns  sums: a wave has 16 NT keys and walks over the queries that see them, S = Q K^T, so that a lane's sums are
//            those of its keys; chunks of the queries, which `sum` adds up where there are several.
//   stream   the same for up to 64 queries of a cache head (rows of 256 bytes): a wave has all of them and streams keys, S^T = K Q^T, whose
//            rows it adds up across the lanes.
//
// No atomics: the same bits every time.  What a wave has is in its registers; what is walked over passes through LDS in
// whole rows, the next ones read ahead.  A prompt is bound by the exponentials and the products of both passes; a few
// queries over a long cache by the reading of the keys.
#include <algorithm>
#include <type_traits>

#include "attn_rows.hpp"

namespace lrqk {

constexpr int kAwWaves = 4, kAwThreads = kAwWaves * kWave;
constexpr float kAwNone = -3.0e38f;    // maximum of no scores
constexpr float kAwMuch = 4096.0f;      // a lane's exponentials of a tile may add up to this before the maximum is looked for
constexpr int kAwTile = 32;             // rows of a tile that is walked over
constexpr int kAwPart = 16;             // tiles of which a lane's sum is one number, before it joins the others

struct WeightArgs {
  const void *q, *k;
  const int32_t* lengths;
  const float* lse;        // natural logarithms of the caller's, or those of base 2 of the first pass
  float lse_scale;         // what makes them base 2
  float* lse2;             // first pass: [b][hq][t]
  float* part;             // first pass: [parts][b][hq][t][2]; second pass: [chunks][b][hc][n]
  const float* weights;    // or null
  float* out;
  int64_t kv_b, kv_h, kv_r;
  int n, hq, hc, t, d, parts, per, groups, chunks;   // per: tiles of a part
  uint32_t heads;           // of the cache, of all sequences
  float scale_log2e;
};

__device__ __forceinline__ int weights_len(const WeightArgs& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.n) : a.n; }

// Rows on their way through LDS.
template <typename T, int DP>
struct WeightTile {
  static constexpr int STEPS = DP * (int)sizeof(T) / 64, CH = 4 * STEPS;      // 16-byte pieces of a row
  static constexpr int LOADS = (kAwTile * CH + kAwThreads - 1) / kAwThreads;  // of a thread for a tile
  static constexpr int SIZE = kAwTile * CH;
  // rows 0 .. last of `base`, `step` bytes apart (a row beyond stands for the last one)
  static __device__ __forceinline__ void load(const void* base, int64_t step, int last, int pieces, ar_u4 (&g)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = min(i * kAwThreads + (int)threadIdx.x, SIZE - 1);
      g[i] = *(const ar_u4*)((const char*)base + min(at / CH, last) * step + 16 * min(at % CH, pieces - 1));
    }
  }
  static __device__ __forceinline__ void store(ar_u4* tile, int pieces, ar_u4 (&g)[LOADS]) {
    if (pieces < CH) {   // (a head of a width between two of the kernels')
#pragma unroll
      for (int i = 0; i < LOADS; ++i) g[i] = (i * kAwThreads + (int)threadIdx.x) % CH < pieces ? g[i] : ar_u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = i * kAwThreads + (int)threadIdx.x;
      if (SIZE % kAwThreads == 0 || at < SIZE) tile[ar_place<CH>(at / CH, at % CH)] = g[i];
    }
  }
  // A wave's own 16 rows r0 .. as operands, through 16 rows of LDS of its own.
  static constexpr int OWN = 16 * CH, OWN_LOADS = OWN / kWave;
  static __device__ __forceinline__ void load_own(const void* base, int64_t step, int64_t r0, int64_t last, int pieces, ar_u4 (&g)[OWN_LOADS]) {
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < OWN_LOADS; ++i) {
      const int at = i * kWave + lane;
      g[i] = *(const ar_u4*)((const char*)base + min(r0 + at / CH, last) * step + 16 * min(at % CH, pieces - 1));
    }
  }
  static __device__ __forceinline__ void own(ar_u4* room, int pieces, const ar_u4 (&g)[OWN_LOADS], ar_u4 (&x)[STEPS]) {
    const int lane = lane_id();
    ar_wave_sync();
#pragma unroll
    for (int i = 0; i < OWN_LOADS; ++i) {
      const int at = i * kWave + lane;
      room[ar_place<CH>(at / CH, at % CH)] = at % CH < pieces ? g[i] : ar_u4{0, 0, 0, 0};
    }
    ar_wave_sync();
#pragma unroll
    for (int c = 0; c < STEPS; ++c) x[c] = room[ar_place<CH>(lane & 15, 4 * c + (lane >> 4))];
  }
};

// Item (head, part, group of 64 NT rows) of a workgroup: its queries' maximum and sum over its part of the keys.  Bound by
// the exponentials beside the products: 8192 tokens of 32 / 8 heads of 128, 275 GFLOP in 313 to 350 us, the vector ALUs 59 %
// busy, the matrix cores 37 %; `merge` 8.
template <typename T, int DP, int NT>
__global__ __launch_bounds__(kAwThreads, 2) void weights_rows_kernel(WeightArgs a) {
  using Tile = WeightTile<T, DP>;
  constexpr int STEPS = Tile::STEPS, CH = Tile::CH, NE = kAwTile / 4, NU = kAwTile / 16;
  constexpr int ROOM = 2 * Tile::SIZE > kAwWaves * Tile::OWN ? 2 * Tile::SIZE : kAwWaves * Tile::OWN;
  __shared__ ar_u4 smem[ROOM];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  // (the heads of a place follow each other: with 8 of them, or a divisor, a head's workgroups are on one XCD, whose L2 holds
  // its keys)
  const int item = (int)(blockIdx.x / a.heads), head = (int)(blockIdx.x % a.heads), b = head / a.hc, hc = head % a.hc;
  // (part by part: dealt out by their number, workgroups of one part would meet on the same CUs, and a prompt's last parts
  // are empty for most groups: 400 instead of 360 us for 8K tokens)
  const int part = item / a.groups, group = a.groups - 1 - item % a.groups;
  const int gc = a.hq / a.hc, M = gc * a.t, row0 = (group * kAwWaves + wave) * 16 * NT;
  const int len = weights_len(a, b), behind = len - a.t;   // query i sees the keys up to behind + i
  const T* q = (const T*)a.q + ((int64_t)b * a.hq + (int64_t)hc * gc) * a.t * a.d;
  const T* k = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
  const int pieces = a.d * (int)sizeof(T) / 16;
  const int64_t q_step = (int64_t)a.d * (int)sizeof(T), k_step = a.kv_r * (int)sizeof(T);
  // keys that the workgroup walks over: to the last row of a head that it has, or its last one
  const int g0 = group * kAwWaves * 16 * NT, g1 = min(g0 + kAwWaves * 16 * NT, M) - 1;
  const int walk = max(0, (g0 / a.t != g1 / a.t ? len - 1 : behind + g1 % a.t) + 1);
  const int begin = part * a.per, end = min((walk + kAwTile - 1) / kAwTile, begin + a.per);
  if (begin >= end) {   // (the merging looks at all parts)
    if (threadIdx.x < 64 * NT && g0 + (int)threadIdx.x < M) {
      const int64_t at = (int64_t)head * M + g0 + threadIdx.x;
      if (a.parts == 1)
        a.lse2[at] = -INFINITY;
      else
        ((float2*)a.part)[(int64_t)part * a.heads * M + at] = make_float2(kAwNone, 0.0f);
    }
    return;
  }
  ar_u4 qf[NT][STEPS];
  {
    ar_u4 own[2][Tile::OWN_LOADS];
    Tile::load_own(q, q_step, row0, M - 1, pieces, own[0]);
#pragma unroll
    for (int m = 0; m < NT; ++m) {
      if (m + 1 < NT) Tile::load_own(q, q_step, row0 + 16 * (m + 1), M - 1, pieces, own[(m + 1) & 1]);
      Tile::own(smem + wave * Tile::OWN, pieces, own[m & 1], qf[m]);
    }
  }
  int last[NT];   // last key that the lane's query sees
  int most = -1, least = a.n;
  float top[NT], part_sum[NT];
  double sum[NT];   // of kAwPart tiles at a time: thousands of addends to one fp32 number would lose its last bits
  int held = 0;
#pragma unroll
  for (int m = 0; m < NT; ++m) {
    last[m] = behind + min(row0 + 16 * m + col, M - 1) % a.t;
    most = max(most, last[m]);
    least = min(least, last[m]);
    top[m] = kAwNone;
    part_sum[m] = 0.0f;
    sum[m] = 0.0;
  }
  // keys that a query of the wave sees, and that all of them see
  most = (int)wave_reduce_u32((uint32_t)(most + 1), [](uint32_t x, uint32_t y) { return max(x, y); });
  least = (int)(wave_reduce_u32((uint32_t)least ^ 0x80000000u, [](uint32_t x, uint32_t y) { return min(x, y); }) ^ 0x80000000u);
  ar_u4 g[2][Tile::LOADS];   // two tiles on their way
  auto load = [&](int tile, ar_u4 (&x)[Tile::LOADS]) {
    const int first = min(tile, end - 1) * kAwTile;
    Tile::load((const char*)k + first * k_step, k_step, walk - 1 - first, pieces, x);
  };
  auto work = [&](auto buffer, int tile) {
    const ar_u4* keys = smem + decltype(buffer)::value * Tile::SIZE;
    const int first = tile * kAwTile;
    if (first >= most) return;
    float x[NT][NE];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      ar_u4 kf[STEPS];
#pragma unroll
      for (int c = 0; c < STEPS; ++c) kf[c] = keys[ar_place<CH>(16 * u + col, 4 * c + quad)];
      ar_f4 s[NT] = {};
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int m = 0; m < NT; ++m) s[m] = ar_step<T>(kf[c], qf[m][c], s[m]);
#pragma unroll
      for (int m = 0; m < NT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[m][4 * u + r] = s[m][r];
    }
    if (first + kAwTile - 1 > least) {
#pragma unroll
      for (int m = 0; m < NT; ++m)
#pragma unroll
        for (int e = 0; e < NE; ++e) x[m][e] = first + 16 * (e >> 2) + 4 * quad + (e & 3) <= last[m] ? x[m][e] : -INFINITY;
    }
    // as long as a lane's exponentials add up to little the maximum that it has serves
    float add[NT];
    bool more = false;
#pragma unroll
    for (int m = 0; m < NT; ++m) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const float p = ar_exp2(fmaf(x[m][e], a.scale_log2e, -top[m]));
        add[m] = e == 0 ? p : add[m] + p;
      }
      more = more | !(add[m] <= kAwMuch);
    }
    if (__ballot(more)) {
#pragma unroll
      for (int m = 0; m < NT; ++m) {
        float now = x[m][0];
#pragma unroll
        for (int e = 1; e < NE; ++e) now = fmaxf(now, x[m][e]);
        now = fmaxf(top[m], now * a.scale_log2e);
        const float f = ar_exp2(top[m] - now);
        part_sum[m] *= f;
        sum[m] *= f;
        top[m] = now;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const float p = ar_exp2(fmaf(x[m][e], a.scale_log2e, -now));
          add[m] = e == 0 ? p : add[m] + p;
        }
      }
    }
#pragma unroll
    for (int m = 0; m < NT; ++m) part_sum[m] += add[m];
    if (++held == kAwPart) {
      held = 0;
#pragma unroll
      for (int m = 0; m < NT; ++m) {
        sum[m] += part_sum[m];
        part_sum[m] = 0.0f;
      }
    }
  };
  load(begin, g[0]);
  load(begin + 1, g[1]);
  __syncthreads();   // (the rooms of the queries make place)
  Tile::store(smem, pieces, g[0]);
  __syncthreads();
  for (int tile = begin; tile < end; tile += 2) {   // (a tile behind the last is the last one again, and not worked on)
    load(tile + 2, g[0]);
    work(std::integral_constant<int, 0>{}, tile);
    Tile::store(smem + Tile::SIZE, pieces, g[1]);
    __syncthreads();
    if (tile + 1 >= end) break;
    load(tile + 3, g[1]);
    work(std::integral_constant<int, 1>{}, tile + 1);
    Tile::store(smem, pieces, g[0]);
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < NT; ++m) {
    const float all = ar_quad_max(top[m]);
    const float total = ar_quad_sum((float)(sum[m] + part_sum[m]) * ar_exp2(top[m] - all));
    const int row = row0 + 16 * m + col;
    if (quad != 0 || row >= M) continue;
    const int64_t at = (int64_t)head * M + row;
    if (a.parts == 1) {
      a.lse2[at] = total == 0.0f ? -INFINITY : all + log2f(total);
    } else {
      ((float2*)a.part)[(int64_t)part * a.heads * M + at] = make_float2(all, total);
    }
  }
}

// 16 rows a workgroup, 16 threads a row.
__global__ __launch_bounds__(kAwThreads) void weights_merge_kernel(WeightArgs a, int64_t rows) {
  __shared__ float red[2][16][16];
  const int col = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int64_t row = (int64_t)blockIdx.x * 16 + col, at = min(row, rows - 1);
  const float2* p = (const float2*)a.part + at;
  float top = kAwNone, sum = 0.0f;
#pragma unroll 4
  for (int i = group; i < a.parts; i += 16) {
    const float2 x = p[i * rows];
    const float now = fmaxf(top, x.x);
    sum = sum * ar_exp2(top - now) + x.y * ar_exp2(x.x - now);
    top = now;
  }
  red[0][group][col] = top;
  red[1][group][col] = sum;
  __syncthreads();
  if (group != 0 || row >= rows) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, red[0][i][col]);
  sum = 0.0f;
  for (int i = 0; i < 16; ++i) sum += red[1][i][col] * ar_exp2(red[0][i][col] - top);
  a.lse2[row] = sum == 0.0f ? -INFINITY : top + log2f(sum);
}

// 64 NT keys and a chunk of the queries a workgroup.  Bound as the rows are: 8192 tokens, 352 to 390 us, vector ALUs 51 %,
// matrix cores 33 %, no bank conflicts, and `sum` 5.  (Keys in registers and queries through LDS: the other way round a wave's
// sums would be rows' and cross the lanes for every tile.  Products of 16 keys placed between the exponentials of the 16 before:
// no difference; 64 queries a tile, half the barriers: 425 us, the registers do not hold them.)
template <typename T, int DP, int NT>
__global__ __launch_bounds__(kAwThreads, 2) void weights_columns_kernel(WeightArgs a) {
  using Tile = WeightTile<T, DP>;
  constexpr int STEPS = Tile::STEPS, CH = Tile::CH, KEYS = 16 * NT, NU = kAwTile / 16;
  constexpr int ROOM = 2 * Tile::SIZE > kAwWaves * Tile::OWN ? 2 * Tile::SIZE : kAwWaves * Tile::OWN;
  __shared__ ar_u4 smem[ROOM];
  __shared__ ar_f4 lse_s[2][kAwTile / 4];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  const int head = (int)(blockIdx.x % a.heads), b = head / a.hc, hc = head % a.hc, place = (int)(blockIdx.x / a.heads);
  const int chunk = place % a.chunks, first0 = place / a.chunks * kAwWaves * KEYS;   // (the most queries first)
  const int first = first0 + wave * KEYS;
  const int gc = a.hq / a.hc, M = gc * a.t;
  const int len = weights_len(a, b), behind = len - a.t;
  const T* q = (const T*)a.q + ((int64_t)b * a.hq + (int64_t)hc * gc) * a.t * a.d;
  const T* k = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
  const float* lse = a.lse + (int64_t)head * M;
  const int pieces = a.d * (int)sizeof(T) / 16;
  const int64_t q_step = (int64_t)a.d * (int)sizeof(T), k_step = a.kv_r * (int)sizeof(T);
  const int64_t row = (int64_t)head * a.n + first;
  float sum[NT], part[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) sum[j] = part[j] = 0.0f;
  if (first0 < len) {   // (the same for all waves)
    // tiles of queries: of one query head each, from the first that sees a key of the workgroup; or, of heads with less than a
    // tile, of several heads (16 tokens of 128 heads over 64K of one: 78 us instead of 174; from 32 tokens on no faster)
    const bool packed = a.t < kAwTile;
    const int t0 = packed ? 0 : max(0, first0 - behind) / kAwTile;
    const int per = packed ? 1 : (a.t + kAwTile - 1) / kAwTile - t0;
    const int items = packed ? (M + kAwTile - 1) / kAwTile : gc * per;
    const int begin = (int)((int64_t)items * chunk / a.chunks), end = (int)((int64_t)items * (chunk + 1) / a.chunks);
    // two tiles on their way, and what the one in LDS is
    struct Next {
      ar_u4 g[Tile::LOADS];
      float lse;
      int base, stop, at;   // rows base .. min(base + 32, stop) - 1 of the head's; query `at` of its head is the first
    } next[2];
    struct {
      int base, stop, at;
      bool none;   // some of its queries saw nothing: they give nothing, whatever they hold
    } now{};
    int h = packed ? 0 : begin / per, tt = packed ? begin : t0 + begin % per, left = end - begin;
    auto load = [&](Next& x) {   // the next tile (behind the last one that one again)
      x.base = h * a.t + kAwTile * tt;
      x.stop = packed ? M : (h + 1) * a.t;
      x.at = packed ? 0 : kAwTile * tt;
      if (--left > 0) {
        ++tt;
        if (!packed && tt == t0 + per) {
          ++h;
          tt = t0;
        }
      }
      Tile::load((const char*)q + x.base * q_step, q_step, x.stop - 1 - x.base, pieces, x.g);
      x.lse = lse[min(x.base + (int)(threadIdx.x % kAwTile), x.stop - 1)];
    };
    auto store = [&](auto buffer, Next& x) {
      const float l = x.lse * a.lse_scale;
      now = {x.base, x.stop, x.at, __any(l == -INFINITY) != 0};
      Tile::store(smem + decltype(buffer)::value * Tile::SIZE, pieces, x.g);
      if (threadIdx.x < kAwTile) ((float*)lse_s[decltype(buffer)::value])[threadIdx.x] = l;
    };
    if (begin < end) {
      load(next[0]);
      load(next[1]);
    }
    ar_u4 kf[NT][STEPS];
    {
      ar_u4 own[2][Tile::OWN_LOADS];
      Tile::load_own(k, k_step, first, len - 1, pieces, own[0]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (j + 1 < NT) Tile::load_own(k, k_step, first + 16 * (j + 1), len - 1, pieces, own[(j + 1) & 1]);
        Tile::own(smem + wave * Tile::OWN, pieces, own[j & 1], kf[j]);
      }
    }
    int held = 0;
    auto work = [&](auto buffer) {
      const ar_u4* rows = smem + decltype(buffer)::value * Tile::SIZE;
      const int base = now.base, stop = now.stop, at = now.at;
      if (first >= len || (!packed && behind + at + kAwTile - 1 < first)) return;   // (no query sees a key of the wave)
      const bool whole = base + kAwTile <= stop && first + KEYS - 1 <= behind + at && !now.none;
      auto add = [&](auto is_whole) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          ar_u4 qf[STEPS];
#pragma unroll
          for (int c = 0; c < STEPS; ++c) qf[c] = rows[ar_place<CH>(16 * u + col, 4 * c + quad)];
          const ar_f4 l2 = lse_s[decltype(buffer)::value][4 * u + quad];
          ar_f4 s[NT] = {};
#pragma unroll
          for (int c = 0; c < STEPS; ++c)
#pragma unroll
            for (int j = 0; j < NT; ++j) s[j] = ar_step<T>(qf[c], kf[j][c], s[j]);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) p[r] = ar_exp2(fmaf(s[j][r], a.scale_log2e, -l2[r]));
            if constexpr (!decltype(is_whole)::value) {
#pragma unroll
              for (int r = 0; r < 4; ++r) {   // (& and not &&: no branch, see tree_mask)
                const int i = 16 * u + 4 * quad + r, last = behind + (packed ? (base + i) % a.t : at + i);
                const bool sees = (base + i < stop) & (first + 16 * j + col <= last) & (l2[r] != -INFINITY);
                p[r] = sees ? p[r] : 0.0f;
              }
            }
            part[j] += (p[0] + p[1]) + (p[2] + p[3]);
          }
        }
      };
      if (whole)
        add(std::true_type{});
      else
        add(std::false_type{});
      if (++held == kAwPart) {   // (sums of sums, as above)
        held = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          sum[j] += part[j];
          part[j] = 0.0f;
        }
      }
    };
    using First = std::integral_constant<int, 0>;
    using Second = std::integral_constant<int, 1>;
    if (begin < end) {
      __syncthreads();   // (the rooms of the keys make place)
      store(First{}, next[0]);
      __syncthreads();
      for (int item = begin; item < end; item += 2) {
        load(next[0]);
        work(First{});
        store(Second{}, next[1]);
        __syncthreads();
        if (item + 1 >= end) break;
        load(next[1]);
        work(Second{});
        store(First{}, next[0]);
        __syncthreads();
      }
    }
  }
  if (first >= a.n) return;
  float* out = (a.chunks == 1 ? a.out : a.part + (int64_t)chunk * a.heads * a.n) + row;
  const float* had = a.chunks == 1 && a.weights ? a.weights + row : nullptr;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    sum[j] = ar_quad_sum(sum[j] + part[j]);
    if (quad == 0 && first + 16 * j + col < a.n) out[16 * j + col] = had ? had[16 * j + col] + sum[j] : sum[j];
  }
}

// All queries of a cache head, up to 16 NT, and every fourth tile of 32 keys of a split for each of the four waves.  Bound
// by the reading of the keys: 5 tokens over 2 x 64K, 32 / 8 heads of 128 bf16 elements, 268 MB in 57 us, 4.7 TB/s.  (Four
// workgroups per CU take 128 registers a thread; with 136 three fit, and the fourth ran alone: 49 instead of 46 us for 32
// queries a cache head over 64K.)  The two kernels of many queries take 58 + 5 us for 16, 32 or 64 queries a cache head over
// 64K keys where this one takes 44, 46 and 51, and 18 + 5 for 64 over 8K instead of 12.
template <typename T, int DP, int NT>
__global__ __launch_bounds__(kAwThreads, DP * (int)sizeof(T) <= 256 && NT <= 2 ? 4 : DP * (int)sizeof(T) <= 512 ? 2 : 1) void weights_stream_kernel(WeightArgs a) {
  using Tile = WeightTile<T, DP>;
  constexpr int STEPS = Tile::STEPS, CH = Tile::CH, NU = kAwTile / 16, LOADS = kAwTile * CH / kWave;
  __shared__ ar_u4 smem[kAwWaves][kAwTile * CH];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  const int head = (int)(blockIdx.x % a.heads), b = head / a.hc, hc = head % a.hc;
  const int M = a.hq / a.hc * a.t;
  const int len = weights_len(a, b), behind = len - a.t;
  const T* q = (const T*)a.q + (int64_t)head * M * a.d;
  const T* k = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
  const int pieces = a.d * (int)sizeof(T) / 16;
  const int64_t k_step = a.kv_r * (int)sizeof(T);
  ar_u4* rows = smem[wave];
  float l2[NT];
  int last[NT];   // last key that the lane's query sees
  ar_u4 qf[NT][STEPS];
  bool nones = false;
#pragma unroll
  for (int m = 0; m < NT; ++m) {
    const int row = min(16 * m + col, M - 1);
    l2[m] = a.lse[(int64_t)head * M + row] * a.lse_scale;
    const bool none = l2[m] == -INFINITY;   // (a query that saw nothing gives nothing, whatever it holds)
    last[m] = ((16 * m + col < M) & !none) ? behind + row % a.t : -1;
    nones = nones | none;
    ar_row(q + (int64_t)row * a.d, quad, pieces, qf[m]);
  }
  const float* had = a.weights ? a.weights + (int64_t)head * a.n : nullptr;
  float* out = a.out + (int64_t)head * a.n;
  const int tiles = (a.n + kAwTile - 1) / kAwTile;
  const int tile0 = (int)(blockIdx.x / a.heads) * a.per + wave, end = min(tiles, (int)(blockIdx.x / a.heads + 1) * a.per);
  // (few queries see a part of the keys of the last tiles, and of the smaller heads' tiles have rows that are none)
  const int wholes = M == 16 * NT && !__any(nones) ? max(0, behind + 1) / kAwTile : 0;
  const int piece = lane % CH, krow = lane / CH, keys = max(len, 1);
  ar_u4 g[LOADS];
  float w = 0.0f;
  auto load = [&](int tile) {   // (of a tile behind the sequence its last key, which is not looked at)
    const int first = min(tile, (keys - 1) / kAwTile) * kAwTile, most = keys - 1 - first;
    const char* src = (const char*)k + first * k_step + 16 * min(piece, pieces - 1);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) g[i] = *(const ar_u4*)(src + min(i * (kWave / CH) + krow, most) * k_step);
    if (had) w = had[min(tile * kAwTile + lane % kAwTile, a.n - 1)];
  };
  if (tile0 < end) load(tile0);
  for (int tile = tile0; tile < end; tile += kAwWaves) {
    const int first = tile * kAwTile;
    const float before = w;
    ar_wave_sync();
    if (pieces < CH) {   // (a head of a width between two of the kernels')
#pragma unroll
      for (int i = 0; i < LOADS; ++i) g[i] = piece < pieces ? g[i] : ar_u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) rows[ar_place<CH>(i * (kWave / CH) + krow, piece)] = g[i];
    ar_wave_sync();
    load(min(tile + kAwWaves, tiles - 1));
    float p[NU][4] = {};   // of key 16 u + 4 quad + r, over the lane's queries
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      ar_u4 kf[STEPS];
#pragma unroll
      for (int c = 0; c < STEPS; ++c) kf[c] = rows[ar_place<CH>(16 * u + col, 4 * c + quad)];
#pragma unroll
      for (int m = 0; m < NT; ++m) {
        ar_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) s = ar_step<T>(kf[c], qf[m][c], s);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = ar_exp2(fmaf(s[r], a.scale_log2e, -l2[m]));
          const bool sees = (tile < wholes) | (first + 16 * u + 4 * quad + r <= last[m]);
          p[u][r] += sees ? x : 0.0f;
        }
      }
    }
    // the 16 queries of a quad's lanes; key 16 u + 4 quad + i is written by lane 16 u + 4 quad + i
    float v = 0.0f;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = row_reduce(p[u][r], [](float f, float h) { return f + h; });
        const float y = __shfl(x, (lane >> 2 & 3) * 16, kWave);
        v = lane >> 4 == u && (lane & 3) == r ? y : v;
      }
    if (lane < kAwTile && first + lane < a.n) out[first + lane] = before + v;
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
  int dp, rows_nt, groups, parts, per, nt, chunks, few_per;
  bool few;
  int64_t lse2, part;   // floats
  int64_t keys_blocks(int64_t n) const { return (n + 16 * nt * kAwWaves - 1) / (16 * nt * kAwWaves); }
  // workgroups of the largest launch, for a head (that of few queries has a thousand; the joining ones less than these)
  int64_t most_blocks(int64_t n) const { return std::max((int64_t)groups * parts, few ? 0 : keys_blocks(n) * chunks); }
  int64_t part_at() const { return (lse2 + 3) / 4 * 4; }
  int64_t bytes() const { return (part_at() + part) * (int64_t)sizeof(float); }
};
static WeightPlan weights_plan(int b, int hq, int hc, int t, int64_t n, int d, int dtype, bool have_lse) {
  WeightPlan p{};
  p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t M = (int64_t)(hq / hc) * t, heads = (int64_t)b * hc;
  const int row = p.dp * (int)elem_size(dtype);
  const int most = row <= 256 ? 4 : row <= 512 ? 2 : 1;   // 16 keys, or queries, that a wave has registers for
  // 64 keys a wave where the products are many (8K prompt of 32 / 8 heads of 128: 352 us with 64, 362 with 32; 512 tokens over
  // 64K: 395, 420), 32 where workgroups that load while others multiply count for more (4K prompt: 133, 106; 512 tokens over
  // 8K: 68, 63; 200 over 32K: 115, 108; 200 over 1K: 29, 19)
  p.nt = (double)heads * (double)M * (double)(n - t / 2) >= 0x1p29 ? most : std::min(most, 2);
  p.few = M <= (row <= 256 ? 64 : row <= 512 ? 32 : 16);   // (what a wave has room for; both kernels measured at weights_stream_kernel)
  if (p.few) {
    // four workgroups per CU, two tiles for each of a workgroup's waves at least
    const int64_t tiles = (n + kAwTile - 1) / kAwTile, splits = std::max<int64_t>(1, 1024 / heads);
    p.few_per = (int)std::max<int64_t>(2 * kAwWaves, (tiles + splits - 1) / splits);
  }
  // two thousand workgroups of keys and chunks of queries (half of a prompt's have little to do; one thousand: no faster),
  // eight tiles of queries for each
  const int64_t blocks = p.keys_blocks(n), items = (M + 15) / 16;
  p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(2048 / (blocks * heads), items / 16));
  if (!p.few && p.chunks > 1) p.part = heads * n * p.chunks;
  if (have_lse) return p;
  // (lse over 8192 keys: 64 queries a cache head 7.8 us with 16 a wave, 12.7 with 64; 128 9.0 and 13; 1024 34 and 29;
  // both passes of an 8K prompt: 665 us with 64, 694 with 32)
  p.rows_nt = M <= 128 ? 1 : most;
  p.groups = (int)((M + 64 * p.rows_nt - 1) / (64 * p.rows_nt));
  // parts of one length, however many keys a group of queries sees (a prompt's first ones few): four thousand, with eight
  // tiles of 32 keys at least.  (One part a group, 8K tokens: a quarter of the GPU waited for the longest ones; two thousand
  // parts: 368 instead of 359 us.)
  const int64_t tiles = (n + kAwTile - 1) / kAwTile;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>((tiles + 7) / 8, 4096 / (heads * p.groups)));
  p.per = (int)((tiles + parts - 1) / parts);
  p.parts = (int)((tiles + p.per - 1) / p.per);
  p.lse2 = heads * M;
  if (p.parts > 1) p.part = std::max(p.part, heads * M * p.parts * 2);   // (the passes follow each other)
  return p;
}

template <typename T, int DP>
static int weights_rows_launch(const WeightArgs& a, const WeightPlan& p, int heads, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.groups * p.parts * heads));
  constexpr int MOST = DP * (int)sizeof(T) <= 256 ? 4 : DP * (int)sizeof(T) <= 512 ? 2 : 1;
  if constexpr (MOST >= 4)
    if (p.rows_nt == 4) hipLaunchKernelGGL((weights_rows_kernel<T, DP, 4>), grid, dim3(kAwThreads), 0, st, a);
  if constexpr (MOST == 2)
    if (p.rows_nt == 2) hipLaunchKernelGGL((weights_rows_kernel<T, DP, 2>), grid, dim3(kAwThreads), 0, st, a);
  if (p.rows_nt == 1) hipLaunchKernelGGL((weights_rows_kernel<T, DP, 1>), grid, dim3(kAwThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  if (p.parts > 1) {
    const int64_t rows = p.lse2;
    hipLaunchKernelGGL(weights_merge_kernel, dim3((unsigned)((rows + 15) / 16)), dim3(kAwThreads), 0, st, a, rows);
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
  if (p.few) {
    a.per = p.few_per;
    const int tiles = (a.n + kAwTile - 1) / kAwTile, M = a.hq / a.hc * a.t;
    const dim3 grid((unsigned)((int64_t)((tiles + a.per - 1) / a.per) * heads));
    constexpr int ROW = DP * (int)sizeof(T);
    if (M <= 16) hipLaunchKernelGGL((weights_stream_kernel<T, DP, 1>), grid, dim3(kAwThreads), 0, st, a);
    if constexpr (ROW <= 512)
      if (M > 16 && M <= 32) hipLaunchKernelGGL((weights_stream_kernel<T, DP, 2>), grid, dim3(kAwThreads), 0, st, a);
    if constexpr (ROW <= 256)
      if (M > 32) hipLaunchKernelGGL((weights_stream_kernel<T, DP, 4>), grid, dim3(kAwThreads), 0, st, a);
    LRQK_HIP_CHECK(hipGetLastError());
    return LRQK_OK;
  }
  const dim3 grid((unsigned)(p.keys_blocks(a.n) * p.chunks * heads));
  constexpr int ROW = DP * (int)sizeof(T);
  if constexpr (ROW <= 256)
    if (p.nt == 4) hipLaunchKernelGGL((weights_columns_kernel<T, DP, 4>), grid, dim3(kAwThreads), 0, st, a);
  if constexpr (ROW <= 512)
    if (p.nt == 2) hipLaunchKernelGGL((weights_columns_kernel<T, DP, 2>), grid, dim3(kAwThreads), 0, st, a);
  if constexpr (ROW > 512) hipLaunchKernelGGL((weights_columns_kernel<T, DP, 1>), grid, dim3(kAwThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  if (p.chunks == 1) return LRQK_OK;   // (the columns have added to the weights themselves)
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
  return p.bytes();
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
  const int64_t need = p.bytes();
  LRQK_REQUIRE(workspace_bytes >= need && (workspace || need == 0), LRQK_EINVAL, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes,
               (long long)need);
  LRQK_REQUIRE(p.most_blocks(n) * b * hc <= kMaxThreads / kAwThreads, LRQK_ELIMIT,
               "%lld keys of %d heads and %d queries are more than a launch has places for", (long long)n, b * hc, t);
  WeightArgs a{q, k, lengths, lse, kLog2e, (float*)workspace, (float*)workspace + p.part_at(), weights, out, k_batch_stride, k_head_stride,
               k_row_stride, (int)n, hq, hc, t, d, p.parts, p.per, p.groups, p.chunks, (uint32_t)(b * hc), scale * kLog2e};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LRQK_F32) return weights_launch_dp<float>(a, p, b * hc, st);
  return weights_launch_dp<bf16_t>(a, p, b * hc, st);
}
