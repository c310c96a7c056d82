// Attention of a tree of drafted tokens: the t new tokens of a sequence attend to its cached tokens, all of them, and to
// each other as a mask says,
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = log sum_j exp(scale q_i.k_j)
//
// over j < length of the cache and the drafted j with mask[i][j].  One pass over K and V: a running maximum and sum per
// query, the axis of the keys split over the GPU and the parts joined by a second launch.
//
// The query heads that read one head of the cache make its rows: M = (heads / cache heads) t of them, 16 MT in a
// workgroup.  S^T = K Q^T leaves a query in a lane's column, so maximum, sum and rescaling need no exchange but two
// between the quads, and the probabilities are the operand of O^T = V^T P^T as they lie: the rows of K are dealt to the
// lanes such that a quad's scores are those of successive keys, whose V rows the same quad loads, 16 lanes one whole row.
// Bf16 V is transposed between those lanes' registers; bf16 probabilities are the sum of two bf16 numbers (16 bits), so
// that the one rounding to bf16 is the output's.
#include <algorithm>

#include "attn_rows.hpp"

namespace lrqk {

constexpr int kTrWaves = 4, kTrThreads = kTrWaves * kWave;
constexpr int kTrCombThreads = 1024;
constexpr int kTrMaxSplits = 256;
constexpr float kTrNone = -3.0e38f;   // running maximum of a query that has seen no key yet
constexpr float kTrSlack = 8.0f;      // a maximum may be exceeded by 2^8 before the sums are rescaled to the new one

struct TreeArgs {
  const void *q, *k, *v, *k_new, *v_new;
  const uint8_t* mask;
  const int32_t* lengths;   // or null: n each
  void* out;
  float* lse;               // or null
  float *part, *part_ml;
  int32_t* odd;             // per workgroup: whether its drafted rows of V hold infinities or NaN
  int64_t kv_b, kv_h, kv_r; // elements between sequences, heads and rows of the cache
  int64_t mask_b;
  int n, hq, hc, hn, t, d, S, row_blocks, units;
  float scale_log2e;
};

// One row's part of V for a lane: elements VW i .. of row `row`.
template <typename T, int VW>
struct TreeV {
  static constexpr int DW = VW * (int)sizeof(T) / 4;
  uint32_t w[DW];
  __device__ __forceinline__ void load(const T* row, int i, int d) {
    if constexpr (DW >= 4) {
#pragma unroll
      for (int p = 0; p < DW / 4; ++p) {
        const int piece = min(i * (DW / 4) + p, d * (int)sizeof(T) / 16 - 1);
        const ar_u4 x = ((const ar_u4*)row)[piece];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * p + e] = x[e];
      }
    } else {
      const int at = i * DW < d * (int)sizeof(T) / 4 ? i * DW : 0;   // (beyond the head: something that is not used)
      if constexpr (DW == 2) {
        const ar_u2 x = *(const ar_u2*)((const uint32_t*)row + at);
        w[0] = x[0];
        w[1] = x[1];
      } else {
        w[0] = ((const uint32_t*)row)[at];
      }
    }
  }
};

// Takes infinities and NaN out of a register of V; whether there were any.
template <typename T>
__device__ __forceinline__ bool tree_clean(uint32_t& w) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t low = (w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u, high = (w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
    w &= ~(low | high);
    return (low | high) != 0;
  } else {
    const bool odd = (w & 0x7f800000u) == 0x7f800000u;
    if (odd) w = 0;
    return odd;
  }
}

// Eight scores of a lane as a bf16 operand.
__device__ __forceinline__ ar_bf8 tree_pack(const float* p) {
  ar_bf8 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (__bf16)p[e];
  return x;
}

template <typename T, int DP, int MT>
struct TreeTile {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int NU = BF ? 2 : 1;             // 16-key blocks of a tile
  static constexpr int KT = 16 * NU, NE = 4 * NU;   // keys of a tile, and of a quad in it
  static constexpr int STEPS = DP * (int)sizeof(T) / 64;
  static constexpr int VW = DP / 16;

  // o[j] += v_j^T p for the keys of the tile; p[e]: probability of the quad's key e for the lane's query
  static __device__ __forceinline__ void add(const TreeV<T, VW> (&v)[NE], const float (&p)[MT][NE], ar_f4 (&o)[MT][VW]) {
    if constexpr (BF) {
      ar_bf8 hi[MT], lo[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        hi[m] = tree_pack(p[m]);
        float rest[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = p[m][e] - (float)hi[m][e];   // exact
        lo[m] = tree_pack(rest);
      }
#pragma unroll
      for (int w = 0; w < VW / 2; ++w) {
        ar_u4 a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = __builtin_amdgcn_perm(v[2 * e + 1].w[w], v[2 * e].w[w], 0x05040100u);
          b[e] = __builtin_amdgcn_perm(v[2 * e + 1].w[w], v[2 * e].w[w], 0x07060302u);
        }
        const ar_bf8 va = __builtin_bit_cast(ar_bf8, a), vb = __builtin_bit_cast(ar_bf8, b);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          o[m][2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, lo[m], o[m][2 * w], 0, 0, 0);
          o[m][2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, lo[m], o[m][2 * w + 1], 0, 0, 0);
          o[m][2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, hi[m], o[m][2 * w], 0, 0, 0);
          o[m][2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, hi[m], o[m][2 * w + 1], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < VW; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < NE; ++e)
            o[m][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[e].w[j]), p[m][e], o[m][j], 0, 0, 0);
    }
  }
};

// The parts of a workgroup: [unit][row block] MT VW float4 a lane, and (maximum, sum) of 16 MT queries.
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kTrThreads) void tree_part_kernel(TreeArgs a) {
  using Tile = TreeTile<T, DP, MT>;
  constexpr int NU = Tile::NU, KT = Tile::KT, NE = Tile::NE, STEPS = Tile::STEPS, VW = Tile::VW;
  constexpr int JC = 2;   // output blocks that the waves join at a time
  __shared__ ar_f4 joint[kTrWaves][MT * JC][kWave];
  __shared__ float ml[kTrWaves][MT][16][2];
  const int lane = lane_id(), wave = wave_id(), col = lane & 15, quad = lane >> 4;
  // the row blocks of a unit (a split of a head) follow each other 8 workgroups apart: on one XCD, whose L2 then has the
  // rows of K and V that the first of them brought
  const int rb = (int)blockIdx.x % (8 * a.row_blocks) / 8;
  const int unit = (int)blockIdx.x / (8 * a.row_blocks) * 8 + (int)blockIdx.x % 8;
  if (unit >= a.units) return;
  const int split = unit % a.S, head = unit / a.S, b = head / a.hc, hc = head % a.hc;
  const int gc = a.hq / a.hc, M = gc * a.t, row0 = rb * 16 * MT;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.n) : a.n;

  const T* q = (const T*)a.q + ((int64_t)b * a.hq + (int64_t)hc * gc) * a.t * a.d;
  const T* kc = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
  const T* vc = (const T*)a.v + b * a.kv_b + hc * a.kv_h;
  const int64_t hn = (int64_t)b * a.hn + hc / (a.hc / a.hn);
  const T* kn = (const T*)a.k_new + hn * a.t * a.d;
  const T* vn = (const T*)a.v_new + hn * a.t * a.d;
  const int pieces = a.d * (int)sizeof(T) / 16;

  ar_u4 qf[MT][STEPS];
  int ti[MT];   // drafted token of the lane's query
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(row0 + 16 * m + col, M - 1);
    ti[m] = row % a.t;
    ar_row(q + (int64_t)row * a.d, quad, pieces, qf[m]);
  }
  ar_f4 o[MT][VW] = {};
  float top[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = kTrNone;
    sum[m] = 0.0f;
  }
  const int cached = (len + KT - 1) / KT, tiles = cached + (a.t + KT - 1) / KT;
  const int per = (tiles + a.S - 1) / a.S;
  const int end = min(tiles, (split + 1) * per);
  bool odd = false;
  for (int tile = split * per + __builtin_amdgcn_readfirstlane(wave); tile < end; tile += kTrWaves) {
    const bool draft = tile >= cached;
    const int first = (draft ? tile - cached : tile) * KT;
    const int valid = min(KT, (draft ? a.t : len) - first);
    const int64_t step = draft ? a.d : a.kv_r;
    const T* kt = (draft ? kn : kc) + first * step;
    const T* vt = (draft ? vn : vc) + first * step;
    ar_u4 kf[NU][STEPS];
#pragma unroll
    for (int u = 0; u < NU; ++u)
      ar_row(kt + min((col >> 2) * NE + 4 * u + (col & 3), valid - 1) * step, quad, pieces, kf[u]);
    TreeV<T, VW> v[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e].load(vt + min(quad * NE + e, valid - 1) * step, col, a.d);

    float p[MT][NE];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        ar_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) s = ar_step<T>(kf[u][c], qf[m][c], s);
#pragma unroll
        for (int r = 0; r < 4; ++r) p[m][4 * u + r] = s[r];
      }
    const bool whole = !draft && valid == KT;
    if (!whole) {
      // (every byte is read, from a place that exists, and then counts or not: reading under a condition compiled to a
      // branch per key, in which the masked score was lost)
      const uint8_t* seen = a.mask + b * a.mask_b + (draft ? first : 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int key = quad * NE + e;
          const uint32_t byte = seen[(int64_t)ti[m] * a.t + (draft ? min(key, valid - 1) : 0)];
          const bool sees = (key < valid) & (!draft | (byte != 0));
          p[m][e] = sees ? p[m][e] : -INFINITY;
        }
    }
    bool more = false;
    float high[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float x = p[m][0];
#pragma unroll
      for (int e = 1; e < NE; ++e) x = fmaxf(x, p[m][e]);
      high[m] = ar_quad_max(x) * a.scale_log2e;
      more = more || high[m] > top[m] + kTrSlack;
    }
    if (__ballot(more)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float now = fmaxf(top[m], high[m]);
        const float f = ar_exp2(top[m] - now);
        top[m] = now;
        sum[m] *= f;
#pragma unroll
        for (int j = 0; j < VW; ++j) o[m][j] *= f;
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        p[m][e] = ar_exp2(fmaf(p[m][e], a.scale_log2e, -top[m]));
        sum[m] += p[m][e];
      }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < NE; ++e)
#pragma unroll
        for (int w = 0; w < TreeV<T, VW>::DW; ++w) {
          if (quad * NE + e >= valid) v[e].w[w] = 0;   // (a row that stands for one beyond the end)
          // queries that do not see a drafted token must not meet what its V holds: the joining launch adds that
          if (draft) odd = tree_clean<T>(v[e].w[w]) || odd;
        }
    }
    Tile::add(v, p, o);
  }

  // the four waves' sums, each over its own keys, to one maximum and together
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    sum[m] = ar_quad_sum(sum[m]);
    if (quad == 0) {
      ml[wave][m][col][0] = top[m];
      ml[wave][m][col][1] = sum[m];
    }
  }
  const int64_t at = (int64_t)unit * a.row_blocks + rb;
  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) a.odd[at] = odd;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    float all = ml[0][m][col][0];
#pragma unroll
    for (int w = 1; w < kTrWaves; ++w) all = fmaxf(all, ml[w][m][col][0]);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kTrWaves; ++w) total += ml[w][m][col][1] * ar_exp2(ml[w][m][col][0] - all);
    const float f = ar_exp2(top[m] - all);
#pragma unroll
    for (int j = 0; j < VW; ++j) o[m][j] *= f;
    if (wave == 0 && quad == 0 && row0 + 16 * m + col < M) {
      float* dst = a.part_ml + (at * MT + m) * 32 + col * 2;
      dst[0] = all;
      dst[1] = total;
    }
  }
  for (int j0 = 0; j0 < VW; j0 += JC) {
    // (the block number is compared, so that o stays in registers)
#pragma unroll
    for (int j = 0; j < VW; ++j)
      if (j >= j0 && j < j0 + JC) {
#pragma unroll
        for (int m = 0; m < MT; ++m) joint[wave][m * JC + (j & (JC - 1))][lane] = o[m][j];
      }
    __syncthreads();
    for (int s = wave; s < MT * JC; s += kTrWaves) {
      ar_f4 x = joint[0][s][lane];
#pragma unroll
      for (int w = 1; w < kTrWaves; ++w) x += joint[w][s][lane];
      const int m = s / JC, j = j0 + s % JC;
      if (row0 + 16 * m + col < M) ((ar_f4*)a.part)[((at * MT + m) * VW + j) * kWave + lane] = x;
    }
    __syncthreads();
  }
}

// One workgroup per 16 queries of a cache head joins the S parts: wave -> (block j of the output, group of splits).
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kTrCombThreads) void tree_join_kernel(TreeArgs a) {
  constexpr int VW = DP / 16, NW = kTrCombThreads / kWave, G = NW / VW;
  __shared__ float f_s[kTrMaxSplits][16];
  __shared__ float red[kTrCombThreads / 16][16];
  __shared__ float top_s[16], sum_s[16];
  __shared__ ar_f4 joint[NW][kWave];
  const int lane = lane_id(), wave = wave_id(), col = lane & 15;
  const int rb = (int)blockIdx.x / MT % a.row_blocks, m = (int)blockIdx.x % MT, head = (int)blockIdx.x / MT / a.row_blocks;
  const int gc = a.hq / a.hc, M = gc * a.t, row0 = rb * 16 * MT + 16 * m;
  if (row0 >= M) return;
  const int64_t at0 = (int64_t)head * a.S * a.row_blocks + rb;   // + split * row_blocks
  const int c = threadIdx.x & 15, s0 = threadIdx.x >> 4;
  const bool mine = row0 + c < M;
  float top = kTrNone;
  bool odd = false;
  for (int s = s0; s < a.S; s += kTrCombThreads / 16) {
    odd = odd || a.odd[at0 + (int64_t)s * a.row_blocks];
    const float x = mine ? a.part_ml[((at0 + (int64_t)s * a.row_blocks) * MT + m) * 32 + c * 2] : kTrNone;
    f_s[s][c] = x;
    top = fmaxf(top, x);
  }
  red[s0][c] = top;
  odd = __syncthreads_or(odd);
  if (threadIdx.x < 16) {
    float x = red[0][c];
    for (int i = 1; i < min(a.S, kTrCombThreads / 16); ++i) x = fmaxf(x, red[i][c]);
    top_s[c] = x;
  }
  __syncthreads();
  float total = 0.0f;
  for (int s = s0; s < a.S; s += kTrCombThreads / 16) {
    const float f = ar_exp2(f_s[s][c] - top_s[c]);
    f_s[s][c] = f;
    if (mine) total += f * a.part_ml[((at0 + (int64_t)s * a.row_blocks) * MT + m) * 32 + c * 2 + 1];
  }
  red[s0][c] = total;
  __syncthreads();
  if (threadIdx.x < 16) {
    float x = red[0][c];
    for (int i = 1; i < min(a.S, kTrCombThreads / 16); ++i) x += red[i][c];
    sum_s[c] = x;
  }
  __syncthreads();
  {
    const int j = wave % VW, g = wave / VW;
    ar_f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row0 + col < M) {
#pragma unroll 8
      for (int s = g; s < a.S; s += G)
        x += ((const ar_f4*)a.part)[(((at0 + (int64_t)s * a.row_blocks) * MT + m) * VW + j) * kWave + lane] * f_s[s][col];
    }
    joint[wave][lane] = x;
  }
  __syncthreads();
  const int64_t row = (int64_t)head * M + row0;   // rows of all heads follow each other
  for (int e = threadIdx.x; e < 16 * DP; e += kTrCombThreads) {
    const int r = e / DP, x = e % DP;
    if (x >= a.d || row0 + r >= M) continue;
    const int j = x % VW, at = x / VW;   // output rows 4 quad + i of block j
    float v = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) v += joint[g * VW + j][(at >> 2) * 16 + r][at & 3];
    if (odd) {
      const int b = head / a.hc, hn = head % a.hc / (a.hc / a.hn);
      const T* vn = (const T*)a.v_new + ((int64_t)b * a.hn + hn) * a.t * a.d + x;
      const uint8_t* sees = a.mask + b * a.mask_b + (int64_t)((row0 + r) % a.t) * a.t;
      for (int i = 0; i < a.t; ++i) {
        const float y = ld_f32(vn, (int64_t)i * a.d);
        if (sees[i] && !(fabsf(y) < INFINITY)) v += y;
      }
    }
    st_f32((T*)a.out, (row + r) * a.d + x, sum_s[r] == 0.0f ? 0.0f : v / sum_s[r]);
  }
  if (a.lse && threadIdx.x < 16 && mine)
    a.lse[row + c] = sum_s[c] == 0.0f ? -INFINITY : (top_s[c] + log2f(sum_s[c])) * kLn2;
}

// How a call is cut up, from its sizes alone.
struct TreePlan {
  int dp, mt, row_blocks, S, units;
  int64_t part, ml, odd;   // words of 4 bytes
};
static TreePlan tree_plan(int b, int hq, int hc, int t, int64_t n, int d, int dtype) {
  TreePlan p;
  p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t M = (int64_t)(hq / hc) * t;
  p.mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  if (p.dp == 256) p.mt = std::min(p.mt, dtype == LRQK_BF16 ? 2 : 1);   // (more queries' sums would not fit the registers)
  p.row_blocks = (int)((M + 16 * p.mt - 1) / (16 * p.mt));
  const int kt = dtype == LRQK_BF16 ? 32 : 16;
  const int64_t tiles = (n + kt - 1) / kt + (t + kt - 1) / kt;
  const int64_t heads = (int64_t)b * hc;
  // two workgroups per CU, four tiles for each of a workgroup's waves at least
  int64_t S = std::max<int64_t>(1, 512 / (heads * p.row_blocks));
  S = std::min<int64_t>(S, (tiles + 4 * kTrWaves - 1) / (4 * kTrWaves));
  p.S = (int)std::max<int64_t>(1, std::min<int64_t>(S, kTrMaxSplits));
  p.units = (int)(heads * p.S);
  const int64_t groups = (int64_t)p.units * p.row_blocks * p.mt;
  p.part = groups * 16 * p.dp;
  p.ml = groups * 32;
  p.odd = (int64_t)p.units * p.row_blocks;
  return p;
}

template <typename T, int DP, int MT>
static int tree_launch(const TreeArgs& a, hipStream_t st) {
  const int64_t grid = (int64_t)(a.units + 7) / 8 * 8 * a.row_blocks;
  hipLaunchKernelGGL((tree_part_kernel<T, DP, MT>), dim3((unsigned)grid), dim3(kTrThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL((tree_join_kernel<T, DP, MT>), dim3((unsigned)(a.units / a.S * a.row_blocks * MT)), dim3(kTrCombThreads), 0, st,
                     a);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
template <typename T, int DP>
static int tree_launch_mt(const TreeArgs& a, int mt, hipStream_t st) {
  if constexpr (DP == 256) {
    if constexpr (sizeof(T) == 2)
      if (mt == 2) return tree_launch<T, DP, 2>(a, st);
    return tree_launch<T, DP, 1>(a, st);
  } else {
    if (mt == 1) return tree_launch<T, DP, 1>(a, st);
    if (mt == 2) return tree_launch<T, DP, 2>(a, st);
    return tree_launch<T, DP, 4>(a, st);
  }
}
template <typename T>
static int tree_launch_dp(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
  if (p.dp == 32) return tree_launch_mt<T, 32>(a, p.mt, st);
  if (p.dp == 64) return tree_launch_mt<T, 64>(a, p.mt, st);
  if (p.dp == 128) return tree_launch_mt<T, 128>(a, p.mt, st);
  return tree_launch_mt<T, 256>(a, p.mt, st);
}

static int tree_check(int b, int hq, int hc, int t, int64_t n, int d, int dtype) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(b > 0 && hq > 0 && hc > 0 && t > 0 && n >= 0 && d > 0, LRQK_EINVAL, "bad sizes b=%d hq=%d hc=%d t=%d n=%lld d=%d", b,
               hq, hc, t, (long long)n, d);
  LRQK_REQUIRE(hq % hc == 0, LRQK_EINVAL, "%d query heads over %d cache heads", hq, hc);
  LRQK_REQUIRE(d * (int)elem_size(dtype) % 16 == 0 && d <= 256, LRQK_ELIMIT,
               "head_dim %d unsupported (rows of whole 16-byte pieces, at most 256 elements)", d);
  LRQK_REQUIRE(t <= 1024 && n <= (1 << 30) && (int64_t)b * hq <= 65535, LRQK_ELIMIT,
               "t=%d (at most 1024), n=%lld (2^30), b * hq=%lld (65535)", t, (long long)n, (long long)b * hq);
  return LRQK_OK;
}

}  // namespace lrqk

using namespace lrqk;

extern "C" int64_t lrqk_tree_attention_workspace(int b, int hq, int hc, int t, int64_t n, int d, int dtype) {
  const int rc = tree_check(b, hq, hc, t, n, d, dtype);
  if (rc) return rc;
  const TreePlan p = tree_plan(b, hq, hc, t, n, d, dtype);
  return (p.part + p.ml + p.odd) * (int64_t)sizeof(float);
}

extern "C" int lrqk_tree_attention(const void* q, const void* k_cache, const void* v_cache, int64_t kv_batch_stride,
                                   int64_t kv_head_stride, int64_t kv_row_stride, int64_t n, const int32_t* lengths,
                                   const void* k_new, const void* v_new, const uint8_t* mask, int64_t mask_batch_stride, void* out,
                                   float* lse, int b, int hq, int hc, int hn, int t, int d, float scale, void* workspace,
                                   int64_t workspace_bytes, int dtype, void* stream) {
  int rc = tree_check(b, hq, hc, t, n, d, dtype);
  if (rc) return rc;
  LRQK_REQUIRE(hn > 0 && hc % hn == 0, LRQK_EINVAL, "%d cache heads over %d heads of drafted tokens", hc, hn);
  LRQK_REQUIRE(q && k_new && v_new && mask && out && workspace && (n == 0 || (k_cache && v_cache)), LRQK_EINVAL, "null pointer");
  LRQK_REQUIRE(scale > 0.0f && scale < INFINITY, LRQK_EINVAL, "scale=%g has to be positive and finite", (double)scale);
  const int vec = 16 / (int)elem_size(dtype);
  LRQK_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k_cache % 16 == 0 && (uintptr_t)v_cache % 16 == 0 && (uintptr_t)k_new % 16 == 0 &&
                   (uintptr_t)v_new % 16 == 0 && (uintptr_t)workspace % 16 == 0 && kv_batch_stride % vec == 0 &&
                   kv_head_stride % vec == 0 && kv_row_stride % vec == 0,
               LRQK_EINVAL, "pointers and rows must be 16-byte aligned");
  const TreePlan p = tree_plan(b, hq, hc, t, n, d, dtype);
  const int64_t need = (p.part + p.ml + p.odd) * (int64_t)sizeof(float);
  LRQK_REQUIRE(workspace_bytes >= need, LRQK_EINVAL, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes,
               (long long)need);
  TreeArgs a{q, k_cache, v_cache, k_new, v_new, mask, lengths, out, lse, (float*)workspace, (float*)workspace + p.part,
             (int32_t*)workspace + p.part + p.ml,
             kv_batch_stride, kv_head_stride, kv_row_stride, mask_batch_stride, (int)n, hq, hc, hn, t, d, p.S, p.row_blocks, p.units,
             scale * kLog2e};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LRQK_F32) return tree_launch_dp<float>(a, p, st);
  return tree_launch_dp<bf16_t>(a, p, st);
}
