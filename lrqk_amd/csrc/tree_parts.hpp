// What the attention of drafted tokens is made of, over a cache in the activations' type and over one in 8 bits: rows of V as
// the operand that they lie in, products of tiles, masks, and the joining of what waves and workgroups have.
#pragma once
#include <algorithm>
#include <type_traits>

#include "attn_rows.hpp"

namespace lrqk {

constexpr int kTrWaves = 4, kTrThreads = kTrWaves * kWave;
constexpr int kTrMaxSplits = 256;
constexpr int kTrLong = 512;          // tiles of a split, at most, for each row block (tree_plan)
constexpr float kTrNone = -3.0e38f;   // running maximum of a query that has seen no key yet
constexpr float kTrMuch = 4096.0f;    // a lane's probabilities of a tile may add up to this before the maximum is looked for

struct TreeArgs {
  const void *q, *k, *v, *k_new, *v_new;
  const uint8_t* mask;
  const int32_t* lengths;   // or null: n each
  void* out;
  float* lse;               // or null
  float *part, *part_ml;    // of 16 queries of a split: VW float4 a lane, and of each query the maximum, the sum and that of
                            // the probabilities as they were multiplied (3 x 16)
  int32_t* odd;             // per workgroup of a split: whether its drafted rows of V hold infinities or NaN
  int32_t* cut;             // of a sequence: the number of its first split, and how many it has
  int64_t kv_b, kv_h, kv_r; // elements between sequences, heads and rows of the cache
  int64_t mask_b;
  // splits: of all sequences together, for a cache head; least: tiles of a split, at least; rows: of a row block
  // most: tiles of a split, at most
  int b, n, hq, hc, hn, t, d, splits, least, most, row_blocks, rows, row_tiles, units;
  float scale_log2e;
};

template <typename V>
__device__ __forceinline__ V tree_at(const void* base, uint32_t bytes) {   // (an address of the wave's and 32 bits of the lane's)
  return *reinterpret_cast<const V*>((const char*)base + bytes);
}

// One row's part of V for a lane: elements VW i .. (of a head's d; what is beyond them is something that is not used).
template <typename T, int VW>
struct TreeV {
  static constexpr int DW = VW * (int)sizeof(T) / 4;
  uint32_t w[DW];
  // bytes from the row's beginning to piece p of the lane
  static __device__ __forceinline__ uint32_t place(int i, int d, int p) {
    if constexpr (DW >= 4) return 16u * (uint32_t)min(i * (DW / 4) + p, d * (int)sizeof(T) / 16 - 1);
    return i * DW < d * (int)sizeof(T) / 4 ? 4u * (uint32_t)(i * DW) : 0u;
  }
  // (places: the lane's pieces, as above)
  __device__ __forceinline__ void load(const void* base, uint32_t row, const uint32_t (&places)[DW >= 4 ? DW / 4 : 1]) {
    if constexpr (DW >= 4) {
#pragma unroll
      for (int p = 0; p < DW / 4; ++p) {
        const ar_u4 x = tree_at<ar_u4>(base, row + places[p]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * p + e] = x[e];
      }
    } else if constexpr (DW == 2) {
      const ar_u2 x = tree_at<ar_u2>(base, row + places[0]);
      w[0] = x[0];
      w[1] = x[1];
    } else {
      w[0] = tree_at<uint32_t>(base, row + places[0]);
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

// Eight probabilities as the sum of two bf16 operands: the upper half of each number, and what that leaves, rounded (16 bits
// in all).  Cut off rather than rounded, the first takes half the instructions.
typedef float tr_f8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void tree_split(const float (&p)[8], ar_bf8& hi, ar_bf8& lo) {
  ar_u4 h;
  tr_f8 rest;
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __builtin_amdgcn_perm(__float_as_uint(p[2 * e + 1]), __float_as_uint(p[2 * e]), 0x07060302u);
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = p[e] - __uint_as_float(__float_as_uint(p[e]) & 0xffff0000u);   // exact
  hi = __builtin_bit_cast(ar_bf8, h);
  lo = __builtin_convertvector(rest, ar_bf8);
}

typedef short tr_v4s __attribute__((ext_vector_type(4)));
typedef tr_v4s __attribute__((address_space(3))) * tr_lds_v4s;

template <typename T, int DP, int MT>
struct TreeTile {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int NU = BF ? 2 : 1;             // 16-key blocks of a tile
  static constexpr int KT = 16 * NU, NE = 4 * NU;   // keys of a tile, and of a quad in it
  static constexpr int STEPS = DP * (int)sizeof(T) / 64;
  static constexpr int VW = DP / 16;
  static constexpr int CH = 4 * STEPS;              // 16-byte pieces of a row
  static constexpr int KL = KT * CH / kWave;        // loads of a wave for the tile's rows of K

  // A row of K is kept in LDS where the operand that has it looks: the 16 rows of block u, row m of them with key
  // (m / 4) NE + 4 u + m % 4.
  static __device__ __forceinline__ int place(int key) { return (key % NE) / 4 * 16 + key / NE * 4 + key % 4; }

  // o[j] += v_j^T p for the keys of the tile; p[e]: probability of the quad's key e for the lane's query
  static __device__ __forceinline__ void add(const TreeV<T, VW> (&v)[NE], const float (&p)[MT][NE], ar_f4 (&o)[MT][VW]) {
    if constexpr (BF) {
      ar_bf8 hi[MT], lo[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) tree_split(p[m], hi[m], lo[m]);
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
// Takes what a query does not see out of a tile that is not a whole one of the cache.
template <int MT, int NE>
__device__ __forceinline__ void tree_mask(float (&p)[MT][NE], const TreeArgs& a, int b, const int (&ti)[MT], int quad, int valid,
                                          bool draft, int first) {
  // The bytes are read, from a place that exists, and then count or not.  As if (key >= valid || (draft && !seen[key])) p = -inf
  // the assignment is lost (clang 22 of ROCm 7.2.0): the scores are elements of a vector, the compiler makes the vector with
  // -inf in front of the condition, and in the block of the inner one it copies the unmasked vector over it, for the lanes
  // that see the key and for those that do not.  All that is left of the assignment is an empty block, which
  // tests/test_csrc_cpu.py looks for in the whole library.  Conditions of & and | have no blocks.  (1024 drafts alone: a quad's
  // bytes in one load 78 us, one by one 99.)
  static_assert(NE == 4 || NE == 8, "bytes of a word");
  const uint8_t* masks = a.mask + b * a.mask_b;
  const int key0 = quad * NE;   // the lane's first key of the tile
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint8_t* seen = masks + (int64_t)ti[m] * a.t;
    uint64_t bytes = 0;
    if (a.t >= NE) {
      const int at = draft ? min(first + key0, a.t - NE) : 0;
      if constexpr (NE == 8) {
        __builtin_memcpy(&bytes, seen + at, 8);
      } else {
        uint32_t four;
        __builtin_memcpy(&four, seen + at, 4);
        bytes = four;
      }
      bytes >>= 8 * (draft ? min(first + key0 - at, NE - 1) : 0);   // (further ones have no key in sight)
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e) bytes |= (uint64_t)seen[draft ? min(first + key0 + e, a.t - 1) : 0] << (8 * e);
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const bool sees = (key0 + e < valid) & (!draft | (((uint32_t)(bytes >> (8 * e)) & 0xffu) != 0));
      p[m][e] = sees ? p[m][e] : -INFINITY;
    }
  }
}

// The four waves' sums, each over its own keys, to one maximum and together, and into the scratch as the part of row block
// `rb` of a unit of the grid.  JC: output blocks that the waves join at a time (two barriers each).  smem: room for kTrWaves x
// JC MT x 64 pieces of 16 bytes, which no wave reads any more behind the first barrier here.
template <int MT, int VW, int JC>
__device__ __forceinline__ void tree_leave(const TreeArgs& a, ar_f4 (&o)[MT][VW], const float (&top)[MT], float (&sum)[MT], bool odd,
                                           int unit, int rb, int M, ar_u4* smem, float (*ml)[MT][16][2]) {
  const int lane = lane_id(), wave = wave_id(), col = lane & 15, quad = lane >> 4, row0 = rb * 16 * MT;
  __syncthreads();
  ar_f4(*joint)[MT * JC][kWave] = (ar_f4(*)[MT * JC][kWave])smem;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    sum[m] = ar_quad_sum(sum[m]);
    if (quad == 0) {
      ml[wave][m][col][0] = top[m];
      ml[wave][m][col][1] = sum[m];
    }
  }
  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) a.odd[(int64_t)unit * a.row_blocks + rb] = odd;
  const int64_t tile16 = (int64_t)unit * a.row_tiles + row0 / 16;
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
      float* dst = a.part_ml + (tile16 + m) * 48 + col;
      dst[0] = all;
      dst[16] = dst[32] = total;
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
      if (row0 + 16 * m + col < M) ((ar_f4*)a.part)[((tile16 + m) * VW + j) * kWave + lane] = x;
    }
    __syncthreads();
  }
}

// Blocks of 16 elements of the head that a workgroup of the join has.
constexpr int tree_join_blocks(int blocks, int threads) { return threads == 512 && blocks > 4 ? 4 : blocks; }

// A workgroup joins the splits' parts of 16 queries of a cache head, VB blocks of a quad of the lanes that hold them (a
// quarter of the head): 16 threads with a query each for (block j, every G-th split).  SHARED: which of the two kernels left
// the parts, whose lanes have other elements.  Its time is a chain of reads that wait for each other and barriers, so the
// reads are few in a row, and what 16 queries of all waves make is added up by every thread that wants it.
template <typename T, int DP, bool SHARED, int THREADS>
static __global__ __launch_bounds__(THREADS) void tree_join_kernel(TreeArgs a) {   // (static: each file that includes this has its own)
  constexpr int VW = DP / 16, VB = tree_join_blocks(VW, THREADS), JS = VW / VB;
  constexpr int GROUPS = THREADS / 16, G = GROUPS / VB, FIRST = 4, NW = THREADS / kWave;
  __shared__ float f_s[kTrMaxSplits][16];
  __shared__ float red[3][NW][16];
  __shared__ ar_f4 joint[G][VB][16];
  const int col = threadIdx.x & 15, group = threadIdx.x >> 4, wave = wave_id();
  const int quad = (int)blockIdx.x & 3, j0 = (int)(blockIdx.x >> 2) % JS * VB, place = (int)(blockIdx.x >> 2) / JS;
  const int tile = place % a.row_tiles, head = place / a.row_tiles;
  const int M = a.hq / a.hc * a.t, row0 = 16 * tile, b = head / a.hc;
  const int slot0 = a.b == 1 ? 0 : a.cut[2 * b], slots = a.units / a.hc;
  const int64_t unit0 = (int64_t)slot0 * a.hc + head % a.hc;   // + split * hc
  const bool mine = row0 + col < M;
  // (the first parts are asked for before it is known how many there are: the scratch has room for `slots`, and what is
  // behind the sequence's is not looked at)
  const int j = group % VB, g = group / VB;
  const ar_f4* part = (const ar_f4*)a.part + ((unit0 * a.row_tiles + tile) * VW + j0 + j) * kWave + quad * 16 + col;
  const int64_t next = (int64_t)a.hc * a.row_tiles * VW * kWave;
  const float* ml = a.part_ml + (unit0 * a.row_tiles + tile) * 48 + col;
  const int64_t ml_next = (int64_t)a.hc * a.row_tiles * 48;
  const int32_t* odd_at = a.odd + unit0 * a.row_blocks + row0 / a.rows;
  ar_f4 early[FIRST];
#pragma unroll
  for (int i = 0; i < FIRST; ++i) early[i] = part[min(g + i * G, slots - 1 - slot0) * next];
  // maximum, sums and flag of the thread's first split
  const int s1 = min(group, slots - 1 - slot0);
  const float top1 = ml[s1 * ml_next], sum1 = ml[s1 * ml_next + 16], norm1 = ml[s1 * ml_next + 32];
  const int odd1 = odd_at[(int64_t)s1 * a.hc * a.row_blocks];
  const int S = a.cut[2 * b + 1];
  float top = (mine & (group < S)) ? top1 : kTrNone;
  bool odd = (group < S) & (odd1 != 0);
  for (int s = group + GROUPS; s < S; s += GROUPS) {
    odd = odd | (odd_at[(int64_t)s * a.hc * a.row_blocks] != 0);
    top = fmaxf(top, mine ? ml[s * ml_next] : kTrNone);
  }
  top = ar_quad_max(top);
  if (lane_id() < 16) red[0][wave][col] = top;
  odd = __syncthreads_or(odd);
#pragma unroll
  for (int w = 0; w < NW; ++w) top = fmaxf(top, red[0][w][col]);
  float total = 0.0f, norm = 0.0f;
  if (group < S) {
    const float f = mine ? ar_exp2(top1 - top) : 0.0f;
    f_s[group][col] = f;
    total = mine ? f * sum1 : 0.0f;
    norm = mine ? f * norm1 : 0.0f;
  }
  for (int s = group + GROUPS; s < S; s += GROUPS) {
    const float f = mine ? ar_exp2(ml[s * ml_next] - top) : 0.0f;
    f_s[s][col] = f;
    if (mine) {
      total += f * ml[s * ml_next + 16];
      norm += f * ml[s * ml_next + 32];
    }
  }
  total = ar_quad_sum(total);
  norm = ar_quad_sum(norm);
  if (lane_id() < 16) {
    red[1][wave][col] = total;
    red[2][wave][col] = norm;
  }
  __syncthreads();
  ar_f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
  if (mine) {
#pragma unroll
    for (int i = 0; i < FIRST; ++i)
      if (g + i * G < S) x += early[i] * f_s[g + i * G][col];
#pragma unroll 4
    for (int s = g + FIRST * G; s < S; s += G) x += part[s * next] * f_s[s][col];
  }
  joint[g][j][col] = x;
  __syncthreads();
  const int64_t row = (int64_t)head * M + row0;   // rows of all heads follow each other
  for (int e = threadIdx.x; e < 16 * 4 * VB; e += THREADS) {
    const int r = e / (4 * VB), y = e % (4 * VB);
    const int blk = SHARED ? y / 4 : y % VB, i = SHARED ? y % 4 : y / VB;
    const int d = SHARED ? 16 * (j0 + blk) + 4 * quad + i : 4 * VW * quad + VW * i + j0 + blk;
    if (d >= a.d || row0 + r >= M) continue;
    float v = 0.0f, all = 0.0f;
#pragma unroll
    for (int h = 0; h < G; ++h) v += joint[h][blk][r][i];
#pragma unroll
    for (int w = 0; w < NW; ++w) all += red[2][w][r];
    if (odd) {
      const int hn = head % a.hc / (a.hc / a.hn);
      const T* vn = (const T*)a.v_new + ((int64_t)b * a.hn + hn) * a.t * a.d + d;
      const uint8_t* sees = a.mask + b * a.mask_b + (int64_t)((row0 + r) % a.t) * a.t;
      for (int k = 0; k < a.t; ++k) {
        const float z = ld_f32(vn, (int64_t)k * a.d);
        if (sees[k] && !(fabsf(z) < INFINITY)) v += z;
      }
    }
    st_f32((T*)a.out, (row + r) * a.d + d, all == 0.0f ? 0.0f : v / all);
  }
  if (a.lse && quad == 0 && j0 == 0 && threadIdx.x < 16 && mine) {
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += red[1][w][col];
    a.lse[row + col] = all == 0.0f ? -INFINITY : (top + log2f(all)) * kLn2;
  }
}
// (few workgroups: more threads for the splits of each, and more workgroups.  Of 64 workgroups 6.5 us instead of 10, of 256
// 10.3 instead of 12.6; of 1024 13.4 instead of 9.9)
template <typename T, int DP, bool SHARED>
static void tree_join_launch(const TreeArgs& a, dim3 grid, hipStream_t st) {
  if (grid.x <= 512)
    hipLaunchKernelGGL((tree_join_kernel<T, DP, SHARED, 512>), dim3(grid.x * (DP / 16 / tree_join_blocks(DP / 16, 512))), dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((tree_join_kernel<T, DP, SHARED, 256>), grid, dim3(256), 0, st, a);
}

}  // namespace lrqk
