// Attention over a cache held in 8 bits (byte_cache.hpp): the t tokens of a query head attend to the cached ones, all of them,
// and to each other as a mask says,
//
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  k_j = s_B c_j,  v_j = s'_B c'_j  for the tokens j of a block B.
//
// A block's scale leaves the sums: scores are (q_i.c_j) s_B, and o += s'_B (sum over the block of p_ij c'_j), one product an
// element of o for 64 keys.  Codes are whole numbers up to 127 or e4m3 numbers, both exact in fp16, so fp16 products take
// them, and probabilities of 11 bits where bf16 would have 8.  A query is scaled by a power of two to where fp16 holds it
// (bf16 ones exactly but for elements 2^-28 of the largest; fp32 ones as the sum of two fp16 numbers, as their probabilities).
// Probabilities are formed 2^8 too large, so that those of 2^-22 of the largest keep all bits and those of 2^-33 are not lost.
// (Of more than 64 bf16 queries a cache head less: where a block's scale of V is 2^-n of another one's near it, n up to 9, its
// probabilities are 2^n smaller, full to 2^(n-22) and lost beyond 2^(n-33); they are sums' parts in fp32 all the same.)
//
// As in tree_attention.hip a query is a lane's column of S^T = C Q^T, and the probabilities are the operand of O^T = C'^T P^T
// as they lie: row m of the i-th 16 keys of a block is key 16 (m / 4) + 4 i + m % 4, so that a quad's scores are those of 16
// successive keys, whose codes of an element of V are the 16 bytes that the same quad loads.  Nothing passes through LDS.
// The tokens that are not in a complete block, and the drafted ones, are multiplied in their own type.
#include "byte_cache.hpp"
#include "tree_parts.hpp"

namespace lrqk {

typedef _Float16 by_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 by_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 by_h4 __attribute__((ext_vector_type(4)));
typedef float by_f8 __attribute__((ext_vector_type(8)));
typedef float by_f4 __attribute__((ext_vector_type(4)));

constexpr float kByUp = 8.0f;          // binary orders that probabilities are formed too large
constexpr float kByMost = 15.0f;       // binary logarithm of the largest one before they are formed anew (fp16 ends at 2^16)
constexpr int kByLong = 256;           // blocks of a split, at most
constexpr float kByLargest = 0x1p24f, kByBelow = 0x1p-60f;   // unit that outputs are held in, at most, and over the largest scale, at least

struct ByteArgs {
  TreeArgs tree;             // queries, drafted tokens, outputs, scratch; n: tokens that the cache has room for
  const void *k, *v;         // codes
  const float *ks, *vs;      // scales
  const void *k_tail, *v_tail;
  int blocks, drafts;        // of a head; drafted tokens: t or none
  bool apart;                // the tokens of no complete block and the drafted ones have a split of their own
};

// Eight codes as fp16 numbers, exactly.
template <bool FP8>
__device__ __forceinline__ by_h8 by_unpack(uint32_t a, uint32_t b) {
  union {
    by_h8 all;
    by_h2 two[4];
  } x;
  if constexpr (FP8) {
    x.two[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
    x.two[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    x.two[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
    x.two[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
  } else {
    // 1024 + u is an fp16 number whose low byte is u, of u = code + 128
    const by_h2 away = {(_Float16)1152.0f, (_Float16)1152.0f};
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    x.two[0] = __builtin_bit_cast(by_h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - away;
    x.two[1] = __builtin_bit_cast(by_h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - away;
    x.two[2] = __builtin_bit_cast(by_h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - away;
    x.two[3] = __builtin_bit_cast(by_h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - away;
  }
  return x.all;
}

__device__ __forceinline__ ar_f4 by_step(by_h8 a, by_h8 b, ar_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Eight numbers as fp16, and what that leaves of them.
template <bool TWO>
__device__ __forceinline__ void by_halves(const float (&x)[8], by_h8& hi, by_h8& lo) {
  by_f8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[e];
  hi = __builtin_convertvector(v, by_h8);
  if constexpr (TWO) lo = __builtin_convertvector(v - __builtin_convertvector(hi, by_f8), by_h8);
}

// Before scores x become probabilities 2^(x f + shift - top); f: of each query.  top is not the maximum so far but what serves
// as one: as long as no probability is above 2^kByMost it stays, and only where one would be it becomes the maximum less
// kByUp, o and the sums rescaled to it.
template <int MT, int NE, int VW>
__device__ __forceinline__ void by_top(const float (&x)[MT][NE], const float (&f)[MT], float shift, float (&top)[MT], float (&sum)[MT],
                                       ar_f4 (&o)[MT][VW]) {
  float high[MT];
  bool more = false;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    high[m] = x[m][0];
#pragma unroll
    for (int e = 1; e < NE; ++e) high[m] = fmaxf(high[m], x[m][e]);
    high[m] = fmaf(high[m], f[m], shift);
    more = more | !(high[m] - top[m] <= kByMost);
  }
  if (__ballot(more)) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float now = fmaxf(top[m], ar_quad_max(high[m]) - kByUp), g = ar_exp2(top[m] - now);
      top[m] = now;
      sum[m] *= g;
#pragma unroll
      for (int j = 0; j < VW; ++j) o[m][j] *= g;
    }
  }
}

// What a wave has of its queries: 16 MT of them, scaled by powers of two into fp16 (up: back, and to the exponents' base), and
// of their outputs.  FOLD: these are held in units of a block's scale of V, and the products add to them as they are: the next
// block's scale over that goes into the probabilities' exponents, as far as it costs fp16 no more than 8 of its bits (2^-8 .. 2);
// one beyond becomes the unit itself.  (A unit that is kept while larger scales come ends in infinities: blocks of zeros have
// 2^-100.)  Far below the largest scale so far, kByBelow, outputs have no room for it in fp32: the products of such a block, as of all
// without FOLD, are multiplied and added.  At most the unit is kByLargest, so that no ratio of a scale to it leaves fp32's
// range.  It pays where the matrix cores bound (256 queries
// over up to 64K of four sequences: 223 us, without 233; 100 over 128K 98 and 101) and costs where loads do, of whose registers
// it needs some (64 over 32K in byte_stream_kernel: 29.4 us, without 27.2; a token over 32K 19.0 and 18.2).  Sums of fp32
// tensors do not take it: the matrix cores cut off what they add to them.
template <typename T, int DP, int MT, bool FOLD>
struct ByteWave {
  static constexpr int VW = DP / 16, CH = DP / 64;
  static constexpr bool TWO = sizeof(T) == 4;
  by_h8 qh[MT][2 * CH], ql[TWO ? MT : 1][2 * CH];   // elements 64 c + 16 quad + 8 h .. in [2 c + h]
  float up[MT], top[MT], sum[MT];
  ar_f4 o[MT][VW];
  float unit, log_unit, most;   // (most: the largest scale so far)

  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] = kTrNone;
      sum[m] = 0.0f;
#pragma unroll
      for (int j = 0; j < VW; ++j) o[m][j] = ar_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    unit = most = 0x1p-100f;   // (the least scale)
    log_unit = -100.0f;
  }
  __device__ __forceinline__ void queries(const T* q, int row0, int M, int d, float scale_log2e) {
    const int col = lane_id() & 15, quad = lane_id() >> 4;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const T* row = q + (int64_t)min(row0 + 16 * m + col, M - 1) * d;
      float x[2 * CH][8], high = 0.0f;
#pragma unroll
      for (int s = 0; s < 2 * CH; ++s) {
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
          const int e = 64 * (s / 2) + 16 * quad + 8 * (s % 2) + N * i;
          Vec16<T> p;
          p.load(row + min(e, d - N));
          float y[N];
          p.unpack(y);
#pragma unroll
          for (int r = 0; r < N; ++r) {
            x[s][N * i + r] = e < d ? y[r] : 0.0f;
            high = fmaxf(high, fabsf(x[s][N * i + r]));
          }
        }
      }
      // a power of two that brings the largest element to 2^14 .. 2^15
      const uint32_t bits = __float_as_uint(fmaxf(ar_quad_max(high), 0x1p-100f)) & 0x7f800000u;   // 2^E
      const float to = __uint_as_float(((127u + 14u + 127u) << 23) - bits);
      up[m] = __uint_as_float(bits) * 0x1p-14f * scale_log2e;
#pragma unroll
      for (int s = 0; s < 2 * CH; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] *= to;
        by_halves<TWO>(x[s], qh[m][s], ql[TWO ? m : 0][s]);
      }
    }
  }
  float x[MT][16];   // scores of a block's keys, key 16 quad + 4 u + r in [4 u + r]
  // Scores of its u-th 16 keys, whose operands are kf.
  __device__ __forceinline__ void scores(int u, const by_h8 (&kf)[2 * CH]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      ar_f4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < 2 * CH; ++s) {
        if constexpr (TWO) c = by_step(kf[s], ql[m][s], c);
        c = by_step(kf[s], qh[m][s], c);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[m][4 * u + r] = c[r];
    }
  }
  // What a block's scales make of its scores and products.
  struct Scales {
    float f[MT], from[MT], less, by;
    bool apart;
  };
  __device__ __forceinline__ Scales scales(float ks, float vs) {
    Scales g;
    float shift = 0.0f;
    if constexpr (FOLD) {
      const float log_vs = __builtin_amdgcn_logf(vs);
      shift = log_vs - log_unit;
      most = fmaxf(most, vs);
      if (shift > 1.0f || (shift < -8.0f && vs >= most * kByBelow)) {
        const float now = fminf(vs, kByLargest), less = unit / now;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < VW; ++j) o[m][j] *= less;
        unit = now;
        log_unit = __builtin_amdgcn_logf(now);
        shift = log_vs - log_unit;
      }
    }
    g.apart = !FOLD || !(shift >= -8.0f && shift <= 1.0f);
    g.less = g.apart ? 1.0f : unit * __builtin_amdgcn_rcpf(vs);
    g.by = FOLD ? vs / unit : vs;
    shift = g.apart ? 0.0f : shift;
#pragma unroll
    for (int m = 0; m < MT; ++m) g.f[m] = up[m] * ks;
    by_top<MT, 16, VW>(x, g.f, shift, top, sum, o);
#pragma unroll
    for (int m = 0; m < MT; ++m) g.from[m] = shift - top[m];
    return g;
  }
  // Probabilities of keys 4 u .. 4 u + 3 of every quad, in p: 16-bit halves of [m][u / 2].
  __device__ __forceinline__ void probabilities(int u, const Scales& g, float (&part)[MT], by_h4 (&ph)[MT][4], by_h4 (&pl)[TWO ? MT : 1][4]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      by_f4 p;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = ar_exp2(fmaf(x[m][4 * u + r], g.f[m], g.from[m]));
        part[m] = u + r == 0 ? p[0] : part[m] + p[r];
      }
      ph[m][u] = __builtin_convertvector(p, by_h4);
      if constexpr (TWO) pl[m][u] = __builtin_convertvector(p - __builtin_convertvector(ph[m][u], by_f4), by_h4);
    }
  }
  // o += of the j-th 16 elements; v0, v1: V's operands of the first and the last 8 keys of every quad
  __device__ __forceinline__ void products(int j, by_h8 v0, by_h8 v1, const Scales& g, const by_h4 (&ph)[MT][4], const by_h4 (&pl)[TWO ? MT : 1][4]) {
    auto both = [](by_h4 a, by_h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); };
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      ar_f4 c = FOLD ? o[m][j] : ar_f4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (TWO) {
        c = by_step(v0, both(pl[m][0], pl[m][1]), c);
        c = by_step(v1, both(pl[m][2], pl[m][3]), c);
      }
      c = by_step(v0, both(ph[m][0], ph[m][1]), c);
      c = by_step(v1, both(ph[m][2], ph[m][3]), c);
      if constexpr (FOLD) {
        o[m][j] = c;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[m][j][r] = fmaf(c[r], g.by, o[m][j][r]);
      }
    }
  }
  // Around the products of a block whose scale is far from any unit (FOLD): what there is waits in memory meanwhile.  (A
  // branch with products of its own costs every block the copying of all outputs from register to register.)
  struct Waiting {
    volatile float o[FOLD ? MT * VW * 4 : 1];
  };
  __device__ __forceinline__ void put_by(const Scales& g, Waiting& w) {
    if constexpr (FOLD)
      if (__builtin_expect(g.apart, 0)) {
#pragma unroll
        for (int i = 0; i < MT * VW * 4; ++i) {
          w.o[i] = o[i / 4 / VW][i / 4 % VW][i % 4];
          o[i / 4 / VW][i / 4 % VW][i % 4] = 0.0f;
        }
      }
  }
  __device__ __forceinline__ void take_up(const Scales& g, Waiting& w) {
    if constexpr (FOLD)
      if (__builtin_expect(g.apart, 0)) {
#pragma unroll
        for (int i = 0; i < MT * VW * 4; ++i) o[i / 4 / VW][i / 4 % VW][i % 4] = fmaf(o[i / 4 / VW][i / 4 % VW][i % 4], g.by, w.o[i]);
      }
  }
  __device__ __forceinline__ void end() {
    if constexpr (FOLD) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < VW; ++j) o[m][j] *= unit;
    }
  }
};

// How the sequences are cut into splits of so many complete blocks each.  What is not in a complete block is a split of its
// own, a sequence's first (apart), or what the last one does when it is through with its blocks.  From the lengths alone, by
// every wave for itself.
struct ByteCut {
  int b, len, split, splits, slot0, per;
  static __device__ __forceinline__ int length(const TreeArgs& a, int b) { return min(max(a.lengths[b], 0), a.n); }
  static __device__ __forceinline__ int share(const TreeArgs& a, int all) {
    return max(a.least, min((int)(((uint32_t)all + (uint32_t)a.splits - 1u) / (uint32_t)a.splits), a.most));
  }
  static __device__ __forceinline__ int parts(int blocks, int per, bool apart) {
    const int n = (blocks + per - 1) / per;
    return apart ? 1 + n : max(n, 1);
  }
  __device__ __forceinline__ bool find(const TreeArgs& a, int slot, bool apart) {
    if (a.b == 1) {
      b = slot0 = 0;
      len = length(a, 0);
      per = share(a, len / kByBlock);
      splits = parts(len / kByBlock, per, apart);
      split = slot;
      return slot < splits;
    }
    const int lane = lane_id();
    int all = 0;   // (blocks of all sequences: by_check holds them below 2^31)
    for (int i = lane; i < a.b; i += kWave) all += length(a, i) / kByBlock;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) all += __shfl_xor(all, off, kWave);
    per = __builtin_amdgcn_readfirstlane(share(a, all));
    int before = 0;
    for (int base = 0; base < a.b; base += kWave) {
      const int i = base + lane;
      const int mine = i < a.b ? parts(length(a, min(i, a.b - 1)) / kByBlock, per, apart) : 0;
      const int end = before + wave_inclusive_sum(mine);
      const unsigned long long hit = __ballot(slot < end);
      if (hit) {
        const int at = __ffsll(hit) - 1;
        b = base + at;
        splits = __builtin_amdgcn_readlane(mine, at);
        slot0 = __builtin_amdgcn_readlane(end, at) - splits;
        split = slot - slot0;
        len = length(a, b);
        return true;
      }
      before = __builtin_amdgcn_readlane(end, kWave - 1);
    }
    return false;
  }
};

// The tokens that are not in a complete block (of the tail) and the drafted ones: every `step`-th tile of them.
template <typename T, int DP, int MT>
__device__ __forceinline__ void by_dense(const ByteArgs& ba, const ByteCut& cut, int hc, int row0, int M, const T* q, int from, int step,
                                         float (&top)[MT], float (&sum)[MT], ar_f4 (&o)[MT][DP / 16], bool& odd) {
  const TreeArgs& a = ba.tree;
  using Tile = TreeTile<T, DP, MT>;
  constexpr int NU = Tile::NU, KT = Tile::KT, NE = Tile::NE, STEPS = Tile::STEPS, VW = Tile::VW, E = (int)sizeof(T);
  constexpr int VP = TreeV<T, VW>::DW >= 4 ? TreeV<T, VW>::DW / 4 : 1;
  const int lane = lane_id(), col = lane & 15, quad = lane >> 4, pieces = a.d * E / 16;
  const int late = cut.len % kByBlock, cached = (late + KT - 1) / KT, tiles = cached + (ba.drafts + KT - 1) / KT;
  const int64_t tail0 = (((int64_t)cut.b * a.hc + hc) * kByTail + (cut.len - late) % kByTail) * a.d;
  const int64_t new0 = ((int64_t)cut.b * a.hn + hc / (a.hc / a.hn)) * a.t * a.d;
  const float f1 = a.scale_log2e;
  float f[MT];
  int ti[MT];   // drafted token of the lane's query
  ar_u4 qf[MT][STEPS];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    f[m] = f1;
    ti[m] = min(row0 + 16 * m + col, M - 1) % a.t;
    ar_row(q + (int64_t)min(row0 + 16 * m + col, M - 1) * a.d, quad, pieces, qf[m]);
  }
  uint32_t vplace[VP];
#pragma unroll
  for (int i = 0; i < VP; ++i) vplace[i] = TreeV<T, VW>::place(col, a.d, i);
  const uint32_t rs = (uint32_t)a.d * E;
  for (int tile = from; tile < tiles; tile += step) {
    const bool draft = tile >= cached;
    const int first = (draft ? tile - cached : tile) * KT, valid = min(KT, (draft ? ba.drafts : late) - first);
    const T* ks = (draft ? (const T*)a.k_new + new0 : (const T*)ba.k_tail + tail0) + (int64_t)first * a.d;
    const T* vs = (draft ? (const T*)a.v_new + new0 : (const T*)ba.v_tail + tail0) + (int64_t)first * a.d;
    TreeV<T, VW> v[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e].load(vs, (uint32_t)min(quad * NE + e, valid - 1) * rs, vplace);
    float x[MT][NE];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      ar_u4 kf[STEPS];
      ar_row((const char*)ks + (uint32_t)min(col / 4 * NE + 4 * u + col % 4, valid - 1) * rs, quad, pieces, kf);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        ar_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) s = ar_step<T>(kf[c], qf[m][c], s);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[m][4 * u + r] = s[r];
      }
    }
    if (draft) {
      tree_mask<MT, NE>(x, a, cut.b, ti, quad, valid, true, first);
    } else {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < NE; ++e) x[m][e] = quad * NE + e < valid ? x[m][e] : -INFINITY;
    }
    by_top<MT, NE, VW>(x, f, 0.0f, top, sum, o);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float part = 0.0f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        x[m][e] = ar_exp2(fmaf(x[m][e], f[m], -top[m]));
        part += x[m][e];
      }
      sum[m] += part;
    }
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int w = 0; w < TreeV<T, VW>::DW; ++w) {
        v[e].w[w] = quad * NE + e < valid ? v[e].w[w] : 0u;   // (a row that stands for one beyond the end)
        // queries that do not see a drafted token must not meet what its V holds: the joining launch adds that
        if (draft) odd = tree_clean<T>(v[e].w[w]) | odd;
      }
    Tile::add(v, x, o);
  }
}

// Where a workgroup is, and whose queries and keys it has.
struct BytePlace {
  int rb, unit, hc, M;
  ByteCut cut;
  __device__ __forceinline__ bool find(const TreeArgs& a, bool apart) {   // false: nothing to do
    // the row blocks of a unit (a split of a head) follow each other 8 workgroups apart: on one XCD, whose L2 then has the
    // codes that the first of them brought
    rb = (int)blockIdx.x % (8 * a.row_blocks) / 8;
    unit = (int)blockIdx.x / (8 * a.row_blocks) * 8 + (int)blockIdx.x % 8;
    if (unit >= a.units || !cut.find(a, unit / a.hc, apart)) return false;
    if (cut.split == 0 && unit % a.hc == 0 && rb == 0 && threadIdx.x == 0) {
      a.cut[2 * cut.b] = cut.slot0;
      a.cut[2 * cut.b + 1] = cut.splits;
    }
    hc = unit % a.hc;
    M = a.hq / a.hc * a.t;
    return true;
  }
};

// Few queries: the four waves of a workgroup take the blocks of its split in turn, each for itself, its codes as operands from
// memory; a block's keys are asked for when the one's before have become scores, its values when those have become products.
// Reading bounds it: a token over 32K (int8, 8 heads of 128, bf16) is 67 MB in 15.2 us, 4.4 TB/s where the largest reads reach
// 5.5, and 16 over 1K .. 8K 158 MB in 31.3 (5.1 TB/s); the joining launch makes them 18 and 43.  Small ones are bound by their
// chain of waits: 7 fp32 queries of 28 heads over 4K, 4.2 MB of codes, take 9.8.  Heads of 256 need more than the 256 registers that two
// waves a SIMD have each (a token over 32K: 37.6 us in all, with two waves 45; fp32 39 and 67).
template <typename T, bool FP8, int DP, int MT>
__global__ __launch_bounds__(kTrThreads, DP == 256 ? 1 : 2) void byte_stream_kernel(ByteArgs ba) {
  const TreeArgs& a = ba.tree;
  using Wave = ByteWave<T, DP, MT, false>;
  constexpr int VW = Wave::VW, CH = Wave::CH;
  constexpr int JC = 8 / MT < VW ? 8 / MT : VW;   // (32 KB; with two blocks at a time a token over 32K took 1.5 us more)
  __shared__ ar_u4 smem[kTrWaves * MT * JC * kWave];
  __shared__ float ml[kTrWaves][MT][16][2];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  BytePlace at;
  if (!at.find(a, ba.apart)) return;
  const ByteCut& cut = at.cut;
  const int row0 = at.rb * 16 * MT;
  const T* q = (const T*)a.q + ((int64_t)cut.b * a.hc + at.hc) * at.M * a.d;
  Wave w;
  w.begin();
  bool odd = false;
  const int before = cut.split - ba.apart;   // splits of blocks in front of this one
  if (before >= 0) {
    const int64_t block0 = ((int64_t)cut.b * a.hc + at.hc) * ba.blocks;
    int block = before * cut.per + wave;
    const int end = min(cut.len / kByBlock, (before + 1) * cut.per);
    // what a lane reads of a block: CH pieces of 4 x 16 keys, and VW pieces of V
    const uint32_t kat = (uint32_t)((col >> 2) * 16 + (col & 3)) * DP + quad * 16, vat = (uint32_t)(VW * col) * kByBlock + quad * 16;
    ar_u4 kg[4][CH], vg[VW];
    float ks_next = 0.0f, vs_next = 0.0f;
    auto load_k = [&](int i) {
      const char* src = (const char*)ba.k + (block0 + i) * (kByBlock * DP);
      ks_next = ba.ks[block0 + i];
      vs_next = ba.vs[block0 + i];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int c = 0; c < CH; ++c) kg[u][c] = tree_at<ar_u4>(src + u * 4 * DP + c * 64, kat);
    };
    auto load_v = [&](int i) {
      const char* src = (const char*)ba.v + (block0 + i) * (kByBlock * DP);
#pragma unroll
      for (int j = 0; j < VW; ++j) vg[j] = tree_at<ar_u4>(src + j * kByBlock, vat);
    };
    if (block < end) {
      load_k(block);
      load_v(block);
      w.queries(q, row0, at.M, a.d, a.scale_log2e);
    }
    for (; block < end; block += kTrWaves) {
      const int next = block + kTrWaves < end ? block + kTrWaves : block;   // (the next one, or this one again)
      const float ks = ks_next, vs = vs_next;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        by_h8 kf[2 * CH];
#pragma unroll
        for (int s = 0; s < 2 * CH; ++s) kf[s] = by_unpack<FP8>(kg[u][s / 2][s % 2 * 2], kg[u][s / 2][s % 2 * 2 + 1]);
        w.scores(u, kf);
      }
      load_k(next);
      const typename Wave::Scales g = w.scales(ks, vs);
      float part[MT];
      by_h4 ph[MT][4], pl[Wave::TWO ? MT : 1][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w.probabilities(u, g, part, ph, pl);
#pragma unroll
      for (int m = 0; m < MT; ++m) w.sum[m] = fmaf(part[m], g.less, w.sum[m]);
#pragma unroll
      for (int j = 0; j < VW; ++j) w.products(j, by_unpack<FP8>(vg[j][0], vg[j][1]), by_unpack<FP8>(vg[j][2], vg[j][3]), g, ph, pl);
      load_v(next);
    }
  }
  if (cut.split == (ba.apart ? 0 : cut.splits - 1))
    by_dense<T, DP, MT>(ba, cut, at.hc, row0, at.M, q, wave, kTrWaves, w.top, w.sum, w.o, odd);
  tree_leave<MT, VW, JC>(a, w.o, w.top, w.sum, odd, at.unit, at.rb, at.M, smem, ml);
}

// Many queries: the four waves have 16 MT of them each and share the blocks.  Each wave makes a quarter of a block's codes
// fp16 operands and leaves them in LDS, in the order in which lanes read them.  While a block's probabilities are formed the
// next one's scores are multiplied, 16 keys at a time into the registers that those 16 leave, since a wave's exponentials and
// products run side by side only if they are next to each other: so LDS has a block's values and the next one's keys, and
// those that follow are written meanwhile; one barrier a block.
//
// What bounds it is what a SIMD has to issue for a block, products, exponentials and reads of LDS, which overlap in part: 256
// queries of each of four sequences over up to 64K, 148K .. 214K tokens in all (int8, 8 heads of 128), are 155 .. 224 GFLOP in
// 207 .. 284 us with the join's 11, 720 .. 800 TFLOP/s (a large product of the library reaches 1075), 100 over 128K 54 in 92.6,
// 580, or 740 with the rows up to 128 that are multiplied too.  The matrix cores are busy a third of all cycles in both.  Two
// waves a SIMD are what registers allow.  64 queries a wave moved
// operands between register files (150 us for the 100), eight waves of a workgroup on the same blocks 210 us for the first and
// 157 for the second, two blocks asked for ahead spilled.
// From 65 queries on: up to 64 the other kernel's waves, which each read the codes, are faster (64 over 32K 27.2 us, here 36.2);
// fp32 queries of long caches and heads of 256 come here from 33 on.
template <typename T, bool FP8, int DP, int MT>
__global__ __launch_bounds__(kTrThreads, 2) void byte_share_kernel(ByteArgs ba) {
  const TreeArgs& a = ba.tree;
  using Wave = ByteWave<T, DP, MT, sizeof(T) == 2 && MT == 2>;
  constexpr int VW = Wave::VW, CH = Wave::CH, VL = VW / kTrWaves;   // pieces of V of a wave (of K: CH)
  __shared__ by_h8 keys[2][4 * 2 * CH][kWave], values[2][VW * 2][kWave];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  BytePlace at;
  if (!at.find(a, true)) return;
  const ByteCut& cut = at.cut;
  const int row0 = (at.rb * kTrWaves + wave) * 16 * MT;
  const T* q = (const T*)a.q + ((int64_t)cut.b * a.hc + at.hc) * at.M * a.d;
  Wave w;
  w.begin();
  bool odd = false;
  if (cut.split == 0) {
    if (row0 < at.M) by_dense<T, DP, MT>(ba, cut, at.hc, row0, at.M, q, 0, 1, w.top, w.sum, w.o, odd);
  } else {
    const int64_t block0 = ((int64_t)cut.b * a.hc + at.hc) * ba.blocks;
    const int begin = (cut.split - 1) * cut.per, last = min(cut.len / kByBlock, begin + cut.per) - 1;   // (a split has a block at least)
    const uint32_t kat = (uint32_t)((col >> 2) * 16 + (col & 3)) * DP + quad * 16, vat = (uint32_t)(VW * col) * kByBlock + quad * 16;
    ar_u4 kg[CH], vg[VL];   // the wave's part of the next keys and values to be written
    auto load_k = [&](int i) {   // (behind the last block it comes again)
      const char* src = (const char*)ba.k + (block0 + min(i, last)) * (kByBlock * DP) + wave * 4 * DP;
#pragma unroll
      for (int c = 0; c < CH; ++c) kg[c] = tree_at<ar_u4>(src + c * 64, kat);
    };
    auto load_v = [&](int i) {
      const char* src = (const char*)ba.v + (block0 + min(i, last)) * (kByBlock * DP) + wave * VL * kByBlock;
#pragma unroll
      for (int j = 0; j < VL; ++j) vg[j] = tree_at<ar_u4>(src + j * kByBlock, vat);
    };
    auto leave_k = [&](int side) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) keys[side][wave * 2 * CH + 2 * c + h][lane] = by_unpack<FP8>(kg[c][2 * h], kg[c][2 * h + 1]);
    };
    auto leave_v = [&](int side) {
#pragma unroll
      for (int j = 0; j < VL; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) values[side][(wave * VL + j) * 2 + h][lane] = by_unpack<FP8>(vg[j][2 * h], vg[j][2 * h + 1]);
    };
    auto operands = [&](int side, int u, by_h8 (&kf)[2 * CH]) {
#pragma unroll
      for (int s = 0; s < 2 * CH; ++s) kf[s] = keys[side][u * 2 * CH + s][lane];
    };
    load_k(begin);
    load_v(begin);
    w.queries(q, row0, at.M, a.d, a.scale_log2e);
    leave_k(0);
    load_k(begin + 1);
    leave_v(0);
    load_v(begin + 1);
    leave_k(1);
    load_k(begin + 2);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      by_h8 kf[2 * CH];
      operands(0, u, kf);
      w.scores(u, kf);
    }
    __syncthreads();
    // (a block's scales are asked for a block ahead: a wait for them is one for all of LDS's reads too)
    float ks = ba.ks[block0 + begin], vs = ba.vs[block0 + begin];
    for (int block = begin; block <= last; ++block) {
      const int side = (block - begin) & 1;
      const typename Wave::Scales g = w.scales(ks, vs);
      ks = ba.ks[block0 + min(block + 1, last)];
      vs = ba.vs[block0 + min(block + 1, last)];
      typename Wave::Waiting put;
      w.put_by(g, put);
      float part[MT];
      by_h4 ph[MT][4], pl[Wave::TWO ? MT : 1][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        by_h8 kf[2 * CH];
        operands(side ^ 1, u, kf);
        w.probabilities(u, g, part, ph, pl);
        w.scores(u, kf);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) w.sum[m] = fmaf(part[m], g.less, w.sum[m]);
      leave_v(side ^ 1);
      load_v(block + 2);
      leave_k(side);
      load_k(block + 3);
#pragma unroll
      for (int j = 0; j < VW; ++j) w.products(j, values[side][2 * j][lane], values[side][2 * j + 1][lane], g, ph, pl);
      w.take_up(g, put);
      __syncthreads();
    }
    w.end();
  }
  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) a.odd[(int64_t)at.unit * a.row_blocks + at.rb] = odd;
  const int64_t tile16 = (int64_t)at.unit * a.row_tiles + row0 / 16;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (row0 + 16 * m + col >= at.M) continue;
    const float sum = ar_quad_sum(w.sum[m]);
    if (quad == 0) {
      float* dst = a.part_ml + (tile16 + m) * 48 + col;
      dst[0] = w.top[m];
      dst[16] = dst[32] = sum;
    }
#pragma unroll
    for (int j = 0; j < VW; ++j) ((ar_f4*)a.part)[((tile16 + m) * VW + j) * kWave + lane] = w.o[m][j];
  }
}

struct BytePlan {
  int dp, mt;
  bool share, apart;
  int rows, row_blocks, row_tiles, splits, least, most, units;
  int64_t part, ml, odd, cut;   // words of 4 bytes
};
static BytePlan byte_plan(int b, int hq, int hc, int t, int64_t blocks, int d, int dtype) {
  BytePlan p;
  p.dp = by_width(d);
  const int64_t M = (int64_t)(hq / hc) * t;
  p.share = M > (p.dp == 256 || (dtype == LRQK_F32 && blocks > 512) ? 32 : 64);
  // 16 queries a wave: all there are, or all that registers have room for; or few blocks, which one workgroup per 16 queries is
  // through sooner (32 queries over 8K: 14.5 us, with 32 a wave 17.1; over 64K 41.5 and 36.5, 64 over 64K 74 and 52)
  p.mt = M <= 16 || p.dp == 256 || dtype == LRQK_F32 || (!p.share && b * hc * blocks <= 2048) ? 1 : 2;
  // Many sequences are enough workgroups without those (64 tokens over 1 .. 1K 35 us, without 30; 48 of 16 over 1K .. 8K 51 and
  // 47, a token of each 44 and 43); of fewer they are done beside the others (8 tokens over 1K .. 8K 25 us, otherwise 26).
  p.apart = p.share || b < 16;
  p.rows = 16 * p.mt * (p.share ? kTrWaves : 1);
  p.row_blocks = (int)((M + p.rows - 1) / p.rows);
  p.row_tiles = p.row_blocks * (p.rows / 16);
  // Workgroups, those of what is not in complete blocks among them: two per CU, which keep each other's time filled.  A single
  // sequence is cut evenly, and of few queries one per CU then reads as fast and leaves less to be joined (a token over 32K:
  // 18 us, with two 21, with three 23); of many sequences with one tile of queries three per CU hide that their lengths differ
  // (16 tokens over 1K .. 8K 42.7 us, with two 44.3, with four 42.4; 32 over up to 2K 26.6, 28.7 and 27.9).
  // Where blocks are shared and a workgroup would have no more than 12 of them, what it leaves costs more than a second one per
  // CU gains (100 queries over 16K, 32K, 64K: 29.8, 38.7, 60.8 us, with one 26.7, 36.6, 63.0); of heads of 256 registers have
  // room for one alone (64 over 64K: 92 us, 82.5).
  const bool one = p.share ? p.dp == 256 || (int64_t)b * hc * blocks * p.row_blocks <= 12 * 512 : b == 1;
  const int wanted = one ? 256 : !p.share && p.mt == 1 && b >= 8 ? 768 : 512;
  p.splits = (int)std::max<int64_t>(b, wanted / ((int64_t)hc * p.row_blocks) - b);
  p.least = (int)std::max<int64_t>(kTrWaves, (blocks + kTrMaxSplits - 2) / (kTrMaxSplits - 1));
  // (where the heads alone fill the GPU: sums of fp32 numbers over no more than kByLong blocks, in splits of one length)
  const int64_t longest = std::max<int64_t>(p.least, kByLong), parts = (blocks + longest - 1) / longest;
  p.most = parts ? (int)((blocks + parts - 1) / parts) : 1;
  p.most = std::max(p.most, p.least);
  const int64_t slots = b + std::min<int64_t>(std::max<int64_t>((int64_t)p.splits + b, b * parts), b * ((blocks + p.least - 1) / p.least));
  p.units = (int)std::min<int64_t>(hc * slots, INT32_MAX);
  const int64_t groups = (int64_t)p.units * p.row_tiles;
  p.part = groups * 16 * p.dp;
  p.ml = groups * 48;
  p.odd = (int64_t)p.units * p.row_blocks;
  p.cut = 2 * (int64_t)b;
  return p;
}

template <typename T, bool FP8, int DP>
static int byte_launch(const ByteArgs& a, const BytePlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)p.units + 7) / 8 * 8 * p.row_blocks));
  constexpr int SHARE = DP < 256 && sizeof(T) == 2 ? 2 : 1;
  if (p.share) {
    hipLaunchKernelGGL((byte_share_kernel<T, FP8, DP, SHARE>), grid, dim3(kTrThreads), 0, st, a);
  } else {
    if constexpr (SHARE == 2)
      if (p.mt == 2) hipLaunchKernelGGL((byte_stream_kernel<T, FP8, DP, 2>), grid, dim3(kTrThreads), 0, st, a);
    if (p.mt == 1) hipLaunchKernelGGL((byte_stream_kernel<T, FP8, DP, 1>), grid, dim3(kTrThreads), 0, st, a);
  }
  LRQK_HIP_CHECK(hipGetLastError());
  tree_join_launch<T, DP, false>(a.tree, dim3((unsigned)((int64_t)a.tree.b * a.tree.hc * a.tree.row_tiles * 4)), st);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
template <typename T, bool FP8>
static int byte_launch_dp(const ByteArgs& a, const BytePlan& p, hipStream_t st) {
  if (p.dp == 64) return byte_launch<T, FP8, 64>(a, p, st);
  if (p.dp == 128) return byte_launch<T, FP8, 128>(a, p, st);
  return byte_launch<T, FP8, 256>(a, p, st);
}

static int byte_check(int b, int hq, int hc, int t, int64_t blocks, int d, int dtype) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(b > 0 && hq > 0 && hc > 0 && t > 0 && blocks > 0 && d > 0, LRQK_EINVAL, "bad sizes b=%d hq=%d hc=%d t=%d blocks=%lld d=%d", b,
               hq, hc, t, (long long)blocks, d);
  LRQK_REQUIRE(hq % hc == 0, LRQK_EINVAL, "%d query heads over %d cache heads", hq, hc);
  LRQK_REQUIRE(d * (int)elem_size(dtype) % 16 == 0 && d <= 256, LRQK_ELIMIT,
               "head_dim %d unsupported (rows of whole 16-byte pieces, at most 256 elements)", d);
  LRQK_REQUIRE(t <= 1024 && blocks <= (1 << 24) && (int64_t)b * hq <= 65535 && b * blocks <= INT32_MAX, LRQK_ELIMIT,
               "t=%d (at most 1024), blocks=%lld (2^24 a sequence, 2^31 in all), b * hq=%lld (65535)", t, (long long)blocks, (long long)b * hq);
  return LRQK_OK;
}

}  // namespace lrqk

using namespace lrqk;

extern "C" int64_t lrqk_byte_attention_workspace(int b, int hq, int hc, int t, int64_t blocks, int d, int dtype) {
  const int rc = byte_check(b, hq, hc, t, blocks, d, dtype);
  if (rc) return rc;
  const BytePlan p = byte_plan(b, hq, hc, t, blocks, d, dtype);
  return (p.part + p.ml + p.odd + p.cut) * (int64_t)sizeof(float);
}

extern "C" int lrqk_byte_attention(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                                   const void* k_tail, const void* v_tail, int64_t blocks, const int32_t* lengths, const void* k_new,
                                   const void* v_new, const uint8_t* mask, int64_t mask_batch_stride, void* out, float* lse, int b,
                                   int hq, int hc, int hn, int t, int d, float scale, int kind, void* workspace,
                                   int64_t workspace_bytes, int dtype, void* stream) {
  int rc = byte_check(b, hq, hc, t, blocks, d, dtype);
  if (rc) return rc;
  LRQK_REQUIRE(kind == LRQK_CODE_INT8 || kind == LRQK_CODE_FP8, LRQK_EINVAL, "kind=%d", kind);
  LRQK_REQUIRE(q && k && v && k_scale && v_scale && k_tail && v_tail && lengths && out && workspace, LRQK_EINVAL, "null pointer");
  LRQK_REQUIRE(!k_new == !v_new && !k_new == !mask, LRQK_EINVAL, "drafted keys, values and their mask come together");
  LRQK_REQUIRE(!k_new || (hn > 0 && hc % hn == 0), LRQK_EINVAL, "%d cache heads over %d heads of drafted tokens", hc, hn);
  LRQK_REQUIRE(scale > 0.0f && scale < INFINITY, LRQK_EINVAL, "scale=%g has to be positive and finite", (double)scale);
  LRQK_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)k_tail % 16 == 0 &&
                   (uintptr_t)v_tail % 16 == 0 && (uintptr_t)k_new % 16 == 0 && (uintptr_t)v_new % 16 == 0 && (uintptr_t)workspace % 16 == 0,
               LRQK_EINVAL, "pointers must be 16-byte aligned");
  const BytePlan p = byte_plan(b, hq, hc, t, blocks, d, dtype);
  const int64_t need = (p.part + p.ml + p.odd + p.cut) * (int64_t)sizeof(float);
  LRQK_REQUIRE(workspace_bytes >= need, LRQK_EINVAL, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes,
               (long long)need);
  LRQK_REQUIRE(((int64_t)p.units + 7) / 8 * 8 * p.row_blocks <= kMaxThreads / kTrThreads, LRQK_ELIMIT,
               "%lld blocks of %d heads and %d tokens are more than a launch has places for", (long long)blocks, b * hc, t);
  float* ws = (float*)workspace;
  ByteArgs a{};
  a.tree = TreeArgs{q, nullptr, nullptr, k_new, v_new, mask, lengths, out, lse, ws, ws + p.part, (int32_t*)ws + p.part + p.ml,
                    (int32_t*)ws + p.part + p.ml + p.odd, 0, 0, 0, mask_batch_stride, b, (int)(blocks * kByBlock), hq, hc, k_new ? hn : hc, t, d,
                    p.splits, p.least, p.most, p.row_blocks, p.rows, p.row_tiles, p.units, scale * kLog2e};
  a.apart = p.apart;
  a.k = k;
  a.v = v;
  a.ks = k_scale;
  a.vs = v_scale;
  a.k_tail = k_tail;
  a.v_tail = v_tail;
  a.blocks = (int)blocks;
  a.drafts = k_new ? t : 0;
  hipStream_t st = (hipStream_t)stream;
  const bool fp8 = kind == LRQK_CODE_FP8;
  if (dtype == LRQK_F32) return fp8 ? byte_launch_dp<float, true>(a, p, st) : byte_launch_dp<float, false>(a, p, st);
  return fp8 ? byte_launch_dp<bf16_t, true>(a, p, st) : byte_launch_dp<bf16_t, false>(a, p, st);
}
