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
// Bf16 V is transposed between those lanes' registers; bf16 probabilities are the sum of two bf16 numbers (off by up to
// 2^-15 of them), so that the one rounding to bf16 is the output's (but for very many queries: tree_share_kernel).
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

// How the sequences are cut into splits: of equal length, whatever the lengths of the sequences, as many as the grid was
// made for (every sequence's last one may be shorter, so there are up to b more).  From the lengths alone, by every wave
// for itself; a sequence's first workgroup leaves what the joining launch wants to know of it.
struct TreeCut {
  int b, len, split, splits, slot0, per;   // splits of the sequence, the number of its first
  static __device__ __forceinline__ int tiles(const TreeArgs& a, int len, int kt) { return (len + kt - 1) / kt + (a.t + kt - 1) / kt; }
  static __device__ __forceinline__ int length(const TreeArgs& a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.n) : a.n;
  }
  // tiles of a split (32 bits divide four times as fast as 64)
  static __device__ __forceinline__ int share(const TreeArgs& a, int64_t all) {
    const int x = all <= INT32_MAX ? (int)(((uint32_t)all + (uint32_t)a.splits - 1u) / (uint32_t)a.splits) : (int)((all + a.splits - 1) / a.splits);
    return max(a.least, min(x, a.most));
  }
  // the split of number `slot` of all; false: there is none
  __device__ __forceinline__ bool find(const TreeArgs& a, int kt, int slot) {
    if (!a.lengths || a.b == 1) {
      len = length(a, 0);
      per = share(a, (int64_t)a.b * tiles(a, len, kt));
      splits = (tiles(a, len, kt) + per - 1) / per;
      b = slot / splits;
      slot0 = b * splits;
      split = slot - slot0;
      return b < a.b;
    }
    const int lane = lane_id();
    long long all = 0;
    for (int i = lane; i < a.b; i += kWave) all += tiles(a, length(a, i), kt);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) all += __shfl_xor(all, off, kWave);
    per = __builtin_amdgcn_readfirstlane(share(a, all));
    int before = 0;
    for (int base = 0; base < a.b; base += kWave) {
      const int i = base + lane;
      const int mine = i < a.b ? (tiles(a, length(a, min(i, a.b - 1)), kt) + per - 1) / per : 0;
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

// What the workgroups of both kernels have in common: where they are and whose keys they read.
template <typename T>
struct TreePlace {
  int rb, unit, b, M, len, begin, end;   // tiles of the split
  const T *q, *kc, *vc, *kn, *vn;
  __device__ __forceinline__ bool find(const TreeArgs& a, int kt) {   // false: nothing to do
    // the row blocks of a unit (a split of a head) follow each other 8 workgroups apart: on one XCD, whose L2 then has the
    // rows of K and V that the first of them brought
    rb = (int)blockIdx.x % (8 * a.row_blocks) / 8;
    unit = (int)blockIdx.x / (8 * a.row_blocks) * 8 + (int)blockIdx.x % 8;
    if (unit >= a.units) return false;
    TreeCut cut;
    if (!cut.find(a, kt, unit / a.hc)) return false;
    if (cut.split == 0 && unit % a.hc == 0 && rb == 0 && threadIdx.x == 0) {
      a.cut[2 * cut.b] = cut.slot0;
      a.cut[2 * cut.b + 1] = cut.splits;
    }
    b = cut.b;
    len = cut.len;
    begin = cut.split * cut.per;
    end = min(TreeCut::tiles(a, len, kt), begin + cut.per);
    const int hc = unit % a.hc, gc = a.hq / a.hc;
    M = gc * a.t;
    q = (const T*)a.q + ((int64_t)b * a.hq + (int64_t)hc * gc) * a.t * a.d;
    kc = (const T*)a.k + b * a.kv_b + hc * a.kv_h;
    vc = (const T*)a.v + b * a.kv_b + hc * a.kv_h;
    const int64_t hn = (int64_t)b * a.hn + hc / (a.hc / a.hn);
    kn = (const T*)a.k_new + hn * a.t * a.d;
    vn = (const T*)a.v_new + hn * a.t * a.d;
    return true;
  }
};

// A tile's scores x become probabilities p = 2^(x scale - top), and the running sums.  The maximum is not looked for: as
// long as a lane's probabilities add up to little the one that is there serves, and where one of them does not (a larger
// score, or the first) the tile is done again with the maximum, o and the sums rescaled to it.  (A maximum per tile was a
// quarter of the vector instructions, which this kernel is bound by.)
template <int MT, int NE, int VW>
__device__ __forceinline__ void tree_softmax(const float (&x)[MT][NE], float (&p)[MT][NE], float (&top)[MT], float (&sum)[MT],
                                             ar_f4 (&o)[MT][VW], float scale_log2e) {
  float part[MT];
  bool more = false;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      p[m][e] = ar_exp2(fmaf(x[m][e], scale_log2e, -top[m]));
      part[m] = e == 0 ? p[m][0] : part[m] + p[m][e];
    }
    more = more | !(part[m] <= kTrMuch);
  }
  if (__ballot(more)) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float high = x[m][0];
#pragma unroll
      for (int e = 1; e < NE; ++e) high = fmaxf(high, x[m][e]);
      const float now = fmaxf(top[m], ar_quad_max(high) * scale_log2e);
      const float f = ar_exp2(top[m] - now);
      top[m] = now;
      sum[m] *= f;
#pragma unroll
      for (int j = 0; j < VW; ++j) o[m][j] *= f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        p[m][e] = ar_exp2(fmaf(x[m][e], scale_log2e, -now));
        part[m] = e == 0 ? p[m][0] : part[m] + p[m][e];
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) sum[m] += part[m];
}

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

// Few queries: the four waves of a workgroup take the tiles of its split in turn, each for itself.  Bound by the reading of
// K and V: a token over 32K of 8 cache heads of 128 bf16 elements, 134 MB in 27 us, 5.0 TB/s, and the join 5.  (Of few tokens
// by the chain of the first reads: 2112 of 32 heads, 10 us.)  Up to 32 queries a cache head: tree_share_kernel takes 58 us
// for 16 or 32 of them where this one takes 51 (32K tokens, after 256 MB of writes), of fp32 40 instead of 29 and 35 (8K).
template <typename T, int DP, int MT>
__global__ __launch_bounds__(kTrThreads, MT == 2 && DP == 128 ? 2 : 1) void tree_stream_kernel(TreeArgs a) {
  using Tile = TreeTile<T, DP, MT>;
  constexpr int NU = Tile::NU, KT = Tile::KT, NE = Tile::NE, STEPS = Tile::STEPS, VW = Tile::VW;
  constexpr int JC = 2;   // output blocks that the waves join at a time
  constexpr int CH = Tile::CH, KL = Tile::KL;
  constexpr int KB = KT * CH * kTrWaves, JB = kTrWaves * MT * JC * kWave;   // 16-byte pieces: of K, and of the joining
  __shared__ ar_u4 smem[KB > JB ? KB : JB];
  __shared__ float ml[kTrWaves][MT][16][2];
  const int lane = lane_id(), wave = wave_id(), col = lane & 15, quad = lane >> 4;
  TreePlace<T> at;
  if (!at.find(a, KT)) return;
  const int M = at.M, row0 = at.rb * 16 * MT, len = at.len;
  const int pieces = a.d * (int)sizeof(T) / 16;

  ar_u4 qf[MT][STEPS];
  int ti[MT];   // drafted token of the lane's query
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(row0 + 16 * m + col, M - 1);
    ti[m] = row % a.t;
    ar_row(at.q + (int64_t)row * a.d, quad, pieces, qf[m]);
  }
  ar_f4 o[MT][VW] = {};
  float top[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = kTrNone;
    sum[m] = 0.0f;
  }
  const int cached = (len + KT - 1) / KT, begin = at.begin, end = at.end;
  bool odd = false;
  // A wave reads whole rows, 64 / CH at a time; K and V of the next tile are on their way while this one is worked on.
  ar_u4* k_s = smem + wave * KT * CH;
  const int piece = lane % CH, krow = lane / CH;
  ar_u4 kg[KL];
  TreeV<T, VW> v[NE];
  constexpr int E = (int)sizeof(T), RPL = kWave / CH;   // bytes of an element, rows of a load
  constexpr int VP = TreeV<T, VW>::DW >= 4 ? TreeV<T, VW>::DW / 4 : 1;
  uint32_t vplace[VP];
#pragma unroll
  for (int i = 0; i < VP; ++i) vplace[i] = TreeV<T, VW>::place(col, a.d, i);
  const uint32_t kplace = 16u * (uint32_t)min(piece, pieces - 1), krs = (uint32_t)a.kv_r * E;
  const uint32_t kwhole = (uint32_t)krow * krs + kplace, vwhole = (uint32_t)(quad * NE) * krs;
  // a whole tile of the cache: the wave's address and offsets that do not change
  auto load_k = [&](int tile) {
    const char* src = (const char*)at.kc + (int64_t)tile * KT * krs;
#pragma unroll
    for (int i = 0; i < KL; ++i) kg[i] = tree_at<ar_u4>(src + (int64_t)(i * RPL) * krs, kwhole);
  };
  auto load_v = [&](int tile) {
    const char* src = (const char*)at.vc + (int64_t)tile * KT * krs;
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e].load(src + (int64_t)e * krs, vwhole, vplace);
  };
  // kg and v are the tile's; valid keys, the first of them drafted token `first` if draft
  auto work = [&](auto is_whole, int valid, bool draft, int first, auto next_k, auto next_v) {
    constexpr bool WHOLE = decltype(is_whole)::value;
    ar_wave_sync();
    if (pieces < CH) {   // (a head of a width between two of the kernels')
#pragma unroll
      for (int i = 0; i < KL; ++i) kg[i] = piece < pieces ? kg[i] : ar_u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < KL; ++i) k_s[ar_place<CH>(Tile::place(i * RPL + krow), piece)] = kg[i];
    ar_wave_sync();
    next_k();
    float x[MT][NE], p[MT][NE];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      ar_u4 kf[STEPS];
#pragma unroll
      for (int c = 0; c < STEPS; ++c) kf[c] = k_s[ar_place<CH>(16 * u + col, 4 * c + quad)];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        ar_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) s = ar_step<T>(kf[c], qf[m][c], s);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[m][4 * u + r] = s[r];
      }
    }
    if constexpr (!WHOLE) tree_mask<MT, NE>(x, a, at.b, ti, quad, valid, draft, first);
    tree_softmax<MT, NE, VW>(x, p, top, sum, o, a.scale_log2e);
    if constexpr (!WHOLE) {
#pragma unroll
      for (int e = 0; e < NE; ++e)
#pragma unroll
        for (int w = 0; w < TreeV<T, VW>::DW; ++w) {
          v[e].w[w] = quad * NE + e < valid ? v[e].w[w] : 0u;   // (a row that stands for one beyond the end)
          // queries that do not see a drafted token must not meet what its V holds: the joining launch adds that
          if (draft) odd = tree_clean<T>(v[e].w[w]) | odd;
        }
    }
    Tile::add(v, p, o);
    next_v();
  };
  int tile = begin + __builtin_amdgcn_readfirstlane(wave);
  const int wholes = min(end, len / KT);
  if (tile < wholes) {
    load_k(tile);
    load_v(tile);
  }
  for (; tile < wholes; tile += kTrWaves) {   // (the next tile, or this one again)
    const int next = tile + kTrWaves < wholes ? tile + kTrWaves : tile;
    work(std::true_type{}, KT, false, 0, [&] { load_k(next); }, [&] { load_v(next); });
  }
  for (; tile < end; tile += kTrWaves) {      // the last tile of the cache, if it is not whole, and the drafted ones
    const bool draft = tile >= cached;
    const int first = (draft ? tile - cached : tile) * KT, valid = min(KT, (draft ? a.t : len) - first);
    const uint32_t rs = draft ? (uint32_t)a.d * E : krs;
    const char* ks = (const char*)(draft ? at.kn : at.kc) + (int64_t)first * rs;
    const char* vs = (const char*)(draft ? at.vn : at.vc) + (int64_t)first * rs;
#pragma unroll
    for (int i = 0; i < KL; ++i) kg[i] = tree_at<ar_u4>(ks, (uint32_t)min(i * RPL + krow, valid - 1) * rs + kplace);
#pragma unroll
    for (int e = 0; e < NE; ++e) v[e].load(vs, (uint32_t)min(quad * NE + e, valid - 1) * rs, vplace);
    work(std::false_type{}, valid, draft, first, [] {}, [] {});
  }
  __syncthreads();   // (the rows of K make room for the sums)
  ar_f4(*joint)[MT * JC][kWave] = (ar_f4(*)[MT * JC][kWave])smem;

  // the four waves' sums, each over its own keys, to one maximum and together
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    sum[m] = ar_quad_sum(sum[m]);
    if (quad == 0) {
      ml[wave][m][col][0] = top[m];
      ml[wave][m][col][1] = sum[m];
    }
  }
  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) a.odd[(int64_t)at.unit * a.row_blocks + at.rb] = odd;
  const int64_t tile16 = (int64_t)at.unit * a.row_tiles + row0 / 16;
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

constexpr int kTlWaves = 4, kTlThreads = kTlWaves * kWave;

// Many queries: WR x WK waves, WR with 16 MT queries each that share the keys, WK groups of them with every WK-th tile of
// the split; K and V of the groups' tiles pass through LDS, whole rows read ahead into registers, one barrier a tile.  Two
// workgroups per CU, whose waves are at different places, so that one forms exponentials while the other multiplies (as
// one workgroup of eight waves they did both at the same time: twice as slow).  V's operand is read transposed
// (ds_read_b64_tr_b16: four keys of one element a lane).
//
// FINE: bf16 probabilities as the sum of two bf16 numbers, as in tree_stream_kernel.  Beyond 128 queries a cache head this
// is bound by the products, and half of those with V are the second number's (64 drafts over 4 x 64K, 32 / 8 heads, three
// ragged sets of lengths: 311, 222 and 226 us a call without it, 372, 258 and 276 with it; 25 drafts over 128K, bound by the
// reading: 108 instead of 112).  There a probability is rounded to bf16, by up to 2^-8 of it, each for itself, and what they
// are divided by is the sum of the rounded ones (one more block of o), so that an output moves by up to 2^-8 of the mean of
// |v - out|, and by its own rounding; lse keeps the exact ones' sum.  Those 64 drafts: 0.00215 of the output's norm off a
// result in 64 bits, 0.00166 with two numbers, which is the output's rounding alone.
template <typename T, int DP, int WR>
struct TreeShare {
  static constexpr int MT = DP == 256 ? 1 : 2, WK = kTlWaves / WR;
  using Tile = TreeTile<T, DP, MT>;
  static constexpr int KT = Tile::KT, CH = Tile::CH, KL = Tile::KL;
  static constexpr int ROWS = WR * 16 * MT;
  static constexpr int TILE = 2 * KT * CH;                          // 16-byte pieces of a tile's K and V
  static constexpr int LPW = (2 * KL + WR - 1) / WR;                // loads of a wave for a tile
  static constexpr int AHEAD = LPW <= 4 ? 2 : 1;                    // steps whose rows are on their way
  static constexpr int JC = 2, JOINT = WK > 1 ? kTlWaves * MT * JC * kWave : 0;
  static constexpr int SMEM = 2 * WK * TILE > JOINT ? 2 * WK * TILE : JOINT;

  // Where piece `piece` of V's row is: moved within the row so that what a transposing read takes (32 bytes of rows r ..
  // r + 3 and r + 8 .. r + 11) or an fp32 operand (64 bytes of rows r, r + 4 ..) comes from different banks.
  static __device__ __forceinline__ int v_place(int row, int piece) {
    int x;
    if constexpr (sizeof(T) == 4)
      x = (4 * (row >> 2)) & (CH - 1);
    else if constexpr (CH >= 16)
      x = 2 * ((row & 3) | ((row >> 3) & 1) << 2);
    else if constexpr (CH == 8)
      x = 2 * (((row >> 1) & 1) | ((row >> 3) & 1) << 1);
    else
      x = 2 * ((row >> 3) & 1);
    return row * CH + (piece ^ x);
  }
};

template <typename T, int DP, int WR, bool FINE>
__global__ __launch_bounds__(kTlThreads, 2) void tree_share_kernel(TreeArgs a) {
  using Share = TreeShare<T, DP, WR>;
  constexpr int MT = Share::MT, WK = Share::WK;
  using Tile = TreeTile<T, DP, MT>;
  constexpr int NU = Tile::NU, KT = Tile::KT, NE = Tile::NE, STEPS = Tile::STEPS, VW = Tile::VW, CH = Tile::CH, KL = Tile::KL;
  constexpr int E = (int)sizeof(T), RPL = kWave / CH, LPW = Share::LPW, JC = Share::JC;
  __shared__ ar_u4 smem[Share::SMEM];
  __shared__ float ml[kTlWaves][MT][16][3];
  TreePlace<T> at;
  if (!at.find(a, KT)) return;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), col = lane & 15, quad = lane >> 4;
  const int wr = wave % WR, wk = wave / WR;
  const int M = at.M, row0 = at.rb * Share::ROWS + wr * 16 * MT, len = at.len;
  const int pieces = a.d * E / 16;
  ar_u4 qf[MT][STEPS];
  int ti[MT];   // drafted token of the lane's query
  constexpr int OB = VW + (FINE ? 0 : 1);   // blocks of o, the last one of the sums
  ar_f4 o[MT][OB] = {};
  float top[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(row0 + 16 * m + col, M - 1);
    ti[m] = row % a.t;
    ar_row(at.q + (int64_t)row * a.d, quad, pieces, qf[m]);
    top[m] = kTrNone;
    sum[m] = 0.0f;
  }
  const int cached = (len + KT - 1) / KT, begin = at.begin, end = at.end, steps = (end - begin + WK - 1) / WK;
  bool odd = false;
  // this wave's share of a tile: loads l0 .. l0 + LPW of its K and then V rows
  const int mine = wave % WK, l0 = wave / WK * LPW;
  const int piece = lane % CH, krow = lane / CH;
  const uint32_t place = 16u * (uint32_t)min(piece, pieces - 1), krs = (uint32_t)a.kv_r * E;
  ar_u4 ring[Share::AHEAD][LPW];
  uint32_t from[LPW];   // of a whole tile of the cache: bytes from its first row of K or V
#pragma unroll
  for (int i = 0; i < LPW; ++i) from[i] = (uint32_t)(min(l0 + i, 2 * KL - 1) % KL * RPL + krow) * krs + place;
  auto load_whole = [&](int step, ar_u4 (&g)[LPW]) {
    const int64_t at_tile = (int64_t)(begin + step * WK + mine) * KT * krs;
    const char *ks = (const char*)at.kc + at_tile, *vs = (const char*)at.vc + at_tile;
#pragma unroll
    for (int i = 0; i < LPW; ++i) g[i] = tree_at<ar_u4>(min(l0 + i, 2 * KL - 1) < KL ? ks : vs, from[i]);
  };
  auto load = [&](int step, ar_u4 (&g)[LPW]) {
    // (always from a place that exists: loads under a condition were waited for one by one)
    const int tile = min(begin + step * WK + mine, end - 1);
    const bool draft = tile >= cached;
    const int first = (draft ? tile - cached : tile) * KT, last = (draft ? a.t : len) - first - 1;
    const uint32_t rs = draft ? (uint32_t)a.d * E : krs;
    const char* ks = (const char*)(draft ? at.kn : at.kc) + (int64_t)first * rs;
    const char* vs = (const char*)(draft ? at.vn : at.vc) + (int64_t)first * rs;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int l = min(l0 + i, 2 * KL - 1);
      g[i] = tree_at<ar_u4>(l < KL ? ks : vs, (uint32_t)min(l % KL * RPL + krow, last) * rs + place);
    }
  };
  // Two versions of a step's work: of whole tiles of the cache, and with everything that the others need.
  uint32_t to[LPW];   // where the loads go within a tile
#pragma unroll
  for (int i = 0; i < LPW; ++i) {
    const int l = min(l0 + i, 2 * KL - 1), row = l % KL * RPL + krow;
    to[i] = (uint32_t)(mine * Share::TILE) + (uint32_t)(l < KL ? ar_place<CH>(Tile::place(row), piece) : KT * CH + Share::v_place(row, piece));
  }
  auto store = [&](auto is_whole, auto buffer, int step, ar_u4 (&g)[LPW]) {
    const int tile = begin + step * WK + mine;
    ar_u4* dst = smem + decltype(buffer)::value * WK * Share::TILE;
    if constexpr (!decltype(is_whole)::value) {
      if (tile >= end) return;
      const bool draft = tile >= cached;
      const int valid = (draft ? a.t : len) - (draft ? tile - cached : tile) * KT;
#pragma unroll
      for (int i = 0; i < LPW; ++i) {
        const int l = min(l0 + i, 2 * KL - 1), row = l % KL * RPL + krow;
#pragma unroll
        for (int w = 0; w < 4; ++w) {   // of V: zeros for a row that stands for one beyond the end
          uint32_t x = ((l < KL) | (row < valid)) ? g[i][w] : 0u;
          // queries that do not see a drafted token must not meet what its V holds: the joining launch adds that
          const uint32_t kept = x;
          const bool found = tree_clean<T>(x) & draft & (l >= KL);
          odd = odd | found;
          g[i][w] = found ? x : kept;
        }
      }
    }
    if (pieces < CH) {   // (a head of a width between two of the kernels')
#pragma unroll
      for (int i = 0; i < LPW; ++i) g[i] = piece < pieces ? g[i] : ar_u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < LPW; ++i) dst[to[i]] = g[i];
  };
  uint32_t vat[Tile::BF ? VW : 1][2];   // bf16: where the lane's part of V's operands is
  if constexpr (Tile::BF) {
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      // keys 8 quad .. + 3 and + 4 .. + 7 of elements 16 j ..: lane i of 16 points to key i / 4, elements 4 (i % 4) ..
      const int row = 8 * quad + (col >> 2), x = 2 * j + ((col >> 1) & 1);
      vat[j][0] = 16u * (uint32_t)(wk * Share::TILE + KT * CH + Share::v_place(row, x)) + 8u * (uint32_t)(col & 1);
      vat[j][1] = 16u * (uint32_t)(wk * Share::TILE + KT * CH + Share::v_place(row + 4, x)) + 8u * (uint32_t)(col & 1);
    }
  }
  uint32_t kat[STEPS];   // where the lane's part of K's operands is (block u: 16 rows further)
#pragma unroll
  for (int c = 0; c < STEPS; ++c) kat[c] = (uint32_t)(wk * Share::TILE + ar_place<CH>(col, 4 * c + quad));
  auto work = [&](auto is_whole, auto buffer, int step) {
    constexpr bool WHOLE = decltype(is_whole)::value;
    const int tile = begin + step * WK + wk;
    if constexpr (!WHOLE)
      if (tile >= end) return;
    const ar_u4* tile_s = smem + decltype(buffer)::value * WK * Share::TILE;   // (the buffer's offset is the instructions')
    float x[MT][NE], p[MT][NE];
    {
      ar_u4 kf[NU][STEPS];
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int u = 0; u < NU; ++u) kf[u][c] = (tile_s + 16 * u * CH)[kat[c]];   // (16 rows on, pieces change places alike)
      ar_f4 s[NU][MT] = {};
#pragma unroll
      for (int c = 0; c < STEPS; ++c)   // (NU MT sums side by side: one waits for none of its own)
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int m = 0; m < MT; ++m) s[u][m] = ar_step<T>(kf[u][c], qf[m][c], s[u][m]);
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[m][4 * u + r] = s[u][m][r];
    }
    if constexpr (!WHOLE) {
      const bool draft = tile >= cached;
      const int first = (draft ? tile - cached : tile) * KT, valid = min(KT, (draft ? a.t : len) - first);
      if (draft || valid < KT) tree_mask<MT, NE>(x, a, at.b, ti, quad, valid, draft, first);
    }
    constexpr int VB = VW < 4 ? VW : 4;   // blocks of V's operands at a time
    auto operand = [&](int j) {
      const tr_v4s b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_lds_v4s)((const char*)tile_s + vat[j][0]));
      const tr_v4s b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_lds_v4s)((const char*)tile_s + vat[j][1]));
      return __builtin_bit_cast(ar_bf8, __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    ar_bf8 v[Tile::BF ? VB : 1];
    if constexpr (Tile::BF) {   // (the first ones are on their way while the exponentials are formed)
#pragma unroll
      for (int j = 0; j < VB; ++j) v[j] = operand(j);
    }
    tree_softmax<MT, NE, OB>(x, p, top, sum, o, a.scale_log2e);
    if constexpr (Tile::BF) {
      ar_bf8 hi[MT], lo[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (FINE) {
          tree_split(p[m], hi[m], lo[m]);
        } else {
          tr_f8 y;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = p[m][e];
          hi[m] = __builtin_convertvector(y, ar_bf8);
          const uint32_t one = 0x3f803f80u;
          o[m][VW] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ar_bf8, ar_u4{one, one, one, one}), hi[m], o[m][VW], 0, 0, 0);
        }
      }
#pragma unroll
      for (int j0 = 0; j0 < VW; j0 += VB) {
#pragma unroll
        for (int j = 0; j < VB; ++j)
#pragma unroll
          for (int m = 0; m < MT; ++m) o[m][j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[j], hi[m], o[m][j0 + j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < VB; ++j) {
          if constexpr (FINE) {
#pragma unroll
            for (int m = 0; m < MT; ++m) o[m][j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[j], lo[m], o[m][j0 + j], 0, 0, 0);
          }
          if (j0 + VB < VW) v[j] = operand(j0 + VB + j);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < VW; ++j)
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const float v = ((const float*)(tile_s + wk * Share::TILE + KT * CH + Share::v_place(4 * quad + e, 4 * j + (col >> 2))))[col & 3];
#pragma unroll
          for (int m = 0; m < MT; ++m) o[m][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[m][e], o[m][j], 0, 0, 0);
        }
    }
  };
  constexpr int AHEAD = Share::AHEAD;
  using First = std::integral_constant<int, 0>;
  using Second = std::integral_constant<int, 1>;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(i, ring[i]);
  store(std::false_type{}, First{}, 0, ring[0]);
  __syncthreads();
  const int wholes = (min(end, len / KT) - begin) / WK;   // steps that have whole tiles only
  int step = 0;
  for (; step + 1 + AHEAD < wholes; step += 2) {
    load_whole(step + AHEAD, ring[0]);
    work(std::true_type{}, First{}, step);
    store(std::true_type{}, Second{}, step + 1, ring[1 % AHEAD]);
    __syncthreads();
    load_whole(step + 1 + AHEAD, ring[1 % AHEAD]);
    work(std::true_type{}, Second{}, step + 1);
    store(std::true_type{}, First{}, step + 2, ring[0]);
    __syncthreads();
  }
  for (; step < steps; step += 2) {   // (steps behind the last have no tile)
    load(step + AHEAD, ring[0]);
    work(std::false_type{}, First{}, step);
    store(std::false_type{}, Second{}, step + 1, ring[1 % AHEAD]);
    __syncthreads();
    load(step + 1 + AHEAD, ring[1 % AHEAD]);
    work(std::false_type{}, Second{}, step + 1);
    store(std::false_type{}, First{}, step + 2, ring[0]);
    __syncthreads();
  }

  odd = __syncthreads_or(odd);
  if (threadIdx.x == 0) a.odd[(int64_t)at.unit * a.row_blocks + at.rb] = odd;
  const int64_t tile16 = (int64_t)at.unit * a.row_tiles + row0 / 16;
#pragma unroll
  for (int m = 0; m < MT; ++m) sum[m] = ar_quad_sum(sum[m]);
  if constexpr (WK > 1) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (quad == 0) {
        ml[wave][m][col][0] = top[m];
        ml[wave][m][col][1] = sum[m];
        ml[wave][m][col][2] = FINE ? sum[m] : o[m][OB - 1][0];   // (every row of that block is the sum)
      }
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    float all = top[m], total = sum[m], norm = FINE ? sum[m] : o[m][OB - 1][0];
    if constexpr (WK > 1) {
      all = ml[wr][m][col][0];
#pragma unroll
      for (int w = 1; w < WK; ++w) all = fmaxf(all, ml[w * WR + wr][m][col][0]);
      total = norm = 0.0f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float f = ar_exp2(ml[w * WR + wr][m][col][0] - all);
        total += ml[w * WR + wr][m][col][1] * f;
        norm += ml[w * WR + wr][m][col][2] * f;
      }
      const float f = ar_exp2(top[m] - all);
#pragma unroll
      for (int j = 0; j < VW; ++j) o[m][j] *= f;
    }
    if (wk == 0 && quad == 0 && row0 + 16 * m + col < M) {
      float* dst = a.part_ml + (tile16 + m) * 48 + col;
      dst[0] = all;
      dst[16] = total;
      dst[32] = norm;
    }
  }
  if constexpr (WK == 1) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < VW; ++j)
        if (row0 + 16 * m + col < M) ((ar_f4*)a.part)[((tile16 + m) * VW + j) * kWave + lane] = o[m][j];
  } else {
    ar_f4(*joint)[MT * JC][kWave] = (ar_f4(*)[MT * JC][kWave])smem;
    for (int j0 = 0; j0 < VW; j0 += JC) {
#pragma unroll
      for (int j = 0; j < VW; ++j)
        if (j >= j0 && j < j0 + JC) {
#pragma unroll
          for (int m = 0; m < MT; ++m) joint[wave][m * JC + (j & (JC - 1))][lane] = o[m][j];
        }
      __syncthreads();
      for (int s = wk; s < MT * JC; s += WK) {
        ar_f4 x = joint[wr][s][lane];
#pragma unroll
        for (int w = 1; w < WK; ++w) x += joint[w * WR + wr][s][lane];
        const int m = s / JC, j = j0 + s % JC;
        if (row0 + 16 * m + col < M) ((ar_f4*)a.part)[((tile16 + m) * VW + j) * kWave + lane] = x;
      }
      __syncthreads();
    }
  }
}

// Blocks of 16 elements of the head that a workgroup of the join has.
constexpr int tree_join_blocks(int blocks, int threads) { return threads == 512 && blocks > 4 ? 4 : blocks; }

// A workgroup joins the splits' parts of 16 queries of a cache head, VB blocks of a quad of the lanes that hold them (a
// quarter of the head): 16 threads with a query each for (block j, every G-th split).  SHARED: which of the two kernels left
// the parts, whose lanes have other elements.  Its time is a chain of reads that wait for each other and barriers, so the
// reads are few in a row, and what 16 queries of all waves make is added up by every thread that wants it.
template <typename T, int DP, bool SHARED, int THREADS>
__global__ __launch_bounds__(THREADS) void tree_join_kernel(TreeArgs a) {
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

// How a call is cut up, from its sizes alone.
struct TreePlan {
  int dp, mt, wr;                    // wr = 0: tree_stream_kernel
  bool fine;
  int rows, row_blocks, row_tiles, splits, least, most, units;
  int64_t part, ml, odd, cut;        // words of 4 bytes
};
static TreePlan tree_plan(int b, int hq, int hc, int t, int64_t n, int d, bool lengths, int dtype) {
  TreePlan p;
  p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t M = (int64_t)(hq / hc) * t;
  p.fine = dtype == LRQK_F32 || M <= 128;
  const int kt = dtype == LRQK_BF16 ? 32 : 16;
  const int64_t tiles = (n + kt - 1) / kt + (t + kt - 1) / kt;
  int64_t groups_wanted, least;
  if (M <= (p.dp == 256 ? 16 : 32)) {
    p.mt = M <= 16 ? 1 : 2;
    p.wr = 0;
    p.rows = 16 * p.mt;
    least = 4 * kTrWaves;   // four tiles for each of a workgroup's waves
  } else {
    p.mt = p.dp == 256 ? 1 : 2;
    p.wr = M <= 32 * p.mt && p.dp != 256 ? 2 : 4;   // (64 queries over 32K: 33 us with two waves of them, 35 with four; fp32, 4K: 29, 32)
    p.rows = 16 * p.mt * p.wr;
    least = 2 * kTlWaves / p.wr;
  }
  // Two workgroups per CU (25 drafts over 128K: 112 + 10 us for the join, four per CU 129 + 16); four where the lengths may
  // differ (64 drafts over 4 sequences of 4 .. 32K: 130 + 17, two per CU 160 + 13; one token over 16 of 2 .. 16K: 110 and 121).
  groups_wanted = b > 1 && lengths ? 1024 : 512;
  p.row_blocks = (int)((M + p.rows - 1) / p.rows);
  p.row_tiles = p.row_blocks * (p.rows / 16);
  p.splits = (int)std::max<int64_t>(b, groups_wanted / ((int64_t)hc * p.row_blocks));
  p.least = (int)std::max<int64_t>(least, (tiles + kTrMaxSplits - 1) / kTrMaxSplits);
  // Where the heads alone fill the GPU a split would be all of a sequence, and one fp32 number the sum over all its keys: with
  // 131072 that round alike lse was 1.2e-4 off and an output 2e-3 (fp32; the matrix cores cut off), with splits of up to 512
  // tiles 2.4e-6 and 8e-6.  Their scratch is 1 % of K and V; more row blocks, which have as much each, have longer splits.  Of
  // a whole cache they are of one length: 64 drafts over 64 sequences of 32K, 1027 tiles as 1024 and 3, took 3.8 ms instead of 2.6.
  const int64_t longest = std::max<int64_t>(p.least, (int64_t)kTrLong * p.row_blocks), parts = (tiles + longest - 1) / longest;
  p.most = (int)((tiles + parts - 1) / parts);
  // the splits that there can be: the wanted ones and the sequences' shorter ones, or those of the longest splits; or what the
  // shortest make
  const int64_t slots = std::min<int64_t>(std::max<int64_t>((int64_t)p.splits + b, b * parts), b * ((tiles + p.least - 1) / p.least));
  p.units = (int)(hc * slots);
  const int64_t groups = (int64_t)p.units * p.row_tiles;
  p.part = groups * 16 * p.dp;
  p.ml = groups * 48;
  p.odd = (int64_t)p.units * p.row_blocks;
  p.cut = 2 * (int64_t)b;
  return p;
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
template <typename T, int DP>
static int tree_launch(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)(a.units + 7) / 8 * 8 * a.row_blocks));
  const dim3 join((unsigned)((int64_t)a.b * a.hc * a.row_tiles * 4));
  // (of the most heads and drafts, 65535 and 1024: 2^24 - 256 workgroups of 256 threads; a launch may have 2^32 - 1 threads)
  if (p.wr == 0) {
    if constexpr (DP < 256)
      if (p.mt == 2) hipLaunchKernelGGL((tree_stream_kernel<T, DP, 2>), grid, dim3(kTrThreads), 0, st, a);
    if (p.mt == 1) hipLaunchKernelGGL((tree_stream_kernel<T, DP, 1>), grid, dim3(kTrThreads), 0, st, a);
    LRQK_HIP_CHECK(hipGetLastError());
    tree_join_launch<T, DP, false>(a, join, st);
  } else {
    if constexpr (DP < 256)
      if (p.wr == 2) hipLaunchKernelGGL((tree_share_kernel<T, DP, 2, true>), grid, dim3(kTlThreads), 0, st, a);
    if constexpr (sizeof(T) == 2)
      if (p.wr == 4 && !p.fine) hipLaunchKernelGGL((tree_share_kernel<T, DP, 4, false>), grid, dim3(kTlThreads), 0, st, a);
    if (p.wr == 4 && p.fine) hipLaunchKernelGGL((tree_share_kernel<T, DP, 4, true>), grid, dim3(kTlThreads), 0, st, a);
    LRQK_HIP_CHECK(hipGetLastError());
    tree_join_launch<T, DP, true>(a, join, st);
  }
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
template <typename T>
static int tree_launch_dp(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
  if (p.dp == 32) return tree_launch<T, 32>(a, p, st);
  if (p.dp == 64) return tree_launch<T, 64>(a, p, st);
  if (p.dp == 128) return tree_launch<T, 128>(a, p, st);
  return tree_launch<T, 256>(a, p, st);
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

extern "C" int64_t lrqk_tree_attention_workspace(int b, int hq, int hc, int t, int64_t n, int d, int have_lengths, int dtype) {
  const int rc = tree_check(b, hq, hc, t, n, d, dtype);
  if (rc) return rc;
  const TreePlan p = tree_plan(b, hq, hc, t, n, d, have_lengths != 0, dtype);
  return (p.part + p.ml + p.odd + p.cut) * (int64_t)sizeof(float);
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
  LRQK_REQUIRE(kv_row_stride >= 0 && kv_row_stride <= (1 << 24), LRQK_ELIMIT, "kv_row_stride=%lld (at most 2^24 elements)",
               (long long)kv_row_stride);
  const TreePlan p = tree_plan(b, hq, hc, t, n, d, lengths != nullptr, dtype);
  const int64_t need = (p.part + p.ml + p.odd + p.cut) * (int64_t)sizeof(float);
  LRQK_REQUIRE(workspace_bytes >= need, LRQK_EINVAL, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes,
               (long long)need);
  LRQK_REQUIRE(((int64_t)p.units + 7) / 8 * 8 * p.row_blocks <= kMaxThreads / kTrThreads, LRQK_ELIMIT,
               "%lld tokens of %d heads and %d drafts are more than a launch has places for", (long long)n, b * hc, t);
  TreeArgs a{q, k_cache, v_cache, k_new, v_new, mask, lengths, out, lse, (float*)workspace, (float*)workspace + p.part,
             (int32_t*)workspace + p.part + p.ml, (int32_t*)workspace + p.part + p.ml + p.odd,
             kv_batch_stride, kv_head_stride, kv_row_stride, mask_batch_stride, b, (int)n, hq, hc, hn, t, d, p.splits, p.least, p.most, p.row_blocks, p.rows,
             p.row_tiles, p.units,
             scale * kLog2e};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LRQK_F32) return tree_launch_dp<float>(a, p, st);
  return tree_launch_dp<bf16_t>(a, p, st);
}
