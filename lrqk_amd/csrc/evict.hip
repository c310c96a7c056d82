// Eviction from a cache by the attention that its tokens got: of a head's n tokens `budget` stay, the `recent` newest
// ones (by their position ids) and, of the others, those with the largest weights (NaN counts as the largest; of equal
// ones those of the lowest slots).  A token that stays in slots 0 .. budget - 1 keeps its slot; the ones that stay of the
// slots behind move, in order, into the slots that became free, in order.  So no row has to wait for another: sources
// and destinations do not overlap, and a cache that is a few tokens over its budget moves a few rows.
//
//   select   one workgroup per head: the budget-th largest 32-bit key by a radix search over histograms in LDS (11, 11 and 10
//            bits; ties by slot), then the list source[slot] of the slots that stay.  Up to 32768 tokens: their keys are in
//            registers.
//   wide     the same for longer heads, several workgroups a head and a launch for every step that needs all of them.
//   move     rows of K and V, weights and ids.  In place and with few tokens over the budget select does that too.
//
// Bound by instructions and the chain of barriers, not by the memory: a wave's instruction takes its SIMD 4 cycles, so each
// one that looks at every key of 32768 takes the one workgroup 0.25 us.  8 heads of 32768 tokens down to 2112: select 22 us
// (reads 3, keys and the first histogram 4, the others 4, counting 3, the lists 5), move 5 us; as wide 38 and 5 (of 40000
// tokens 38, of 131072 39; one workgroup a head that reads them for every look: 200 and 420).  32 heads of 2117 tokens down
// to 2112, in place and in one launch: 10 us (in two: 9 and 5).  Keys of 4, 12 or 32 slots a thread: 2117 tokens 7.6 us
// instead of 20 with 32, 9000 tokens 12.  (A wave's slots one behind the other need no table of counts, but then one or two
// waves have all slots in front of `keep`, which cost most: 24 us.)
#include <algorithm>
#include <initializer_list>

#include "common.hpp"

namespace lrqk {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / kWave;
constexpr int kEvBins = 2048, kEvCopies = 4;    // of a histogram, and how many share a wave's additions
constexpr int kEvMoveThreads = 256;
constexpr int kEvMost = 32 * kEvThreads;         // slots of a head that one workgroup takes
constexpr int kEvWide = 4, kEvMaxBlocks = 512;   // of more: rounds that a workgroup has in registers, workgroups of a head
constexpr int kEvFew = 128;                     // tokens over the budget whose rows select moves itself

struct EvictMove {
  const uint4 *k, *v;
  uint4 *k_out, *v_out;
  const float* w;
  const int32_t* ids;
  float* w_out;
  int32_t* ids_out;
  int cap, cap_out, chunks;   // slots of a head; 16-byte pieces of a row
};

// Order of the tokens: the newest in front of everything, then NaN, then by weight.  (No id is above the newest one, so
// that their difference has 32 bits.)
__device__ __forceinline__ uint32_t evict_key(float w, int32_t id, int32_t newest, int recent) {
  const uint32_t k = w != w ? 0xfffffffeu : score_key(w);
  return (uint32_t)newest - (uint32_t)id < (uint32_t)recent ? 0xffffffffu : k;
}

__device__ __forceinline__ int evict_len(const int32_t* lengths, int b, int cap) {
  return lengths ? min(max(lengths[b], 0), cap) : cap;
}

// Sums over the workgroup's threads in order: of what stands in front of the thread, and of all.  Two barriers (AGAIN: the
// next one may use the same scratch at once), or one.
template <bool AGAIN = true>
__device__ __forceinline__ uint32_t evict_scan(uint32_t v, uint32_t* scratch, uint32_t& total) {
  const uint32_t incl = (uint32_t)wave_inclusive_sum((int)v);
  if (lane_id() == kWave - 1) scratch[wave_id()] = incl;
  __syncthreads();
  uint32_t base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kEvWaves; ++w) {
    const uint32_t c = scratch[w];
    base += w < wave_id() ? c : 0u;
    all += c;
  }
  if (AGAIN) __syncthreads();
  total = all;
  return base + incl - v;
}

// `base` and the lanes of `mask` in front of this one.
__device__ __forceinline__ uint32_t evict_place(unsigned long long mask, uint32_t base) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, base));
}

__device__ __forceinline__ void evict_row(const EvictMove& m, int h, int from_slot, int to_slot, int sub, int step) {
  const int64_t from = (int64_t)h * m.cap + from_slot, to = (int64_t)h * m.cap_out + to_slot;
  for (int c = sub; c < m.chunks; c += step) {
    const uint4 a = m.k[from * m.chunks + c], b = m.v[from * m.chunks + c];
    m.k_out[to * m.chunks + c] = a;
    m.v_out[to * m.chunks + c] = b;
  }
  if (sub == 0) {
    const float w = m.w[from];
    const int32_t id = m.ids[from];
    m.w_out[to] = w;
    m.ids_out[to] = id;
  }
}

// Digit `pass` of the need-th largest key from a histogram (sums of a bin: count(bin)): two bins a thread, the largest
// first.  `equal`: keys that begin like it; `need` counts among those from here on.  Two barriers: the first, within the
// next one's sums, keeps the picked numbers until they have been read.
template <typename F>
__device__ __forceinline__ void evict_pick(F count, int shift, uint32_t& prefix, uint32_t& need, uint32_t& equal, uint32_t* scratch,
                                           uint32_t* pick_s) {
  const int bin = kEvBins - 1 - 2 * (int)threadIdx.x;
  const uint32_t c[2] = {count(bin), count(bin - 1)};
  uint32_t total;
  uint32_t before = evict_scan<false>(c[0] + c[1], scratch, total);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (before < need && need <= before + c[j]) {
      pick_s[0] = (uint32_t)(bin - j);
      pick_s[1] = need - before;
      pick_s[2] = c[j];
    }
    before += c[j];
  }
  __syncthreads();
  prefix |= pick_s[0] << shift;
  need = pick_s[1];
  equal = pick_s[2];
}
__device__ __forceinline__ int evict_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }

// Keys into the histogram of a pass.  A piece is 64 slots of a wave, and the waves' pieces of a round follow each other:
// slot first0 + 1024 c + 64 wave + lane is in key[c].
template <int CHUNKS>
__device__ __forceinline__ void evict_count(const uint32_t (&key)[CHUNKS], int pass, int first0, int n, uint32_t prefix, uint4* hist) {
  uint32_t* mine = (uint32_t*)hist + (lane_id() & (kEvCopies - 1));
  const int shift = evict_shift(pass);
  const uint32_t limit = pass == 1 ? 1u << 21 : 1u << 10;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {   // (what is no slot is in the first bins, which are behind all tokens)
    const uint32_t rest = key[c] ^ prefix;
    if (pass == 0 ? first0 + c * kEvThreads < n : rest < limit) atomicAdd(&mine[kEvCopies * (rest >> shift)], 1u);
  }
}

// The lists of a block of CHUNKS rounds, behind nh holes, nm movers and `ties` keys that are `prefix`, which count on: every
// key from `prefix` on stays, or (TIES) of those that are `prefix` the first `need`.  Lane c has the counts of the wave's
// round c, and the table of all waves' says what is in front of its piece.
template <int CHUNKS, bool TIES>
__device__ __forceinline__ void evict_lists(const uint32_t (&key)[CHUNKS], int first0, int keep, uint32_t prefix, uint32_t need,
                                            uint32_t& ties, uint32_t& nh, uint32_t& nm, uint32_t (*counts)[kEvWaves + 1], int32_t* src,
                                            int32_t* hole, int32_t* mover) {
  static_assert(CHUNKS <= kWave, "a lane for the counts of each round");
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  first0 += wave * kWave;
  // two numbers of lane c, in 16 bits each: `low` and `high` go from the sums in front of the block to those in front of
  // the wave's piece of round c.  -> the sums behind the block
  auto in_front = [&](uint32_t mine, uint32_t& low, uint32_t& high) {
    if (lane < CHUNKS) counts[lane][wave] = mine;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
      const uint32_t x = counts[min(lane, CHUNKS - 1)][i];
      before += i < wave ? x : 0u;
      all += x;
    }
    all = lane < CHUNKS ? all : 0u;   // (of a round: at most 1024 in each half)
    const uint32_t ends = (uint32_t)wave_inclusive_sum((int)(all & 0xffffu)), highs = (uint32_t)wave_inclusive_sum((int)(all >> 16));
    const uint32_t at = low, at_high = high;
    low = at + ends - (all & 0xffffu) + (before & 0xffffu);
    high = at_high + highs - (all >> 16) + (before >> 16);
    __syncthreads();
    return make_uint2(at + (uint32_t)__builtin_amdgcn_readlane((int)ends, kWave - 1),
                      at_high + (uint32_t)__builtin_amdgcn_readlane((int)highs, kWave - 1));
  };
  uint32_t rank = ties;   // of the first tie of lane c's piece
  if constexpr (TIES) {
    int mine = 0;
    uint32_t none = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int tied = __popcll(__ballot(key[c] == prefix));
      mine = lane == c ? tied : mine;
    }
    ties = in_front((uint32_t)mine, rank, none).x;
  }
  auto stays = [&](int c) -> bool {
    if constexpr (!TIES) return key[c] >= prefix;
    const uint32_t r = evict_place(__ballot(key[c] == prefix), (uint32_t)__builtin_amdgcn_readlane((int)rank, c));
    return (key[c] > prefix) | ((key[c] == prefix) & (r < need));
  };
  // (a wave's instructions are what this costs, so the usual pieces, behind `keep`, are apart)
  int mine = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int first = first0 + c * kEvThreads;
    const bool stay = stays(c);
    int both;
    if (first >= keep)
      both = __popcll(__ballot(stay)) << 16;
    else
      both = __popcll(__ballot((first + lane < keep) & !stay)) + (__popcll(__ballot((first + lane >= keep) & stay)) << 16);
    mine = lane == c ? both : mine;
  }
  uint32_t ah = nh, am = nm;
  const uint2 ends = in_front((uint32_t)mine, ah, am);
  nh = ends.x;
  nm = ends.y;
  auto put = [&](int32_t* to, bool which, uint32_t at, int slot) {
    const unsigned long long mask = __ballot(which);
    if (mask && which) to[evict_place(mask, at)] = slot;
  };
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int first = first0 + c * kEvThreads;
    const bool stay = stays(c);
    const uint32_t mover_at = (uint32_t)__builtin_amdgcn_readlane((int)am, c);
    if (first >= keep) {
      put(mover, stay, mover_at, first + lane);
    } else {
      const bool front = first + lane < keep;
      put(hole, front & !stay, (uint32_t)__builtin_amdgcn_readlane((int)ah, c), first + lane);
      put(mover, stay & !front, mover_at, first + lane);
      if (src && (stay & front)) src[first + lane] = first + lane;
    }
  }
}

__device__ __forceinline__ int32_t evict_max(int32_t newest, uint32_t* scratch) {   // over the workgroup's threads; one barrier
  newest = (int32_t)(wave_reduce_u32((uint32_t)newest ^ 0x80000000u, [](uint32_t a, uint32_t b) { return max(a, b); }) ^ 0x80000000u);
  if (lane_id() == 0) scratch[wave_id()] = (uint32_t)newest;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEvWaves; ++i) newest = max(newest, (int32_t)scratch[i]);
  return newest;
}

// One workgroup a head, up to 1024 CHUNKS slots, whose keys are in registers.  source: [bh][budget]; holes, movers:
// [bh][budget] scratch.  lg: 2^lg threads move a row, where this launch moves them (few).
template <int CHUNKS>
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictMove m, const int32_t* lengths, int32_t* new_lengths, int heads,
                                                                  int budget, int recent, int32_t* source, int32_t* holes,
                                                                  int32_t* movers, int few, int lg) {
  __shared__ uint4 hist[kEvBins];   // (four copies of a bin side by side)
  __shared__ uint32_t scratch[kEvWaves];
  __shared__ uint32_t counts[CHUNKS][kEvWaves + 1];   // (rows in different banks)
  __shared__ int32_t few_s[2][kEvFew];
  __shared__ uint32_t pick_s[3];
  const int h = blockIdx.x, tid = threadIdx.x;
  const int n = evict_len(lengths, h / heads, m.cap);
  const int keep = min(n, budget);
  int32_t* src = source + (int64_t)h * budget;
  if (n <= budget) {
    if (!few)
      for (int i = tid; i < keep; i += kEvThreads) src[i] = i;
    else if (h % heads == 0 && tid == 0)
      new_lengths[h / heads] = keep;
    return;
  }
  const float* w = m.w + (int64_t)h * m.cap;
  const int32_t* id = m.ids + (int64_t)h * m.cap;
  for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = make_uint4(0, 0, 0, 0);
  uint32_t key[CHUNKS];
  {
    int32_t y[CHUNKS], newest = INT32_MIN;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {   // (of a slot behind the n-th the last one)
      const int slot = min(c * kEvThreads + tid, n - 1);
      y[c] = id[slot];
      key[c] = __float_as_uint(w[slot]);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) newest = max(newest, y[c]);
    newest = evict_max(newest, scratch);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {   // (0: no slot; the smallest key of a token, -inf's, is 0x007fffff)
      const uint32_t k = evict_key(__uint_as_float(key[c]), y[c], newest, recent);
      key[c] = c * kEvThreads + tid < n ? k : 0u;
    }
  }
  uint32_t prefix = 0, need = (uint32_t)keep, equal = 0;   // the need-th largest of the `equal` keys that begin with `prefix`
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    evict_count<CHUNKS>(key, pass, __builtin_amdgcn_readfirstlane(wave_id()) * kWave, n, prefix, hist);
    __syncthreads();
    evict_pick(
        [&](int bin) {   // (and cleared for the next pass)
          const uint4 four = hist[bin];
          hist[bin] = make_uint4(0, 0, 0, 0);
          return (four.x + four.y) + (four.z + four.w);
        },
        evict_shift(pass), prefix, need, equal, scratch, pick_s);
    if (need == equal) break;   // (all that begin with it stay: mostly two passes)
  }
  // (few: as many movers at most as there are slots behind `keep`; and LDS is nearer)
  int32_t* hole = few ? few_s[0] : holes + (int64_t)h * budget;
  int32_t* mover = few ? few_s[1] : movers + (int64_t)h * budget;
  uint32_t ties = 0, nh = 0, moved = 0;   // (as many movers as holes)
  if (need < equal)
    evict_lists<CHUNKS, true>(key, 0, keep, prefix, need, ties, nh, moved, counts, few ? nullptr : src, hole, mover);
  else
    evict_lists<CHUNKS, false>(key, 0, keep, prefix, need, ties, nh, moved, counts, few ? nullptr : src, hole, mover);
  __threadfence_block();
  __syncthreads();
  if (!few) {
    for (uint32_t i = tid; i < moved; i += kEvThreads) src[hole[i]] = mover[i];
    return;
  }
  for (uint32_t i = tid >> lg; i < moved; i += kEvThreads >> lg) evict_row(m, h, mover[i], hole[i], tid & ((1 << lg) - 1), 1 << lg);
  if (h % heads == 0 && tid == 0) new_lengths[h / heads] = keep;
}

// More slots than that: workgroups of `span` slots each, and a launch for every step that needs all of them.
//   0      newest id of each workgroup's slots; histograms cleared
//   1 2 3  histograms of the digits, added up in memory (integers: the order does not matter)
//   4      of each workgroup's slots, how many are above the key and how many have it, in front of `keep` and behind
//   5      lists
// What the launches before found is formed again by each workgroup that wants it.
struct EvictWide {
  uint32_t* hist;       // [bh][3][kEvBins]
  int32_t* newest;      // [bh][blocks]
  uint4* counts;        // [bh][blocks]: above in front, above behind, the same in front, behind
  uint32_t* moved;      // [bh]
  int blocks, span;
};
template <int STEP>
__global__ __launch_bounds__(kEvThreads) void evict_wide_kernel(EvictMove m, EvictWide x, const int32_t* lengths, int heads, int budget,
                                                                int recent, int32_t* source, int32_t* holes, int32_t* movers) {
  __shared__ uint4 hist[STEP >= 1 && STEP <= 3 ? kEvBins : 1];
  __shared__ uint32_t scratch[kEvWaves];
  __shared__ uint32_t counts[STEP == 5 ? kEvWide : 1][kEvWaves + 1];
  __shared__ uint32_t pick_s[3];
  const int h = blockIdx.y, block = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  const int n = evict_len(lengths, h / heads, m.cap), keep = min(n, budget);
  const int begin = min(n, block * x.span), end = min(n, begin + x.span);
  const float* w = m.w + (int64_t)h * m.cap;
  const int32_t* id = m.ids + (int64_t)h * m.cap;
  uint32_t* digits = x.hist + (int64_t)h * 3 * kEvBins;
  if constexpr (STEP == 0) {
    for (int i = block * kEvThreads + tid; i < 3 * kEvBins; i += x.blocks * kEvThreads) digits[i] = 0;
    int32_t newest = INT32_MIN;
    for (int first = begin; first < end; first += kEvWide * kEvThreads) {
      int32_t y[kEvWide];
#pragma unroll
      for (int c = 0; c < kEvWide; ++c) y[c] = id[min(first + c * kEvThreads + tid, end - 1)];
#pragma unroll
      for (int c = 0; c < kEvWide; ++c) newest = max(newest, y[c]);
    }
    newest = evict_max(newest, scratch);
    if (tid == 0) x.newest[(int64_t)h * x.blocks + block] = newest;
    return;
  }
  int32_t* src = source + (int64_t)h * budget;
  if (n <= budget) {
    if constexpr (STEP == 5) {
      for (int i = begin + tid; i < end; i += kEvThreads) src[i] = i;
      if (block == 0 && tid == 0) x.moved[h] = 0;
    }
    return;
  }
  int32_t newest = INT32_MIN;
  for (int i = tid; i < x.blocks; i += kEvThreads) newest = max(newest, x.newest[(int64_t)h * x.blocks + i]);
  newest = evict_max(newest, scratch);
  __syncthreads();
  uint32_t prefix = 0, need = (uint32_t)keep, equal = 0;
  constexpr int KNOWN = STEP <= 3 ? STEP - 1 : 3;
  bool found = false;
#pragma unroll
  for (int pass = 0; pass < KNOWN; ++pass) {
    if (found) break;
    evict_pick([&](int bin) { return digits[pass * kEvBins + bin]; }, evict_shift(pass), prefix, need, equal, scratch, pick_s);
    found = need == equal;
  }
  auto form = [&](int first, uint32_t (&key)[kEvWide]) {
    int32_t y[kEvWide];
#pragma unroll
    for (int c = 0; c < kEvWide; ++c) {
      const int slot = min(first + c * kEvThreads + tid, n - 1);
      key[c] = __float_as_uint(w[slot]);
      y[c] = id[slot];
    }
#pragma unroll
    for (int c = 0; c < kEvWide; ++c) {   // (0: no slot of the workgroup's)
      const uint32_t k = evict_key(__uint_as_float(key[c]), y[c], newest, recent);
      key[c] = first + c * kEvThreads + tid < end ? k : 0u;
    }
  };
  const int wave_first = __builtin_amdgcn_readfirstlane(wave_id()) * kWave;
  if constexpr (STEP <= 3) {
    if (found || begin >= end) return;
    constexpr int PASS = STEP - 1;
    for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int first = begin; first < end; first += kEvWide * kEvThreads) {
      uint32_t key[kEvWide];
      form(first, key);
      evict_count<kEvWide>(key, PASS, first + wave_first, end, prefix, hist);
    }
    __syncthreads();
    for (int i = tid; i < kEvBins; i += kEvThreads) {
      const uint4 four = hist[i];
      const uint32_t c = (four.x + four.y) + (four.z + four.w);
      if (c) atomicAdd(&digits[PASS * kEvBins + i], c);
    }
    return;
  }
  const bool has_ties = need < equal;
  if constexpr (STEP == 4) {
    uint32_t above[2] = {0, 0}, same[2] = {0, 0};   // in front of `keep` and behind
    for (int first = begin; first < end; first += kEvWide * kEvThreads) {
      uint32_t key[kEvWide];
      form(first, key);
#pragma unroll
      for (int c = 0; c < kEvWide; ++c) {
        const bool behind = first + c * kEvThreads + tid >= keep;
        const bool tie = has_ties & (key[c] == prefix), over = (key[c] >= prefix) & !tie;
        above[0] += (uint32_t)__popcll(__ballot(over & !behind));
        above[1] += (uint32_t)__popcll(__ballot(over & behind));
        same[0] += (uint32_t)__popcll(__ballot(tie & !behind));
        same[1] += (uint32_t)__popcll(__ballot(tie & behind));
      }
    }
    uint32_t total[4];   // (a wave's numbers are the same in its lanes: one of them adds)
    evict_scan(lane == 0 ? above[0] : 0u, scratch, total[0]);
    evict_scan(lane == 0 ? above[1] : 0u, scratch, total[1]);
    evict_scan(lane == 0 ? same[0] : 0u, scratch, total[2]);
    evict_scan(lane == 0 ? same[1] : 0u, scratch, total[3]);
    if (tid == 0) x.counts[(int64_t)h * x.blocks + block] = make_uint4(total[0], total[1], total[2], total[3]);
  }
  if constexpr (STEP == 5) {
    __shared__ uint32_t base_s[3];
    // thread i: workgroup i's counts (512 workgroups at most)
    const uint4 c = x.counts[(int64_t)h * x.blocks + min(tid, x.blocks - 1)];
    const bool in = tid < x.blocks;
    const int front = in ? min(max(keep - tid * x.span, 0), x.span) : 0;
    uint32_t total, moved;
    const uint32_t ties = evict_scan(in ? c.z + c.w : 0u, scratch, total);
    const uint32_t left = need > ties ? need - ties : 0u, tied = min(left, c.z), tied_behind = min(left - tied, c.w);
    const uint32_t nh = evict_scan(in ? (uint32_t)front - c.x - (has_ties ? tied : 0u) : 0u, scratch, total);
    const uint32_t nm = evict_scan(in ? c.y + (has_ties ? tied_behind : 0u) : 0u, scratch, moved);
    if (tid == block) {
      base_s[0] = ties;
      base_s[1] = nh;
      base_s[2] = nm;
    }
    if (block == 0 && tid == 0) x.moved[h] = moved;
    __syncthreads();
    uint32_t at[3] = {base_s[0], base_s[1], base_s[2]};
    int32_t *hole = holes + (int64_t)h * budget, *mover = movers + (int64_t)h * budget;
    for (int first = begin; first < end; first += kEvWide * kEvThreads) {
      uint32_t key[kEvWide];
      form(first, key);
      // (a slot behind the workgroup's last is no hole of its own: `keep` ends there too)
      if (has_ties)
        evict_lists<kEvWide, true>(key, first, min(keep, end), prefix, need, at[0], at[1], at[2], counts, src, hole, mover);
      else
        evict_lists<kEvWide, false>(key, first, min(keep, end), prefix, need, at[0], at[1], at[2], counts, src, hole, mover);
    }
  }
}
__global__ __launch_bounds__(kEvMoveThreads) void evict_pair_kernel(const uint32_t* moved, int budget, int32_t* source, const int32_t* holes,
                                                                    const int32_t* movers) {
  const int64_t head = (int64_t)blockIdx.y * budget;
  const int count = (int)moved[blockIdx.y];
  for (int i = (int)(blockIdx.x * kEvMoveThreads + threadIdx.x); i < count; i += (int)(gridDim.x * kEvMoveThreads))
    source[head + holes[head + i]] = movers[head + i];
}

// Row `slot` of head h takes the row source[slot]; 2^lg threads a row.
__global__ __launch_bounds__(kEvMoveThreads) void evict_move_kernel(EvictMove m, const int32_t* lengths, int32_t* new_lengths, int heads,
                                                                    int budget, int in_place, const int32_t* __restrict__ source,
                                                                    int lg) {
  const int h = blockIdx.y;
  const int keep = min(evict_len(lengths, h / heads, m.cap), budget);
  // (where the new lengths take the place of the old ones, another workgroup may find the new one: it gives the same `keep`)
  if (blockIdx.x == 0 && h % heads == 0 && threadIdx.x == 0) new_lengths[h / heads] = keep;
  const int rpb = kEvMoveThreads >> lg;
  for (int slot = (int)blockIdx.x * rpb + ((int)threadIdx.x >> lg); slot < keep; slot += (int)gridDim.x * rpb) {
    const int s = source[(int64_t)h * budget + slot];
    if (in_place && s == slot) continue;
    evict_row(m, h, s, slot, (int)threadIdx.x & ((1 << lg) - 1), 1 << lg);
  }
}

}  // namespace lrqk

using namespace lrqk;

// Words of 4 bytes: the lists, and what the launches over many slots leave for each other (in front, 16-byte aligned).
struct EvictPlan {
  int blocks = 0, span = 0;
  int64_t counts = 0, hist = 0, newest = 0, moved = 0, lists = 0, words = 0;   // where they begin
};
static EvictPlan evict_plan(int64_t bh, int cap, int budget) {
  EvictPlan p;
  if (cap > kEvMost) {
    const int round = kEvWide * kEvThreads, rounds = (cap + round - 1) / round;
    p.span = round * ((rounds + kEvMaxBlocks - 1) / kEvMaxBlocks);
    p.blocks = (cap + p.span - 1) / p.span;
    p.hist = p.counts + 4 * bh * p.blocks;
    p.newest = p.hist + 3 * bh * kEvBins;
    p.moved = p.newest + bh * p.blocks;
    p.lists = p.moved + bh;
  }
  p.words = p.lists + 3 * bh * std::min(cap, budget);
  return p;
}

static int evict_check(int b, int heads, int cap, int budget) {
  LRQK_REQUIRE(b > 0 && heads > 0 && cap > 0 && budget > 0, LRQK_EINVAL, "bad sizes b=%d heads=%d cap=%d budget=%d", b, heads, cap,
               budget);
  LRQK_REQUIRE((int64_t)b * heads <= 65535, LRQK_ELIMIT, "%d sequences of %d heads: at most 65535 heads in all", b, heads);
  LRQK_REQUIRE(cap <= (1 << 30), LRQK_ELIMIT, "cap=%d", cap);
  return LRQK_OK;
}

extern "C" int64_t lrqk_evict_workspace(int b, int heads, int cap, int budget) {
  const int rc = evict_check(b, heads, cap, budget);
  if (rc) return rc;
  return evict_plan((int64_t)b * heads, cap, budget).words * (int64_t)sizeof(int32_t);
}

extern "C" int lrqk_evict(float* weights, int32_t* ids, void* k, void* v, const int32_t* lengths, int cap, float* weights_out,
                          int32_t* ids_out, void* k_out, void* v_out, int cap_out, int32_t* new_lengths, int b, int heads, int d,
                          int budget, int recent, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(d > 0, LRQK_EINVAL, "bad sizes d=%d", d);
  const int rc = evict_check(b, heads, cap, budget);
  if (rc) return rc;
  LRQK_REQUIRE(recent >= 0 && recent <= budget, LRQK_EINVAL, "recent=%d outside 0..budget=%d", recent, budget);
  LRQK_REQUIRE(weights && ids && k && v && new_lengths && workspace, LRQK_EINVAL, "null pointer");
  const bool in_place = weights_out == nullptr;
  LRQK_REQUIRE(in_place ? !ids_out && !k_out && !v_out : ids_out && k_out && v_out, LRQK_EINVAL,
               "all of weights_out, ids_out, k_out, v_out or none of them");
  LRQK_REQUIRE(in_place || (weights_out != weights && ids_out != ids && k_out != k && v_out != v), LRQK_EINVAL,
               "an output is its own input: leave the outputs out to evict in place");
  LRQK_REQUIRE(in_place || cap_out >= std::min(cap, budget), LRQK_EINVAL, "%d rows for min(cap=%d, budget=%d) tokens", cap_out, cap,
               budget);
  const int row = d * (int)elem_size(dtype);
  LRQK_REQUIRE(row % 16 == 0, LRQK_ELIMIT, "head_dim %d unsupported (rows of whole 16-byte pieces)", d);
  LRQK_REQUIRE((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0 &&
                   (uintptr_t)workspace % 16 == 0,
               LRQK_EINVAL, "pointers must be 16-byte aligned");
  const int64_t need = lrqk_evict_workspace(b, heads, cap, budget);
  LRQK_REQUIRE(workspace_bytes >= need, LRQK_EINVAL, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes,
               (long long)need);
  budget = std::min(budget, cap);
  const int bh = b * heads;
  const EvictPlan p = evict_plan(bh, cap, budget);
  int32_t* words = (int32_t*)workspace;
  int32_t *source = words + p.lists, *holes = source + (int64_t)bh * budget, *movers = holes + (int64_t)bh * budget;
  hipStream_t st = (hipStream_t)stream;
  EvictMove m{(const uint4*)k, (const uint4*)v, (uint4*)(in_place ? k : k_out), (uint4*)(in_place ? v : v_out), weights, ids,
              in_place ? weights : weights_out, in_place ? ids : ids_out, cap, in_place ? cap : cap_out, row / 16};
  int lg = 0;
  while ((1 << lg) < m.chunks && (1 << lg) < kWave) ++lg;
  // (not where the new lengths take the place of the old ones, which the workgroups of the other heads still want to see)
  const int few = in_place && cap <= kEvMost && cap - budget <= kEvFew && new_lengths != lengths ? 1 : 0;
  const dim3 block(kEvThreads);
  if (cap <= kEvMost) {
    auto select = cap <= 4 * kEvThreads    ? evict_select_kernel<4>
                  : cap <= 12 * kEvThreads ? evict_select_kernel<12>
                                           : evict_select_kernel<32>;
    hipLaunchKernelGGL(select, dim3((unsigned)bh), block, 0, st, m, lengths, new_lengths, heads, budget, recent, source, holes, movers, few, lg);
  } else {
    const EvictWide x{(uint32_t*)words + p.hist, words + p.newest, (uint4*)(words + p.counts), (uint32_t*)words + p.moved, p.blocks, p.span};
    const dim3 grid((unsigned)p.blocks, (unsigned)bh);
    for (auto step : {evict_wide_kernel<0>, evict_wide_kernel<1>, evict_wide_kernel<2>, evict_wide_kernel<3>, evict_wide_kernel<4>, evict_wide_kernel<5>}) {
      hipLaunchKernelGGL(step, grid, block, 0, st, m, x, lengths, heads, budget, recent, source, holes, movers);
      LRQK_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(evict_pair_kernel, dim3((unsigned)std::min((budget + kEvMoveThreads - 1) / kEvMoveThreads, 64), (unsigned)bh),
                       dim3(kEvMoveThreads), 0, st, x.moved, budget, source, holes, movers);
  }
  LRQK_HIP_CHECK(hipGetLastError());
  if (few) return LRQK_OK;
  const int rpb = kEvMoveThreads >> lg;
  const int64_t blocks = ((int64_t)budget + rpb - 1) / rpb;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)std::min<int64_t>(blocks, std::max(1, 8192 / bh)), (unsigned)bh),
                     dim3(kEvMoveThreads), 0, st, m, lengths, new_lengths, heads, budget, in_place ? 1 : 0, source, lg);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
