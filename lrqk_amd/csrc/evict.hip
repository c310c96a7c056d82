// Eviction from a cache by the attention that its tokens got: of a head's n tokens `budget` stay, the `recent` newest
// ones (by their position ids) and, of the others, those with the largest weights (NaN counts as the largest; of equal
// ones those of the lowest slots).  A token that stays in slots 0 .. budget - 1 keeps its slot; the ones that stay of the
// slots behind move, in order, into the slots that became free, in order.  So no row has to wait for another: sources
// and destinations do not overlap, and a cache that is a few tokens over its budget moves a few rows.
//
//   select   one workgroup per head: the budget-th largest 32-bit key by a radix search over histograms in LDS (11, 11 and 10
//            bits; ties by slot), then the list source[slot] of the slots that stay.  The keys of up to 32768 tokens are in
//            registers; of more they are formed again for every look.
//   move     rows of K and V, weights and ids.  In place and with few tokens over the budget select does that too.
//
// Bound by the instructions of the one workgroup, not by the memory: a wave's instruction takes its SIMD 4 cycles, so each
// one that looks at every key of 32768 takes 0.25 us.  8 heads of 32768 tokens down to 2112: select 22 us (reads 3, keys and
// the first histogram 4, the others 4, counting 3, the lists 5), move 5 us.  32 heads of 2117 tokens down to 2112, in place
// and in one launch: 10 us, most of it the chain of barriers.  (Several workgroups a head would have to wait for each other
// four times, as launches of some 4 us each.  A wave's slots one behind the other need no table of counts, but then one
// or two waves have all slots in front of `keep`, which cost most: 24 us.  Copies of a histogram per wave instead of per
// lane: no difference.)
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace lrqk {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / kWave;
constexpr int kEvBins = 2048, kEvCopies = 4;    // of a histogram, and how many share a wave's additions
constexpr int kEvMoveThreads = 256;
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

// Sums over the workgroup's threads in order: of what stands in front of the thread, and of all.  Two barriers.
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
  __syncthreads();
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

// A block of slots is CHUNKS rounds of a piece of 64 slots for each wave, whose keys are in registers.  MANY: more slots
// than the largest block has, and the keys are formed again for every look at them.  source: [bh][budget]; holes, movers:
// [bh][budget] scratch.  lg: 2^lg threads move a row, where this launch moves them (few).
template <int CHUNKS, bool MANY>
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictMove m, const int32_t* lengths, int32_t* new_lengths, int heads,
                                                                  int budget, int recent, int32_t* source, int32_t* holes,
                                                                  int32_t* movers, int few, int lg) {
  static_assert(CHUNKS <= kWave, "a lane for the counts of each round");
  __shared__ uint4 hist[kEvBins];   // (four copies of a bin side by side)
  __shared__ uint32_t scratch[kEvWaves];
  __shared__ uint32_t counts[CHUNKS][kEvWaves + 1];   // (rows in different banks)
  __shared__ uint32_t pick_s[3];
  const int h = blockIdx.x, tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
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
  const int blocks = MANY ? (n + CHUNKS * kEvThreads - 1) / (CHUNKS * kEvThreads) : 1;
  // first slot of a round's piece (up to 2^30 slots and a block more)
  auto first_slot = [&](int block, int c) { return (block * CHUNKS + c) * kEvThreads + wave * kWave; };
  uint32_t key[CHUNKS];
  int32_t newest = INT32_MIN;
  {
    int32_t y[CHUNKS];
    auto read = [&](int block) {   // (of a slot behind the n-th the last one)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int slot = min(first_slot(block, c) + lane, n - 1);
        y[c] = id[slot];
        if constexpr (!MANY) key[c] = __float_as_uint(w[slot]);
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) newest = max(newest, y[c]);
    };
    for (int block = 0; block < blocks; ++block) read(block);
    newest = (int32_t)(wave_reduce_u32((uint32_t)newest ^ 0x80000000u, [](uint32_t a, uint32_t b) { return max(a, b); }) ^ 0x80000000u);
    if (lane == 0) scratch[wave] = (uint32_t)newest;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) newest = max(newest, (int32_t)scratch[i]);
    if constexpr (!MANY) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {   // (0: no slot; the smallest key of a token, -inf's, is 0x007fffff)
        const uint32_t k = evict_key(__uint_as_float(key[c]), y[c], newest, recent);
        key[c] = first_slot(0, c) + lane < n ? k : 0u;
      }
    }
  }
  auto form = [&](int block) {
    if constexpr (MANY) {
      int32_t y[CHUNKS];
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int slot = min(first_slot(block, c) + lane, n - 1);
        key[c] = __float_as_uint(w[slot]);
        y[c] = id[slot];
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t k = evict_key(__uint_as_float(key[c]), y[c], newest, recent);
        key[c] = first_slot(block, c) + lane < n ? k : 0u;
      }
    }
  };

  uint32_t prefix = 0, need = (uint32_t)keep, equal = 0;   // the need-th largest of the `equal` keys that begin with `prefix`
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t limit = pass == 1 ? 1u << 21 : 1u << 10;
    for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t* mine = (uint32_t*)hist + (lane & (kEvCopies - 1));
    for (int block = 0; block < blocks; ++block) {
      form(block);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {   // (what is no slot is in the first bins, which are behind all tokens)
        const uint32_t rest = key[c] ^ prefix;
        if (pass == 0 ? first_slot(block, c) < n : rest < limit) atomicAdd(&mine[kEvCopies * (rest >> shift)], 1u);
      }
    }
    __syncthreads();
    // two bins a thread, the largest first
    uint32_t c[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 four = hist[kEvBins - 1 - (2 * tid + j)];
      c[j] = (four.x + four.y) + (four.z + four.w);
    }
    uint32_t total;
    uint32_t before = evict_scan(c[0] + c[1], scratch, total);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (before < need && need <= before + c[j]) {
        pick_s[0] = (uint32_t)(kEvBins - 1 - (2 * tid + j));
        pick_s[1] = need - before;
        pick_s[2] = c[j];
      }
      before += c[j];
    }
    __syncthreads();
    prefix |= pick_s[0] << shift;
    need = pick_s[1];
    equal = pick_s[2];
    if (need == equal) break;   // (all that begin with it stay: mostly two passes)
  }
  // Every key from `prefix` on stays, or where fewer are needed than have it, the first `need` of those.  Lane c has the
  // counts of the wave's round c, and the table of all waves' says what is in front of its piece.
  int32_t* hole = holes + (int64_t)h * budget;
  int32_t* mover = movers + (int64_t)h * budget;
  uint32_t moved = 0;   // (as many movers as holes)
  auto list = [&](auto has_ties) {
    constexpr bool TIES = decltype(has_ties)::value;
    uint32_t ties = 0, nh = 0, nm = 0;   // of the blocks before
    // two numbers of lane c, in 16 bits each: their sums over the pieces in front of the wave's of round c
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
    for (int block = 0; block < blocks; ++block) {
      form(block);
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
      int mine = 0;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int first = first_slot(block, c);
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
        const int first = first_slot(block, c);
        const bool stay = stays(c);
        const uint32_t mover_at = (uint32_t)__builtin_amdgcn_readlane((int)am, c);
        if (first >= keep) {
          put(mover, stay, mover_at, first + lane);
        } else {
          const bool front = first + lane < keep;
          put(hole, front & !stay, (uint32_t)__builtin_amdgcn_readlane((int)ah, c), first + lane);
          put(mover, stay & !front, mover_at, first + lane);
          if (!few && (stay & front)) src[first + lane] = first + lane;
        }
      }
    }
    moved = nm;
  };
  if (need < equal)
    list(std::true_type{});
  else
    list(std::false_type{});
  __threadfence_block();
  __syncthreads();
  if (!few) {
    for (uint32_t i = tid; i < moved; i += kEvThreads) src[hole[i]] = mover[i];
    return;
  }
  for (uint32_t i = tid >> lg; i < moved; i += kEvThreads >> lg) evict_row(m, h, mover[i], hole[i], tid & ((1 << lg) - 1), 1 << lg);
  if (h % heads == 0 && tid == 0) new_lengths[h / heads] = keep;
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

extern "C" int64_t lrqk_evict_workspace(int b, int heads, int cap, int budget) {
  LRQK_REQUIRE(b > 0 && heads > 0 && cap > 0 && budget > 0, LRQK_EINVAL, "bad sizes b=%d heads=%d cap=%d budget=%d", b, heads, cap,
               budget);
  return (int64_t)b * heads * std::min(cap, budget) * 3 * (int64_t)sizeof(int32_t);
}

extern "C" int lrqk_evict(float* weights, int32_t* ids, void* k, void* v, const int32_t* lengths, int cap, float* weights_out,
                          int32_t* ids_out, void* k_out, void* v_out, int cap_out, int32_t* new_lengths, int b, int heads, int d,
                          int budget, int recent, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(b > 0 && heads > 0 && d > 0 && cap > 0 && budget > 0, LRQK_EINVAL, "bad sizes b=%d heads=%d d=%d cap=%d budget=%d",
               b, heads, d, cap, budget);
  LRQK_REQUIRE((int64_t)b * heads <= 65535, LRQK_ELIMIT, "%d sequences of %d heads: at most 65535 heads in all", b, heads);
  LRQK_REQUIRE(cap <= (1 << 30), LRQK_ELIMIT, "cap=%d", cap);
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
  int32_t* source = (int32_t*)workspace;
  int32_t *holes = source + (int64_t)bh * budget, *movers = holes + (int64_t)bh * budget;
  hipStream_t st = (hipStream_t)stream;
  EvictMove m{(const uint4*)k, (const uint4*)v, (uint4*)(in_place ? k : k_out), (uint4*)(in_place ? v : v_out), weights, ids,
              in_place ? weights : weights_out, in_place ? ids : ids_out, cap, in_place ? cap : cap_out, row / 16};
  int lg = 0;
  while ((1 << lg) < m.chunks && (1 << lg) < kWave) ++lg;
  // (not where the new lengths take the place of the old ones, which the workgroups of the other heads still want to see)
  const int few = in_place && cap - budget <= kEvFew && new_lengths != lengths ? 1 : 0;
  const dim3 grid((unsigned)bh), block(kEvThreads);
  auto select = cap <= 4 * kEvThreads    ? evict_select_kernel<4, false>
                : cap <= 12 * kEvThreads ? evict_select_kernel<12, false>
                : cap <= 32 * kEvThreads ? evict_select_kernel<32, false>
                                         : evict_select_kernel<32, true>;
  hipLaunchKernelGGL(select, grid, block, 0, st, m, lengths, new_lengths, heads, budget, recent, source, holes, movers, few, lg);
  LRQK_HIP_CHECK(hipGetLastError());
  if (few) return LRQK_OK;
  const int rpb = kEvMoveThreads >> lg;
  const int64_t blocks = ((int64_t)budget + rpb - 1) / rpb;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)std::min<int64_t>(blocks, std::max(1, 8192 / bh)), (unsigned)bh),
                     dim3(kEvMoveThreads), 0, st, m, lengths, new_lengths, heads, budget, in_place ? 1 : 0, source, lg);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
