// Eviction from a cache by the attention that its tokens got: of a head's n tokens `budget` stay, the `recent` newest
// ones (by their position ids) and, of the others, those with the largest weights (NaN counts as the largest; of equal
// ones those of the lowest slots).  A token that stays in slots 0 .. budget - 1 keeps its slot; the ones that stay of the
// slots behind move, in order, into the slots that became free, in order.  So no row has to wait for another: sources
// and destinations do not overlap, and a cache that is a few tokens over its budget moves a few rows.
//
//   select   one workgroup per head: the budget-th largest 32-bit key by a radix search over histograms in LDS (11, 11 and 10
//            bits; ties by slot), then the list source[slot] of the slots that stay.  The keys of up to 32768 tokens are in
//            registers; of more they are formed again for every pass.
//   move     rows of K and V, weights and ids.  In place and with few tokens over the budget select does that too.
//
// Bound by the latency of one workgroup's passes (32768 tokens: 256 KB to one CU), not by the memory.
#include <algorithm>

#include "common.hpp"

namespace lrqk {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / kWave;
constexpr int kEvPer = 4;                       // slots of a thread per trip: 16 bytes of weights and of ids
constexpr int kEvTrip = kEvThreads * kEvPer;
constexpr int kEvBins = 2048, kEvCopies = 4;    // of a histogram, and how many share the waves' additions
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

// Order of the tokens: the newest in front of everything, then NaN, then by weight.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t id, int32_t newest, int recent) {
  if ((int64_t)id > (int64_t)newest - recent) return 0xffffffffu;
  return w != w ? 0xfffffffeu : score_key(w);
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

// The same for N values a thread, all threads' first ones in front of the second ones.  scratch: 129 words.  Three
// barriers, however many.
template <int N>
__device__ __forceinline__ void evict_scan_trips(uint32_t (&v)[N], uint32_t* scratch, uint32_t& total) {
  static_assert(N * kEvWaves <= 2 * kWave, "two sums a lane");
  uint32_t incl[N];
#pragma unroll
  for (int t = 0; t < N; ++t) {
    incl[t] = (uint32_t)wave_inclusive_sum((int)v[t]);
    if (lane_id() == kWave - 1) scratch[t * kEvWaves + wave_id()] = incl[t];
  }
  __syncthreads();
  if (wave_id() == 0) {
    const int i = 2 * lane_id();
    const uint32_t a = i < N * kEvWaves ? scratch[i] : 0u, b = i < N * kEvWaves ? scratch[i + 1] : 0u;
    const uint32_t end = (uint32_t)wave_inclusive_sum((int)(a + b));
    scratch[i] = end - a - b;
    scratch[i + 1] = end - b;
    if (lane_id() == kWave - 1) scratch[2 * kWave] = end;
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < N; ++t) v[t] = scratch[t * kEvWaves + wave_id()] + incl[t] - v[t];
  total = scratch[2 * kWave];
  __syncthreads();
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

// TRIPS: trips whose keys are in registers (0: none).  source: [bh][budget]; holes, movers: [bh][budget] scratch.  lg: 2^lg
// threads move a row, where this launch moves them (few).
template <int TRIPS>
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictMove m, const int32_t* lengths, int32_t* new_lengths, int heads,
                                                                  int budget, int recent, int32_t* source, int32_t* holes,
                                                                  int32_t* movers, int few, int lg) {
  __shared__ uint32_t hist[kEvCopies][kEvBins];
  __shared__ uint32_t scratch[2 * kWave + 1];
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
  const bool wide = m.cap % 4 == 0 && (uintptr_t)m.w % 16 == 0 && (uintptr_t)m.ids % 16 == 0;
  const int trips = TRIPS > 0 ? TRIPS : (n + kEvTrip - 1) / kEvTrip;
  // weights and ids of the thread's slots of a trip (behind the n-th: the last one's)
  auto read = [&](int trip, float (&x)[kEvPer], int32_t (&y)[kEvPer]) {
    const int i0 = trip * kEvTrip + tid * kEvPer;
    if (wide && i0 + kEvPer <= n) {
      const float4 a = *(const float4*)(w + i0);
      const int4 b = *(const int4*)(id + i0);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      y[0] = b.x; y[1] = b.y; y[2] = b.z; y[3] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < kEvPer; ++j) {
        x[j] = w[min(i0 + j, n - 1)];
        y[j] = id[min(i0 + j, n - 1)];
      }
    }
  };
  constexpr int HELD = TRIPS > 0 ? TRIPS : 1;
  constexpr bool ONCE = TRIPS > 0 && TRIPS <= 3;   // (there is room for the ids too until the newest one is known)
  uint32_t key[HELD][kEvPer];
  int32_t held_id[ONCE ? TRIPS : 1][kEvPer];
  int32_t newest = INT32_MIN;
  if constexpr (ONCE) {
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) {
      float x[kEvPer];
      read(t, x, held_id[t]);
#pragma unroll
      for (int j = 0; j < kEvPer; ++j) {
        key[t][j] = __float_as_uint(x[j]);
        newest = max(newest, held_id[t][j]);
      }
    }
  } else {
#pragma unroll 4
    for (int t = 0; t < trips; ++t) {
      const int i0 = t * kEvTrip + tid * kEvPer;
      if (wide && i0 + kEvPer <= n) {
        const int4 y = *(const int4*)(id + i0);
        newest = max(max(max(newest, y.x), y.y), max(y.z, y.w));
      } else {
#pragma unroll
        for (int j = 0; j < kEvPer; ++j) newest = max(newest, id[min(i0 + j, n - 1)]);
      }
    }
  }
  newest = (int32_t)(wave_reduce_u32((uint32_t)newest ^ 0x80000000u, [](uint32_t a, uint32_t b) { return max(a, b); }) ^ 0x80000000u);
  if (lane_id() == 0) scratch[wave_id()] = (uint32_t)newest;
  __syncthreads();
  newest = (int32_t)scratch[0];
#pragma unroll
  for (int i = 1; i < kEvWaves; ++i) newest = max(newest, (int32_t)scratch[i]);
  // (0: no slot; the smallest key of a token, -inf's, is 0x007fffff)
  if constexpr (TRIPS > 0) {
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) {
      float x[kEvPer];
      int32_t y[kEvPer];
      if constexpr (!ONCE) read(t, x, y);
#pragma unroll
      for (int j = 0; j < kEvPer; ++j) {
        const bool in = t * kEvTrip + tid * kEvPer + j < n;
        const uint32_t k = ONCE ? evict_key(__uint_as_float(key[t][j]), held_id[ONCE ? t : 0][j], newest, recent) : evict_key(x[j], y[j], newest, recent);
        key[t][j] = in ? k : 0u;
      }
    }
  }
  auto keys = [&](int t, uint32_t (&k)[kEvPer]) {
    if constexpr (TRIPS == 0) {
      float x[kEvPer];
      int32_t y[kEvPer];
      read(t, x, y);
#pragma unroll
      for (int j = 0; j < kEvPer; ++j) {
        const bool in = t * kEvTrip + tid * kEvPer + j < n;
        const uint32_t v = evict_key(x[j], y[j], newest, recent);
        k[j] = in ? v : 0u;
      }
    }
  };

  uint32_t prefix = 0, high = 0, need = (uint32_t)keep, equal = 0;   // the need-th largest of the keys that begin with `prefix`
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < kEvCopies * kEvBins; i += kEvThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    uint32_t* mine = hist[wave_id() & (kEvCopies - 1)];
    auto count = [&](const uint32_t (&k)[kEvPer]) {
#pragma unroll
      for (int j = 0; j < kEvPer; ++j)
        if (k[j] != 0u && (k[j] & high) == prefix) atomicAdd(&mine[(k[j] >> shift) & (bins - 1)], 1u);
    };
    if constexpr (TRIPS > 0) {
#pragma unroll
      for (int t = 0; t < TRIPS; ++t) count(key[t]);
    } else {
#pragma unroll 2
      for (int t = 0; t < trips; ++t) {
        uint32_t k[kEvPer];
        keys(t, k);
        count(k);
      }
    }
    __syncthreads();
    // two bins a thread, the largest first
    uint32_t c[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int bin = kEvBins - 1 - (2 * tid + j);
      c[j] = 0;
#pragma unroll
      for (int i = 0; i < kEvCopies; ++i) c[j] += hist[i][bin];
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
    high |= (uint32_t)(bins - 1) << shift;
    need = pick_s[1];
    equal = pick_s[2];
  }
  // every key above `prefix` stays, and the first `need` of the `equal` ones that have it
  int32_t* hole = holes + (int64_t)h * budget;
  int32_t* mover = movers + (int64_t)h * budget;
  uint32_t ties = 0, nh = 0, nm = 0;
  const bool rank_ties = need < equal;
  auto tied = [&](int t, const uint32_t (&k)[kEvPer]) {
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < kEvPer; ++j) mine += ((k[j] == prefix) & (t * kEvTrip + tid * kEvPer + j < n)) ? 1u : 0u;
    return mine;
  };
  // which of the slots' tokens stay (a bit each), and how many holes (low half) and movers (high half) that makes; rank: of
  // the first tie
  auto decide = [&](int t, const uint32_t (&k)[kEvPer], uint32_t rank, uint32_t& bits) {
    uint32_t packed = 0;
    bits = 0;
#pragma unroll
    for (int j = 0; j < kEvPer; ++j) {
      const int slot = t * kEvTrip + tid * kEvPer + j;
      const bool in = slot < n, tie = in & (k[j] == prefix), stay = in & ((k[j] > prefix) | (tie & (rank < need)));
      rank += (rank_ties & tie) ? 1u : 0u;
      bits |= stay ? 1u << j : 0u;
      packed += (in & (slot < keep) & !stay) ? 1u : 0u;
      packed += (stay & (slot >= keep)) ? 0x10000u : 0u;
    }
    return packed;
  };
  auto emit = [&](int t, uint32_t bits, uint32_t ah, uint32_t am) {
#pragma unroll
    for (int j = 0; j < kEvPer; ++j) {
      const int slot = t * kEvTrip + tid * kEvPer + j;
      if (slot >= n) continue;
      if (slot < keep) {
        if (!(bits >> j & 1u)) hole[ah++] = slot;
        else if (!few) src[slot] = slot;
      } else if (bits >> j & 1u) {
        mover[am++] = slot;
      }
    }
  };
  if constexpr (TRIPS > 0) {   // (up to 32767 holes and as many movers: the halves hold them)
    uint32_t at[TRIPS], bits[TRIPS], total;
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) at[t] = 0;
    if (rank_ties) {
#pragma unroll
      for (int t = 0; t < TRIPS; ++t) at[t] = tied(t, key[t]);
      evict_scan_trips<TRIPS>(at, scratch, total);
    }
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) at[t] = decide(t, key[t], at[t], bits[t]);
    evict_scan_trips<TRIPS>(at, scratch, total);
#pragma unroll
    for (int t = 0; t < TRIPS; ++t) emit(t, bits[t], at[t] & 0xffffu, at[t] >> 16);
    nh = total & 0xffffu;
  } else {
    for (int t = 0; t < trips; ++t) {
      uint32_t k[kEvPer], rank = 0, bits, total;
      keys(t, k);
      if (rank_ties) {
        rank = ties + evict_scan(tied(t, k), scratch, total);
        ties += total;
      }
      const uint32_t at = evict_scan(decide(t, k, rank, bits), scratch, total);
      emit(t, bits, nh + (at & 0xffffu), nm + (at >> 16));
      nh += total & 0xffffu;
      nm += total >> 16;
    }
  }
  __threadfence_block();
  __syncthreads();
  // (nh == nm: keep slots hold keep tokens)
  if (!few) {
    for (uint32_t i = tid; i < nh; i += kEvThreads) src[hole[i]] = mover[i];
    return;
  }
  for (uint32_t i = tid >> lg; i < nh; i += kEvThreads >> lg) evict_row(m, h, mover[i], hole[i], tid & ((1 << lg) - 1), 1 << lg);
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
  const int trips = (cap + kEvTrip - 1) / kEvTrip;
  const dim3 grid((unsigned)bh), block(kEvThreads);
  if (trips <= 1)
    hipLaunchKernelGGL((evict_select_kernel<1>), grid, block, 0, st, m, lengths, new_lengths, heads, budget, recent, source, holes, movers,
                       few, lg);
  else if (trips <= 3)
    hipLaunchKernelGGL((evict_select_kernel<3>), grid, block, 0, st, m, lengths, new_lengths, heads, budget, recent, source, holes, movers,
                       few, lg);
  else if (trips <= 8)
    hipLaunchKernelGGL((evict_select_kernel<8>), grid, block, 0, st, m, lengths, new_lengths, heads, budget, recent, source, holes, movers,
                       few, lg);
  else
    hipLaunchKernelGGL((evict_select_kernel<0>), grid, block, 0, st, m, lengths, new_lengths, heads, budget, recent, source, holes, movers,
                       few, lg);
  LRQK_HIP_CHECK(hipGetLastError());
  if (few) return LRQK_OK;
  const int rpb = kEvMoveThreads >> lg;
  const int64_t blocks = ((int64_t)budget + rpb - 1) / rpb;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)std::min<int64_t>(blocks, std::max(1, 8192 / bh)), (unsigned)bh),
                     dim3(kEvMoveThreads), 0, st, m, lengths, new_lengths, heads, budget, in_place ? 1 : 0, source, lg);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
