// Eviction from a cache by the attention that its tokens got: of a head's n tokens `budget` stay, the `recent` newest
// ones (by their position ids) and, of the others, those with the largest weights (NaN counts as the largest; of equal
// ones those of the lowest slots).  A token that stays in slots 0 .. budget - 1 keeps its slot; the ones that stay of the
// slots behind move, in order, into the slots that became free, in order.  So no row has to wait for another: sources
// and destinations do not overlap, and a cache that is a few tokens over its budget moves a few rows.
//
//   select   one workgroup per head: the budget-th largest 32-bit key by a radix search over histograms in LDS (ties by
//            slot), then the list source[slot] of the slots that stay
//   move     rows of K and V, weights and ids
#include <algorithm>

#include "common.hpp"

namespace lrqk {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / kWave;
constexpr int kEvPer = 4;                       // slots of a thread per trip
constexpr int kEvTrip = kEvThreads * kEvPer;
constexpr int kEvMoveThreads = 256;

// Order of the tokens: the newest in front of everything, then NaN, then by weight.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t id, int32_t newest, int recent) {
  if ((int64_t)id > (int64_t)newest - recent) return 0xffffffffu;
  return w != w ? 0xfffffffeu : score_key(w);
}

__device__ __forceinline__ int evict_len(const int32_t* lengths, int b, int cap) {
  return lengths ? min(max(lengths[b], 0), cap) : cap;
}

// exclusive sum over the workgroup's threads in order, and the total; scratch: kEvWaves ints
__device__ __forceinline__ int evict_scan(int v, int* scratch, int& total) {
  const int incl = wave_inclusive_sum(v);
  if (lane_id() == kWave - 1) scratch[wave_id()] = incl;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kEvWaves; ++w) {
    const int c = scratch[w];
    if (w < wave_id()) base += c;
    all += c;
  }
  __syncthreads();
  total = all;
  return base + incl - v;
}

// source: [bh][budget]; holes, movers: [bh][budget] scratch.
__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(const float* __restrict__ weights,
                                                                  const int32_t* __restrict__ ids,
                                                                  const int32_t* __restrict__ lengths, int heads, int cap,
                                                                  int budget, int recent, int32_t* source, int32_t* holes,
                                                                  int32_t* movers) {
  __shared__ uint32_t hist[kEvWaves][256];
  __shared__ int scratch[kEvWaves];
  __shared__ uint32_t pick_s[2];
  const int h = blockIdx.x, tid = threadIdx.x;
  const int n = evict_len(lengths, h / heads, cap);
  const int keep = min(n, budget);
  int32_t* src = source + (int64_t)h * budget;
  if (n <= budget) {
    for (int i = tid; i < keep; i += kEvThreads) src[i] = i;
    return;
  }
  const float* w = weights + (int64_t)h * cap;
  const int32_t* id = ids + (int64_t)h * cap;
  int32_t newest = INT32_MIN;
  for (int i = tid; i < n; i += kEvThreads) newest = max(newest, id[i]);
  newest = (int32_t)(wave_reduce_u32((uint32_t)newest ^ 0x80000000u, [](uint32_t a, uint32_t b) { return max(a, b); }) ^ 0x80000000u);
  if (lane_id() == 0) scratch[wave_id()] = newest;
  __syncthreads();
  newest = scratch[0];
#pragma unroll
  for (int i = 1; i < kEvWaves; ++i) newest = max(newest, scratch[i]);

  uint32_t prefix = 0, need = (uint32_t)keep;   // the need-th largest of the keys that begin with `prefix` is looked for
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < kEvWaves * 256; i += kEvThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int i = tid; i < n; i += kEvThreads) {
      const uint32_t k = evict_key(w[i], id[i], newest, recent);
      if ((k & high) == prefix) atomicAdd(&hist[wave_id()][(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t c = 0;
#pragma unroll
      for (int i = 0; i < kEvWaves; ++i) c += hist[i][tid];
      hist[0][tid] = c;
    }
    __syncthreads();
    if (tid < kWave) {  // four bins a lane, the largest first
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += c[j] = hist[0][255 - (4 * tid + j)];
      uint32_t before = (uint32_t)wave_inclusive_sum((int)sum) - sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (before < need && need <= before + c[j]) {
          pick_s[0] = 255 - (4 * tid + j);
          pick_s[1] = need - before;
        }
        before += c[j];
      }
    }
    __syncthreads();
    prefix |= pick_s[0] << shift;
    need = pick_s[1];
    __syncthreads();
  }
  // every key above `prefix` stays, and the first `need` of those that equal it
  int32_t* hole = holes + (int64_t)h * budget;
  int32_t* mover = movers + (int64_t)h * budget;
  int ties = 0, nh = 0, nm = 0;
  for (int base = 0; base < n; base += kEvTrip) {
    const int i0 = base + tid * kEvPer;
    uint32_t k[kEvPer];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kEvPer; ++j) {
      k[j] = i0 + j < n ? evict_key(w[i0 + j], id[i0 + j], newest, recent) : 0u;
      mine += i0 + j < n && k[j] == prefix;
    }
    int total;
    int rank = ties + evict_scan(mine, scratch, total);
    ties += total;
    bool stay[kEvPer];
    int packed = 0;  // holes in the low half, movers in the high one (a trip has 4096 slots)
#pragma unroll
    for (int j = 0; j < kEvPer; ++j) {
      const bool in = i0 + j < n;
      stay[j] = in && (k[j] > prefix || (k[j] == prefix && rank < (int)need));
      rank += in && k[j] == prefix;
      if (in && i0 + j < keep) packed += !stay[j];
      if (in && i0 + j >= keep) packed += stay[j] ? 0x10000 : 0;
    }
    const int at = evict_scan(packed, scratch, total);
    int ah = nh + (at & 0xffff), am = nm + (at >> 16);
    nh += total & 0xffff;
    nm += total >> 16;
#pragma unroll
    for (int j = 0; j < kEvPer; ++j) {
      const int slot = i0 + j;
      if (slot >= n) continue;
      if (slot < keep) {
        if (stay[j]) src[slot] = slot;
        else hole[ah++] = slot;
      } else if (stay[j]) {
        mover[am++] = slot;
      }
    }
  }
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < nh; i += kEvThreads) src[hole[i]] = mover[i];   // (nh == nm: keep slots hold keep tokens)
}

struct EvictMove {
  const uint4 *k, *v;
  uint4 *k_out, *v_out;
  const float* w;
  const int32_t* ids;
  float* w_out;
  int32_t* ids_out;
  int cap, cap_out, chunks;   // slots of a head; 16-byte pieces of a row
};

// Row `slot` of head h takes the row source[slot]; cpr = 2^lg threads a row, its K and then its V.
__global__ __launch_bounds__(kEvMoveThreads) void evict_move_kernel(EvictMove m, const int32_t* __restrict__ lengths,
                                                                    int32_t* new_lengths, int heads, int budget, int in_place,
                                                                    const int32_t* __restrict__ source, int lg) {
  const int h = blockIdx.y;
  const int n = evict_len(lengths, h / heads, m.cap);
  const int keep = min(n, budget);
  if (blockIdx.x == 0 && h % heads == 0 && threadIdx.x == 0) new_lengths[h / heads] = keep;
  const int rpb = kEvMoveThreads >> lg;
  const int sub = threadIdx.x & ((1 << lg) - 1);
  for (int slot = (int)blockIdx.x * rpb + (threadIdx.x >> lg); slot < keep; slot += gridDim.x * rpb) {
    const int s = source[(int64_t)h * budget + slot];
    if (in_place && s == slot) continue;
    const int64_t from = (int64_t)h * m.cap + s, to = (int64_t)h * m.cap_out + slot;
    for (int c = sub; c < m.chunks; c += 1 << lg) {
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
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)bh), dim3(kEvThreads), 0, st, weights, ids, lengths, heads, cap, budget,
                     recent, source, holes, movers);
  LRQK_HIP_CHECK(hipGetLastError());
  EvictMove m{(const uint4*)k, (const uint4*)v, (uint4*)(in_place ? k : k_out), (uint4*)(in_place ? v : v_out), weights, ids,
              in_place ? weights : weights_out, in_place ? ids : ids_out, cap, in_place ? cap : cap_out, row / 16};
  int lg = 0;
  while ((1 << lg) < m.chunks && (1 << lg) < kWave) ++lg;
  const int rpb = kEvMoveThreads >> lg;
  const int64_t blocks = ((int64_t)budget + rpb - 1) / rpb;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)std::min<int64_t>(blocks, std::max(1, 8192 / bh)), (unsigned)bh),
                     dim3(kEvMoveThreads), 0, st, m, lengths, new_lengths, heads, budget, in_place ? 1 : 0, source, lg);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}
