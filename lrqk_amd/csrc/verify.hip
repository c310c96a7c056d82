// Drafted tokens verified against the target's probabilities (speculative sampling on a tree), from given random numbers.
//
// Node 0 of a sequence's tree is certain; node i > 0 was drawn from row parent[i] of the drafting model's probabilities p, and
// q[i] is the target's distribution behind node i.  A node's children x_1 .. x_k are looked at in order, with what is left of
// the distribution: r_0 = q, Z_0 = 1; x_j is accepted if u_j p(x_j) Z_(j-1) < r_(j-1)(x_j), and if it is not
//
//   r_j = max(r_(j-1) - Z_(j-1) p, 0) = max(q - C_j p, 0),  C_j = C_(j-1) + Z_(j-1), C_0 = 0,  Z_j = sum of r_j,
//
// so that one pass over two rows gives Z_j, and only nodes with several children need one.  Drafts without probabilities have
// p = 1 at their token: r_j is r_(j-1) without it.  Behind the last accepted node the next token is drawn from what is left:
// the lowest x with r(0) + .. + r(x) > u_0 sum(r).  Everything is formed in 64 bits, since a vocabulary's sums in 32 would
// put the border between two tokens elsewhere; what is not a positive number counts as 0.
//
// Three launches: Z of the nodes with several children (trees with p only); the walk, by every workgroup for itself, and the
// sums of what is left by chunks of the vocabulary; the chunk and the token.
#include <algorithm>

#include "common.hpp"

namespace lrqk {

constexpr int kVfThreads = 256, kVfMost = 1024;      // nodes of a tree, at most
constexpr int kVfEach = 8, kVfChunk = kVfThreads * kVfEach;   // elements of a thread, and of a workgroup
constexpr int kVfWide = 1024;                        // threads of the workgroup that has a node's rows for itself

struct VerifyArgs {
  const int32_t *tokens, *parents;   // [b][s]; parents: or null, a chain
  const void *q, *p;                 // rows of the vocabulary; p: or null
  int64_t qb, qr, pb, pr;            // elements between sequences and rows
  const float* u;                    // [b][s]
  int32_t *path, *counts, *next;
  double *cut, *mass;                // [b][s]: C and Z that a node's test is made with (trees with p)
  double* sums;                      // [b][chunks]
  double* left;                      // [b]: C behind the last accepted node
  int32_t* end;                      // [b]: the last accepted node
  int b, s, vocab, chunks;
};

__device__ __forceinline__ double vf_positive(double x) { return x > 0.0 ? x : 0.0; }   // (NaN: 0)

// A tree as the threads of a workgroup see it.
struct VerifyTree {
  int parent[kVfMost];   // -1: not a node that can be reached
  int token[kVfMost];
};

template <int THREADS>
__device__ __forceinline__ void vf_read(const VerifyArgs& a, int b, VerifyTree& tree) {
  for (int i = threadIdx.x; i < a.s; i += THREADS) {
    const int up = a.parents ? a.parents[(int64_t)b * a.s + i] : i - 1, x = a.tokens[(int64_t)b * a.s + i];
    tree.parent[i] = i > 0 && up >= 0 && up < i ? up : -1;
    tree.token[i] = x >= 0 && x < a.vocab ? x : -1;
  }
  __syncthreads();
}

// Sum over the workgroup in an order that does not change; every thread gets it.
template <int THREADS>
__device__ __forceinline__ double vf_sum(double v, double* scratch) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
  __syncthreads();
  if (lane_id() == 0) scratch[wave_id()] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) all += scratch[w];
  return all;
}

// Z of the children of one node, one after the other: a workgroup has both rows for itself.
template <typename T>
__global__ __launch_bounds__(kVfWide) void verify_mass_kernel(VerifyArgs a) {
  __shared__ VerifyTree tree;
  __shared__ double scratch[kVfWide / kWave];
  const int n = blockIdx.x, b = blockIdx.y;
  vf_read<kVfWide>(a, b, tree);
  const T* q = (const T*)a.q + b * a.qb + n * a.qr;
  const T* p = (const T*)a.p + b * a.pb + n * a.pr;
  double cut = 0.0, mass = 1.0;
  bool first = true;
  for (int i = n + 1; i < a.s; ++i) {
    if (tree.parent[i] != n) continue;
    if (!first) {
      cut += mass;
      double sum = 0.0;
      for (int x = threadIdx.x; x < a.vocab; x += kVfWide) sum += vf_positive((double)ld_f32(q, x) - cut * vf_positive((double)ld_f32(p, x)));
      mass = vf_sum<kVfWide>(sum, scratch);
    }
    first = false;
    if (threadIdx.x == 0) {
      a.cut[(int64_t)b * a.s + i] = cut;
      a.mass[(int64_t)b * a.s + i] = mass;
    }
  }
}

// The walk from the root.  Every node is tested, as if its earlier siblings were refused; then the path is followed.
template <typename T>
__device__ __forceinline__ void vf_walk(const VerifyArgs& a, int b, VerifyTree& tree, double* own, int* chosen, int& end, double& cut, int& count) {
  vf_read<kVfThreads>(a, b, tree);
  const T* q = (const T*)a.q + b * a.qb;
  const T* p = (const T*)a.p + b * a.pb;
  for (int i = threadIdx.x; i < a.s; i += kVfThreads) {
    chosen[i] = INT32_MAX;
    const int up = tree.parent[i], x = tree.token[i];
    double mine = up >= 0 && x >= 0 ? vf_positive((double)ld_f32(q + up * a.qr, x)) : 0.0;
    // (without p: a token that an earlier sibling has is gone)
    if (!a.p && a.parents && up >= 0)
      for (int j = up + 1; j < i; ++j)
        if (tree.parent[j] == up && tree.token[j] == x) mine = 0.0;
    own[i] = mine;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.s; i += kVfThreads) {
    const int up = tree.parent[i], x = tree.token[i];
    if (up < 0 || x < 0) continue;
    const double u = (double)a.u[(int64_t)b * a.s + i];
    bool taken;
    if (a.p) {
      const double px = vf_positive((double)ld_f32(p + up * a.pr, x));
      const double c = a.parents ? a.cut[(int64_t)b * a.s + i] : 0.0, mass = a.parents ? a.mass[(int64_t)b * a.s + i] : 1.0;
      taken = u * px * mass < vf_positive(own[i] - c * px);
    } else {
      double mass = 1.0;
      if (a.parents)
        for (int j = up + 1; j < i; ++j)
          if (tree.parent[j] == up) mass -= own[j];
      taken = u * mass < own[i];
    }
    if (taken) atomicMin(&chosen[up], i);
  }
  __syncthreads();
  end = 0;
  count = 1;
  while (chosen[end] != INT32_MAX) {   // (a child stands behind its parent: at most s steps)
    end = chosen[end];
    ++count;
  }
  // what the last node's distribution has lost to its children, all of them refused
  cut = 0.0;
  if (a.p) {
    if (!a.parents)
      cut = end + 1 < a.s ? 1.0 : 0.0;
    else {
      int last = -1;
      for (int i = end + 1; i < a.s; ++i) last = tree.parent[i] == end ? i : last;
      if (last >= 0) cut = a.cut[(int64_t)b * a.s + last] + a.mass[(int64_t)b * a.s + last];
    }
  }
}

// The tokens that refused children of node `end` took with them (drafts without p): in any order, they are only looked for.
// Holds a barrier.
__device__ __forceinline__ void vf_refused(const VerifyArgs& a, const VerifyTree& tree, int end, int* gone, int& gone_n) {
  if (a.p) return;
  for (int i = threadIdx.x; i < a.s; i += kVfThreads)
    if (tree.parent[i] == end && tree.token[i] >= 0) gone[atomicAdd(&gone_n, 1)] = tree.token[i];
  __syncthreads();
}

// What is left of a row, element x.
template <typename T>
struct VerifyRow {
  const T *q, *p;
  double cut;
  const int* gone;
  int gone_n;
  __device__ __forceinline__ double at(int x) const {
    double y = (double)ld_f32(q, x);
    if (p) y -= cut * vf_positive((double)ld_f32(p, x));
    for (int i = 0; i < gone_n; ++i) y = gone[i] == x ? 0.0 : y;
    return vf_positive(y);
  }
};
// (the drafting model's row is not looked at where no child was refused: there may be none for the last node)
template <typename T>
__device__ __forceinline__ VerifyRow<T> vf_row(const VerifyArgs& a, int b, int end, double cut, const int* gone, int gone_n) {
  return {(const T*)a.q + b * a.qb + end * a.qr, a.p && cut != 0.0 ? (const T*)a.p + b * a.pb + end * a.pr : nullptr, cut, gone, gone_n};
}

template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_sums_kernel(VerifyArgs a) {
  __shared__ VerifyTree tree;
  __shared__ double own[kVfMost], scratch[kVfThreads / kWave];
  __shared__ int chosen[kVfMost], gone[kVfMost], gone_n;
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  if (tid == 0) gone_n = 0;
  int end, count;
  double cut;
  vf_walk<T>(a, b, tree, own, chosen, end, cut, count);
  if (chunk == 0) {
    for (int i = count + tid; i < a.s; i += kVfThreads) a.path[(int64_t)b * a.s + i] = -1;
    if (tid == 0) {
      a.counts[b] = count;
      a.end[b] = end;
      a.left[b] = cut;
      for (int i = 0, at = 0; i < count; ++i, at = chosen[at]) a.path[(int64_t)b * a.s + i] = at;
    }
  }
  vf_refused(a, tree, end, gone, gone_n);
  const VerifyRow<T> row = vf_row<T>(a, b, end, cut, gone, gone_n);
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < kVfEach; ++e) {
    const int64_t x = (int64_t)chunk * kVfChunk + e * kVfThreads + tid;
    if (x < a.vocab) sum += row.at((int)x);
  }
  sum = vf_sum<kVfThreads>(sum, scratch);
  if (tid == 0) a.sums[(int64_t)b * a.chunks + chunk] = sum;
}

// Sums over the threads in front of this one and up to it.
__device__ __forceinline__ double vf_scan(double v, double* scratch, double& before, double& all) {
  double x = v;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const double y = __shfl_up(x, off, kWave);
    x += lane_id() >= off ? y : 0.0;
  }
  const double y = __shfl_up(x, 1, kWave);
  __syncthreads();
  if (lane_id() == kWave - 1) scratch[wave_id()] = x;
  __syncthreads();
  double base = 0.0;
  all = 0.0;
#pragma unroll
  for (int w = 0; w < kVfThreads / kWave; ++w) {
    if (w < wave_id()) base += scratch[w];
    all += scratch[w];
  }
  before = base + (lane_id() > 0 ? y : 0.0);
  return base + x;
}

// The first of n numbers whose sum with those in front of it is above a border (the last that is not 0, where rounding hides it;
// -1 if all are), and the border less what stands in front of it.  SHARE: the border is `share` of the sum of all.
struct VerifyPlace {
  int64_t i;
  double rest;
};
template <bool SHARE, typename F>
__device__ __forceinline__ VerifyPlace vf_first(int64_t n, F number, double share, double* scratch, VerifyPlace& found, int* who) {
  const int64_t each = (n + kVfThreads - 1) / kVfThreads, lo = min(threadIdx.x * each, n), hi = min(lo + each, n);
  double mine = 0.0, before, all;
  for (int64_t i = lo; i < hi; ++i) mine += number(i);
  if (threadIdx.x == 0) {
    who[0] = INT32_MAX;
    who[1] = found.i = -1;
  }
  const double upto = vf_scan(mine, scratch, before, all), border = SHARE ? share * all : share;   // (holds barriers)
  if (mine > 0.0) {
    if (upto > border) atomicMin(&who[0], (int)threadIdx.x);
    atomicMax(&who[1], (int)threadIdx.x);
  }
  __syncthreads();
  if ((int)threadIdx.x == (who[0] != INT32_MAX ? who[0] : who[1])) {
    double sum = before;
    for (int64_t i = lo; i < hi; ++i) {
      const double x = number(i);
      if (!(x > 0.0)) continue;
      found = {i, border - sum};
      sum += x;
      if (sum > border) break;
    }
  }
  __syncthreads();
  return found;
}

template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_token_kernel(VerifyArgs a) {
  __shared__ VerifyTree tree;
  __shared__ double scratch[kVfThreads / kWave];
  __shared__ int gone[kVfMost], gone_n, who[2];
  __shared__ VerifyPlace found;
  const int b = blockIdx.x;
  if (threadIdx.x == 0) gone_n = 0;
  vf_read<kVfThreads>(a, b, tree);
  const int end = a.end[b];
  vf_refused(a, tree, end, gone, gone_n);
  const double* sums = a.sums + (int64_t)b * a.chunks;
  const double u = (double)a.u[(int64_t)b * a.s];
  const VerifyPlace chunk = vf_first<true>(a.chunks, [&](int64_t i) { return sums[i]; }, u, scratch, found, who);
  __syncthreads();
  int64_t token;
  if (chunk.i >= 0) {
    const VerifyRow<T> row = vf_row<T>(a, b, end, a.left[b], gone, gone_n);
    const int64_t x0 = chunk.i * kVfChunk;
    token = x0 + vf_first<false>(min((int64_t)kVfChunk, a.vocab - x0), [&](int64_t i) { return row.at((int)(x0 + i)); }, chunk.rest, scratch, found, who).i;
  } else {   // nothing is left: of the target's distribution as it is
    const VerifyRow<T> row = vf_row<T>(a, b, end, 0.0, gone, 0);
    token = vf_first<true>(a.vocab, [&](int64_t i) { return row.at((int)i); }, u, scratch, found, who).i;
  }
  if (threadIdx.x == 0) a.next[b] = (int)token;
}

static int verify_check(int b, int s, int64_t vocab) {
  LRQK_REQUIRE(b > 0 && s > 0 && vocab > 0, LRQK_EINVAL, "bad sizes b=%d s=%d vocab=%lld", b, s, (long long)vocab);
  LRQK_REQUIRE(s <= kVfMost && b <= 65535 && vocab <= (1 << 30), LRQK_ELIMIT, "s=%d (at most %d), b=%d (65535), vocab=%lld (2^30)", s,
               kVfMost, b, (long long)vocab);
  return LRQK_OK;
}
static int64_t verify_chunks(int64_t vocab) { return (vocab + kVfChunk - 1) / kVfChunk; }
// 64-bit words of the scratch
static int64_t verify_words(int b, int s, int64_t vocab) { return b * (2 * (int64_t)s + verify_chunks(vocab) + 2); }

template <typename T>
static int verify_launch(const VerifyArgs& a, hipStream_t st) {
  if (a.p && a.parents && a.s > 1) {
    hipLaunchKernelGGL(verify_mass_kernel<T>, dim3((unsigned)(a.s - 1), (unsigned)a.b), dim3(kVfWide), 0, st, a);
    LRQK_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(verify_sums_kernel<T>, dim3((unsigned)a.chunks, (unsigned)a.b), dim3(kVfThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(verify_token_kernel<T>, dim3((unsigned)a.b), dim3(kVfThreads), 0, st, a);
  LRQK_HIP_CHECK(hipGetLastError());
  return LRQK_OK;
}

}  // namespace lrqk

using namespace lrqk;

extern "C" int64_t lrqk_verify_drafts_workspace(int b, int s, int64_t vocab) {
  const int rc = verify_check(b, s, vocab);
  if (rc) return rc;
  return 8 * verify_words(b, s, vocab);
}

extern "C" int lrqk_verify_drafts(const int32_t* tokens, const int32_t* parents, const void* target, int64_t target_batch_stride,
                                  int64_t target_row_stride, const void* draft, int64_t draft_batch_stride, int64_t draft_row_stride,
                                  const float* uniforms, int32_t* path, int32_t* counts, int32_t* next, int b, int s, int64_t vocab,
                                  void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  const int rc = verify_check(b, s, vocab);
  if (rc) return rc;
  LRQK_REQUIRE(dtype == LRQK_F32 || dtype == LRQK_BF16, LRQK_EINVAL, "dtype=%d", dtype);
  LRQK_REQUIRE(tokens && target && uniforms && path && counts && next && workspace, LRQK_EINVAL, "null pointer");
  LRQK_REQUIRE((uintptr_t)workspace % 16 == 0, LRQK_EINVAL, "the workspace must be 16-byte aligned");
  LRQK_REQUIRE(workspace_bytes >= 8 * verify_words(b, s, vocab), LRQK_EINVAL, "workspace of %lld bytes: %lld are needed",
               (long long)workspace_bytes, (long long)(8 * verify_words(b, s, vocab)));
  double* ws = (double*)workspace;
  const int64_t nodes = (int64_t)b * s, chunks = verify_chunks(vocab);
  VerifyArgs a{tokens, parents, target, draft, target_batch_stride, target_row_stride, draft_batch_stride, draft_row_stride, uniforms, path,
               counts, next, ws, ws + nodes, ws + 2 * nodes, ws + 2 * nodes + b * chunks,
               (int32_t*)(ws + 2 * nodes + b * chunks + b), b, s, (int)vocab, (int)chunks};
  hipStream_t st = (hipStream_t)stream;
  return dtype == LRQK_F32 ? verify_launch<float>(a, st) : verify_launch<bf16_t>(a, st);
}
