// Drafted tokens verified against the target's probabilities (speculative sampling on a tree), from given random numbers.
//
// Node 0 of a sequence's tree is certain; node i > 0 was drawn from row parent[i] of the drafting model's probabilities p, and
// q[i] is the target's distribution behind node i.  A node's children x_1 .. x_k are looked at in order, with what is left of
// the distribution: r_0 = q, Z_0 = 1; x_j is accepted if u_j p(x_j) Z_(j-1) < r_(j-1)(x_j), and if it is not
//
//   r_j = max(r_(j-1) - Z_(j-1) p, 0) = max(q - C_j p, 0),  C_j = C_(j-1) + Z_(j-1), C_0 = 0,  Z_j = sum of r_j,
//
// so that one pass over two rows gives Z_j, and only nodes with several children need one.  Drafts without probabilities have
// p = 1 at their token: r_j is r_(j-1) without it, and Z_j = Z_(j-1) - r_(j-1)(x_j), 1 less what the refused ones had, whatever
// the row adds up to (its sum would be a pass; a row of bf16 probabilities is off by up to 2^-8).  Behind the last accepted node
// the next token is drawn from what is left: the lowest x with r(0) + .. + r(x) > u_0 sum(r).  Everything is formed in 64 bits,
// since a vocabulary's sums in 32 would put the border between two tokens elsewhere; what is not a positive number counts as 0.
//
// Three launches: Z of the nodes with several children (trees with p only); the walk, by every workgroup for itself, and the
// sums of what is left by chunks of the vocabulary; the chunk and the token.
// Bound by launches and their chains of reads: over one fp32 row of 128256 tokens the sums take 3.4 us and the token 4.8 (7.9
// together, as replayed), over 16 trees of 16 nodes without p 7 and 6; an eager call costs the host 14 .. 17.  (One launch
// for both would have its workgroups wait for each other.)
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
  struct VerifyEnd* ends;            // [b]
  int32_t* gone;                     // [b][s]: tokens of the last accepted node's refused children (drafts without p)
  int b, s, vocab, chunks;
};

struct VerifyEnd {   // where a sequence's walk ended
  double cut;        // C there
  int node, gone;    // the last accepted node; how many tokens are gone
};

__device__ __forceinline__ double vf_positive(double x) { return fmax(x, 0.0); }         // (NaN: 0)
__device__ __forceinline__ double vf_probability(float x) { return fmax((double)x, 0.0); }   // (a maximum in fp32 is two instructions)

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

// u p Z < r, with r = max(q - C p, 0).
__device__ __forceinline__ bool vf_accepts(double u, double px, double mass, double qx, double cut) {
  return u * px * mass < vf_positive(fma(-cut, px, qx));
}

// add(q, p) of two rows of n pieces of N elements, by a workgroup, EACH pieces of a thread at a time.  (The end is one such step
// too, with those behind it left out: one after the other they wait for memory as often.)
template <typename T, int N, int EACH, bool END, typename F>
__device__ __forceinline__ void vf_step(const T* q, const T* p, int64_t at, int64_t n, F add) {
  float qs[EACH][N], ps[EACH][N];
  [[maybe_unused]] Vec16<T> qv[EACH], pv[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (END && at - (int)threadIdx.x + e * kVfWide >= n) break;
    const int64_t x = (END ? min(at + e * kVfWide, n - 1) : at + e * kVfWide) * N;
    if constexpr (N == 1) {
      qs[e][0] = ld_f32(q, x);
      ps[e][0] = ld_f32(p, x);
    } else {
      qv[e].load(q + x);
      pv[e].load(p + x);
    }
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (END && at - (int)threadIdx.x + e * kVfWide >= n) break;
    if constexpr (N > 1) {
      qv[e].unpack(qs[e]);
      pv[e].unpack(ps[e]);
    }
    if (END && at + e * kVfWide >= n) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) add(qs[e][i], ps[e][i]);
  }
}
template <typename T, int N, int EACH, typename F>
__device__ __forceinline__ void vf_pass(const T* q, const T* p, int64_t n, F add) {
  int64_t done = 0;
  for (; done + EACH * kVfWide <= n; done += EACH * kVfWide) vf_step<T, N, EACH, false>(q, p, done + threadIdx.x, n, add);
  if (done < n) vf_step<T, N, EACH, true>(q, p, done + threadIdx.x, n, add);
}

// Z of the children of one node, one after the other up to the one that is accepted: a workgroup has both rows for itself.  Bound
// by one CU's arithmetic, 9 us a pass over 128256 tokens, six instructions an element in 64 bits: rows of half the bytes take as
// long, and rows kept in registers and LDS from pass to pass.  (Several CUs would have to wait for each other, or for a launch a
// child; that of the second child alone, at C = 1, is known beforehand.)
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
  for (int base = n + 1; base < a.s; base += kWave) {
    const int mine = base + lane_id();
    unsigned long long children = __ballot(mine < a.s && tree.parent[min(mine, a.s - 1)] == n);
    for (; children; children &= children - 1) {
      const int i = base + __ffsll(children) - 1, x = tree.token[i];
      const int64_t at = (int64_t)b * a.s + i;
      // (asked for before the pass, which they do not wait for)
      const float u = a.u[at], qx = ld_f32(q, max(x, 0)), px = ld_f32(p, max(x, 0));
      if (!first) {
        cut += mass;
        double sum = 0.0;
        auto add = [&](float qy, float py) { sum += vf_positive(fma(-cut, vf_probability(py), (double)qy)); };
        constexpr int N = Vec16<T>::N;
        const int64_t whole = ((uintptr_t)q | (uintptr_t)p) % 16 == 0 ? a.vocab / N : 0;
        vf_pass<T, N, 4>(q, p, whole, add);
        vf_pass<T, 1, 8>(q + whole * N, p + whole * N, a.vocab - whole * N, add);
        mass = vf_sum<kVfWide>(sum, scratch);
      }
      first = false;
      if (threadIdx.x == 0) {
        a.cut[at] = cut;
        a.mass[at] = mass;
      }
      // (behind an accepted child nobody asks: of a node's accepted children the first counts)
      if (x >= 0 && vf_accepts((double)u, vf_probability(px), mass, vf_probability(qx), cut)) return;
    }
  }
}

// The walk from the root.  Every node is tested, as if its earlier siblings were refused; then the path is followed.
template <typename T>
__device__ __forceinline__ void vf_walk(const VerifyArgs& a, int b, VerifyTree& tree, double* own, int* chosen, int& end, double& cut, int& count) {
  end = 0;
  count = 1;
  cut = 0.0;
  if (a.s == 1) return;
  for (int i = threadIdx.x; i < a.s; i += kVfThreads) chosen[i] = INT32_MAX;
  vf_read<kVfThreads>(a, b, tree);   // (holds a barrier)
  const T* q = (const T*)a.q + b * a.qb;
  const T* p = (const T*)a.p + b * a.pb;
  if (a.p) {
    for (int i = threadIdx.x; i < a.s; i += kVfThreads) {
      const int up = tree.parent[i], x = tree.token[i];
      if (up < 0 || x < 0) continue;
      const int64_t at = (int64_t)b * a.s + i;
      const double c = a.parents ? a.cut[at] : 0.0, mass = a.parents ? a.mass[at] : 1.0;
      if (vf_accepts((double)a.u[at], vf_probability(ld_f32(p + up * a.pr, x)), mass, vf_probability(ld_f32(q + up * a.qr, x)), c))
        atomicMin(&chosen[up], i);
    }
  } else {
    for (int i = threadIdx.x; i < a.s; i += kVfThreads) {
      const int up = tree.parent[i], x = tree.token[i];
      const double mine = up >= 0 && x >= 0 ? vf_probability(ld_f32(q + up * a.qr, x)) : 0.0;
      // (a token that an earlier sibling has is gone)
      // (without branches, as below: then the reads of many j are under way at once)
      bool gone = false;
      if (a.parents && up >= 0)
#pragma unroll 8
        for (int j = up + 1; j < i; ++j) gone = gone | ((tree.parent[j] == up) & (tree.token[j] == x));
      own[i] = gone ? 0.0 : mine;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.s; i += kVfThreads) {
      const int up = tree.parent[i];
      if (up < 0 || tree.token[i] < 0) continue;
      double mass = 1.0;
      if (a.parents)
#pragma unroll 8
        for (int j = up + 1; j < i; ++j) {
          const double theirs = own[j];
          mass -= tree.parent[j] == up ? theirs : 0.0;
        }
      if ((double)a.u[(int64_t)b * a.s + i] * mass < own[i]) atomicMin(&chosen[up], i);
    }
  }
  __syncthreads();
  while (chosen[end] != INT32_MAX) {   // (a child stands behind its parent: at most s steps)
    end = chosen[end];
    ++count;
  }
  // what the last node's distribution has lost to its children, all of them refused
  if (a.p) {
    if (!a.parents) {
      cut = end + 1 < a.s ? 1.0 : 0.0;
    } else {
      int last = -1;
      for (int base = end + 1; base < a.s; base += kWave) {
        const int i = base + lane_id();
        const unsigned long long children = __ballot(i < a.s && tree.parent[min(i, a.s - 1)] == end);
        if (children) last = base + 63 - __clzll(children);
      }
      if (last >= 0) cut = a.cut[(int64_t)b * a.s + last] + a.mass[(int64_t)b * a.s + last];
    }
  }
}

// Which elements of a chunk are gone, a bit each.  (Every element held against every token that is gone: 4 sequences of 64
// looked-up siblings took 31 us instead of 16.)
struct VerifyGone {
  uint32_t bits[kVfChunk / 32];
  __device__ __forceinline__ void fill(const int* gone, int n, int64_t first) {   // by the workgroup; holds barriers
    for (int i = threadIdx.x; i < kVfChunk / 32; i += kVfThreads) bits[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kVfThreads) {
      const int64_t x = gone[i] - first;
      if (x >= 0 && x < kVfChunk) atomicOr(&bits[x / 32], 1u << (x % 32));
    }
    __syncthreads();
  }
  __device__ __forceinline__ bool has(int64_t x) const { return bits[x % kVfChunk / 32] >> (x % 32) & 1u; }
};

// What is left of a row, element x.
template <typename T>
struct VerifyRow {
  const T *q, *p;     // p: or null
  double cut;
  // (the drafting model's row is not looked at where no child was refused: there may be none for the last node)
  __device__ __forceinline__ VerifyRow(const VerifyArgs& a, int b, int node, double cut)
      : q((const T*)a.q + b * a.qb + node * a.qr), p(a.p && cut != 0.0 ? (const T*)a.p + b * a.pb + node * a.pr : nullptr), cut(cut) {}
  // N elements from x on, `step` apart, without those that are gone (or null); 0 behind the end
  template <int N>
  __device__ __forceinline__ void load(int64_t x, int step, int64_t end, const VerifyGone* gone, double (&r)[N]) const {
    float qs[N], ps[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t at = x + e * step < end ? x + e * step : end - 1;
      qs[e] = ld_f32(q, at);
      ps[e] = p ? ld_f32(p, at) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      r[e] = vf_positive(fma(-cut, vf_probability(ps[e]), (double)qs[e]));
      if (gone) r[e] = gone->has(x + e * step) ? 0.0 : r[e];
      r[e] = x + e * step < end ? r[e] : 0.0;
    }
  }
};

template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_sums_kernel(VerifyArgs a) {
  __shared__ VerifyTree tree;
  __shared__ VerifyGone out;
  __shared__ double own[kVfMost], scratch[kVfThreads / kWave];
  __shared__ int chosen[kVfMost], gone[kVfMost], gone_n;
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  if (tid == 0) gone_n = 0;
  int end, count;
  double cut;
  vf_walk<T>(a, b, tree, own, chosen, end, cut, count);
  if (!a.p) {   // (in any order: they are only looked for)
    for (int i = end + 1 + tid; i < a.s; i += kVfThreads)
      if (tree.parent[i] == end && tree.token[i] >= 0) gone[atomicAdd(&gone_n, 1)] = tree.token[i];
    __syncthreads();
  }
  const int lost = a.p ? 0 : gone_n;
  if (chunk == 0) {
    for (int i = count + tid; i < a.s; i += kVfThreads) a.path[(int64_t)b * a.s + i] = -1;
    for (int i = tid; i < lost; i += kVfThreads) a.gone[(int64_t)b * a.s + i] = gone[i];
    if (tid == 0) {
      a.counts[b] = count;
      a.ends[b] = {cut, end, lost};
      a.path[(int64_t)b * a.s] = 0;
      for (int i = 1, at = 0; i < count; ++i) a.path[(int64_t)b * a.s + i] = at = chosen[at];
    }
  }
  if (lost) out.fill(gone, lost, (int64_t)chunk * kVfChunk);
  const VerifyRow<T> row(a, b, end, cut);
  double r[kVfEach], sum = 0.0;
  row.load((int64_t)chunk * kVfChunk + tid, kVfThreads, a.vocab, lost ? &out : nullptr, r);
#pragma unroll
  for (int e = 0; e < kVfEach; ++e) sum += r[e];
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

// The first of the workgroup's numbers, kVfEach successive ones a thread, whose sum with those in front of it is above a border
// (the last that is not 0, where rounding hides it; -1 if all are), and the border less what stands in front of it.  SHARE: the
// border is `share` of the sum of all.
struct VerifyPlace {
  int64_t i;
  double rest;
};
struct VerifyFind {
  double scratch[kVfThreads / kWave];
  int first, last;
  VerifyPlace found;
};
template <bool SHARE>
__device__ __forceinline__ VerifyPlace vf_first(const double (&r)[kVfEach], double share, VerifyFind& f) {
  double mine = 0.0, before, all;
#pragma unroll
  for (int e = 0; e < kVfEach; ++e) mine += r[e];
  if (threadIdx.x == 0) {
    f.first = INT32_MAX;
    f.last = -1;
    f.found.i = -1;
  }
  const double upto = vf_scan(mine, f.scratch, before, all), border = SHARE ? share * all : share;   // (holds barriers)
  // the first such thread of each wave and the last one with anything, then of all
  const unsigned long long over = __ballot(mine > 0.0 && upto > border), some = __ballot(mine > 0.0);
  if (lane_id() == 0) {
    if (over) atomicMin(&f.first, (int)threadIdx.x + __ffsll(over) - 1);
    if (some) atomicMax(&f.last, (int)threadIdx.x + 63 - __clzll(some));
  }
  __syncthreads();
  if ((int)threadIdx.x == (f.first != INT32_MAX ? f.first : f.last)) {
    double sum = before;
    bool done = false;
#pragma unroll
    for (int e = 0; e < kVfEach; ++e) {
      if (!done && r[e] > 0.0) f.found = {(int64_t)threadIdx.x * kVfEach + e, border - sum};
      sum += r[e];
      done = done || (r[e] > 0.0 && sum > border);
    }
  }
  __syncthreads();
  return f.found;
}

// The sums of runs of equal length, as many as vf_first looks through at once, that n numbers are made of.
template <typename F>
__device__ __forceinline__ void vf_runs(int64_t n, int64_t run, F number, double (&r)[kVfEach]) {
#pragma unroll
  for (int e = 0; e < kVfEach; ++e) {
    const int64_t lo = min(((int64_t)threadIdx.x * kVfEach + e) * run, n), hi = min(lo + run, n);
    double sum = 0.0;
    for (int64_t i = lo; i < hi; ++i) sum += number(i);
    r[e] = sum;
  }
}

template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_token_kernel(VerifyArgs a) {
  __shared__ VerifyFind find;
  __shared__ VerifyGone out;
  const int b = blockIdx.x, tid = threadIdx.x;
  const VerifyEnd end = a.ends[b];
  const double* sums = a.sums + (int64_t)b * a.chunks;
  const double u = (double)a.u[(int64_t)b * a.s];
  double r[kVfEach];
  const int64_t run = (a.chunks + kVfChunk - 1) / kVfChunk;   // (1 up to 4 million tokens)
  if (run == 1) {
#pragma unroll
    for (int e = 0; e < kVfEach; ++e) r[e] = tid * kVfEach + e < a.chunks ? sums[min(tid * kVfEach + e, a.chunks - 1)] : 0.0;
  } else {
    vf_runs(a.chunks, run, [&](int64_t i) { return sums[i]; }, r);
  }
  VerifyPlace at = vf_first<true>(r, u, find);
  const bool nothing = at.i < 0;   // of the target's distribution as it is, then
  const VerifyRow<T> row(a, b, end.node, nothing ? 0.0 : end.cut);
  int64_t token = -1;
  if (!nothing) {
    if (run > 1) {
      // (the last chunk with anything, where rounding hides the border: there may be zeros behind it)
      double border = at.rest;
      const int64_t stop = min((at.i + 1) * run, (int64_t)a.chunks);
      for (int64_t i = at.i * run; i < stop; ++i) {
        const double x = sums[i];
        if (x > 0.0) at = {i, border};
        if (x > 0.0 && x > border) break;
        border -= x;
      }
    }
    const int64_t x0 = at.i * kVfChunk;
    if (end.gone) out.fill(a.gone + (int64_t)b * a.s, end.gone, x0);
    row.load(x0 + (int64_t)tid * kVfEach, 1, a.vocab, end.gone ? &out : nullptr, r);
    __syncthreads();
    const VerifyPlace place = vf_first<false>(r, at.rest, find);
    token = place.i < 0 ? -1 : x0 + place.i;
  } else {
    const int64_t part = (a.vocab + kVfChunk - 1) / kVfChunk;
    auto number = [&](int64_t i) {
      double one[1];
      row.load(i, 1, a.vocab, nullptr, one);
      return one[0];
    };
    vf_runs(a.vocab, part, number, r);
    __syncthreads();
    const VerifyPlace place = vf_first<true>(r, u, find);
    if (place.i >= 0) {
      double border = place.rest;
      const int64_t stop = min((place.i + 1) * part, (int64_t)a.vocab);
      for (int64_t i = place.i * part; i < stop; ++i) {
        const double x = number(i);
        if (x > 0.0) token = i;
        if (x > 0.0 && x > border) break;
        border -= x;
      }
    }
  }
  if (tid == 0) a.next[b] = (int)token;
}

static int verify_check(int b, int s, int64_t vocab) {
  LRQK_REQUIRE(b > 0 && s > 0 && vocab > 0, LRQK_EINVAL, "bad sizes b=%d s=%d vocab=%lld", b, s, (long long)vocab);
  LRQK_REQUIRE(s <= kVfMost && b <= 65535 && vocab <= (1 << 30), LRQK_ELIMIT, "s=%d (at most %d), b=%d (65535), vocab=%lld (2^30)", s,
               kVfMost, b, (long long)vocab);
  return LRQK_OK;
}
static int64_t verify_chunks(int64_t vocab) { return (vocab + kVfChunk - 1) / kVfChunk; }
// 64-bit words of the scratch
static int64_t verify_words(int b, int s, int64_t vocab) { return b * (2 * (int64_t)s + verify_chunks(vocab) + 2) + ((int64_t)b * s + 1) / 2; }

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
  double* ends = ws + 2 * nodes + b * chunks;
  VerifyArgs a{tokens, parents, target, draft, target_batch_stride, target_row_stride, draft_batch_stride, draft_row_stride, uniforms, path,
               counts, next, ws, ws + nodes, ws + 2 * nodes, (VerifyEnd*)ends, (int32_t*)(ends + 2 * (int64_t)b), b, s, (int)vocab,
               (int)chunks};
  hipStream_t st = (hipStream_t)stream;
  return dtype == LRQK_F32 ? verify_launch<float>(a, st) : verify_launch<bf16_t>(a, st);
}
