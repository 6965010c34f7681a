// Verification of drafted tokens by rejection sampling (the reference accepts by p(token) >= threshold in a host loop
// over sequences, demo/src/execution/cb_executor.py:261-300; this is the rule that keeps the target's distribution):
//   token x of position j is taken while p_j(x) > u_j * q_j(x);
//   at the first refusal one token is drawn from max(p_j - q_j, 0), after n accepted tokens one from p_n.
// A draw with the given number u takes the first i with r_0 + ... + r_i > u * (r_0 + ... + r_{V-1}).
//
// Neighbouring tokens of a large vocabulary are closer in the running sum than fp32 resolves, so differences and
// sums are taken in 64 bits.  What bounds it is HBM for large batches (one or two rows of the vocabulary per sequence)
// and, for small ones, a chain of dependent loads: start -> token -> probability -> row -> the place in the row.
// A cluster of CTAs shares a sequence: each warp sums one contiguous piece of the row, all sums meet in every CTA's
// shared memory over the cluster, and the CTA whose piece holds the draw reads it again (from L2), all its warps side by
// side, to find the token.  One launch, no workspace, no atomics in global memory.
//
// Measured on B200, device time back to back: one sequence of 4 drafts over 32000 tokens 5.2 us; 48 sequences over 151936
// 16 us with new inputs every call (12.2 us from L2); 64 greedy ones over 128256, bf16, 8.8 us.  The same 64 over 1024
// tokens take 5.9 us: that is the chain alone, which leaves 3 us for the rows.  Most of a warp's stalls are loads (half to
// three fifths) and the barriers between the passes; the 64-bit pipe is 9 % busy.  Rows whose length, stride or base is no
// multiple of 16 bytes are read element by element: 48 x 50257 9.2 us against 7.6 for 50256, 48 x 32001 bf16 8.6 against 7.2.
#pragma once
#include <cooperative_groups.h>

#include "common.cuh"

namespace b200moe {

struct VerifyParams {
  const long long* tokens;         // [drafts]
  const void* target;              // [target_rows, V]
  const void* draft;               // [drafts, V] or null: each draft has all its probability on its token
  const float *accept, *sample;    // [drafts], [B]
  const int* start;                // [B+1]
  long long* out;                  // [B, max_draft + 1]
  int* count;                      // [B]
  int* status;                     // may be null
  long long target_stride, draft_stride;
  int B, V, max_draft, num_draft, target_rows;
};

constexpr int kVerifyMaxCluster = 8;
constexpr int kVerifyThreads = 256;
constexpr int kVerifyCtasPerSm = 4;                                    // what 64 registers a thread allow
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyPieces = kVerifyMaxCluster * kVerifyWarps;        // at most; 64

__device__ __forceinline__ double warp_scan_incl(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// E consecutive elements; VEC: one 16-byte load, else what lies before `end`
template <typename T, int E, bool VEC> __device__ __forceinline__ void load_probs(const T* p, int i, int end, float (&f)[E]) {
  if constexpr (VEC) {
    static_assert(E * sizeof(T) == 16, "one vector");
    const uint4 raw = ldg_cached(p + i);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = Elem<T>::to_float(e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = i + k < end ? Elem<T>::to_float(p[i + k]) : 0.0f;
  }
}

// r_i of the draw: what is left of p after the draft's share q (LESS), never negative; `skip` is a token that has none.
// Which elements count is decided in fp32, where the comparison is exact and a NaN counts as nothing; the rest is in
// 64 bits.
template <typename T, int E, bool VEC, bool LESS>
__device__ __forceinline__ void load_rest(const T* p, const T* q, int skip, int i, int end, double (&r)[E]) {
  float f[E];
  load_probs<T, E, VEC>(p, i, end, f);
  if constexpr (LESS) {
    float s[E];
    load_probs<T, E, VEC>(q, i, end, s);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const bool left = f[k] > s[k];
      r[k] = (double)(left ? f[k] : 0.0f) - (double)(left ? s[k] : 0.0f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) r[k] = (double)fmaxf(f[k], 0.0f);
    if ((unsigned)(skip - i) < (unsigned)E) {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (i + k == skip) r[k] = 0.0;
    }
  }
}

// The sum of r over [lo, hi), by a whole warp.
template <typename T, bool VEC, bool LESS> __device__ __forceinline__ double rest_sum(const T* p, const T* q, int skip, int lo, int hi) {
  constexpr int E = 16 / (int)sizeof(T);
  double sum = 0.0;
  // two steps at once: four are slower by 2 us a call (more code to fetch than latency to hide), one by 4
#pragma unroll 2
  for (int i = lo + (threadIdx.x & 31) * E; i < hi; i += 32 * E) {
    double r[E];
    load_rest<T, E, VEC, LESS>(p, q, skip, i, hi, r);
    double part = 0.0;
#pragma unroll
    for (int k = 0; k < E; ++k) part += r[k];
    sum += part;
  }
  return warp_sum(sum);
}

// The first of up to 2 x 32 sums (two per lane, in index order) with which the running sum passes `goal`, and the sum
// before it; without one, the last that is positive.  By a whole warp; -1 when none is positive.
struct Found { int at; bool passed; double before, total; };
__device__ __forceinline__ Found find_sum(double s0, double s1, double base, double u, bool relative, double goal) {
  const int lane = threadIdx.x & 31;
  const double own = s0 + s1, incl = warp_scan_incl(own);
  Found f;
  f.total = __shfl_sync(0xffffffffu, incl, 31);
  if (relative) goal = u * f.total;
  const double run = base + (incl - own);
  const bool h0 = s0 > 0.0 && run + s0 > goal, h1 = s1 > 0.0 && run + s0 + s1 > goal;
  const unsigned has = __ballot_sync(0xffffffffu, h0 || h1);
  f.passed = has != 0;
  if (has) {
    const int src = __ffs(has) - 1;
    f.at = __shfl_sync(0xffffffffu, h0 ? 2 * lane : 2 * lane + 1, src);
    f.before = __shfl_sync(0xffffffffu, h0 ? run : run + s0, src);
  } else {
    f.at = __reduce_max_sync(0xffffffffu, s1 > 0.0 ? 2 * lane + 1 : (s0 > 0.0 ? 2 * lane : -1));
    f.before = 0.0;
  }
  return f;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads, kVerifyCtasPerSm) verify_draft_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int UNIT = 32 * E;                                        // a warp's elements per step
  __shared__ double s_sum[2][kVerifyPieces];
  __shared__ double s_part[kVerifyWarps];
  __shared__ int s_first;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.x / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();

  // --- how many tokens are taken (every CTA for itself: a handful of loads)
  const int base = p.start[b], n = p.start[b + 1] - base;
  const float u = p.sample[b];
  const int width = p.max_draft + 1;
  long long* out = p.out + (long long)b * width;
  const bool bad = base < 0 || n < 0 || n > p.max_draft || base > p.num_draft - n || (long long)base + b + n >= p.target_rows;
  if (bad) {                                                          // the same for the whole cluster
    if (rank == 0) {
      for (int j = threadIdx.x; j < width; j += kVerifyThreads) out[j] = -1;
      if (threadIdx.x == 0) {
        p.count[b] = 0;
        if (p.status) atomicOr(p.status, kDevBadLength);
      }
    }
    return;
  }
  cluster.barrier_arrive();                                           // waited for before the other CTAs' memory is written
  const T* target = reinterpret_cast<const T*>(p.target) + ((long long)base + b) * p.target_stride;
  const T* draft = reinterpret_cast<const T*>(p.draft);
  if (threadIdx.x == 0) s_first = n;
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += kVerifyThreads) {
    const long long x = p.tokens[base + j];
    const float uj = p.accept[base + j];
    bool take = false;
    if (x >= 0 && x < p.V) {
      const double pj = (double)Elem<T>::to_float(target[j * p.target_stride + x]);
      const double qj = draft ? (double)Elem<T>::to_float(draft[((long long)base + j) * p.draft_stride + x]) : 1.0;
      take = pj > (double)uj * qj;                                    // exact in 64 bits; a NaN refuses
    } else if (p.status && rank == 0) {
      atomicOr(p.status, kDevBadToken);
    }
    if (!take) atomicMin(&s_first, j);
  }
  __syncthreads();
  const int taken = s_first;
  if (rank == 0) {
    for (int j = threadIdx.x; j < width; j += kVerifyThreads)
      if (j != taken) out[j] = j < taken ? p.tokens[base + j] : -1;
    if (threadIdx.x == 0) p.count[b] = taken;
  }

  // --- the draw
  const T* row = target + taken * p.target_stride;
  const T* less = taken < n && draft ? draft + ((long long)base + taken) * p.draft_stride : nullptr;
  long long gone = -1;
  if (taken < n && !draft) gone = p.tokens[base + taken];
  int skip = gone >= 0 && gone < p.V ? (int)gone : -1;
  const int pieces = C * kVerifyWarps, piece = rank * kVerifyWarps + warp;
  const int per = ((p.V + pieces - 1) / pieces + E - 1) / E * E;
  const int lo = (int)min((long long)piece * per, (long long)p.V), hi = min(lo + per, p.V);

  for (int round = 0; round < 2; ++round) {
    double sum = less ? rest_sum<T, VEC, true>(row, less, skip, lo, hi) : rest_sum<T, VEC, false>(row, less, skip, lo, hi);
    if (round == 0) cluster.barrier_wait();
    if (lane < C) *cluster.map_shared_rank(&s_sum[round][piece], lane) = sum;
    cluster.sync();
    // every warp finds the piece that holds the draw, or the last with anything in it
    const bool l0 = 2 * lane < pieces, l1 = 2 * lane + 1 < pieces;
    const Found f = find_sum(l0 ? s_sum[round][2 * lane] : 0.0, l1 ? s_sum[round][2 * lane + 1] : 0.0, 0.0, (double)u, true, 0.0);
    if (!(f.total > 0.0)) {                                           // the same in every CTA
      if (round == 0 && (less || skip >= 0)) { less = nullptr; skip = -1; continue; }   // nothing is left of p - q: draw from p
      if (rank == 0 && threadIdx.x == 0) {
        out[taken] = -1;
        if (p.status) atomicOr(p.status, kDevBadProbs);
      }
      return;
    }
    if (f.at / kVerifyWarps != rank) return;
    // this CTA owns it: each warp takes a share of the piece
    const double goal = (double)u * f.total;
    const int plo = (int)min((long long)f.at * per, (long long)p.V), phi = min(plo + per, p.V);
    const int share = ((phi - plo + kVerifyWarps - 1) / kVerifyWarps + E - 1) / E * E;
    const int slo = min(plo + warp * share, phi), shi = min(slo + share, phi);
    sum = less ? rest_sum<T, VEC, true>(row, less, skip, slo, shi) : rest_sum<T, VEC, false>(row, less, skip, slo, shi);
    if (lane == 0) s_part[warp] = sum;
    __syncthreads();
    const Found w = find_sum(lane < kVerifyWarps / 2 ? s_part[2 * lane] : 0.0, lane < kVerifyWarps / 2 ? s_part[2 * lane + 1] : 0.0, f.before, 0.0, false,
                             f.passed ? goal : (double)INFINITY);
    if (w.at != warp) return;
    double before = w.before;
    const bool want = f.passed && w.passed;                           // else the last token with any weight
    int found = -1, last_pos = -1;
    for (int i0 = slo; i0 < shi && found < 0; i0 += UNIT) {
      const int i = i0 + lane * E;
      double r[E], s = 0.0;
#pragma unroll
      for (int k = 0; k < E; ++k) r[k] = 0.0;
      if (i < shi) {
        if (less) load_rest<T, E, VEC, true>(row, less, skip, i, shi, r);
        else load_rest<T, E, VEC, false>(row, less, skip, i, shi, r);
      }
#pragma unroll
      for (int k = 0; k < E; ++k) s += r[k];
      const double inc = warp_scan_incl(s);
      double at = before + (inc - s);
      int here = -1, pos = -1;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        if (r[k] > 0.0) {
          at += r[k];
          pos = i + k;
          if (want && here < 0 && at > goal) here = i + k;
        }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, here >= 0);
      if (hit) found = __shfl_sync(0xffffffffu, here, __ffs(hit) - 1);
      last_pos = max(last_pos, (int)__reduce_max_sync(0xffffffffu, pos));
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) out[taken] = found >= 0 ? found : last_pos;
    return;
  }
}

}  // namespace b200moe
