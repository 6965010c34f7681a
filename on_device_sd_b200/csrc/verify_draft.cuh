// Verification of drafted tokens by rejection sampling (the reference accepts by p(token) >= threshold in a host loop
// over sequences, demo/src/execution/cb_executor.py:261-300; this is the rule that keeps the target's distribution):
//   token x of position j is taken while p_j(x) > u_j * q_j(x);
//   at the first refusal one token is drawn from max(p_j - q_j, 0), after n accepted tokens one from p_n.
// A draw with the given number u takes the first i with r_0 + ... + r_i > u * (r_0 + ... + r_{V-1}).
//
// Neighbouring tokens of a large vocabulary are closer in the running sum than fp32 resolves, so differences and
// sums are taken in 64 bits.  What bounds it is HBM (one or two rows of the vocabulary per sequence) and, for one
// sequence, the chain of dependent loads start -> token -> probability.  A cluster of eight CTAs shares a row: each
// warp sums one contiguous piece, all sums meet in every CTA's shared memory over the cluster, and the warp whose piece
// holds the draw reads it again (from L2) to find the token.  One launch, no workspace, no atomics.
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

constexpr int kVerifyCluster = 8;
constexpr int kVerifyThreads = 512;
constexpr int kVerifyPieces = kVerifyCluster * (kVerifyThreads / 32);

__device__ __forceinline__ double warp_scan_incl(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// E consecutive elements as doubles; VEC: one 16-byte load
template <typename T, int E, bool VEC> __device__ __forceinline__ void load_probs(const T* p, int i, int end, double (&f)[E]) {
  if constexpr (VEC) {
    static_assert(E * sizeof(T) == 16, "one vector");
    const uint4 raw = ldg_cached(p + i);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = (double)Elem<T>::to_float(e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = i + k < end ? (double)Elem<T>::to_float(p[i + k]) : 0.0;
  }
}

// r_i of the draw: what is left of p after the draft's share; `skip` is a token that has none
template <typename T, int E, bool VEC>
__device__ __forceinline__ void load_rest(const T* p, const T* q, int skip, int i, int end, double (&r)[E]) {
  load_probs<T, E, VEC>(p, i, end, r);
  if (q) {
    double s[E];
    load_probs<T, E, VEC>(q, i, end, s);
#pragma unroll
    for (int k = 0; k < E; ++k) r[k] -= s[k];
  }
#pragma unroll
  for (int k = 0; k < E; ++k) r[k] = r[k] > 0.0 && i + k != skip ? r[k] : 0.0;   // a NaN counts as nothing
}

template <typename T, bool VEC>
__global__ void __cluster_dims__(kVerifyCluster, 1, 1) __launch_bounds__(kVerifyThreads) verify_draft_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int WARPS = kVerifyThreads / 32;
  __shared__ double s_sum[2][kVerifyPieces];
  __shared__ int s_first;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / kVerifyCluster;
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
    bool take = false;
    if (x >= 0 && x < p.V) {
      const double pj = (double)Elem<T>::to_float(target[j * p.target_stride + x]);
      const double qj = draft ? (double)Elem<T>::to_float(draft[((long long)base + j) * p.draft_stride + x]) : 1.0;
      take = pj > (double)p.accept[base + j] * qj;                    // exact in 64 bits; a NaN refuses
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
  const int piece = rank * WARPS + warp;
  const int unit = 32 * E;                                            // a warp's elements per step
  const int per = ((p.V + kVerifyPieces - 1) / kVerifyPieces + E - 1) / E * E;
  const int lo = (int)min((long long)piece * per, (long long)p.V), hi = min(lo + per, p.V);

  for (int round = 0; round < 2; ++round) {
    double sum = 0.0;
#pragma unroll 2
    for (int i = lo + lane * E; i < hi; i += unit) {
      double r[E];
      load_rest<T, E, VEC>(row, less, skip, i, hi, r);
#pragma unroll
      for (int k = 0; k < E; ++k) sum += r[k];
    }
    sum = warp_sum(sum);
    if (round == 0) cluster.barrier_wait();
    if (lane < kVerifyCluster) *cluster.map_shared_rank(&s_sum[round][piece], lane) = sum;
    cluster.sync();
    // piece sums in index order: lane holds pieces 4*lane .. +3
    constexpr int PL = kVerifyPieces / 32;
    double mine[PL], own = 0.0;
#pragma unroll
    for (int k = 0; k < PL; ++k) { mine[k] = s_sum[round][lane * PL + k]; own += mine[k]; }
    const double incl = warp_scan_incl(own);
    const double total = __shfl_sync(0xffffffffu, incl, 31);
    if (!(total > 0.0)) {                                             // the same in every CTA
      if (round == 0 && (less || skip >= 0)) { less = nullptr; skip = -1; continue; }   // nothing is left of p - q: draw from p
      if (rank == 0 && threadIdx.x == 0) {
        out[taken] = -1;
        if (p.status) atomicOr(p.status, kDevBadProbs);
      }
      return;
    }
    const double goal = (double)u * total;
    // the first piece whose running sum passes the goal, else the last that holds anything
    double run = incl - own, before = 0.0;
    int first = kVerifyPieces, last = -1;
#pragma unroll
    for (int k = 0; k < PL; ++k) {
      if (mine[k] > 0.0) {
        last = lane * PL + k;
        if (first == kVerifyPieces && run + mine[k] > goal) { first = lane * PL + k; before = run; }
      }
      run += mine[k];
    }
    const unsigned has = __ballot_sync(0xffffffffu, first < kVerifyPieces);
    int target_piece;
    if (has) {
      const int src = __ffs(has) - 1;
      target_piece = __shfl_sync(0xffffffffu, first, src);
      before = __shfl_sync(0xffffffffu, before, src);
    } else {
      target_piece = __reduce_max_sync(0xffffffffu, last);
      before = 0.0;
    }
    if (target_piece != piece) return;
    // this warp's piece holds the draw
    int found = -1, last_pos = -1;
    for (int i0 = lo; i0 < hi && found < 0; i0 += unit) {
      const int i = i0 + lane * E;
      double r[E], s = 0.0;
#pragma unroll
      for (int k = 0; k < E; ++k) r[k] = 0.0;
      if (i < hi) load_rest<T, E, VEC>(row, less, skip, i, hi, r);
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
          if (has && here < 0 && at > goal) here = i + k;
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
