// Attention of one or a few new tokens per sequence over a paged key-value cache (what the reference calls
// flash_attn_with_kvcache and its per-sequence fallback for, demo/src/layers/attention.py:262-349):
//
//   o[t,h] = sum_j softmax_j(scale * q[t,h] . k[j,g]) v[j,g],   g = h / (Hq/Hkv),   j < limit(t)
//   limit(t) = context - n + i + 1     for the i-th of a sequence's n new tokens (the cache already holds them)
//
// One pass over the cache with the running maximum and sum of a softmax.  What bounds it is HBM: a key and a value are
// read once for all query heads of their group and all tokens of the span (rows), 2 flops per row and byte.
//
// Work split.  A unit is (sequence, kv head, tile of R rows); it is cut along the cache into tiles of 64 keys (32 for
// the widest fp32 heads), and the tiles of all units, laid end to end, are dealt to the CTAs in equal contiguous ranges
// computed from the lengths on the device, so ragged batches stay balanced without the host knowing a length.  A CTA
// that holds a whole unit writes the output; otherwise it leaves (m, l, o) of its part in the workspace and
// a second kernel joins the parts in index order (results do not depend on timing).  Short contexts are not cut.
//
// Inside a CTA four key groups take 16 of the 64 keys of a tile each, with a ring of shared memory of their own that
// they fill with cp.async: no barrier of the CTA in the loop (with two row groups, one of 64 threads per stage).  When a
// unit ends, the loads of the next begin before the groups' results meet in the free slots of their rings.
// 16-bit types multiply on mma.sync m16n8k16: rows (padded to 16) x keys, accumulators and the softmax in registers.
// With 16 rows the tensor pipe is 19 % busy when HBM is saturated, with 32 rows 36 %; the hand-over through tensor memory
// that tcgen05 needs between the two products would lengthen the path of the few rows that decoding has.  Past 32 rows
// per kv head it would pay (the cache is then read once per 32 rows, from L2 at best): not built.  A prompt of 2048 tokens, 32
// query heads on 4, takes 478 us, 72 TFLOP/s, a twentieth of what the tensor cores give matrix products.
// fp32 multiplies on the CUDA cores (16 sequences of 300..6000 tokens 95 us, 2.6 times the bytes' time).
//
// Roundings: scores, softmax, sums and accumulators are fp32; p is rounded to the cache's type for the second product
// (the operand type of the tensor cores; the sum l uses the same unrounded p), outputs are rounded once.  That costs at
// most half a step of the type, 2^-8 (bf16) or 2^-11 of sum_j p_j |v_j| / l, besides the output's own; fp32 rounds no p.
//
// Measured on B200, device time back to back, heads of 128: 32 sequences of 21000 tokens, 8 kv heads of 4 queries 414 us
// (6.7 TB/s, the copy rate), with spans of 8 tokens 420; one sequence of 131071, 4 kv heads 48.6 us (5.5 TB/s); 16 of
// 300..6000 25.5 us (4.7 TB/s); 64 spans of 1..5 tokens, 8 queries a kv head, over 800..16384 tokens 233 us.  What is
// left there is fixed cost: about 5 us from the launch to the first products (lengths, page table and cache are three
// dependent loads), 1.5 to 5 us for the join.  A stage of 16 keys is some 1600 cycles of dependent instructions for its
// warp whatever is in flight, which eight warps an SM hide for 16 rows and just about for 32, where heads of 128 also
// spill 48 bytes a thread (92 with pages that are no multiple of 16 slots).  Slower were: bulk copies of a row per lane (by
// 10 to 30 %), rows padded in shared memory instead of permuted (3 to 9 %), a deeper ring (nothing).
#pragma once
#include <type_traits>

#include "common.cuh"
#include "tma.cuh"

namespace b200moe {

struct AttnParams {
  const void *q, *k, *v;
  void* out;
  float* lse;                      // may be null
  const int* tables;               // [B, table_stride]
  const int* context;              // [B]
  const int* qstart;               // [B+1] or null: one token per sequence
  int* status;                     // may be null
  float* ws;                       // parts: [2 * grid][R * D] o, [2 * grid][R][2] (m, l), [grid][R] (token, head), [grid] words
  long long q_tok, q_head, o_tok, o_head, c_block, c_slot, c_head, table_stride;
  float scale_log2;                // scale * log2(e)
  int B, T, Hq, Hkv, group, block_size, num_blocks, max_blocks, span;
  int split;                       // 0: units are not cut
  unsigned page_mul;               // key / block_size = key * page_mul >> page_shift, for keys below 2^31
  int page_shift;
  int tile_shift;                  // a tile holds 1 << tile_shift keys
  int unit_cost;                   // what beginning a unit costs, in tiles
  int grid;                        // CTAs of the attention kernel
  int cuts;                        // whether it leaves its cut units for the join (attn_join_cuts_kernel)
};

// ---------------------------------------------------------------------------------------------
// The work list, as every thread can recompute it from the lengths
// ---------------------------------------------------------------------------------------------
struct AttnSeq {
  int first, n, ctx;               // first query row, new tokens, keys
  int row_tiles, tiles;
};
template <bool AGAIN = false>                      // AGAIN: loaded here and now, whatever has been loaded before
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& p, int b, int r_shift) {   // a row tile holds 1 << r_shift rows
  auto get = [](const int* at) {
    if constexpr (!AGAIN) return *at;
    int v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
    return v;
  };
  AttnSeq s;
  s.first = b; s.n = 1;
  s.ctx = get(p.context + b);
  if (p.qstart) {
    s.first = get(p.qstart + b);
    s.n = get(p.qstart + b + 1) - s.first;
  }
  // lengths that do not fit the tensors: nothing is read or written out of range (reported by attn_report)
  if (s.first < 0 || s.n < 0 || s.first > p.T || s.n > p.T - s.first) s.n = 0;
  const long long cap = (long long)p.max_blocks * p.block_size;
  if (s.ctx < 0) s.ctx = 0;
  if (s.ctx > cap) s.ctx = (int)cap;
  s.row_tiles = (s.n * p.group + (1 << r_shift) - 1) >> r_shift;
  s.tiles = max((s.ctx + (1 << p.tile_shift) - 1) >> p.tile_shift, 1);   // an empty sequence still has rows to write
  return s;
}
__device__ __forceinline__ void attn_report(const AttnParams& p, int b) {
  if (!p.status) return;
  bool bad = p.context[b] < 0 || p.context[b] > (long long)p.max_blocks * p.block_size;
  if (p.qstart) {
    const int f = p.qstart[b], e = p.qstart[b + 1];
    bad = bad || f < 0 || e < f || e > p.T;
  }
  if (bad) atomicOr(p.status, kDevBadLength);
}
// What the join has to know of a unit that goes on behind the CTA that began it: token and query head of its rows, and in
// one word how many there are and which CTA took the last of its tiles (rows | CTA << 8).  Every CTA leaves that word:
// none begins more than one such unit, and one that begins none says 0 rows, so the workspace need not be cleared.
constexpr int kJoinThreads = 256;
constexpr int kJoinMaxGrid = 4 * kJoinThreads;                         // a thread of the join takes four of the words
__host__ __device__ constexpr long long attn_ml_at(int grid, int R, int D) { return 2ll * grid * R * D; }     // in floats
__host__ __device__ constexpr long long attn_row_at(int grid, int R, int D) { return 2ll * grid * R * (D + 2); }
__host__ __device__ constexpr long long attn_word_at(int grid, int R, int D) { return attn_row_at(grid, R, D) + 2ll * grid * R; }
__host__ __device__ constexpr long long attn_ws_floats(int grid, int R, int D) { return attn_word_at(grid, R, D) + (grid + 3) / 4 * 4; }
// A unit weighs its tiles and the cost of beginning it (the weight's first items stand for that).
__device__ __forceinline__ int attn_weight(const AttnParams& p, const AttnSeq& s) { return p.split ? s.tiles + p.unit_cost : 1; }
__device__ __forceinline__ long long attn_work(const AttnParams& p, const AttnSeq& s) { return (long long)s.row_tiles * p.Hkv * attn_weight(p, s); }
__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Work of the sequences [0, b_end), by a whole warp.
__device__ __forceinline__ long long attn_work_before(const AttnParams& p, int b_end, int r_shift) {
  long long w = 0;
  for (int b = threadIdx.x & 31; b < b_end; b += 32) w += attn_work(p, attn_seq(p, b, r_shift));
  return warp_sum_ll(w);
}
// The sequence that holds work item x, and the work before it; by a whole warp.
__device__ __forceinline__ int attn_find(const AttnParams& p, long long x, int r_shift, long long* before) {
  const int lane = threadIdx.x & 31;
  long long base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    const long long w = b < p.B ? attn_work(p, attn_seq(p, b, r_shift)) : 0;
    long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, x < base + inc);
    if (hit) {
      const int src = __ffs(hit) - 1;
      *before = base + __shfl_sync(0xffffffffu, inc - w, src);
      return b0 + src;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  *before = base;
  return p.B;
}
// Division of numbers that are seldom past 32 bits, where it takes a fifth of the time.
__device__ __forceinline__ long long div_ll(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
// CTA c of g takes the items [attn_lo(c), attn_lo(c+1)); item x belongs to CTA attn_owner(x).  g <= W.
__device__ __forceinline__ long long attn_lo(long long W, int g, int c) { return div_ll(W * c, g); }
__device__ __forceinline__ int attn_owner(long long W, int g, long long x) { return (int)div_ll((x + 1) * g - 1, W); }

// ---------------------------------------------------------------------------------------------
// Primitives
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  // a source size of zero fills the 16 bytes with zeros and reads nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 2^x, two units in the last place; results below 2^-126 become 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ bool any_nonfinite2(uint32_t x) {   // either of two packed 16-bit values
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (x & e) == e || ((x >> 16) & e) == e;
}

// Rows of ROWB bytes; 16-byte chunks are permuted within a row so that the eight rows that an ldmatrix or a quarter
// warp reads at one chunk position lie in eight different bank groups.
template <int ROWB> __device__ __forceinline__ uint32_t row_chunk(int row, int chunk) {
  if constexpr (ROWB >= 128) return row * ROWB + ((chunk ^ (row & 7)) << 4);
  else return row * ROWB + ((chunk ^ ((row >> 1) & 3)) << 4);
}

// MT: 16-row tiles of a warp, RG: row groups (warps that share a ring), KG: key groups.
template <typename T, int D, int MT, int RG, int KG, int STAGES_> struct AttnShape {
  static constexpr int R = 16 * MT * RG;
  static constexpr int R_SHIFT = R == 16 ? 4 : 5;
  static_assert(R == 1 << R_SHIFT, "rows");
  static constexpr int STAGES = STAGES_;
  static constexpr int KEYS = 16;                  // keys of a stage
  static constexpr int TILE = KEYS * KG;
  static constexpr int THREADS = 32 * KG * RG;
  static constexpr int ROWB = D * (int)sizeof(T);
  static constexpr int CPR = ROWB / 16;
  static constexpr int HALF_STAGE = KEYS * ROWB;   // K, then V
  static constexpr int SLOT = 2 * HALF_STAGE;
  static constexpr int RING = KG * STAGES * SLOT;
  // At the end of a unit a key group leaves its o in JSLOTS slots of its ring; the others fetch the next unit meanwhile.
  static constexpr int RPS = SLOT / (D * 4);       // rows of o in a slot
  static constexpr int JSLOTS = (R + RPS - 1) / RPS;
  static constexpr int AHEAD = STAGES - JSLOTS < STAGES - 1 ? STAGES - JSLOTS : STAGES - 1;
  static constexpr int QB = R * ROWB;
  static constexpr int Q_OFF = RING;               // two buffers
  static constexpr int ML_OFF = Q_OFF + 2 * QB;
  static constexpr int P_OFF = ML_OFF + KG * R * 8;                        // fp32 only: p [KG][KEYS][16], factors [KG][16]
  static constexpr int SMEM = P_OFF + (sizeof(T) == 4 ? KG * (KEYS + 1) * 16 * 4 : 0);
  static_assert(AHEAD >= 1, "room to fetch ahead");
};

// PAGE16: pages hold a multiple of 16 slots, so that the 16 keys of a stage lie in one page.
template <typename T, int D, int MT, int RG, int KG, int STAGES, int MINB, bool PAGE16>
__global__ void __launch_bounds__(32 * KG * RG, MINB) attn_kernel(const AttnParams p) {
  using S = AttnShape<T, D, MT, RG, KG, STAGES>;
  constexpr int R = S::R, RS = S::R_SHIFT, ROWB = S::ROWB, CPR = S::CPR, KEYS = S::KEYS, THREADS = S::THREADS;
  constexpr bool kMma = sizeof(T) == 2;
  static_assert(kMma || (MT == 1 && RG == 1), "shape");
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kg = warp % KG, rg = warp / KG;
  const uint32_t sbase = smem_addr(smem);
  const uint32_t ring = sbase + kg * (STAGES * S::SLOT);
  float2* s_ml = reinterpret_cast<float2*>(smem + S::ML_OFF);

  pdl_wait();
  pdl_trigger();
  if (p.status)
    for (int b = blockIdx.x * THREADS + tid; b < p.B; b += gridDim.x * THREADS) attn_report(p, b);
  const long long W = attn_work_before(p, p.B, RS);
  const int g = (int)(W < gridDim.x ? W : gridDim.x);
  const int cta = blockIdx.x;
  int* const words = reinterpret_cast<int*>(p.ws + attn_word_at(p.grid, R, D));
  if (p.cuts && cta == 0 && p.grid + tid < (p.grid + 3) / 4 * 4) words[p.grid + tid] = 0;
  if (cta >= g) {
    if (p.cuts && tid == 0) words[cta] = 0;
    return;
  }
  long long lo = attn_lo(W, g, cta);
  const long long hi = attn_lo(W, g, cta + 1);
  long long seq_base;
  int b_next = attn_find(p, lo, RS, &seq_base);
  const T* kc = reinterpret_cast<const T*>(p.k);
  const T* vc = reinterpret_cast<const T*>(p.v);

  // --- this CTA's units, one after the other
  struct Unit {
    int first, ctx, n;             // the sequence: query row, keys, new tokens
    int head, row0, rows;          // rows row0 .. row0 + rows - 1 of the sequence: token-major, then head of the group
    int tile0, ntile, part;        // part: where a cut unit's result goes, -1 for a whole one
    const int* table;
  };
  auto next_unit = [&](Unit* u) -> bool {
    while (lo < hi && b_next < p.B) {
      const AttnSeq sq = attn_seq(p, b_next, RS);
      const long long seq_work = attn_work(p, sq);
      if (lo >= seq_base + seq_work) { seq_base += seq_work; ++b_next; continue; }
      const int weight = attn_weight(p, sq);
      const int unit = (int)div_ll(lo - seq_base, weight), skip = (int)(lo - seq_base - (long long)unit * weight);
      const int take = (int)min(hi - lo, (long long)(weight - skip));
      lo += take;
      int t0 = 0, t1 = sq.tiles;
      if (p.split) {
        t0 = max(skip - p.unit_cost, 0);
        t1 = skip + take - p.unit_cost;
        if (t1 <= t0) continue;    // only the part that stands for the beginning
      }
      u->first = sq.first; u->ctx = sq.ctx; u->n = sq.n;
      u->head = unit / sq.row_tiles;   // row tiles of one head follow each other: the second finds the cache in L2
      u->row0 = unit % sq.row_tiles * R;
      u->rows = min(R, sq.n * p.group - u->row0);
      u->tile0 = t0; u->ntile = t1 - t0;
      // a part that begins inside a unit is this CTA's first, one that ends inside a unit its last
      u->part = t1 - t0 == sq.tiles ? -1 : 2 * cta + (t0 > 0 ? 0 : 1);
      u->table = p.tables + (long long)b_next * p.table_stride;
      return true;
    }
    return false;
  };

  // --- loads: a key group fills slot after slot of its ring with 16 keys and values
  constexpr int STEP = 32 * RG;                                       // lanes that fill a stage
  constexpr int COPIES = (KEYS * CPR + STEP - 1) / STEP;
  const int pt = rg * 32 + lane;
  int page_next = 0;                                                  // page of the next stage to fetch, looked up one stage ahead
  auto block_of = [&](int key) -> int { return (int)(((unsigned long long)(unsigned)key * p.page_mul) >> p.page_shift); };
  auto page_of = [&](const Unit& u, int t) -> int {                   // of this lane's key of tile t
    const int key = (u.tile0 + t) * S::TILE + kg * KEYS + (PAGE16 ? 0 : lane % KEYS);
    return (t < u.ntile && key < u.ctx) ? u.table[block_of(key)] : -1;
  };
  auto issue = [&](const Unit& u, int t, int slot_at, int page) {
    if (t < u.ntile) {
      const int key0 = (u.tile0 + t) * S::TILE + kg * KEYS;
      const uint32_t dst = ring + slot_at * S::SLOT;
      const T* kh = kc + u.head * p.c_head;
      const T* vh = vc + u.head * p.c_head;
      const int key = key0 + (PAGE16 ? 0 : lane % KEYS);              // the key whose page this lane looked up
      const bool in = key < u.ctx;
      const bool ok = in && page >= 0 && page < p.num_blocks;
      if (in && !ok && p.status) atomicOr(p.status, kDevBadPage);
      const long long off = ok ? page * p.c_block + (long long)(key - block_of(key) * p.block_size) * p.c_slot : 0;
      if constexpr (PAGE16) {
        // a lane's rows are STEP/CPR apart at one chunk (or, in rows longer than a step, its chunks STEP apart)
        constexpr int DROW = CPR <= STEP ? STEP / CPR : 0;
        const long long e = off + (pt / CPR) * p.c_slot + (pt % CPR) * (16 / (int)sizeof(T));
        const T* ks = kh + e;
        const T* vs = vh + e;
        auto place = [&](int i, int* row, int* ch, long long* delta) {
          const int idx = pt + i * STEP;
          *row = idx / CPR;
          *ch = idx % CPR;
          *delta = DROW ? (long long)(i * DROW) * p.c_slot : (long long)(*row - pt / CPR) * p.c_slot + (*ch - pt % CPR) * (16 / (int)sizeof(T));
        };
        int row, ch;
        long long delta;
        if (ok && key0 + KEYS <= u.ctx && KEYS * CPR % STEP == 0) {
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            place(i, &row, &ch, &delta);
            const uint32_t d = dst + row_chunk<ROWB>(row, ch);
            cp_async16(d, ks + delta);
            cp_async16(d + S::HALF_STAGE, vs + delta);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < COPIES; ++i) {
            place(i, &row, &ch, &delta);
            if (row < KEYS) {
              const bool there = ok && key0 + row < u.ctx;
              const uint32_t d = dst + row_chunk<ROWB>(row, ch);
              cp_async16(d, there ? ks + delta : kc, there);
              cp_async16(d + S::HALF_STAGE, there ? vs + delta : vc, there);
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
          const int idx = pt + i * STEP;
          const int row = idx / CPR, ch = idx % CPR;
          const long long o = __shfl_sync(0xffffffffu, ok ? off : -1, row % KEYS);
          if (KEYS * CPR % STEP == 0 || idx < KEYS * CPR) {
            const long long e = o + ch * (16 / (int)sizeof(T));
            const uint32_t d = dst + row_chunk<ROWB>(row, ch);
            cp_async16(d, o < 0 ? kc : kh + e, o >= 0);
            cp_async16(d + S::HALF_STAGE, o < 0 ? vc : vh + e, o >= 0);
          }
        }
      }
    }
    cp_async_commit();
  };
  auto slot_after = [](int at, int d) { return at + d >= STAGES ? at + d - STAGES : at + d; };   // d <= STAGES
  // the queries of a unit (into one of two buffers) and its first stages
  auto begin = [&](const Unit& u, int at, int qbuf) {
    int pages[S::AHEAD];                                              // all at once: one after the other they cost 0.4 us each
#pragma unroll
    for (int t = 0; t < S::AHEAD; ++t) pages[t] = page_of(u, t);
    page_next = page_of(u, S::AHEAD);
    for (int i = tid; i < R * CPR; i += THREADS) {
      const int r = i / CPR, ch = i % CPR;
      const int token = u.first + (u.row0 + r) / p.group, h = u.head * p.group + (u.row0 + r) % p.group;
      const T* src = reinterpret_cast<const T*>(p.q) + token * p.q_tok + h * p.q_head + ch * (16 / (int)sizeof(T));
      cp_async16(sbase + S::Q_OFF + qbuf * S::QB + row_chunk<ROWB>(r, ch), r < u.rows ? src : reinterpret_cast<const T*>(p.q), r < u.rows);
    }
#pragma unroll
    for (int t = 0; t < S::AHEAD; ++t) issue(u, t, slot_after(at, t), pages[t]);
  };
  // where row r, column c of key group k's o lies while the groups meet: `at` is the ring slot of the next stage
  auto o_place = [&](int k, int r, int c, int at) -> float* {
    const int slot = slot_after(at, S::AHEAD + r / S::RPS);
    const int unit32 = (c >> 3) ^ (r & (D / 8 < 8 ? D / 8 - 1 : 7));  // 32-byte units permuted: the 8 rows of a fragment in different banks
    return reinterpret_cast<float*>(smem + (k * STAGES + slot) * S::SLOT + (r % S::RPS) * (D * 4) + unit32 * 32 + (c & 7) * 4);
  };

  Unit u;
  bool more = next_unit(&u);
  int at = 0, qbuf = 0;                                               // ring slot of the stage in hand, buffer of the queries
  if (more) begin(u, at, qbuf);
  if (p.cuts && warp == 0) {       // while the first loads are under way: the unit that this CTA begins and does not end
    long long base;
    const AttnSeq sq = attn_seq(p, attn_find(p, hi - 1, RS, &base), RS);
    const int weight = attn_weight(p, sq), unit = (int)div_ll(hi - 1 - base, weight);
    const long long tiles_at = base + (long long)unit * weight + p.unit_cost;     // work item of its first tile
    const bool cut = hi > tiles_at && hi < tiles_at + sq.tiles && attn_lo(W, g, cta) <= tiles_at;
    const int row = unit % sq.row_tiles * R + lane, rows = cut ? min(R, sq.n * p.group - unit % sq.row_tiles * R) : 0;
    if (lane < rows)
      reinterpret_cast<int2*>(p.ws + attn_row_at(p.grid, R, D))[cta * R + lane] =
          make_int2(sq.first + row / p.group, unit / sq.row_tiles * p.group + row % p.group);
    if (lane == 0) words[cta] = cut ? attn_owner(W, g, tiles_at + sq.tiles - 1) << 8 | rows : 0;
  }
  while (more) {
#pragma unroll
    for (int t = S::AHEAD; t < STAGES - 1; ++t) {
      issue(u, t, slot_after(at, t), page_next);
      page_next = page_of(u, t + 1);
    }
    cp_async_wait<STAGES - 2>();                                      // the queries have come with the first stage
    __syncthreads();
    const int rows = u.rows, row0 = u.row0;
    const int lim0 = u.ctx - u.n + 1 + row0 / p.group;                // keys that the first (and least seeing) row sees
    auto limit = [&](int r) { return u.ctx - u.n + 1 + (row0 + min(r, rows - 1)) / p.group; };
    Unit nu;

    if constexpr (kMma) {
      // rows lane/4 and lane/4 + 8 of each 16-row tile, columns 2*(lane%4), +1 of each 8-column tile.  Row tiles go to the
      // row groups in turn; tiles without a row are left out.
      const int mts = min(MT, ((rows + 15) / 16 - rg + RG - 1) / RG);
      float o[MT][D / 8][4];
      float m[MT][2], l[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.0f;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          m[mt][hh] = -INFINITY; l[mt][hh] = 0.0f;
        }
      }
      // Fragment addresses: a step of 16 columns is two chunks, and an exclusive or with it keeps the permutation.
      const uint32_t q_off = sbase + S::Q_OFF + qbuf * S::QB + row_chunk<ROWB>(rg * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
      const uint32_t k_off = row_chunk<ROWB>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
      const uint32_t v_off = S::HALF_STAGE + row_chunk<ROWB>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
      constexpr bool kQRegs = MT == 1 && RG == 1 && D <= 128;         // else the registers are needed for o
      uint32_t qf[kQRegs ? D / 16 : 1][4];
      if constexpr (kQRegs) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) ldsm4(qf[ks], q_off ^ (ks << 5));
      }

      // One stage (16 keys) for the first M row tiles of this warp
      auto stage = [&](auto tiles, uint32_t base, int key0) {
        constexpr int M = decltype(tiles)::value;
        float s[M][2][4];
#pragma unroll
        for (int mt = 0; mt < M; ++mt)
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t kf[4];
          ldsm4(kf, (base + k_off) ^ (ks << 5));
#pragma unroll
          for (int mt = 0; mt < M; ++mt) {
            if constexpr (kQRegs) {
              mma16816<T>(s[mt][0], qf[ks], kf[0], kf[1]);
              mma16816<T>(s[mt][1], qf[ks], kf[2], kf[3]);
            } else {
              uint32_t a[4];
              ldsm4(a, (q_off ^ (ks << 5)) + mt * (RG * 16 * ROWB));
              mma16816<T>(s[mt][0], a, kf[0], kf[1]);
              mma16816<T>(s[mt][1], a, kf[2], kf[3]);
            }
          }
        }

        const bool masked = key0 + KEYS > lim0;
        // keys that this lane's row hh of row tile mt sees (recomputed in the few stages that need it: registers are scarce)
        auto row_limit = [&](int mt, int hh) { return limit((mt * RG + rg) * 16 + hh * 8 + (lane >> 2)); };
        if (masked) {
#pragma unroll
          for (int mt = 0; mt < M; ++mt)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const int lim = row_limit(mt, hh);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key0 + (i >> 1) * 8 + 2 * (lane & 3) + (i & 1) >= lim) s[mt][i >> 1][2 * hh + (i & 1)] = -INFINITY;
            }
        }
        // m is the reference that p is taken against, l and o are relative to the same one.  It lies kLift powers of two
        // below a maximum of the row and is renewed only when the row has outgrown that by kLag, so that o is seldom
        // rescaled: the largest p is between 2^kLift and 2^(kLift + kLag).  bf16 has fp32's range.  fp16 ends at 2^-24, so
        // there p goes up to 2^12 (2^4 are left to its largest number): what is lost of a key is at most 2^-33 of the
        // largest p, 2^-16 in all over 131071 keys.  Without the lift 60000 keys of 2^-26 each vanished beside one.
        constexpr float kLift = std::is_same<T, __half>::value ? 8.0f : 0.0f, kLag = std::is_same<T, __half>::value ? 4.0f : 8.0f;
        bool grew = false;
        float top[M][2];
#pragma unroll
        for (int mt = 0; mt < M; ++mt) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float x = fmaxf(fmaxf(s[mt][0][2 * hh], s[mt][0][2 * hh + 1]), fmaxf(s[mt][1][2 * hh], s[mt][1][2 * hh + 1]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            top[mt][hh] = x * p.scale_log2;
            grew = grew || top[mt][hh] > m[mt][hh] + (kLift + kLag);
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int mt = 0; mt < M; ++mt) {
            float fac[2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const bool renew = top[mt][hh] > m[mt][hh] + (kLift + kLag);
              const float next = top[mt][hh] - kLift;
              fac[hh] = renew ? ex2(m[mt][hh] - next) : 1.0f;
              if (renew) m[mt][hh] = next;
              l[mt][hh] *= fac[hh];
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              o[mt][i][0] *= fac[0]; o[mt][i][1] *= fac[0];
              o[mt][i][2] *= fac[1]; o[mt][i][3] *= fac[1];
            }
          }
        }
        uint32_t pf[M][4];
#pragma unroll
        for (int mt = 0; mt < M; ++mt) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const float ref = m[mt][hh] == -INFINITY ? 0.0f : m[mt][hh];      // a row that has seen nothing yet
            const float x0 = ex2(fmaf(s[mt][0][2 * hh], p.scale_log2, -ref)), x1 = ex2(fmaf(s[mt][0][2 * hh + 1], p.scale_log2, -ref));
            const float x2 = ex2(fmaf(s[mt][1][2 * hh], p.scale_log2, -ref)), x3 = ex2(fmaf(s[mt][1][2 * hh + 1], p.scale_log2, -ref));
            l[mt][hh] += (x0 + x1) + (x2 + x3);
            pf[mt][hh] = pack2<T>(x0, x1);
            pf[mt][2 + hh] = pack2<T>(x2, x3);
          }
        }
        // A key that some rows may not see has p = 0 there, which a product with an infinity or NaN turns into NaN.
        // Such values are looked for in the few stages where rows differ; there the keys then go one by one and rows
        // that do not see a key keep what they had.
        bool odd = false;
        if (masked) {
          for (int i = lane; i < KEYS * CPR; i += 32) {
            const uint4 x = *reinterpret_cast<const uint4*>(smem + (base - sbase) + S::HALF_STAGE + i * 16);
            odd = odd || any_nonfinite2<T>(x.x) || any_nonfinite2<T>(x.y) || any_nonfinite2<T>(x.z) || any_nonfinite2<T>(x.w);
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
          for (int dn = 0; dn < D / 16; ++dn) {
            uint32_t vf[4];
            ldsm4_t(vf, (base + v_off) ^ (dn << 5));
#pragma unroll
            for (int mt = 0; mt < M; ++mt) {
              mma16816<T>(o[mt][2 * dn], pf[mt], vf[0], vf[1]);
              mma16816<T>(o[mt][2 * dn + 1], pf[mt], vf[2], vf[3]);
            }
          }
        } else {
          int lim[M][2];
#pragma unroll
          for (int mt = 0; mt < M; ++mt) { lim[mt][0] = row_limit(mt, 0); lim[mt][1] = row_limit(mt, 1); }
#pragma unroll 1
          for (int j = 0; j < KEYS; ++j) {
            // this lane holds keys 2*(lane%4), +1 (registers 0, 1 of A; 0, 2 of B) and those + 8 (2, 3; 1, 3)
            const uint32_t keep = (j & 7) / 2 == (lane & 3) ? (j & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
            const uint32_t k_lo = j < 8 ? keep : 0u, k_hi = j < 8 ? 0u : keep;
#pragma unroll
            for (int dn = 0; dn < D / 16; ++dn) {
              uint32_t vf[4];
              ldsm4_t(vf, (base + v_off) ^ (dn << 5));
#pragma unroll
              for (int mt = 0; mt < M; ++mt) {
                const uint32_t a[4] = {pf[mt][0] & k_lo, pf[mt][1] & k_lo, pf[mt][2] & k_hi, pf[mt][3] & k_hi};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  float (&acc)[4] = o[mt][2 * dn + half];
                  float next[4] = {acc[0], acc[1], acc[2], acc[3]};
                  mma16816<T>(next, a, vf[2 * half] & k_lo, vf[2 * half + 1] & k_hi);
                  if (key0 + j < lim[mt][0]) { acc[0] = next[0]; acc[1] = next[1]; }
                  if (key0 + j < lim[mt][1]) { acc[2] = next[2]; acc[3] = next[3]; }
                }
              }
            }
          }
        }
      };

      for (int t = 0; t < u.ntile; ++t) {
        cp_async_wait<STAGES - 2>();
        if constexpr (RG > 1) bar_sync(1 + kg, 32 * RG); else __syncwarp();
        issue(u, t + STAGES - 1, slot_after(at, STAGES - 1), page_next);
        page_next = page_of(u, t + STAGES);
        const uint32_t base = ring + at * S::SLOT;
        at = slot_after(at, 1);
        const int key0 = (u.tile0 + t) * S::TILE + kg * KEYS;
        if (key0 >= u.ctx) continue;                                  // nothing of the last tile in this group
        if constexpr (MT == 2) {
          if (mts == 2) stage(std::integral_constant<int, 2>{}, base, key0);
          else if (mts == 1) stage(std::integral_constant<int, 1>{}, base, key0);
        } else {
          if (RG == 1 || mts == 1) stage(std::integral_constant<int, 1>{}, base, key0);
        }
      }
      if constexpr (RG > 1) bar_sync(1 + kg, 32 * RG); else __syncwarp();   // the ring is free
      more = next_unit(&nu);
      if (more) begin(nu, at, qbuf ^ 1);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int r = (mt * RG + rg) * 16 + hh * 8 + (lane >> 2);
          float sum = l[mt][hh];
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if ((lane & 3) == 0) s_ml[kg * R + r] = make_float2(m[mt][hh], sum);
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(o_place(kg, r, i * 8 + 2 * (lane & 3), at)) = make_float2(o[mt][i][2 * hh], o[mt][i][2 * hh + 1]);
        }
      }
    } else {
      // fp32: for the scores a lane is one key and every other row, for the second product D/32 columns and all rows.  What
      // bounds it are the loads from shared memory (five of 16 bytes for 16 products), so rows go in groups of 4, 8 or 16
      // and are not padded to 16 as on the tensor cores.
      constexpr int C = D / 32;                                       // output columns of a lane
      float* s_p = reinterpret_cast<float*>(smem + S::P_OFF) + kg * (KEYS + 1) * 16;
      float* s_f = s_p + KEYS * 16;
      const int key_l = lane % 16, half = lane / 16;                  // score rows half, half + 2, ...
      const int my_limit = limit(key_l);                              // of row lane % 16
      float o[16][C], m[8], l[8];
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int i = 0; i < C; ++i) o[r][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) { m[i] = -INFINITY; l[i] = 0.0f; }
      const unsigned char* s_q = smem + S::Q_OFF + qbuf * S::QB;
      // One stage for the first 2 * NP rows
      auto stage = [&](auto pairs, const unsigned char* ks_base, int key0) {
        constexpr int NP = decltype(pairs)::value;
        const unsigned char* vs_base = ks_base + S::HALF_STAGE;
        float s[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) s[i] = 0.0f;
#pragma unroll 4
        for (int ch = 0; ch < CPR; ++ch) {
          const float4 kv = *reinterpret_cast<const float4*>(ks_base + row_chunk<ROWB>(key_l, ch));
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float4 qv = *reinterpret_cast<const float4*>(s_q + row_chunk<ROWB>(2 * i + half, ch));
            s[i] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[i]))));
          }
        }
        const bool masked = key0 + KEYS > lim0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (masked) {
            const int lim = __shfl_sync(0xffffffffu, my_limit, 2 * i + half);
            if (key0 + key_l >= lim) s[i] = -INFINITY;
          }
          float top = s[i] * p.scale_log2;
#pragma unroll
          for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          const float mn = fmaxf(m[i], top);
          const float ref = mn == -INFINITY ? 0.0f : mn;
          const float f = ex2(m[i] - ref);
          m[i] = mn;
          const float x = ex2(fmaf(s[i], p.scale_log2, -ref));
          l[i] = l[i] * f + x;
          s_p[key_l * 16 + 2 * i + half] = x;
          if (key_l == 0) s_f[2 * i + half] = f;
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 2 * NP; ++r) {
          const float f = s_f[r];
#pragma unroll
          for (int i = 0; i < C; ++i) o[r][i] *= f;
        }
#pragma unroll 2
        for (int j = 0; j < KEYS; ++j) {
          float v[C];
#pragma unroll
          for (int i = 0; i < C; ++i) {
            // the lane's columns are adjacent: C floats from column lane*C on
            const int col = lane * C + i;
            v[i] = *reinterpret_cast<const float*>(vs_base + row_chunk<ROWB>(j, col / 4) + (col % 4) * 4);
          }
          float w[2 * NP];
#pragma unroll
          for (int r = 0; r < 2 * NP; r += 4) {
            const float4 x = *reinterpret_cast<const float4*>(s_p + j * 16 + r);
            w[r] = x.x; w[r + 1] = x.y; w[r + 2] = x.z; w[r + 3] = x.w;
          }
          // rows that do not see the key are left alone (0 * inf is not 0)
          const unsigned seen = masked ? __ballot_sync(0xffffffffu, key0 + j < my_limit) : 0xffffffffu;
          if (seen == 0xffffffffu) {
#pragma unroll
            for (int r = 0; r < 2 * NP; ++r)
#pragma unroll
              for (int i = 0; i < C; ++i) o[r][i] = fmaf(w[r], v[i], o[r][i]);
          } else if (seen) {
#pragma unroll
            for (int r = 0; r < 2 * NP; ++r)
#pragma unroll
              for (int i = 0; i < C; ++i) o[r][i] = (seen >> r) & 1 ? fmaf(w[r], v[i], o[r][i]) : o[r][i];
          }
        }
        __syncwarp();
      };
      for (int t = 0; t < u.ntile; ++t) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        issue(u, t + STAGES - 1, slot_after(at, STAGES - 1), page_next);
        page_next = page_of(u, t + STAGES);
        const unsigned char* base = smem + (ring - sbase) + at * S::SLOT;
        at = slot_after(at, 1);
        const int key0 = (u.tile0 + t) * S::TILE + kg * KEYS;
        if (key0 >= u.ctx) continue;
        if (rows <= 4) stage(std::integral_constant<int, 2>{}, base, key0);
        else if (rows <= 8) stage(std::integral_constant<int, 4>{}, base, key0);
        else stage(std::integral_constant<int, 8>{}, base, key0);
      }
      more = next_unit(&nu);
      if (more) begin(nu, at, qbuf ^ 1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float sum = l[i];
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (key_l == 0) s_ml[kg * R + 2 * i + half] = make_float2(m[i], sum);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int i = 0; i < C; ++i) *o_place(kg, r, lane * C + i, at) = o[r][i];
    }
    __syncthreads();

    // --- join the key groups; write the output of a whole unit or the part of a cut one
    for (int i = tid; i < rows * (D / 4); i += THREADS) {
      const int r = i / (D / 4), c = i % (D / 4);
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < KG; ++k) top = fmaxf(top, s_ml[k * R + r].x);
      const float ref = top == -INFINITY ? 0.0f : top;
      float l = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const float2 ml = s_ml[k * R + r];
        const float f = ex2(ml.x - ref);
        const float4 x = *reinterpret_cast<const float4*>(o_place(k, r, c * 4, at));
        l = fmaf(ml.y, f, l);
        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
      }
      if (u.part < 0) {
        const int token = u.first + (row0 + r) / p.group, h = u.head * p.group + (row0 + r) % p.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;                // a row that sees no key gives zeros
        T* dst = reinterpret_cast<T*>(p.out) + token * p.o_tok + h * p.o_head + c * 4;
        if constexpr (kMma) {
          uint2 v;
          v.x = pack2<T>(acc.x * inv, acc.y * inv);
          v.y = pack2<T>(acc.z * inv, acc.w * inv);
          *reinterpret_cast<uint2*>(dst) = v;
        } else {
          *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
        if (p.lse && c == 0) p.lse[(long long)token * p.Hq + h] = l == 0.0f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(p.ws + ((long long)u.part * R + r) * D + c * 4) = acc;
        if (c == 0) reinterpret_cast<float2*>(p.ws + attn_ml_at(p.grid, R, D))[(long long)u.part * R + r] = make_float2(top, l);
      }
    }
    qbuf ^= 1;
    u = nu;
    __syncthreads();                                                  // before the slots that held o are filled again
  }
}

// ---------------------------------------------------------------------------------------------
// The join of the units that attn_kernel cut, in the order of the CTAs
// ---------------------------------------------------------------------------------------------
struct JoinRow {
  int c0, c1, r;                   // the CTAs that began and ended the row's unit (c1 < c0: there is nothing to join), the row in it
  int token, h;
};
// Four parts of a row (every WPR-th from `c` on), their loads side by side whether or not there are four.
template <int C> struct JoinParts {
  float2 ml[4];
  float x[4][C];
  template <int D, int WPR> __device__ __forceinline__ void load(const AttnParams& p, const JoinRow& j, int R, int c) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int ck = c + k * WPR;
      const long long part = (long long)(2 * ck + (ck == j.c0 ? 1 : 0)) * R + j.r;
      ml[k] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int i = 0; i < C; ++i) x[k][i] = 0.0f;
      if (ck <= j.c1) {
        ml[k] = reinterpret_cast<const float2*>(p.ws + attn_ml_at(p.grid, R, D))[part];
        const float* src = p.ws + part * D + lane * C;
        if constexpr (C >= 4) {
#pragma unroll
          for (int i = 0; i < C; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + i);
            x[k][i] = v.x; x[k][i + 1] = v.y; x[k][i + 2] = v.z; x[k][i + 3] = v.w;
          }
        } else if constexpr (C == 2) {
          const float2 v = *reinterpret_cast<const float2*>(src);
          x[k][0] = v.x; x[k][1] = v.y;
        } else {
          x[k][0] = *src;
        }
      }
    }
  }
};
// (m, l, o) of what has been joined of a row; C columns of o a lane
template <int C> struct JoinSum {
  float top = -INFINITY, l = 0.0f, acc[C];
  __device__ __forceinline__ JoinSum() {
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.0f;
  }
  __device__ __forceinline__ void add(const JoinParts<C>& q) {
    float mn = top;
#pragma unroll
    for (int k = 0; k < 4; ++k) mn = fmaxf(mn, q.ml[k].x);
    const float ref = mn == -INFINITY ? 0.0f : mn, f0 = ex2(top - ref);
    l *= f0;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] *= f0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = ex2(q.ml[k].x - ref);
      l = fmaf(q.ml[k].y, f, l);
#pragma unroll
      for (int i = 0; i < C; ++i) acc[i] = fmaf(q.x[k][i], f, acc[i]);
    }
    top = mn;
  }
};
template <typename T, int D> __device__ __forceinline__ void join_store(const AttnParams& p, const JoinRow& j, const JoinSum<D / 32>& s) {
  constexpr int C = D / 32;
  const int lane = threadIdx.x & 31;
  const float inv = s.l == 0.0f ? 0.0f : 1.0f / s.l;
  T* dst = reinterpret_cast<T*>(p.out) + j.token * p.o_tok + j.h * p.o_head + lane * C;
  if constexpr (sizeof(T) == 2 && C >= 2) {
    uint32_t v[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; ++i) v[i] = pack2<T>(s.acc[2 * i] * inv, s.acc[2 * i + 1] * inv);
    if constexpr (C == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
    else if constexpr (C == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
    else *reinterpret_cast<uint32_t*>(dst) = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) dst[i] = Elem<T>::from_float(s.acc[i] * inv);
  }
  if (p.lse && lane == 0) p.lse[(long long)j.token * p.Hq + j.h] = s.l == 0.0f ? -INFINITY : (s.top + log2f(s.l)) * 0.6931471805599453f;
}

// 64 bits that lengths which differ share by an accident of 2^-64.
__device__ __forceinline__ unsigned long long join_digest(unsigned long long d, const AttnSeq& s) {
  d = d * 0x9e3779b97f4a7c15ull + ((unsigned long long)(unsigned)s.ctx << 32 | (unsigned)s.first);
  return d * 0xd1b54a32d192ed03ull + (unsigned)s.n;
}
__device__ __forceinline__ unsigned long long join_lengths(const AttnParams& p, int r_shift) {
  unsigned long long d = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + (int)(threadIdx.x & 31);
    AttnSeq sq = {};
    if (b < p.B) sq = attn_seq<true>(p, b, r_shift);
    d = join_digest(d, sq);
  }
  return d;
}

// What became of an output row, from the lengths; by a whole warp.  Starts need not be in order (spans that fit nothing stand
// between): the row belongs to the first sequence that holds it.
// *seen: a digest of this lane's part of the lengths (join_lengths).
__device__ __forceinline__ void join_find(const AttnParams& p, int r_shift, JoinRow* j, unsigned long long* seen) {
  const int lane = threadIdx.x & 31;
  long long all = 0, before = 0;   // of this lane's sequences: work, and work in front of the row's sequence
  int first = 0, n = 0, tiles = 0, row_tiles = 0, weight = 0;
  bool have = false;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    long long w = 0;
    AttnSeq sq = {};
    if (b < p.B) {
      sq = attn_seq<true>(p, b, r_shift);
      w = attn_work(p, sq);
    }
    *seen = join_digest(*seen, sq);
    all += w;
    if (have) continue;
    const unsigned hit = __ballot_sync(0xffffffffu, j->token >= sq.first && j->token - sq.first < sq.n);
    const int src = hit ? __ffs(hit) - 1 : 32;
    if (lane < src) before += w;
    if (hit) {
      have = true;
      first = __shfl_sync(0xffffffffu, sq.first, src);
      n = __shfl_sync(0xffffffffu, sq.n, src);
      tiles = __shfl_sync(0xffffffffu, sq.tiles, src);
      row_tiles = __shfl_sync(0xffffffffu, sq.row_tiles, src);
      weight = tiles + p.unit_cost;
    }
  }
  j->c0 = 0; j->c1 = -1; j->r = 0;
  if (!have) return;
  all = warp_sum_ll(all);
  before = warp_sum_ll(before);
  const int g = (int)(all < p.grid ? all : p.grid);
  const int r_all = (j->token - first) * p.group + j->h % p.group;
  const long long at = before + (long long)(j->h / p.group * row_tiles + (r_all >> r_shift)) * weight + p.unit_cost;
  const int c0 = attn_owner(all, g, at), c1 = attn_owner(all, g, at + tiles - 1);
  if (c0 == c1) return;                                               // one CTA had it all and has written the output
  j->c0 = c0; j->c1 = c1; j->r = r_all & ((1 << r_shift) - 1);
}

// For calls of few rows: WPR warps (2, 4 or 8) of the CTA's 8 share an output row, and find out from the lengths what became of
// it, as far as they can before the wait for attn_kernel.  But only the wait promises that the lengths can be seen; so what
// was found is a guess, by which the first parts are fetched behind the wait, and while they are on their way the lengths
// are read again.  Where they differ, which no run has shown, the parts are fetched anew.
template <typename T, int D, int WPR>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnParams p, int r_shift) {
  constexpr int RPC = 8 / WPR, C = D / 32;
  static_assert(WPR > 1, "one warp a row: attn_join_cuts_kernel");
  const int R = 1 << r_shift;
  __shared__ float s_acc[8][D];
  __shared__ float2 s_ml[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  const unsigned row = blockIdx.x * RPC + warp / WPR;                 // (token, head), below 2^31
  JoinRow j = {0, -1, 0, (int)(row / (unsigned)p.Hq), (int)(row % (unsigned)p.Hq)};
  unsigned long long seen = 0;
  if (j.token < p.T) join_find(p, r_shift, &j, &seen);
  pdl_wait();
  JoinParts<C> q;
  q.template load<D, WPR>(p, j, R, j.c0 + warp % WPR);
  if (j.token < p.T) {
    if (__any_sync(0xffffffffu, join_lengths(p, r_shift) != seen)) {
      const JoinRow guess = j;
      join_find(p, r_shift, &j, &seen);
      if (j.c0 != guess.c0 || j.c1 != guess.c1 || j.r != guess.r) q.template load<D, WPR>(p, j, R, j.c0 + warp % WPR);
    }
  }
  JoinSum<C> sum;
  for (int c = j.c0 + warp % WPR;;) {
    sum.add(q);
    c += 4 * WPR;
    if (c > j.c1) break;
    q.template load<D, WPR>(p, j, R, c);
  }
#pragma unroll
  for (int i = 0; i < C; ++i) s_acc[warp][lane * C + i] = sum.acc[i];
  if (lane == 0) s_ml[warp] = make_float2(sum.top, sum.l);
  __syncthreads();
  if (warp % WPR != 0 || j.c1 < j.c0) return;
  JoinSum<C> whole;
#pragma unroll
  for (int w = 0; w < WPR; ++w) whole.top = fmaxf(whole.top, s_ml[warp + w].x);
  const float ref = whole.top == -INFINITY ? 0.0f : whole.top;
#pragma unroll
  for (int w = 0; w < WPR; ++w) {
    const float f = ex2(s_ml[warp + w].x - ref);
    whole.l = fmaf(s_ml[warp + w].y, f, whole.l);
#pragma unroll
    for (int i = 0; i < C; ++i) whole.acc[i] = fmaf(s_acc[warp + w][lane * C + i], f, whole.acc[i]);
  }
  join_store<T, D>(p, j, whole);
}

// For calls of many rows: a warp a row, and only the rows that were cut, from what attn_kernel's CTAs left.  Every CTA adds the
// counts up and takes its place among the cut rows, however many sequences there are and wherever their rows lie.  That is
// a load and a scan in front of the parts' loads, but no work that grows with rows x sequences: 1024 sequences of up to
// 600 tokens, 8 kv heads: 243 us, with every row looked up from the lengths 284.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) attn_join_cuts_kernel(const AttnParams p, int r_shift) {
  constexpr int C = D / 32;
  const int R = 1 << r_shift;
  __shared__ int s_rows[8];
  __shared__ int3 s_at[8];                                            // per warp: c0, c1, r
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  if (threadIdx.x < 8) s_at[threadIdx.x] = make_int3(0, -1, 0);
  pdl_wait();
  const int c_own = threadIdx.x * 4;
  int4 v = make_int4(0, 0, 0, 0);
  if (c_own < p.grid) v = *reinterpret_cast<const int4*>(p.ws + attn_word_at(p.grid, R, D) + c_own);
  const int word[4] = {v.x, v.y, v.z, v.w};
  const int mine = (v.x & 255) + (v.y & 255) + (v.z & 255) + (v.w & 255);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) s_rows[warp] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;                                // cut rows before this thread's, and all of them
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before += w < warp ? s_rows[w] : 0;
    total += s_rows[w];
  }
  // One round, but where spans that do not fit make sequences share rows: then there can be more cut rows than rows.
  for (int first = (int)blockIdx.x * 8; first < total; first += (int)gridDim.x * 8) {
    int at = before - first;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = word[i] & 255;
      for (int k = max(at, 0); k < min(at + n, 8); ++k) s_at[k] = make_int3(c_own + i, word[i] >> 8, k - at);
      at += n;
    }
    __syncthreads();
    JoinRow j = {s_at[warp].x, s_at[warp].y, s_at[warp].z, 0, 0};
    if (j.c1 >= j.c0) {
      const int2 dest = reinterpret_cast<const int2*>(p.ws + attn_row_at(p.grid, R, D))[j.c0 * R + j.r];
      JoinSum<C> sum;
      for (int c = j.c0; c <= j.c1; c += 4) {
        JoinParts<C> q;
        q.template load<D, 1>(p, j, R, c);
        sum.add(q);
      }
      j.token = dest.x;
      j.h = dest.y;
      join_store<T, D>(p, j, sum);
    }
    if (first + (int)gridDim.x * 8 >= total) break;
    __syncthreads();
    if (threadIdx.x < 8) s_at[threadIdx.x] = make_int3(0, -1, 0);
    __syncthreads();
  }
}

}  // namespace b200moe
