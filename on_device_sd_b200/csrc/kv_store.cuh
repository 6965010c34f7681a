// Writes new keys and values into the paged cache, with the head norm and the rotary embedding of queries and keys in
// the same pass (the reference runs q_norm / k_norm, the rotary embedding and store_kvcache_kernel one after the
// other, demo/src/layers/attention.py:32-79):
//   y = x * rsqrt(mean(x^2) + eps) * w          (only with norm weights)
//   z = (y1*cos - y2*sin, y2*cos + y1*sin)      y1, y2 the halves of the head, angles by position
//   q_out[t] = z(q);  cache[slot[t]] = z(k), v  (slot -1: nothing is stored)
// Everything between the load and the store is fp32 and each output is rounded once.
//
// What bounds it: one launch for the few tokens of a decoding step, HBM for a prompt.  D/16 lanes hold one head, each
// lane 8 elements of either half, so a rotation pairs registers of one lane, loads are 16 bytes and the norm's sum is
// a few shuffles.  A lane group takes kHeads heads of one token after the other and keeps the token's angles in
// registers: the fp32 table row is twice a 16-bit head.  8191 tokens of 32 + 2 x 8 heads of 128, fp16, take 35.7 us
// (5.8 TB/s) with four heads, in fp32 68 us (6.0 TB/s); two were 4 % and eight 27 % slower.
#pragma once
#include "common.cuh"

namespace b200moe {

struct StoreKvParams {
  const void *q, *k, *v;
  void* q_out;
  void *k_cache, *v_cache;
  const void *positions, *slots;
  const float* cos_sin;            // [max_position, D]: cosines of the D/2 angles, then sines
  const void *q_weight, *k_weight; // [D] or null
  int* status;                     // may be null
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;   // element strides
  long long c_block, c_slot, c_head;
  long long num_slots;             // num_blocks * block_size
  int T, Hq, Hkv, block_size, max_position;
  int positions64, slots64;
  float eps;
};

__device__ __forceinline__ long long load_index(const void* p, int i, int is64) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

template <typename T> __device__ __forceinline__ void store_chunk(T* dst, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

constexpr int kStoreThreads = 64;     // small CTAs: 8191 tokens 35.7 us, with 128 threads 36.5, with 256 37.8

// Heads 0..Hq-1 are queries, then Hkv keys, then Hkv values.  Lane group = (token, kHeads consecutive heads).
template <typename T, int D, int kHeads>
__global__ void __launch_bounds__(kStoreThreads) store_kv_kernel(const StoreKvParams p) {
  constexpr int L = D / 16;                        // lanes of a head
  constexpr int HALF = D / 2;
  pdl_trigger();
  pdl_wait();
  const int heads = p.Hq + 2 * p.Hkv;
  const unsigned groups = (unsigned)(heads + kHeads - 1) / kHeads;
  const unsigned item = blockIdx.x * (unsigned)(kStoreThreads / L) + threadIdx.x / L;   // below 2^32, as the caller checks
  const int sub = threadIdx.x % L;
  const bool live = item < p.T * groups;              // whole lane groups; idle ones still take part in the shuffles
  const int t = live ? (int)(item / groups) : 0;
  const int h0 = live ? (int)(item % groups) * kHeads : heads;

  const long long slot = p.slots ? load_index(p.slots, t, p.slots64) : -1;
  const bool rotate = p.cos_sin != nullptr;
  long long pos = 0;
  bool bad_pos = false;
  if (rotate) {
    pos = load_index(p.positions, t, p.positions64);
    bad_pos = pos < 0 || pos >= p.max_position;
  }
  const bool bad_slot = slot < -1 || slot >= p.num_slots;
  if (p.status && live && sub == 0 && h0 == 0 && (bad_pos || bad_slot))
    atomicOr(p.status, (bad_pos ? kDevBadPosition : 0) | (bad_slot ? kDevBadSlot : 0));
  const bool keep = slot >= 0 && !bad_slot && !bad_pos;
  long long cache_off = 0;
  if (keep) {
    if (slot <= 0xffffffffll) {                       // a 64-bit division costs as much as the rest of a head
      const unsigned s32 = (unsigned)slot, blk = s32 / (unsigned)p.block_size;
      cache_off = blk * p.c_block + (s32 - blk * p.block_size) * p.c_slot;
    } else {
      cache_off = (slot / p.block_size) * p.c_block + (slot % p.block_size) * p.c_slot;
    }
  }

  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = 1.0f; s[i] = 0.0f; }
  if (rotate && !bad_pos && h0 < p.Hq + p.Hkv) {
    const float* row = p.cos_sin + pos * D + sub * 8;
    Chunk<float> cc, sc;
    cc.template load<false>(row);
    sc.template load<false>(row + HALF);
    cc.unpack(c);
    sc.unpack(s);
  }

  Chunk<T> xa[kHeads], xb[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    xa[i].zero();
    xb[i].zero();
    if (h >= heads) continue;
    const T* src;
    if (h < p.Hq) src = reinterpret_cast<const T*>(p.q) + t * p.q_tok + h * p.q_head;
    else if (h < p.Hq + p.Hkv) src = reinterpret_cast<const T*>(p.k) + t * p.k_tok + (h - p.Hq) * p.k_head;
    else src = reinterpret_cast<const T*>(p.v) + t * p.v_tok + (h - p.Hq - p.Hkv) * p.v_head;
    if (h >= p.Hq && !keep) continue;
    // plain loads: q_out may be q itself, so the read-only path is not for these
    if constexpr (sizeof(T) == 4) {
      xa[i].a = *reinterpret_cast<const uint4*>(src + sub * 8); xa[i].b = *reinterpret_cast<const uint4*>(src + sub * 8 + 4);
      xb[i].a = *reinterpret_cast<const uint4*>(src + HALF + sub * 8); xb[i].b = *reinterpret_cast<const uint4*>(src + HALF + sub * 8 + 4);
    } else {
      xa[i].a = *reinterpret_cast<const uint4*>(src + sub * 8);
      xb[i].a = *reinterpret_cast<const uint4*>(src + HALF + sub * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
    float a[8], b[8];
    xa[i].unpack(a);
    xb[i].unpack(b);
    const void* weight = is_q ? p.q_weight : (is_v ? nullptr : p.k_weight);
    if (p.q_weight || p.k_weight) {                // uniform over the grid: every lane takes part in the shuffles
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (weight && h < heads) {
        const float r = __frsqrt_rn(ss * (1.0f / D) + p.eps);
        Chunk<T> wa, wb;
        float fa[8], fb[8];
        wa.template load<false>(reinterpret_cast<const T*>(weight) + sub * 8);
        wb.template load<false>(reinterpret_cast<const T*>(weight) + HALF + sub * 8);
        wa.unpack(fa);
        wb.unpack(fb);
#pragma unroll
        for (int j = 0; j < 8; ++j) { a[j] = a[j] * r * fa[j]; b[j] = b[j] * r * fb[j]; }
      }
    }
    if (h >= heads || (!is_q && !keep)) continue;
    if (rotate && !is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y1 = a[j], y2 = b[j];
        a[j] = y1 * c[j] - y2 * s[j];
        b[j] = y2 * c[j] + y1 * s[j];
      }
    }
    T* dst;
    if (is_q) {
      dst = reinterpret_cast<T*>(p.q_out) + t * p.o_tok + h * p.o_head;
      if (bad_pos) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.0f;
      }
    } else if (!is_v) {
      dst = reinterpret_cast<T*>(p.k_cache) + cache_off + (h - p.Hq) * p.c_head;
    } else {
      dst = reinterpret_cast<T*>(p.v_cache) + cache_off + (h - p.Hq - p.Hkv) * p.c_head;
    }
    store_chunk<T>(dst + sub * 8, a);
    store_chunk<T>(dst + HALF + sub * 8, b);
  }
}

}  // namespace b200moe
