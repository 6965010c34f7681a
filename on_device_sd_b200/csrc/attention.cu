// C entry points of the attention side of a decoding step: b200moe_store_kv, b200moe_paged_attention.
#include "../../include/b200moe.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "kv_store.cuh"
#include "paged_attention.cuh"

using namespace b200moe;

namespace {

constexpr int kMaxDevices = 64;

bool unaligned(const void* p) { return ((uintptr_t)p & 15u) != 0; }
size_t elem_bytes(int dtype) { return dtype == B200MOE_F32 ? 4 : 2; }
bool odd_stride(int64_t s, int dtype) { return ((size_t)s * elem_bytes(dtype)) % 16 != 0; }
bool known_head_dim(int d) { return d == 32 || d == 64 || d == 128 || d == 256; }

int current_device(const char* who, int* dev) {
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return b200moe_fail_global(B200MOE_E_CUDA, "%s: no CUDA device: %s (there is no CPU path)", who, cudaGetErrorString(e));
  if (*dev < 0 || *dev >= kMaxDevices) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: device ordinal %d not supported", who, *dev);
  return B200MOE_OK;
}

int sm_count(int dev, cudaError_t* err) {
  static std::atomic<int> known[kMaxDevices];      // two threads that ask at once store the same number
  int n = known[dev].load(std::memory_order_acquire);
  if (n) return n;
  *err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (*err == cudaSuccess) known[dev].store(n, std::memory_order_release);
  return n;
}

// Every kernel here waits for its predecessor itself (pdl_wait), so it may be launched while that one drains.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---------------------------------------------------------------------------------------------
// b200moe_store_kv
// ---------------------------------------------------------------------------------------------
template <typename T, int D> cudaError_t launch_store(const StoreKvParams& p, int dev, cudaStream_t s) {
  constexpr int L = D / 16;
  const int heads = p.Hq + 2 * p.Hkv;
  cudaError_t e = cudaSuccess;
  const int sms = sm_count(dev, &e);
  if (e != cudaSuccess) return e;
  // One head per lane group until that fills the GPU about twice (SMs x 2048 threads), four from there on.
  const bool wide = (long long)p.T * heads * L >= 2ll * sms * 2048;
  const long long groups = (long long)p.T * (wide ? (heads + 3) / 4 : heads);
  const unsigned grid = (unsigned)((groups * L + kStoreThreads - 1) / kStoreThreads);
  return wide ? launch(store_kv_kernel<T, D, 4>, grid, kStoreThreads, 0, s, p) : launch(store_kv_kernel<T, D, 1>, grid, kStoreThreads, 0, s, p);
}
template <typename T> cudaError_t dispatch_store(const StoreKvParams& p, int D, int dev, cudaStream_t s) {
  switch (D) {
    case 32: return launch_store<T, 32>(p, dev, s);
    case 64: return launch_store<T, 64>(p, dev, s);
    case 128: return launch_store<T, 128>(p, dev, s);
    default: return launch_store<T, 256>(p, dev, s);
  }
}

// ---------------------------------------------------------------------------------------------
// b200moe_paged_attention
// ---------------------------------------------------------------------------------------------
// Whether a call's units are cut along the cache over the whole grid, from what the host knows: B sequences of at most
// max_blocks * block_size slots.  Uncut, a unit belongs to one CTA, which takes about 0.9 us for a tile when it has the
// time to itself (fp32 3.2); cut, a second kernel joins the parts, and the division costs every unit kUnitCost.  us uncut /
// cut, all lengths equal, 4 kv heads of 128 with 8 queries each:
//   16-bit, one token a sequence   1 x 33 slots 5.4 / 6.5, 120 6.3 / 6.6, 250 7.9 / 6.6;  16 x 250 8.2 / 9.0, 500 11.3 / 10.0
//   16-bit, spans of 5             1 x 120 8.9 / 9.0, 250 10.9 / 9.2, 500 15.0 / 9.8;     16 x 250 11.6 / 14.6, 500 15.7 / 17.2
//   units that just fill the GPU   64 x 250 9.8 / 13.8, 500 13.4 / 17.9, 1000 26.9 / 30.2
//   fp32                           1 x 60 8.1 / 9.5, 120 11.4 / 9.3;  16 x 120 11.5 / 14.3, 500 30.8 / 23.2;  64 x 500 62 / 65
// One sequence breaks even at 2 or 3 tiles, several at 6 to 20, but lengths lie anywhere below the table's width, and of ragged
// ones the longest sets the uncut time: 4 tiles, 8 where the units just fill the GPU, are between the two.  So short spans
// of one sequence pay up to 2 us (250 slots), and equal lengths past 8 tiles, or in fp32 past one, up to 3 or 4.
constexpr int kUncutTiles = 4, kUncutTilesFull = 8, kUncutTilesF32 = 1;
// What beginning a unit costs a CTA, in tiles of 64 keys, for the equal division of the work.  (32 spans over 100..2500
// tokens: 55 us at 0, 48 at 1, 44 at 2, 43 at 3; equal lengths do not care.)
constexpr int kUnitCost = 3;

struct AttnPlan {
  int64_t ws_bytes = 0;            // 0: units are not cut
};

// MINB CTAs fit an SM: they are what the grid holds, so that all parts of a call run at once.
template <typename T, int D, int MT, int RG, int KG, int STAGES, int MINB, int REGB = MINB> struct AttnVariant {
  using S = AttnShape<T, D, MT, RG, KG, STAGES>;
  static_assert(MINB * (S::SMEM + 1024) <= 228 * 1024, "shared memory of an SM");

  template <bool PAGE16> static cudaError_t start(const AttnParams& p, unsigned grid, int dev, cudaStream_t s) {
    static std::atomic<bool> ready[kMaxDevices];
    auto k = attn_kernel<T, D, MT, RG, KG, STAGES, REGB, PAGE16>;
    if (!ready[dev].load(std::memory_order_acquire)) {
      cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
      if (e != cudaSuccess) return e;
      ready[dev].store(true, std::memory_order_release);
    }
    return launch(k, grid, S::THREADS, S::SMEM, s, p);
  }
  static cudaError_t run(AttnParams* p, int dev, AttnPlan* plan, cudaStream_t s, bool plan_only) {
    cudaError_t e = cudaSuccess;
    const int sms = sm_count(dev, &e), full = MINB * sms;
    if (e != cudaSuccess) return e;
    // as far as comparisons need them
    const long long row_tiles = std::min(((long long)p->span * p->group + S::R - 1) / S::R, 1ll << 20);
    const long long units = (long long)std::min(p->B, 1 << 24) * p->Hkv * row_tiles;
    const long long tiles = ((long long)p->max_blocks * p->block_size + S::TILE - 1) / S::TILE;
    const bool cut = full <= kJoinMaxGrid && tiles > (sizeof(T) == 4 ? kUncutTilesF32 : units * 2 >= full && units <= full ? kUncutTilesFull : kUncutTiles);
    plan->ws_bytes = cut ? attn_ws_floats(full, S::R, D) * 4 : 0;
    if (plan_only) return cudaSuccess;
    p->split = cut && p->ws != nullptr;
    p->grid = full;
    p->tile_shift = S::TILE == 64 ? 6 : 5;
    static_assert(S::TILE == 64 || S::TILE == 32, "tile");
    p->unit_cost = kUnitCost;
    const unsigned grid = (unsigned)(!p->split && units < full ? units : full);
    // division by the page size as a multiplication, exact for keys below 2^31: page_mul = floor(2^(31+s) / d) + 1, 2^s >= d
    int sh = 0;
    while ((1ll << sh) < p->block_size) ++sh;
    p->page_shift = 31 + sh;
    p->page_mul = (unsigned)((1ull << (31 + sh)) / (unsigned)p->block_size + 1);
    const long long rows = (long long)p->T * p->Hq;
    p->cuts = p->split && rows > 8 * sms;
    e = p->block_size % 16 == 0 ? start<true>(*p, grid, dev, s) : start<false>(*p, grid, dev, s);
    if (e != cudaSuccess || !p->split) return e;
    // Few rows are cut into many parts each: up to eight warps per row, in up to two CTAs of eight on every SM.
    if (rows <= 2 * sms) return launch(attn_join_kernel<T, D, 8>, (unsigned)rows, 256, 0, s, *p, S::R_SHIFT);
    if (rows <= 4 * sms) return launch(attn_join_kernel<T, D, 4>, (unsigned)((rows + 1) / 2), 256, 0, s, *p, S::R_SHIFT);
    if (!p->cuts) return launch(attn_join_kernel<T, D, 2>, (unsigned)((rows + 3) / 4), 256, 0, s, *p, S::R_SHIFT);
    // no more rows are cut than there are, or than the CTAs can begin units of
    return launch(attn_join_cuts_kernel<T, D>, (unsigned)((std::min(rows, (long long)(full - 1) * S::R) + 7) / 8), kJoinThreads, 0, s, *p, S::R_SHIFT);
  }
};

// Rows that share a kv head's keys: tokens of the span x query heads of the group, in tiles of 16 or 32.  More than 32
// read the cache once per tile, the further times from L2: a tile of 64 rows would leave one CTA of 8 warps on an SM and
// was slower (64 spans of 1..5 tokens, 8 heads a group, over ~8000: 343 us against 229; 64 rows everywhere: equal).
// Heads of 256 need two warps' registers for 32 rows (32 spans of 4 over 10000: 77 us, with tiles of 16 rows 105).
template <typename T> cudaError_t dispatch_attn(AttnParams* p, int D, int dev, AttnPlan* plan, cudaStream_t s, bool po) {
  const long long rows = (long long)p->span * p->group;
  if constexpr (sizeof(T) == 4) {
    switch (D) {
      case 32: return AttnVariant<T, 32, 1, 1, 4, 4, 2>::run(p, dev, plan, s, po);
      case 64: return AttnVariant<T, 64, 1, 1, 4, 3, 2>::run(p, dev, plan, s, po);
      case 128: return AttnVariant<T, 128, 1, 1, 4, 3, 1>::run(p, dev, plan, s, po);
      default: return AttnVariant<T, 256, 1, 1, 2, 3, 1>::run(p, dev, plan, s, po);
    }
  } else {
    switch (D) {
      case 32:
        if (rows <= 16) return AttnVariant<T, 32, 1, 1, 4, 6, 4>::run(p, dev, plan, s, po);
        return AttnVariant<T, 32, 2, 1, 4, 6, 3>::run(p, dev, plan, s, po);
      case 64:
        if (rows <= 16) return AttnVariant<T, 64, 1, 1, 4, 4, 3>::run(p, dev, plan, s, po);
        return AttnVariant<T, 64, 2, 1, 4, 4, 3>::run(p, dev, plan, s, po);
      case 128:
        if (rows <= 16) return AttnVariant<T, 128, 1, 1, 4, 3, 2, 3>::run(p, dev, plan, s, po);
        return AttnVariant<T, 128, 2, 1, 4, 3, 2>::run(p, dev, plan, s, po);
      default:
        if (rows <= 16) return AttnVariant<T, 256, 1, 1, 4, 3, 1>::run(p, dev, plan, s, po);
        return AttnVariant<T, 256, 1, 2, 4, 3, 1>::run(p, dev, plan, s, po);
    }
  }
}

int run_attn(AttnParams* p, int dtype, int D, int dev, AttnPlan* plan, cudaStream_t s, bool plan_only, const char* who) {
  cudaError_t e;
  switch (dtype) {
    case B200MOE_F32: e = dispatch_attn<float>(p, D, dev, plan, s, plan_only); break;
    case B200MOE_F16: e = dispatch_attn<__half>(p, D, dev, plan, s, plan_only); break;
    default: e = dispatch_attn<__nv_bfloat16>(p, D, dev, plan, s, plan_only); break;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return b200moe_fail_global(B200MOE_E_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  }
  return B200MOE_OK;
}

int check_heads(const char* who, int dtype, int Hq, int Hkv, int D) {
  if (dtype < B200MOE_F32 || dtype > B200MOE_BF16) return b200moe_fail_global(B200MOE_E_ARG, "%s: unknown dtype %d", who, dtype);
  if (!known_head_dim(D)) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: head_dim %d (32, 64, 128 or 256)", who, D);
  if (Hq <= 0 || Hkv <= 0 || Hq > 65536 || Hkv > 65536) return b200moe_fail_global(B200MOE_E_ARG, "%s: head counts must be in 1..65536", who);
  if (Hq % Hkv) return b200moe_fail_global(B200MOE_E_ARG, "%s: %d query heads are not a multiple of %d key-value heads", who, Hq, Hkv);
  return B200MOE_OK;
}

}  // namespace

extern "C" int b200moe_store_kv(const b200moe_store_kv_args* a, void* stream) {
  const char* who = "b200moe_store_kv";
  if (!a) return b200moe_fail_global(B200MOE_E_ARG, "%s: null arguments", who);
  const bool has_q = a->query != nullptr;
  const int dt = a->dtype;
  if (int rc = check_heads(who, dt, has_q ? a->num_heads : a->num_kv_heads, a->num_kv_heads, a->head_dim)) return rc;
  if (a->num_tokens < 0 || a->num_blocks < 0 || a->block_size <= 0) return b200moe_fail_global(B200MOE_E_ARG, "%s: negative size", who);
  if (a->num_tokens == 0) return B200MOE_OK;
  if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->slots) return b200moe_fail_global(B200MOE_E_ARG, "%s: null pointer", who);
  if (has_q && !a->query_out) return b200moe_fail_global(B200MOE_E_ARG, "%s: query given without query_out", who);
  if (a->cos_sin && (!a->positions || a->max_position <= 0)) return b200moe_fail_global(B200MOE_E_ARG, "%s: an angle table needs positions and its length", who);
  const void* ptrs[] = {a->query, a->key, a->value, a->query_out, a->k_cache, a->v_cache, a->cos_sin, a->q_norm_weight, a->k_norm_weight};
  for (const void* p : ptrs)
    if (unaligned(p)) return b200moe_fail_global(B200MOE_E_ARG, "%s: data pointers must be 16-byte aligned", who);
  const int64_t strides[] = {a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride,
                             a->o_token_stride, a->o_head_stride, a->cache_block_stride, a->cache_slot_stride, a->cache_head_stride};
  for (int64_t s : strides)
    if (odd_stride(s, dt)) return b200moe_fail_global(B200MOE_E_ARG, "%s: strides must be multiples of 16 bytes", who);
  // heads are numbered in 32 bits, up to the end of the last CTA
  if ((int64_t)a->num_tokens * ((has_q ? a->num_heads : 0) + 2ll * a->num_kv_heads) > (1ll << 31))
    return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: more than 2^31 tokens x heads", who);
  int dev;
  if (int rc = current_device(who, &dev)) return rc;
  StoreKvParams p = {};
  p.q = a->query; p.k = a->key; p.v = a->value; p.q_out = a->query_out; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.positions = a->positions; p.slots = a->slots; p.cos_sin = a->cos_sin; p.q_weight = has_q ? a->q_norm_weight : nullptr; p.k_weight = a->k_norm_weight;
  p.status = a->status;
  p.q_tok = a->q_token_stride; p.q_head = a->q_head_stride; p.k_tok = a->k_token_stride; p.k_head = a->k_head_stride;
  p.v_tok = a->v_token_stride; p.v_head = a->v_head_stride; p.o_tok = a->o_token_stride; p.o_head = a->o_head_stride;
  p.c_block = a->cache_block_stride; p.c_slot = a->cache_slot_stride; p.c_head = a->cache_head_stride;
  p.num_slots = (long long)a->num_blocks * a->block_size;
  p.T = a->num_tokens; p.Hq = has_q ? a->num_heads : 0; p.Hkv = a->num_kv_heads; p.block_size = a->block_size; p.max_position = a->max_position;
  p.positions64 = a->positions_are_int64; p.slots64 = a->slots_are_int64; p.eps = a->eps;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  switch (dt) {
    case B200MOE_F32: e = dispatch_store<float>(p, a->head_dim, dev, s); break;
    case B200MOE_F16: e = dispatch_store<__half>(p, a->head_dim, dev, s); break;
    default: e = dispatch_store<__nv_bfloat16>(p, a->head_dim, dev, s); break;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return b200moe_fail_global(B200MOE_E_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  }
  return B200MOE_OK;
}

extern "C" int b200moe_paged_attention_workspace(int dtype, int num_seqs, int num_heads, int num_kv_heads, int head_dim, int max_query_len,
                                                 int max_blocks_per_seq, int block_size, int64_t* bytes_out) {
  const char* who = "b200moe_paged_attention_workspace";
  if (!bytes_out) return b200moe_fail_global(B200MOE_E_ARG, "%s: null pointer", who);
  if (int rc = check_heads(who, dtype, num_heads, num_kv_heads, head_dim)) return rc;
  if (num_seqs < 0 || max_query_len < 0 || max_blocks_per_seq < 0 || block_size <= 0) return b200moe_fail_global(B200MOE_E_ARG, "%s: negative size", who);
  *bytes_out = 0;
  int dev;
  if (int rc = current_device(who, &dev)) return rc;
  AttnParams p = {};
  p.B = num_seqs; p.Hkv = num_kv_heads; p.group = num_heads / num_kv_heads; p.span = max_query_len > 0 ? max_query_len : 1;
  p.max_blocks = max_blocks_per_seq; p.block_size = block_size;
  AttnPlan plan;
  if (int rc = run_attn(&p, dtype, head_dim, dev, &plan, nullptr, true, who)) return rc;
  *bytes_out = plan.ws_bytes;
  return B200MOE_OK;
}

extern "C" int b200moe_paged_attention(const b200moe_paged_attention_args* a, void* stream) {
  const char* who = "b200moe_paged_attention";
  if (!a) return b200moe_fail_global(B200MOE_E_ARG, "%s: null arguments", who);
  const int dt = a->dtype;
  if (int rc = check_heads(who, dt, a->num_heads, a->num_kv_heads, a->head_dim)) return rc;
  if (a->num_tokens < 0 || a->num_seqs < 0 || a->num_blocks < 0 || a->block_size <= 0 || a->max_blocks_per_seq < 0 || a->max_query_len < 0)
    return b200moe_fail_global(B200MOE_E_ARG, "%s: negative size", who);
  if (!a->query_start && a->num_tokens != a->num_seqs)
    return b200moe_fail_global(B200MOE_E_ARG, "%s: without query_start there is one token per sequence (%d tokens, %d sequences)", who, a->num_tokens, a->num_seqs);
  if (a->num_tokens == 0 || a->num_seqs == 0) return B200MOE_OK;
  const bool has_cache = a->num_blocks > 0 && a->max_blocks_per_seq > 0;
  if (!a->query || !a->out || !a->context_lens || (has_cache && (!a->k_cache || !a->v_cache || !a->block_tables)))
    return b200moe_fail_global(B200MOE_E_ARG, "%s: null pointer", who);
  if (unaligned(a->query) || unaligned(a->out) || unaligned(a->k_cache) || unaligned(a->v_cache) || unaligned(a->workspace))
    return b200moe_fail_global(B200MOE_E_ARG, "%s: data pointers must be 16-byte aligned", who);
  const int64_t strides[] = {a->q_token_stride, a->q_head_stride, a->o_token_stride, a->o_head_stride, a->cache_block_stride, a->cache_slot_stride,
                             a->cache_head_stride};
  for (int64_t s : strides)
    if (odd_stride(s, dt)) return b200moe_fail_global(B200MOE_E_ARG, "%s: strides must be multiples of 16 bytes", who);
  if (!(a->scale > 0.0f) || a->scale > 1.0e30f) return b200moe_fail_global(B200MOE_E_ARG, "%s: scale must be positive and at most 1e30", who);
  const int64_t max_context = (int64_t)a->max_blocks_per_seq * a->block_size;
  if (max_context > (1ll << 30)) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: block tables span more than 2^30 slots", who);
  // the join's grid and the row numbers are 32-bit
  if ((int64_t)a->num_tokens * a->num_heads > (1ll << 30)) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: more than 2^30 tokens x heads", who);
  // work items are tiles of at least 32 keys x 16 rows, numbered in 64 bits and multiplied by the grid (at most 2^10)
  const double rows16 = (double)a->num_tokens * (a->num_heads / a->num_kv_heads) / 16 + std::min(a->num_tokens, a->num_seqs);
  if (rows16 * a->num_kv_heads * ((double)max_context / 32 + 1 + kUnitCost) > 4503599627370496.0)
    return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: more than 2^52 tiles of work", who);
  int dev;
  if (int rc = current_device(who, &dev)) return rc;
  AttnParams p = {};
  p.q = a->query; p.k = a->k_cache; p.v = a->v_cache; p.out = a->out; p.lse = a->lse_out;
  p.tables = a->block_tables; p.context = a->context_lens; p.qstart = a->query_start; p.status = a->status; p.ws = (float*)a->workspace;
  p.q_tok = a->q_token_stride; p.q_head = a->q_head_stride; p.o_tok = a->o_token_stride; p.o_head = a->o_head_stride;
  p.c_block = a->cache_block_stride; p.c_slot = a->cache_slot_stride; p.c_head = a->cache_head_stride; p.table_stride = a->block_table_stride;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.B = a->num_seqs; p.T = a->num_tokens; p.Hq = a->num_heads; p.Hkv = a->num_kv_heads; p.group = a->num_heads / a->num_kv_heads;
  p.block_size = a->block_size; p.num_blocks = a->num_blocks; p.max_blocks = has_cache ? a->max_blocks_per_seq : 0;
  p.span = a->query_start && a->max_query_len > 0 ? a->max_query_len : 1;
  AttnPlan plan;
  if (p.ws) {
    if (int rc = run_attn(&p, dt, a->head_dim, dev, &plan, nullptr, true, who)) return rc;
    if (a->workspace_bytes < plan.ws_bytes)
      return b200moe_fail_global(B200MOE_E_ARG, "%s: workspace of %lld bytes, %lld are needed (b200moe_paged_attention_workspace)", who,
                                 (long long)a->workspace_bytes, (long long)plan.ws_bytes);
  }
  return run_attn(&p, dt, a->head_dim, dev, &plan, (cudaStream_t)stream, false, who);
}
