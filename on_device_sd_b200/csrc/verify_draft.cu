// C entry point b200moe_verify_draft.
#include "../../include/b200moe.h"

#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "verify_draft.cuh"

using namespace b200moe;

namespace {

constexpr int kMaxDevices = 64;

// How many clusters of the given size run at once, as the device says (its groups of SMs are not filled to the end: 71 of
// eight CTAs on a B200 whose SMs would hold 74).  Asked once per kernel, device and size.
int clusters_at_once(const void* kernel, std::atomic<int>* known, cudaLaunchConfig_t cfg) {
  int n = known->load(std::memory_order_acquire);
  if (n > 0) return n;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  known->store(n, std::memory_order_release);
  return n;
}

template <typename T> cudaError_t launch_verify(const VerifyParams& p, int dev, cudaStream_t s) {
  // rows that all start on a 16-byte boundary are read as vectors, others element by element
  const bool vec = (p.V * sizeof(T)) % 16 == 0 && (p.target_stride * sizeof(T)) % 16 == 0 && ((uintptr_t)p.target & 15u) == 0 &&
                   (!p.draft || ((p.draft_stride * sizeof(T)) % 16 == 0 && ((uintptr_t)p.draft & 15u) == 0));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  // As many CTAs per sequence, up to eight, as let all sequences run at once: clusters that have to wait for others cost more
  // than wider ones gain.  Of eight, the last sixteenth waits all the same where launches follow each other.  32000 tokens,
  // bf16, us: 66 sequences with 8 CTAs 7.2, 70 9.1, 74 9.8; 70 with 4 6.7, 140 7.4, 146 10.3; 146 with 2 7.6, 296 9.2; 297
  // with 1 12.1.
  static std::atomic<int> known[kMaxDevices][2][4];
  const void* kernel = vec ? (const void*)verify_draft_kernel<T, true> : (const void*)verify_draft_kernel<T, false>;
  unsigned cluster = kVerifyMaxCluster;
  for (int i = 0; cluster > 1; ++i, cluster /= 2) {
    attr[1].val.clusterDim.x = cluster;
    cfg.gridDim = dim3(cluster);
    const int room = clusters_at_once(kernel, &known[dev][vec][i], cfg);
    if (p.B <= room - (i == 0 ? (room + 15) / 16 : 0)) break;
  }
  attr[1].val.clusterDim.x = cluster;
  cfg.gridDim = dim3((unsigned)p.B * cluster);
  return vec ? cudaLaunchKernelEx(&cfg, verify_draft_kernel<T, true>, p) : cudaLaunchKernelEx(&cfg, verify_draft_kernel<T, false>, p);
}

}  // namespace

extern "C" int b200moe_verify_draft(const b200moe_verify_draft_args* a, void* stream) {
  const char* who = "b200moe_verify_draft";
  if (!a) return b200moe_fail_global(B200MOE_E_ARG, "%s: null arguments", who);
  if (a->dtype < B200MOE_F32 || a->dtype > B200MOE_BF16) return b200moe_fail_global(B200MOE_E_ARG, "%s: unknown dtype %d", who, a->dtype);
  if (a->num_seqs < 0 || a->vocab_size <= 0 || a->max_draft_len < 0 || a->num_draft_tokens < 0 || a->num_target_rows < 0)
    return b200moe_fail_global(B200MOE_E_ARG, "%s: negative size or empty vocabulary", who);
  // indices of a row, and the step past its end, are 32-bit
  if (a->vocab_size > (1 << 30)) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: vocabulary of more than 2^30", who);
  if (a->num_seqs > (1 << 24) || a->max_draft_len > (1 << 24)) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: more than 2^24 sequences or drafts", who);
  if (a->num_seqs == 0) return B200MOE_OK;
  if (!a->target_probs || !a->sample_uniform || !a->draft_start || !a->tokens_out || !a->accepted_out ||
      (a->num_draft_tokens > 0 && (!a->draft_tokens || !a->accept_uniform)))
    return b200moe_fail_global(B200MOE_E_ARG, "%s: null pointer", who);
  int dev;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return b200moe_fail_global(B200MOE_E_CUDA, "%s: no CUDA device: %s (there is no CPU path)", who, cudaGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) return b200moe_fail_global(B200MOE_E_UNSUPPORTED, "%s: device ordinal %d not supported", who, dev);
  VerifyParams p = {};
  p.tokens = (const long long*)a->draft_tokens; p.target = a->target_probs; p.draft = a->draft_probs;
  p.accept = a->accept_uniform; p.sample = a->sample_uniform; p.start = a->draft_start;
  p.out = (long long*)a->tokens_out; p.count = a->accepted_out; p.status = a->status;
  p.target_stride = a->target_stride; p.draft_stride = a->draft_stride;
  p.B = a->num_seqs; p.V = a->vocab_size; p.max_draft = a->max_draft_len; p.num_draft = a->num_draft_tokens; p.target_rows = a->num_target_rows;
  cudaStream_t s = (cudaStream_t)stream;
  switch (a->dtype) {
    case B200MOE_F32: e = launch_verify<float>(p, dev, s); break;
    case B200MOE_F16: e = launch_verify<__half>(p, dev, s); break;
    default: e = launch_verify<__nv_bfloat16>(p, dev, s); break;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return b200moe_fail_global(B200MOE_E_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  }
  return B200MOE_OK;
}
