// C entry point b200moe_verify_draft.
#include "../../include/b200moe.h"

#include <cuda_runtime.h>

#include "common.cuh"
#include "internal.h"
#include "verify_draft.cuh"

using namespace b200moe;

namespace {

template <typename T> cudaError_t launch_verify(const VerifyParams& p, cudaStream_t s) {
  // rows that all start on a 16-byte boundary are read as vectors, others element by element
  const bool vec = (p.V * sizeof(T)) % 16 == 0 && (p.target_stride * sizeof(T)) % 16 == 0 && ((uintptr_t)p.target & 15u) == 0 &&
                   (!p.draft || ((p.draft_stride * sizeof(T)) % 16 == 0 && ((uintptr_t)p.draft & 15u) == 0));
  cudaLaunchConfig_t cfg = {};
  // eight CTAs per sequence until four on every SM (what the registers allow) are taken, fewer for larger batches
  unsigned cluster = kVerifyMaxCluster;
  while (cluster > 1 && (long long)p.B * cluster > kVerifyCtasPerSm * 148) cluster /= 2;
  cfg.gridDim = dim3((unsigned)p.B * cluster);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
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
  VerifyParams p = {};
  p.tokens = (const long long*)a->draft_tokens; p.target = a->target_probs; p.draft = a->draft_probs;
  p.accept = a->accept_uniform; p.sample = a->sample_uniform; p.start = a->draft_start;
  p.out = (long long*)a->tokens_out; p.count = a->accepted_out; p.status = a->status;
  p.target_stride = a->target_stride; p.draft_stride = a->draft_stride;
  p.B = a->num_seqs; p.V = a->vocab_size; p.max_draft = a->max_draft_len; p.num_draft = a->num_draft_tokens; p.target_rows = a->num_target_rows;
  cudaStream_t s = (cudaStream_t)stream;
  switch (a->dtype) {
    case B200MOE_F32: e = launch_verify<float>(p, s); break;
    case B200MOE_F16: e = launch_verify<__half>(p, s); break;
    default: e = launch_verify<__nv_bfloat16>(p, s); break;
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return b200moe_fail_global(B200MOE_E_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  }
  return B200MOE_OK;
}
