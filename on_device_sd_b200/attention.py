"""The attention side of a decoding step over a paged key-value cache: the cache write (with head norms and rotary
embedding in the same launch) and the attention of new tokens, single ones (draft step) or spans (verify step).

The cache tensors are the reference's, [num_blocks, block_size, kv_heads, head_dim] (demo/src/memory/paged_kv_cache.py:228),
and stay the caller's.  All calls run on the current stream of their tensors' device, never synchronise and can be
captured into CUDA graphs; there are no gradients.  `status`, where given, is an int32 tensor of one element on the
same device that the kernels OR DEV_* bits into (include/b200moe.h); the caller zeroes and reads it.  Arguments are
checked in csrc/bindings.cpp: ValueError / TypeError for tensors that do not fit together, B200MoEError for what the
library refuses."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._lib import load_step


def rotary_table(head_dim: int, max_position: int, base: float = 1e6, device: Optional[torch.device] = None) -> torch.Tensor:
    """The fp32 angle table [max_position, head_dim] that rope_store_kvcache takes: cos of the position's head_dim/2 angles,
    then sin.  Angles are formed in fp64, where a far position times a frequency still has all its digits."""
    inv = base ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=-1).float().to(device or "cpu")


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                  status: Optional[torch.Tensor] = None) -> None:
    """key, value [T, kv_heads, D] -> rows slot_mapping[t] of the caches; slot -1 stores nothing (the reference's function of
    this name, demo/src/layers/attention.py:56-79).  The slots of one call are distinct, k_cache and v_cache share no memory,
    and key and value are not rows that the call writes."""
    load_step().store_kv(None, key, value, None, None, k_cache, v_cache, slot_mapping, None, None, 0.0, None, status)


def rope_store_kvcache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *, q_norm_weight: Optional[torch.Tensor] = None,
                       k_norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, out: Optional[torch.Tensor] = None,
                       status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What the reference's attention layer does between the projection and the attention, in one launch: per-head RMS norm
    of queries and keys (where weights are given), rotary embedding at `positions`, keys and values into the cache.

    query [T, heads, D], key and value [T, kv_heads, D] may be views of one projection row; positions and slot_mapping are
    int64 or int32 [T]; cos_sin is rotary_table's.  Returns the rotated queries [T, heads, D] (`out` when given, which may
    be `query` itself and otherwise shares no memory with the other tensors).  fp32 inside, each output rounded once."""
    if query is None or cos_sin is None or positions is None:
        raise ValueError("rope_store_kvcache needs query, positions and cos_sin (store_kvcache stores keys and values alone)")
    return load_step().store_kv(query, key, value, positions, cos_sin, k_cache, v_cache, slot_mapping, q_norm_weight, k_norm_weight, eps, out, status)


def paged_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                    query_start: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of new tokens over their sequences' cached keys and values (theirs included), causal within a span.

    query [T, heads, D]; block_tables int32 [B, max_blocks]; context_lens int32 [B].  Without query_start there is one token
    per sequence (T == B, the draft step); with it (int32 [B+1]) sequence b owns rows query_start[b]:query_start[b+1] and
    its last row sees all context_lens[b] keys (the verify step).  max_query_len, the longest span, picks the row tile; any
    value gives right results.  scale defaults to D ** -0.5.

    Scores, softmax and sums are fp32.  With 16-bit tensors each probability is rounded to their type before its product with
    the value (half a step: 2^-8 of the weighted mean of |v| in bf16, 2^-11 in fp16), and the output once more.

    Returns out [T, heads, D] (with return_lse also the fp32 log-sum-exp [T, heads]).  A row that sees no key gives zeros
    and -inf; rows behind query_start[B] are not written (nor initialised unless `out` was given).  `out` may be
    `query` itself; otherwise it shares no memory with it or the caches."""
    return load_step().paged_attention(query, k_cache, v_cache, block_tables, context_lens, query_start, max_query_len, scale, out, return_lse, status)
