"""The end of a speculative step: drafted tokens against the target's probabilities.

The engine accepts by a threshold in a host loop over sequences (_execute_accept, demo/src/execution/cb_executor.py:261-300);
verify_draft does rejection sampling for the whole batch in one launch, with the random numbers as inputs, so that the
tokens follow the target's distribution and a run can be repeated."""
from __future__ import annotations

from ctypes import byref
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import VerifyDraftArgs, check
from .attention import _need, _on, _status_ptr
from .context import _stream, dtype_tag


def verify_draft(draft_tokens: torch.Tensor, target_probs: torch.Tensor, draft_probs: Optional[torch.Tensor], accept_uniform: torch.Tensor,
                 sample_uniform: torch.Tensor, *, draft_start: torch.Tensor, max_draft_len: int,
                 status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (tokens int64 [B, max_draft_len + 1], accepted int32 [B]).

    Sequence b drafted draft_tokens[draft_start[b]:draft_start[b+1]] (int64; draft_start int32 [B+1]); target_probs holds one
    row more per sequence (rows draft_start[b] + b on): the distribution of every drafted position and of the one behind
    them.  Position j's draft x is accepted while p_j(x) > accept_uniform[j] * q_j(x).  At the first refusal the next token is
    drawn from max(p_j - q_j, 0), after a fully accepted span from the last row, both by inverse cumulative sum at
    sample_uniform[b].  draft_probs None means greedy drafts: q is 1 on the drafted token.  Rows of `tokens` hold the accepted
    tokens, the drawn one, then -1.  Both uniforms are float32; probabilities float32, float16 or bfloat16 (one type for
    both), after the caller's temperature and top-k / top-p."""
    dev, dt = target_probs.device, target_probs.dtype
    tag = dtype_tag(dt)
    _need(target_probs, "target_probs", dev, dt, 2)
    rows, vocab = target_probs.shape
    _need(draft_tokens, "draft_tokens", dev, torch.int64, 1)
    n = draft_tokens.shape[0]
    _need(accept_uniform, "accept_uniform", dev, torch.float32, 1)
    _need(sample_uniform, "sample_uniform", dev, torch.float32, 1)
    _need(draft_start, "draft_start", dev, torch.int32, 1)
    B = sample_uniform.shape[0]
    if max_draft_len < 0:
        raise ValueError("max_draft_len must not be negative")
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    if accept_uniform.shape[0] != n or draft_start.shape[0] != B + 1:
        raise ValueError(f"accept_uniform must be [{n}] and draft_start [{B + 1}]")
    for name, t in (("draft_tokens", draft_tokens), ("accept_uniform", accept_uniform), ("sample_uniform", sample_uniform), ("draft_start", draft_start)):
        if t.shape[0] > 1 and t.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")
    if target_probs.stride(1) != 1 and vocab > 1:
        raise ValueError("the rows of target_probs must be contiguous")
    draft_ptr, draft_stride = None, 0
    if draft_probs is not None:
        _need(draft_probs, "draft_probs", dev, dt, 2)
        if draft_probs.shape != (n, vocab) or (draft_probs.stride(1) != 1 and vocab > 1):
            raise ValueError(f"draft_probs must be [{n}, {vocab}] with contiguous rows, got {tuple(draft_probs.shape)}")
        draft_stride = draft_probs.stride(0)
        # without drafts there is no row to point at, but the rule is the sampled one all the same
        draft_ptr = draft_probs.data_ptr() or target_probs.data_ptr()
    tokens = torch.empty(B, max_draft_len + 1, dtype=torch.int64, device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    args = VerifyDraftArgs(draft_tokens.data_ptr(), target_probs.data_ptr(), draft_ptr, accept_uniform.data_ptr(), sample_uniform.data_ptr(),
                           draft_start.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), _status_ptr(status, dev), target_probs.stride(0), draft_stride,
                           B, vocab, max_draft_len, n, rows, tag)
    with _on(dev):
        check(None, _lib.load().b200moe_verify_draft(byref(args), _stream(dev)))
    return tokens, accepted
