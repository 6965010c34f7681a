"""The end of a speculative step: drafted tokens against the target's probabilities.

The engine accepts by a threshold in a host loop over sequences (_execute_accept, demo/src/execution/cb_executor.py:261-300);
verify_draft does rejection sampling for the whole batch in one launch, with the random numbers as inputs, so that the
tokens follow the target's distribution and a run can be repeated."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import VerifyDraftArgs
from .attention import _call, _need, _status_ptr, _tag


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
    tag, dev, dt = _tag(target_probs, "target_probs"), target_probs.device, target_probs.dtype
    (rows, vocab), ts = _need(target_probs, "target_probs", dev, dt, 2), target_probs.stride()
    n, = _need(draft_tokens, "draft_tokens", dev, torch.int64, 1)
    B, = _need(sample_uniform, "sample_uniform", dev, torch.float32, 1)
    if max_draft_len < 0:
        raise ValueError("max_draft_len must not be negative")
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    if _need(accept_uniform, "accept_uniform", dev, torch.float32, 1)[0] != n or _need(draft_start, "draft_start", dev, torch.int32, 1)[0] != B + 1:
        raise ValueError(f"accept_uniform must be [{n}] and draft_start [{B + 1}]")
    if not (draft_tokens.is_contiguous() and accept_uniform.is_contiguous() and sample_uniform.is_contiguous() and draft_start.is_contiguous()):
        raise ValueError("draft_tokens, accept_uniform, sample_uniform and draft_start must be contiguous")
    if ts[1] != 1 and vocab > 1:
        raise ValueError("the rows of target_probs must be contiguous")
    draft_ptr, draft_stride = None, 0
    if draft_probs is not None:
        ds = draft_probs.stride()
        if _need(draft_probs, "draft_probs", dev, dt, 2) != (n, vocab) or (ds[1] != 1 and vocab > 1):
            raise ValueError(f"draft_probs must be [{n}, {vocab}] with contiguous rows, got {tuple(draft_probs.shape)}")
        # without drafts there is no row to point at, but the rule is the sampled one all the same
        draft_ptr, draft_stride = draft_probs.data_ptr() or target_probs.data_ptr(), ds[0]
    tokens = torch.empty(B, max_draft_len + 1, dtype=torch.int64, device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    _call(_lib.load().b200moe_verify_draft,
          VerifyDraftArgs(draft_tokens.data_ptr(), target_probs.data_ptr(), draft_ptr, accept_uniform.data_ptr(), sample_uniform.data_ptr(),
                          draft_start.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), None if status is None else _status_ptr(status, dev), ts[0],
                          draft_stride, B, vocab, max_draft_len, n, rows, tag), dev)
    return tokens, accepted
