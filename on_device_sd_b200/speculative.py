"""The end of a speculative step: drafted tokens against the target's probabilities.

The engine accepts by a threshold in a host loop over sequences (_execute_accept, demo/src/execution/cb_executor.py:261-300);
verify_draft does rejection sampling for the whole batch in one launch, with the random numbers as inputs, so that the
tokens follow the target's distribution and a run can be repeated."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._lib import load_step


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
    both), after the caller's temperature and top-k / top-p.  Errors and `status` as in attention.py; a sequence whose rows
    do not fit the tensors (fewer target rows than draft_start[b+1] + b + 1 among them, a span longer than max_draft_len)
    gets a row of -1 and 0 accepted, and shows only there and in `status`."""
    return load_step().verify_draft(draft_tokens, target_probs, draft_probs, accept_uniform, sample_uniform, draft_start, max_draft_len, status)
