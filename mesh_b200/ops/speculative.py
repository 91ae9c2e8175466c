"""Verification of drafted tokens against the target model's probabilities."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

VERIFY_MAX_DRAFTS = 31  # drafts a session, as in the kernel


def verify_drafts(logits: torch.Tensor, draft_ids: torch.Tensor, uniforms: torch.Tensor,
                  inv_t: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None,
                  draft_lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accept or replace the tokens each session proposed ahead, so that what comes out is distributed as the
    target alone would give it.

    logits [B, K+1, V] fp32 or bf16: row k is the target's after k drafts (over the whole vocabulary);
    draft_ids [B, K] int32; uniforms [B, K+1] fp32 in [0, 1): one per draft, and the last for the token drawn;
    inv_t [B] fp32, 1/T per session, 0 = greedy (default: 1); draft_probs [B, K, V] fp32 or bf16, what the drafts
    were drawn from (default: guesses, of probability 1); draft_lens [B] int32, drafts of each session (default: K).

    Draft k is accepted while ``u_k q_k(x_k) < p_k(x_k)``; the token after the accepted ones is drawn from
    max(p - q, 0) of the first refused row (from p there if nothing is left, and after the last draft), as the
    first index whose running mass exceeds ``u_K`` of the whole. Greedy sessions compare with the row's first
    maximum. NaN logits and draft probabilities count as none; a draft outside the vocabulary is refused; a row
    with nothing to choose draws -1.

    Returns (tokens [B, K+1] int32: accepted drafts, the new token, then -1; accepted [B] int32; probs [B, K] fp32:
    the target's probability of each draft, 0 past a session's drafts)."""
    from . import _count, ext
    if logits.dim() != 3 or logits.shape[1] < 1:
        raise ValueError(f"logits [B, K+1, V] expected, got {tuple(logits.shape)}")
    out = ext().verify_drafts(logits, draft_ids, uniforms, inv_t, draft_probs, draft_lens)
    _count(2)
    return out
