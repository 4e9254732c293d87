"""Verification of drafted tokens (speculative decoding), C ABI ``qi4_verify_draft``."""

from __future__ import annotations

import torch

from .paged import _ops


def b200_verify_draft(draft_tokens, target_probs, uniforms, *, draft_probs=None,
                      draft_counts=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens [B, K + 1] int64, accepted [B] int32) for K drafted tokens per sequence.

    draft_tokens [B, K] int64; target_probs [B, K + 1, V] and draft_probs
    [B, K, V] (FP32, BF16 or FP16): position i's distributions, given the
    drafts before it; draft_probs None: drafts without a distribution (taken
    as certain); uniforms [B, K + 1] FP32 in [0, 1); draft_counts [B] int32:
    drafts of each sequence (None: K).

    Draft i stands while ``uniforms[b, i] * q_i(t_i) < p_i(t_i)`` and all
    before it stand. A row of ``tokens`` is the standing drafts, the token
    drawn after them at ``uniforms[b, K]`` (from max(p - q, 0) where
    a draft was refused, from p where none was: the tokens are then
    distributed as the target's own), and -1. The draw sums the weights as
    whole numbers of 2^-40, so equal inputs give equal tokens in any order of
    the sum; a draw from nothing is -1.
    """
    return _ops().verify_draft(draft_tokens, target_probs, uniforms, draft_probs, draft_counts)
