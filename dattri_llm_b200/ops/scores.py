"""Scores of tokens from logits: log-probabilities, entropies, best alternatives."""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from dattri_llm_b200.ops import error_word, native, use_native
from dattri_llm_b200.ops.losses import _check_logits

MAX_ALTERNATIVES = 32  # of a row (kMostTop of csrc/token_scores.cuh)


class TokenScores(NamedTuple):
    """``logps (B, T)`` of the labels and ``entropy (B, T)`` of the distributions, in nats, which
    backpropagate into the logits; the ``top_k`` likeliest tokens ``top_ids (B, T, K)`` with
    their log-probabilities ``top_logps (B, T, K)``, which do not.  Where a label is ignored:
    0, and -1 among the ids."""

    logps: torch.Tensor
    entropy: torch.Tensor
    top_logps: torch.Tensor
    top_ids: torch.Tensor


def _scores_torch(logits, labels, top_k, temperature, ignore) -> TokenScores:
    valid = labels != ignore
    if bool(((labels < 0) | (labels >= logits.shape[2]))[valid].any()):
        raise ValueError(f"labels must be {ignore} or in [0, {logits.shape[2]})")
    raw = (logits if logits.dtype == torch.float64 else logits.float()).masked_fill(~valid.unsqueeze(-1), 0.0)
    base = raw.detach().amax(-1, keepdim=True)  # off before the division, which would round it
    logs = torch.log_softmax((raw - torch.where(torch.isfinite(base), base, 0.0)) / temperature, -1)
    p = logs.exp()
    # a token that cannot come (p = 0) adds nothing, though its log-probability may be -inf
    entropy = -torch.where(p > 0, p * torch.where(p > 0, logs, 0.0), p).sum(-1)
    logps = logs.gather(2, labels.masked_fill(~valid, 0).unsqueeze(-1)).squeeze(-1)
    ids = torch.sort(raw.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
    top = logs.detach().gather(2, ids)
    off = ~valid.unsqueeze(-1)
    return TokenScores(logps.masked_fill(~valid, 0.0), entropy.masked_fill(~valid, 0.0), top.masked_fill(off, 0.0),
                       ids.masked_fill(off, -1))


def token_scores(logits: torch.Tensor, labels: torch.Tensor, *, top_k: int = 0, temperature: float = 1.0,
                 ignore_index: int = -100) -> TokenScores:
    """Log-probability of each label, entropy of each distribution and its *top_k* likeliest
    tokens, under ``softmax(logits / temperature)``, in one pass over the logits
    (``csrc/token_scores.cu``; statistics in fp32).

    Args:
        logits: ``(B, T, V)``, any batch and token strides; bf16, fp16 or fp32 on the GPU.
        labels: ``(B, T)``, the token that ``logits[b, t]`` predicts or *ignore_index*.  The
            logits of ignored positions are not read.
        top_k: alternatives of each token, at most 32; the lowest index first among equal logits.

    Returns:
        :class:`TokenScores`.  A label outside the vocabulary is left out and reported by
        :func:`~dattri_llm_b200.ops.check_device_errors` (raised at once on CPU).  A row with a
        NaN or an infinity above all has NaN for its numbers; NaN counts as the largest logit.
    """
    if use_native(logits):
        return TokenScores(*native().token_scores(logits, labels, top_k, temperature, ignore_index, error_word(logits.device)))
    logits, labels = _check_logits(logits, labels)
    if not 0 <= top_k <= min(MAX_ALTERNATIVES, logits.shape[2]):
        raise ValueError(f"top_k must be between 0 and {MAX_ALTERNATIVES} and no more than the vocabulary, got {top_k}")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive, got {temperature}")
    return _scores_torch(logits, labels, top_k, temperature, ignore_index)
