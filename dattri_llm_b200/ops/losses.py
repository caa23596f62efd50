"""Losses of post-training: preference pairs, clipped policy updates, router balance.

Each takes logits and returns a loss that backpropagates into them:

* :func:`preference_loss` -- paired log ratios of chosen and rejected sequences against a
  reference model (sigmoid, hinge or squared form);
* :func:`policy_loss` -- the clipped surrogate of sampled tokens with a KL term;
* :func:`router_balance_loss` -- the auxiliary loss of an expert router, with the number of
  tokens each expert received.

On sm_100 they run the kernels of ``csrc/logit_loss.cu`` and ``csrc/router_balance.cu``
(bf16, fp16 or fp32 logits; fp32 softmax statistics, sums over tokens in fp64), which have
no forward-mode derivatives and refuse inputs with tangents; the same formulas in PyTorch
serve CPU tensors.  The reference has neither: its losses are the
user's own.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F

from dattri_llm_b200.ops import error_word, native, use_native

PAIR_LOSSES = ("sigmoid", "hinge", "ipo")


class PreferenceLoss(NamedTuple):
    """``loss`` (a scalar, or ``(P,)`` with ``reduction="none"``) and the policy's log-probability
    of each sequence ``logps (2P,)``; both backpropagate into the logits."""

    loss: torch.Tensor
    logps: torch.Tensor


class PolicyLoss(NamedTuple):
    """``loss`` (scalar) and the policy's token log-probabilities ``logps (B, T)`` (0 where
    ignored), which backpropagate; the mean ``kl`` and the ``clip_fraction`` over the tokens
    that count, which do not."""

    loss: torch.Tensor
    logps: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


class BalanceLoss(NamedTuple):
    """``loss`` of every group (the leading shape of the logits), which backpropagates, and the
    tokens each expert received, ``counts (..., E)`` int64."""

    loss: torch.Tensor
    counts: torch.Tensor


def _constant(name: str, x: torch.Tensor | None, logits: torch.Tensor) -> torch.Tensor | None:
    """*x* in 32 bits, or in the 64 of *logits*, or an error if it would need a gradient."""
    if x is None:
        return None
    if x.requires_grad:
        raise ValueError(f"{name} is a constant of the loss: detach it")
    return x.to(torch.promote_types(logits.dtype, torch.float32))


def _check_logits(logits: torch.Tensor, labels: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    if logits.dim() != 3 or not logits.is_floating_point():
        raise ValueError(f"logits must be floating (B, T, V), got {logits.dtype} {tuple(logits.shape)}")
    if labels.shape != logits.shape[:2] or labels.is_floating_point() or labels.dtype == torch.bool:
        raise ValueError(f"labels must be whole numbers (B, T) = {tuple(logits.shape[:2])}, got {labels.dtype} "
                         f"{tuple(labels.shape)}")
    if logits.shape[2] == 0:
        raise ValueError("logits need a vocabulary of at least one entry")
    if labels.device != logits.device:
        raise ValueError(f"labels are on {labels.device}, logits on {logits.device}")
    if logits.stride(2) != 1:
        logits = logits.contiguous()
    return logits, labels.long().contiguous()


def _token_logps(logits: torch.Tensor, labels: torch.Tensor, ignore: int,
                 temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(log-probabilities of the labels, 0 where ignored, which tokens count)`` in PyTorch."""
    valid = labels != ignore
    if bool(((labels < 0) | (labels >= logits.shape[2]))[valid].any()):
        raise ValueError(f"labels must be {ignore} or in [0, {logits.shape[2]})")
    x = logits if logits.dtype == torch.float64 else logits.float()
    x = x.masked_fill(~valid.unsqueeze(-1), 0.0)  # an ignored row may hold anything
    if temperature != 1.0:
        x = x / temperature  # not in a half type, which would round the quotient
    logps = torch.log_softmax(x, -1).gather(2, labels.masked_fill(~valid, 0).unsqueeze(-1)).squeeze(-1)
    return logps.masked_fill(~valid, 0.0), valid


# ---------------------------------------------------------------- preference


def _preference_torch(logits, labels, ref, kind, beta, smoothing, average, reduction, ignore) -> PreferenceLoss:
    tokens, valid = _token_logps(logits, labels, ignore)
    logps = tokens.sum(1)
    if average:
        logps = logps / valid.sum(1).clamp(min=1)
    chosen, rejected = (logps - ref).chunk(2)
    m = chosen - rejected
    if kind == "sigmoid":
        loss = -(1 - smoothing) * F.logsigmoid(beta * m)
        if smoothing:
            loss = loss - smoothing * F.logsigmoid(-beta * m)
    elif kind == "hinge":
        loss = torch.relu(1 - beta * m)
    else:
        loss = (m - 1 / (2 * beta)).square()
    return PreferenceLoss(loss if reduction == "none" else loss.mean() if reduction == "mean" else loss.sum(), logps)


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: torch.Tensor, *, beta: float = 0.1,
                    kind: str = "sigmoid", label_smoothing: float = 0.0, average_logps: bool = False,
                    reduction: str = "mean", ignore_index: int = -100) -> PreferenceLoss:
    """Preference loss of ``P`` pairs: sequences ``0 .. P-1`` of the batch are the chosen ones,
    sequence ``P + i`` is the one rejected against sequence ``i``.

    With ``L_b`` the summed (*average_logps*: mean) log-probability of sequence *b*'s labels
    and ``m = (L_i - ref_i) - (L_{P+i} - ref_{P+i})``:

    * ``"sigmoid"``: ``-(1 - s) log sigmoid(beta m) - s log sigmoid(-beta m)``, ``s`` = *label_smoothing*;
    * ``"hinge"``: ``max(0, 1 - beta m)``;
    * ``"ipo"``: ``(m - 1 / (2 beta))^2``.

    Args:
        logits: ``(2P, T, V)``, any batch and token strides.
        labels: ``(2P, T)``, the token that ``logits[b, t]`` predicts (shift the labels, not
            the logits: a shifted slice of the logits costs a copy of their gradient) or
            *ignore_index*.  The logits of ignored positions are not read.
        ref_logps: ``(2P,)`` the reference model's ``L_b``; a constant.
        reduction: ``"mean"`` or ``"sum"`` over pairs, or ``"none"``.

    Returns:
        :class:`PreferenceLoss`.  A label outside the vocabulary is left out and reported by
        :func:`~dattri_llm_b200.ops.check_device_errors` (raised at once on CPU).
    """
    if use_native(logits):
        return PreferenceLoss(*native().preference_loss(logits, labels, ref_logps, kind, beta, label_smoothing, average_logps,
                                                        reduction, ignore_index, error_word(logits.device)))
    logits, labels = _check_logits(logits, labels)
    b = logits.shape[0]
    if b < 2 or b % 2:
        raise ValueError(f"a preference loss needs an even number of sequences (chosen, then rejected), got {b}")
    if kind not in PAIR_LOSSES:
        raise ValueError(f"kind must be one of {PAIR_LOSSES}, got {kind!r}")
    if reduction not in ("none", "mean", "sum"):
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if not (beta > 0 and math.isfinite(beta)):
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0 <= label_smoothing < 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"label_smoothing must be in [0, 0.5), and 0 unless kind is 'sigmoid', got {label_smoothing}")
    if ref_logps.shape != (b,):
        raise ValueError(f"ref_logps must be ({b},), got {tuple(ref_logps.shape)}")
    ref = _constant("ref_logps", ref_logps, logits)
    return _preference_torch(logits, labels, ref, kind, beta, label_smoothing, average_logps, reduction, ignore_index)


# ---------------------------------------------------------------- policy


def _policy_torch(logits, labels, adv, old, ref, lo, hi, kl_coef, temperature, reduction, ignore) -> PolicyLoss:
    logps, valid = _token_logps(logits, labels, ignore, temperature)
    adv = adv if adv.dim() == 2 else adv.unsqueeze(1)
    base = logps.detach() if old is None else old
    ratio = torch.exp((logps - base).masked_fill(~valid, 0.0))
    free, held = ratio * adv, ratio.clamp(lo, hi) * adv
    loss = -torch.where(free <= held, free, held)
    kl = torch.zeros_like(logps)
    if ref is not None:
        d = (ref - logps).masked_fill(~valid, 0.0)
        kl = torch.expm1(d) - d
        if kl_coef:  # an infinite distance that is only reported leaves the loss alone
            loss = loss + kl_coef * kl
    loss = loss.masked_fill(~valid, 0.0)
    n = valid.sum().clamp(min=1)
    if reduction == "token_mean":
        total = loss.sum() / n
    elif reduction == "sequence_mean":
        total = (loss.sum(1) / valid.sum(1).clamp(min=1)).mean()
    else:
        total = loss.sum()
    clipped = ((held < free) & valid).sum().to(logps.dtype) / n
    return PolicyLoss(total, logps, kl.detach().masked_fill(~valid, 0.0).sum() / n, clipped)


def policy_loss(logits: torch.Tensor, labels: torch.Tensor, advantages: torch.Tensor,
                old_logps: torch.Tensor | None = None, ref_logps: torch.Tensor | None = None, *,
                clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0, temperature: float = 1.0,
                reduction: str = "token_mean", ignore_index: int = -100) -> PolicyLoss:
    """Clipped policy loss of sampled tokens with a KL term.

    With ``logp`` the log-probability of a label under ``softmax(logits / temperature)``,
    ``r = exp(logp - old)`` and ``d = ref - logp``, each token that counts adds
    ``-min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (exp(d) - d - 1)``.

    On the GPU the gradient is written along with the loss (memory of the logits' size from the
    forward on, unless the logits need none) and given out where the loss ends the graph; under
    any other loss gradient (a scaled loss, accumulation) and in a second backward the backward
    computes it from the logits, in 32 bits and rounded once.

    Args:
        logits: ``(B, T, V)``, any batch and token strides.
        labels: ``(B, T)``, the sampled token that ``logits[b, t]`` predicts or *ignore_index*.
            The logits of ignored positions are not read.
        advantages: ``(B,)`` or ``(B, T)``; a constant.
        old_logps: ``(B, T)`` log-probabilities at sampling time, or ``None`` for an on-policy
            step (``r = 1``, whose gradient is ``-A``); a constant.
        ref_logps: ``(B, T)`` log-probabilities under the reference model, or ``None``: no KL
            term (then *kl_coef* must be 0); a constant.
        reduction: ``"token_mean"`` over all tokens that count, ``"sequence_mean"`` (the mean
            of the sequences' means; one without tokens adds 0), or ``"sum"``.

    Returns:
        :class:`PolicyLoss`.  A label outside the vocabulary is left out and reported by
        :func:`~dattri_llm_b200.ops.check_device_errors` (raised at once on CPU).
    """
    if use_native(logits):
        return PolicyLoss(*native().policy_loss(logits, labels, advantages, old_logps, ref_logps, clip[0], clip[1], kl_coef,
                                                temperature, reduction, ignore_index, error_word(logits.device)))
    logits, labels = _check_logits(logits, labels)
    b, t = labels.shape
    if b == 0:
        raise ValueError("a policy loss needs at least one sequence")
    if advantages.shape not in ((b,), (b, t)):
        raise ValueError(f"advantages must be ({b},) or ({b}, {t}), got {tuple(advantages.shape)}")
    for name, x in (("old_logps", old_logps), ("ref_logps", ref_logps)):
        if x is not None and x.shape != (b, t):
            raise ValueError(f"{name} must be ({b}, {t}), got {tuple(x.shape)}")
    if reduction not in ("token_mean", "sequence_mean", "sum"):
        raise ValueError(f"reduction must be 'token_mean', 'sequence_mean' or 'sum', got {reduction!r}")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive, got {temperature}")
    if not (0 <= clip[0] <= 1 and clip[1] >= 0):
        raise ValueError(f"clip must be (low in [0, 1], high >= 0), got {clip}")
    if kl_coef and ref_logps is None:
        raise ValueError("a KL term needs ref_logps")
    lo, hi = 1.0 - clip[0], 1.0 + clip[1]
    consts = (_constant(n, x, logits) for n, x in (("advantages", advantages), ("old_logps", old_logps),
                                                   ("ref_logps", ref_logps)))
    return _policy_torch(logits, labels, *consts, lo, hi, kl_coef, temperature, reduction, ignore_index)


# ---------------------------------------------------------------- router balance


def _balance_torch(logits, ids, mask, top_k, z_coef) -> BalanceLoss:
    g, n, e = logits.shape
    x = logits if logits.dtype == torch.float64 else logits.float()
    keep = torch.ones(g, n, dtype=torch.bool, device=x.device) if mask is None else mask
    x = x.masked_fill(~keep.unsqueeze(-1), 0.0)  # a masked token may hold anything
    if ids is None:
        ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
    elif bool(((ids < 0) | (ids >= e))[keep].any()):
        raise ValueError(f"expert_ids must be in [0, {e})")
    chosen = keep.unsqueeze(-1).expand_as(ids)
    counts = torch.zeros(g, e, dtype=torch.int64, device=x.device)
    counts.scatter_add_(1, torch.where(chosen, ids, 0).reshape(g, n * top_k), chosen.reshape(g, n * top_k).long())
    tokens = keep.sum(1).clamp(min=1).unsqueeze(-1)
    mean_p = torch.softmax(x, -1).masked_fill(~keep.unsqueeze(-1), 0.0).sum(1) / tokens
    loss = e * (counts / tokens * mean_p).sum(1)
    if z_coef:
        lse = torch.logsumexp(x, -1).masked_fill(~keep, 0.0)
        loss = loss + z_coef * lse.square().sum(1) / tokens.squeeze(-1)
    return BalanceLoss(loss, counts)


def router_balance_loss(logits: torch.Tensor, top_k: int, expert_ids: torch.Tensor | None = None,
                        mask: torch.Tensor | None = None, *, z_coef: float = 0.0) -> BalanceLoss:
    """Auxiliary balance loss of an expert router, for every group of tokens by itself.

    With ``p = softmax(logits)``, ``f_e`` the choices of expert *e* per token and ``P_e`` the
    mean of ``p_e``, both over the tokens that count, a group's loss is
    ``E sum_e f_e P_e + z_coef mean(logsumexp(logits)^2)``; it is ``top_k`` when all experts
    are used alike.  ``f`` carries no gradient.  A group without tokens has loss 0.

    Args:
        logits: ``(..., N, E)``; each index of the leading axes (layers, sequences) is a group.
        top_k: choices of each token.
        expert_ids: ``(..., N, top_k)`` the experts chosen, or ``None``: the largest logits, the
            lowest index where they tie.
        mask: ``(..., N)`` bool, the tokens that count, or ``None``: all.  The others get no
            gradient, whatever their logits hold.

    Returns:
        :class:`BalanceLoss`.  An expert id outside ``[0, E)`` is left out and reported by
        :func:`~dattri_llm_b200.ops.check_device_errors` (raised at once on CPU).
    """
    if use_native(logits):
        return BalanceLoss(*native().balance_loss(logits, expert_ids, mask, top_k, z_coef, error_word(logits.device)))
    if logits.dim() < 2 or not logits.is_floating_point():
        raise ValueError(f"router logits must be floating (..., N, E), got {logits.dtype} {tuple(logits.shape)}")
    lead, (n, e) = logits.shape[:-2], logits.shape[-2:]
    if not 1 <= top_k <= e:
        raise ValueError(f"top_k must be between 1 and the number of experts {e}, got {top_k}")
    if expert_ids is not None:
        if expert_ids.shape != (*lead, n, top_k) or expert_ids.is_floating_point() or expert_ids.dtype == torch.bool:
            raise ValueError(f"expert_ids must be whole numbers {(*lead, n, top_k)}, got {expert_ids.dtype} "
                             f"{tuple(expert_ids.shape)}")
        expert_ids = expert_ids.long().contiguous()
    if mask is not None:
        if mask.shape != (*lead, n):
            raise ValueError(f"mask must be {(*lead, n)}, got {tuple(mask.shape)}")
        mask = (mask if mask.dtype == torch.bool else mask != 0).contiguous()
    x = logits.reshape(math.prod(lead), n, e)
    loss, counts = _balance_torch(x, None if expert_ids is None else expert_ids.view(*x.shape[:2], top_k),
                                  None if mask is None else mask.view(x.shape[:2]), top_k, z_coef)
    return BalanceLoss(loss.reshape(lead), counts.reshape(*lead, e))
