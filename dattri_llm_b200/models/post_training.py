"""Losses of models trained on preference pairs or on their own rollouts.

``loss_fn(model, batch)`` callables like :func:`~dattri_llm_b200.models.llama.token_sum_loss`,
for any causal LM whose output has ``.logits`` (or is the logits), over the fused losses of
:mod:`dattri_llm_b200.ops.losses`.  They sum over pairs or tokens by default, so that a
capture's per-sample gradients are each sequence's own.  The labels are shifted here, not the
logits: the gradient of a shifted slice would be copied once more.

A pair is two rows of the batch: the chosen sequences come first, then the rejected ones in
the same order, and the gradient of pair *i* is the sum of the captured rows ``i`` and ``P + i``.
"""

from __future__ import annotations

import torch
from torch import nn

from dattri_llm_b200.ops.losses import BalanceLoss, PolicyLoss, PreferenceLoss, policy_loss, preference_loss, router_balance_loss
from dattri_llm_b200.ops.scores import TokenScores, token_scores

IGNORE = -100


def shift_labels(labels: torch.Tensor) -> torch.Tensor:
    """The labels that ``logits[:, t]`` predicts: ``labels[:, t + 1]``, nothing at the last position."""
    return torch.cat([labels[:, 1:], torch.full_like(labels[:, :1], IGNORE)], dim=1)


def _logits(model: nn.Module, batch: dict) -> torch.Tensor:
    out = model(input_ids=batch["input_ids"], attention_mask=batch.get("attention_mask"))
    return out.logits if hasattr(out, "logits") else out


@torch.no_grad()
def token_logps(model: nn.Module, batch: dict, *, temperature: float = 1.0) -> torch.Tensor:
    """Log-probabilities ``(B, T)`` of the batch's labels under *model*, at the position that
    predicts them, 0 where ignored: a reference model's (summed over tokens) for
    :func:`preference_pair_loss`, or the sampling policy's for :func:`policy_token_loss`."""
    labels = shift_labels(batch["labels"])
    zero = torch.zeros(labels.shape[0], device=labels.device)
    return policy_loss(_logits(model, batch), labels, zero, temperature=temperature, ignore_index=IGNORE).logps


@torch.no_grad()
def token_quality(model: nn.Module, batch: dict, *, top_k: int = 0, temperature: float = 1.0) -> TokenScores:
    """:func:`~dattri_llm_b200.ops.token_scores` of the batch's labels under *model*, at the position that
    predicts them: how likely and how uncertain the model finds each token, and what it would
    have said instead (for choosing samples, or for reading an attribution)."""
    return token_scores(_logits(model, batch), shift_labels(batch["labels"]), top_k=top_k, temperature=temperature,
                        ignore_index=IGNORE)


def entropy_regularized_loss(model: nn.Module, batch: dict, *, coef: float = 0.0, temperature: float = 1.0) -> torch.Tensor:
    """Summed next-token loss less *coef* times the summed entropy of the predictions, in one pass over the logits."""
    scores = token_scores(_logits(model, batch), shift_labels(batch["labels"]), temperature=temperature, ignore_index=IGNORE)
    return -scores.logps.sum() - coef * scores.entropy.sum()


def preference_pair_loss(model: nn.Module, batch: dict, *, reduction: str = "sum", **options) -> torch.Tensor:
    """Preference loss of a batch ``{"input_ids", "labels", "ref_logps", ["attention_mask"]}`` of
    ``2P`` sequences (*options*: those of :func:`~dattri_llm_b200.ops.preference_loss`)."""
    return preference_pair_terms(model, batch, reduction=reduction, **options).loss


def preference_pair_terms(model: nn.Module, batch: dict, **options) -> PreferenceLoss:
    """:func:`preference_pair_loss` with the sequences' log-probabilities."""
    return preference_loss(_logits(model, batch), shift_labels(batch["labels"]), batch["ref_logps"],
                           ignore_index=IGNORE, **options)


def policy_token_loss(model: nn.Module, batch: dict, *, reduction: str = "sum", **options) -> torch.Tensor:
    """Clipped policy loss of rollouts ``{"input_ids", "labels", "advantages", ["old_logps"],
    ["ref_logps"], ["attention_mask"]}``; the log-probabilities are :func:`token_logps`'s, at the
    predicting position (*options*: those of :func:`~dattri_llm_b200.ops.policy_loss`)."""
    return policy_token_terms(model, batch, reduction=reduction, **options).loss


def policy_token_terms(model: nn.Module, batch: dict, **options) -> PolicyLoss:
    """:func:`policy_token_loss` with the token log-probabilities, the mean KL and the clip fraction."""
    return policy_loss(_logits(model, batch), shift_labels(batch["labels"]), batch["advantages"],
                       batch.get("old_logps"), batch.get("ref_logps"), ignore_index=IGNORE, **options)


def stacked_balance_loss(router_logits, top_k: int, attention_mask: torch.Tensor | None = None, *,
                         z_coef: float = 0.0) -> BalanceLoss:
    """Balance loss of every layer from the ``router_logits`` a Hugging Face expert model
    returns (one ``(B * T, E)`` tensor for each layer), padded tokens left out.

    One loss for each layer; Hugging Face's own auxiliary loss joins the tokens of all layers
    first.  The experts are chosen again from the logits, the lowest index where they tie: 16-bit
    logits tie often and ``torch.topk`` promises no order, so the counts need not be those of
    the model's routing (:func:`~dattri_llm_b200.ops.router_balance_loss` takes the model's ids)."""
    logits = torch.stack([x.reshape(-1, x.shape[-1]) for x in router_logits])
    mask = None
    if attention_mask is not None:
        mask = attention_mask.reshape(1, -1).bool().expand(logits.shape[0], -1)
    return router_balance_loss(logits, top_k, mask=mask, z_coef=z_coef)
