"""The gated delta rule: chunked for training and prefill, token by token for decoding.

Linear attention whose state forgets by a gate and overwrites what a key read before
(Yang, Kautz & Hatamizadeh 2025, "Gated Delta Networks"): with rows of *k* scaled to length
one and rows of *q* to length *scale*,

    ``g = -exp(a_log) softplus(a + dt_bias)``, ``beta = sigmoid(b)``,
    ``S <- exp(g) S``, ``S <- S + k (beta (v - S^T k))^T``, ``o = S^T q``

for every value head, ``H / Hk`` of which share a key head.  On sm_100 the kernels of
``csrc/delta_*.cu``; the same formulas in PyTorch serve CPU tensors.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from dattri_llm_b200.ops import error_word, native, use_native

CHUNK = 64
MAX_KEY_DIM = 128  # of a head on the GPU (kMostKeyDim of csrc/delta_rule.cuh)
MAX_GROUP = 8      # value heads of a key head on the GPU (kMostGroup)


def _check(q, k, v, a, b, a_log, dt_bias, scale) -> float:
    if q.dim() != 4 or q.shape != k.shape or v.dim() != 4 or v.shape[:2] != q.shape[:2]:
        raise ValueError("q and k must be (B, T, Hk, dk), v (B, T, H, dv) with the same B and T")
    hk, h = q.shape[2], v.shape[2]
    if hk == 0 or h == 0 or h % hk:
        raise ValueError(f"v must have a multiple of the {hk} heads of q and k, got {h}")
    if a.shape != v.shape[:3] or b.shape != v.shape[:3]:
        raise ValueError(f"a and b must be (B, T, H) = {tuple(v.shape[:3])}")
    if a_log.shape != (h,) or dt_bias.shape != (h,):
        raise ValueError(f"a_log and dt_bias must be ({h},)")
    if any(x.dtype != q.dtype for x in (k, v, a, b)):
        raise TypeError("q, k, v, a and b must be of one type")
    if scale is None:
        return 1.0 / math.sqrt(q.shape[3])
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive, got {scale}")
    return scale


def _check_state(name: str, state, q, v) -> None:
    want = (q.shape[0], v.shape[2], q.shape[3], v.shape[3])
    if state.shape != want:
        raise ValueError(f"{name} must be (B, H, dk, dv) = {want}, got {tuple(state.shape)}")
    if state.dtype != torch.promote_types(q.dtype, torch.float32):
        raise TypeError(f"{name} must be float32, got {state.dtype}")


def _overlaps(state) -> bool:
    """Whether elements of a state share memory."""
    reach, nested = 0, True
    for step, size in sorted(zip(state.stride(), state.shape, strict=True)):
        if size > 1:  # each axis steps further than those of smaller steps reach together
            nested = nested and step > reach
            reach += (size - 1) * step
    if nested or state.numel() == 0:
        return False
    place = torch.zeros((), dtype=torch.int64)
    for step, size in zip(state.stride(), state.shape, strict=True):
        place = place.unsqueeze(-1) + step * torch.arange(size)
    return place.unique().numel() < state.numel()


def _parts(q, k, v, a, b, a_log, dt_bias, scale):
    """Scaled rows of every value head, values, log-decays and write strengths, in 32 bits or more."""
    wide = torch.promote_types(q.dtype, torch.float32)
    q, k, v, a, b, a_log, dt_bias = (x.to(wide) for x in (q, k, v, a, b, a_log, dt_bias))

    def unit(x):
        return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6)

    group = v.shape[2] // q.shape[2]
    q, k = (unit(x).repeat_interleave(group, 2) for x in (q, k))
    return q * scale, k, v, (-a_log.exp() * F.softplus(a + dt_bias)).clamp(min=-1e4), torch.sigmoid(b)


def _rule_torch(q, k, v, g, beta, state):
    t = v.shape[1]
    pad = -t % CHUNK
    q, k, v = (F.pad(x.transpose(1, 2), (0, 0, 0, pad)).unflatten(2, (-1, CHUNK)) for x in (q, k, v))
    g, beta = (F.pad(x.transpose(1, 2), (0, pad)).unflatten(2, (-1, CHUNK)) for x in (g, beta))
    total = g.double().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=v.device).tril()
    decay = (total.unsqueeze(-1) - total.unsqueeze(-2)).masked_fill(~lower, -math.inf).exp().to(v.dtype)
    grown = total.exp().to(v.dtype).unsqueeze(-1)
    left = (total[..., -1:] - total).exp().to(v.dtype).unsqueeze(-1)
    mix = ((k @ k.mT) * decay).tril(-1) * beta.unsqueeze(-2)
    attend = (q @ k.mT) * decay
    outs = []
    for c in range(v.shape[2]):
        rhs = v[:, :, c] - grown[:, :, c] * (k[:, :, c] @ state)
        new = beta[:, :, c].unsqueeze(-1) * torch.linalg.solve_triangular(mix[:, :, c], rhs, upper=False, unitriangular=True)
        outs.append(grown[:, :, c] * (q[:, :, c] @ state) + attend[:, :, c] @ new)
        state = grown[:, :, c, -1:] * state + (left[:, :, c] * k[:, :, c]).mT @ new
    out = torch.stack(outs, 2).flatten(2, 3)[:, :, :t] if outs else v.flatten(2, 3)[:, :, :0]
    return out.transpose(1, 2), state


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                     a_log: torch.Tensor, dt_bias: torch.Tensor, *, initial_state: torch.Tensor | None = None,
                     output_final_state: bool = False,
                     scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The rule over whole sequences, in chunks of 64 tokens.

    Args:
        q, k: ``(B, T, Hk, dk)``, not normalised.  On the GPU ``dk`` is a multiple of 8, 128 at
            most; any strides with a contiguous last axis (slices of one projection).
        v: ``(B, T, H, dv)``; ``H`` is a multiple of ``Hk`` (8 times at most on the GPU) and
            head *h* reads key head ``h // (H // Hk)``; ``dv`` a multiple of 8, 1024 at most.
        a, b: ``(B, T, H)``, the gates' projections, of the type of *q*, *k* and *v* (bf16 or fp16 on the GPU).
        a_log, dt_bias: ``(H,)``, bf16, fp16 or fp32.
        initial_state: ``(B, H, dk, dv)`` fp32, or ``None``: zeros.
        scale: length of the rows of *q*, ``dk ** -0.5`` unless given.

    Returns:
        ``(out (B, T, H, dv), final state (B, H, dk, dv) fp32 or None)``.  Both backpropagate into
        all inputs.  For the backward the forward keeps the state before every chunk and the chunks'
        matrices: 2.3 KB a token and value head of 128 x 128 on the GPU, where two value heads share a
        key head.  Operands of the products carry 16 bits there: a final state is 1e-6 to 6e-6 of its norm off.  A token
        with ``b = -inf`` writes nothing; one with ``a = +inf`` forgets everything before it.
    """
    if use_native(q):
        return native().gated_delta_rule(q, k, v, a, b, a_log, dt_bias, initial_state, output_final_state, scale,
                                         error_word(q.device))
    scale = _check(q, k, v, a, b, a_log, dt_bias, scale)
    parts = _parts(q, k, v, a, b, a_log, dt_bias, scale)
    if initial_state is None:
        state = parts[2].new_zeros(q.shape[0], v.shape[2], q.shape[3], v.shape[3])
    else:
        _check_state("initial_state", initial_state, q, v)
        state = initial_state
    out, state = _rule_torch(*parts, state)
    return out.to(v.dtype), state if output_final_state else None


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                     a_log: torch.Tensor, dt_bias: torch.Tensor, state: torch.Tensor, *,
                     scale: float | None = None) -> torch.Tensor:
    """The rule for one or a few new tokens: *state* ``(B, H, dk, dv)`` fp32 is updated in place.

    The other arguments are :func:`gated_delta_rule`'s (fp32 too on the GPU).  No gradient; one
    launch that reads and writes the state once whatever the number of tokens.
    """
    if use_native(q):
        return native().gated_delta_step(q, k, v, a, b, a_log, dt_bias, state, scale, error_word(q.device))
    scale = _check(q, k, v, a, b, a_log, dt_bias, scale)
    _check_state("state", state, q, v)
    if _overlaps(state):
        raise ValueError("state: the heads must not overlap")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v, a, b, a_log, dt_bias, state)):
        raise RuntimeError("gated_delta_step has no gradient: call it under torch.no_grad(), or gated_delta_rule")
    q32, k32, v32, g, beta = _parts(q, k, v, a, b, a_log, dt_bias, scale)
    outs = []
    for t in range(v.shape[1]):
        state.mul_(g[:, t, :, None, None].exp())
        e = beta[:, t, :, None] * (v32[:, t] - torch.einsum("bhkv,bhk->bhv", state, k32[:, t]))
        state.add_(k32[:, t].unsqueeze(-1) * e.unsqueeze(-2))
        outs.append(torch.einsum("bhkv,bhk->bhv", state, q32[:, t]))
    return (torch.stack(outs, 1) if outs else v32).to(v.dtype)
