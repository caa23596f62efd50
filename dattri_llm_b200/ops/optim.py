"""Native optimizer-geometry kernels (``csrc/rows.cu``)."""

from __future__ import annotations

import torch


def adam_direction(g: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, *, step: int,
                   beta1: float, beta2: float, eps: float) -> torch.Tensor:
    """Per-sample Adam update direction of ``g (..., p)`` (fp32): ``m_hat / (sqrt(v_hat) + eps)``
    with ``m = beta1 m0 + (1 - beta1) g`` and ``v = beta2 v0 + (1 - beta2) g^2`` for the
    optimizer's moments ``m0, v0`` (flattened to ``p``) -- one fused pass (the update
    ``torch.optim.Adam`` would take next if *g* were the whole batch's gradient).
    Reference: ``dattri_llm/gradient/ops/optimizer.py`` (Adam preconditioner)."""
    from dattri_llm_b200.ops import count_launch, native

    p = g.shape[-1]
    m0 = exp_avg.detach().reshape(-1).to(g.device, torch.float32).contiguous()
    v0 = exp_avg_sq.detach().reshape(-1).to(g.device, torch.float32).contiguous()
    if m0.numel() != p or v0.numel() != p:
        raise ValueError(f"optimizer moments have {m0.numel()} entries for a {p}-wide gradient")
    g32 = g.to(torch.float32).contiguous()
    if p % 4:
        raise ValueError("adam_direction: the width must be a multiple of 4")
    count_launch()
    return native().adam_direction(g32.reshape(-1, p), m0, v0, float(beta1), float(beta2), int(step),
                                   float(eps)).view(g.shape)


MOMENT_BLOCK = 256  # elements that share a scale of an 8-bit moment (kMomentBlock of csrc/adamw.cuh)
_F8_MAX = 448.0
_F8_TINY = 2.0 ** -9  # the smallest e4m3 code that is not zero


def _to_blocks(x: torch.Tensor) -> torch.Tensor:
    """The elements in the order of memory as ``(blocks, MOMENT_BLOCK)``, zeros behind the last one."""
    flat = x.as_strided((x.numel(),), (1,))
    return torch.nn.functional.pad(flat, (0, -flat.numel() % MOMENT_BLOCK)).view(-1, MOMENT_BLOCK)


def _spread(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """``codes * scale`` of each block, laid out like *codes*."""
    flat = codes.as_strided((codes.numel(),), (1,)).float()
    return (flat * scale.repeat_interleave(MOMENT_BLOCK)[:flat.numel()]).as_strided(codes.shape, codes.stride())


def _encode(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, root: bool) -> None:
    blocks = _to_blocks(x)
    top = blocks.abs().amax(1) if blocks.numel() else blocks.new_zeros(0)
    scale.copy_(torch.where(top > 0, (top / _F8_MAX).clamp(min=1e-37), top))
    ratio = blocks / torch.where(scale > 0, scale, 1.0).unsqueeze(1)
    if root:
        ratio = torch.where(blocks > 0, ratio.clamp(min=_F8_TINY), ratio)
    flat = ratio.clamp(-_F8_MAX, _F8_MAX).to(torch.float8_e4m3fn).view(-1)[:x.numel()]
    codes.as_strided((codes.numel(),), (1,)).copy_(flat)


def adamw_state(param: torch.Tensor, bits: int = 32) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``(exp_avg, exp_avg_sq, scales)`` of zeros for *param*, as :func:`adamw_step` takes them:
    fp32 and ``None`` with 32 *bits*, e4m3 codes and fp32 scales ``(2, blocks)`` with 8."""
    if bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits, got {bits}")
    dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
    m, v = (torch.zeros_like(param, dtype=dtype, requires_grad=False) for _ in range(2))
    blocks = -(-param.numel() // MOMENT_BLOCK)
    return m, v, None if bits == 32 else torch.zeros(2, blocks, device=param.device)


def adamw_moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor,
                  scales: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    """The moments ``(m, v)`` in fp32 that a state stands for."""
    if scales is None:
        return exp_avg, exp_avg_sq
    return _spread(exp_avg, scales[0]), _spread(exp_avg_sq, scales[1]).square()


def adamw_state_like(param: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor,
                     scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A state of 8-bit moments in the layout of *param*.  Blocks go by the order of memory: where that differs, the
    moments are written as codes once more."""
    if [t for n, t in zip(param.shape, exp_avg.stride(), strict=True) if n > 1] == [
            t for n, t in zip(param.shape, param.stride(), strict=True) if n > 1]:
        return *(torch.empty_like(param, dtype=x.dtype, requires_grad=False).copy_(x) for x in (exp_avg, exp_avg_sq)), scales
    m, v, s = adamw_state(param, 8)
    for codes, to, row in ((exp_avg, m, 0), (exp_avg_sq, v, 1)):
        wide = torch.empty_like(param, dtype=torch.float32, requires_grad=False).copy_(_spread(codes, scales[row]))
        _encode(wide, to, s[row], bool(row))
    return m, v, s


def _adamw_torch(p, g, exp_avg, exp_avg_sq, scales, step, lr, betas, eps, weight_decay, maximize) -> None:
    wide = torch.promote_types(p.dtype, torch.float32)
    m, v = (x.to(wide) for x in adamw_moments(exp_avg, exp_avg_sq, scales))
    g = -g.to(wide) if maximize else g.to(wide)
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    root = v.sqrt()
    bias2 = 1 - betas[1] ** step
    p.copy_(p.to(wide) * (1 - lr * weight_decay) - lr / (1 - betas[0] ** step) * m / (root / bias2 ** 0.5 + eps))
    if scales is None:
        exp_avg.copy_(m)
        exp_avg_sq.copy_(v)
    else:
        _encode(m.as_strided(p.shape, p.stride()) if m.stride() == p.stride() else torch.empty_like(p, dtype=wide).copy_(m),
                exp_avg, scales[0], False)
        _encode(root if root.stride() == p.stride() else torch.empty_like(p, dtype=wide).copy_(root),
                exp_avg_sq, scales[1], True)


@torch.no_grad()
def adamw_step(params: list[torch.Tensor], grads: list[torch.Tensor], exp_avgs: list[torch.Tensor],
               exp_avg_sqs: list[torch.Tensor], scales: list[torch.Tensor] | None = None, *, step: int, lr: float,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               maximize: bool = False) -> None:
    """One AdamW update of many tensors, in place and in one launch for each pair of types
    (``csrc/adamw.cu``): ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
    ``p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)``, computed in fp32 and
    rounded once.

    Args:
        params: bf16, fp16 or fp32, dense in memory in any order of their axes, on one device.
        grads: of the parameters' types, or fp32.
        exp_avgs, exp_avg_sqs: the moments, laid out like the parameters: fp32, or with *scales*
            e4m3 codes, 256 elements to a scale (see :func:`adamw_state`).  What stands for ``v``
            is its root; a root that is not zero keeps a code that is not zero.  A gradient whose square
            is infinite in fp32 makes NaN of its block's moments, as an infinite one does.
        scales: ``None``, or for each parameter fp32 ``(2, blocks)``.
        step: the number of this update, from 1 on.  A captured graph repeats the update of the
            step that it was captured with.

    A parameter, a moment or scales given twice raise; so do sparse gradients.
    """
    from dattri_llm_b200.ops import native, use_native

    if step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0):
        raise ValueError(f"betas must be in [0, 1) and eps not negative, got {betas} and {eps}")
    if params and use_native(params[0]):
        native().adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales, step, lr, betas[0], betas[1], eps,
                            weight_decay, maximize)
        return
    lists = (params, grads, exp_avgs, exp_avg_sqs, *(() if scales is None else (scales,)))
    if len({len(x) for x in lists}) != 1:
        raise ValueError("every parameter needs a gradient and both moments (and scales of both, or of none)")
    written = [x.data_ptr() for x in (*params, *exp_avgs, *exp_avg_sqs) if x.numel()]
    if len(set(written)) != len(written):
        raise ValueError("a parameter or a moment is given twice")
    written += [s.data_ptr() for s in scales or () if s.numel()]
    if len(set(written)) != len(written):
        raise ValueError("scales are given twice")
    moment = torch.float32 if scales is None else torch.float8_e4m3fn
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, strict=True)):
        if g.layout != torch.strided:
            raise NotImplementedError(f"a gradient must be dense, got {g.layout}")
        if g.shape != p.shape or any(x.shape != p.shape or x.stride() != p.stride() for x in (m, v)):
            raise ValueError("gradients must have their parameter's shape, moments its strides too")
        if m.dtype != v.dtype or (m.dtype != moment and not (p.dtype == m.dtype == torch.float64)):
            raise TypeError(f"moments must be {moment}, got {m.dtype} and {v.dtype}")
        if scales is not None and scales[i].shape != (2, -(-p.numel() // MOMENT_BLOCK)):
            raise ValueError(f"scales must be (2, blocks of {MOMENT_BLOCK} elements), got {tuple(scales[i].shape)}")
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, strict=True)):
        _adamw_torch(p, g, m, v, None if scales is None else scales[i], step, lr, betas, eps, weight_decay, maximize)
