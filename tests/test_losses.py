"""Preference and policy losses and the router's balance loss against their definitions in 64 bits.

Tolerances.  A softmax in 32 bits with arguments below 64 in base two: rounding the argument
moves a term by at most ``64 ln 2 2^-24 < 3e-6`` of itself, the exponential and the sums by
less, so a log-probability is within ``1e-5 + 2^-22 |logp|`` and a probability within ``1e-5``
of itself.  A gradient is a coefficient (a smooth function of log-probabilities, whose own
error is below ``2e-5`` of its bound) times a probability: ``4e-5`` of the coefficient's bound
in 32 bits, and half a unit in the last place of the type it is rounded to (``2^-9`` bf16,
``2^-12`` fp16, of which values below the normal range keep ``2^-25``).  The tests allow the
unit itself.
"""

import math

import pytest
import torch

from dattri_llm_b200 import ops
from dattri_llm_b200.ops import losses

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 4e-5, torch.bfloat16: 2**-8, torch.float16: 2**-11}
FLOOR = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2**-24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _close(got, want, rtol, atol):
    torch.testing.assert_close(got.detach().double().cpu(), want.detach().double().cpu(), rtol=rtol, atol=atol,
                               equal_nan=True)


def _labels(b, t, v, seed, masked=0.3):
    g = _gen(seed)
    y = torch.randint(0, v, (b, t), generator=g)
    return torch.where(torch.rand(b, t, generator=g) < masked, -100, y)


def _logits(b, t, v, dtype, seed, layout="plain", device="cpu", spread=3.0):
    """Logits of a layout: the values are the same in each."""
    x = (spread * torch.randn(b, t, v, generator=_gen(seed))).to(dtype).to(device)
    if layout == "sliced":  # rows of a longer sequence and a wider, oddly offset table
        wide = torch.full((b, t + 2, v + 3), 7.0, dtype=dtype, device=device)
        wide[:, 1:t + 1, 2:v + 2] = x
        x = wide[:, 1:t + 1, 2:v + 2]
    elif layout == "shifted":
        long = torch.full((b, t + 1, v), 7.0, dtype=dtype, device=device)
        long[:, 1:] = x
        x = long[:, 1:]
    elif layout == "time_first":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "vocab_strided":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    return x.detach().requires_grad_()


# ---------------------------------------------------------------- definitions in 64 bits


def _logps64(x, labels, temperature=1.0):
    """Label log-probabilities, 0 where ignored, of fp64 logits whose ignored rows may hold anything."""
    keep = labels != -100
    x = torch.where(keep[..., None], x, 0.0) / temperature
    top = x.amax(-1, keepdim=True)
    lse = (x - top).exp().sum(-1).log() + top[..., 0]
    return torch.where(keep, x.gather(2, labels.clamp(min=0)[..., None])[..., 0] - lse, 0.0), keep


def preference64(x, labels, ref, beta=0.1, kind="sigmoid", label_smoothing=0.0, average_logps=False, reduction="mean"):
    tokens, keep = _logps64(x, labels)
    logps = tokens.sum(1)
    if average_logps:
        logps = logps / keep.sum(1).clamp(min=1)
    p = len(logps) // 2
    m = (logps[:p] - ref[:p]) - (logps[p:] - ref[p:])
    if kind == "sigmoid":
        loss = (1 - label_smoothing) * torch.log1p((-beta * m).exp()) + label_smoothing * torch.log1p((beta * m).exp())
    elif kind == "hinge":
        loss = (1 - beta * m).clamp(min=0)
    else:
        loss = (m - 0.5 / beta) ** 2
    return {"mean": loss.mean(), "sum": loss.sum(), "none": loss}[reduction], logps


def policy64(x, labels, adv, old, ref, clip=(0.2, 0.2), kl_coef=0.0, temperature=1.0, reduction="token_mean"):
    logps, keep = _logps64(x, labels, temperature)
    adv = adv if adv.dim() == 2 else adv[:, None].expand(labels.shape)
    r = ((logps - (logps.detach() if old is None else old)) * keep).exp()
    free = r * adv
    held = r.detach().clamp(1 - clip[0], 1 + clip[1]) * adv
    use = free <= held
    loss = -torch.where(use, free, held)
    kl = torch.zeros_like(logps)
    if ref is not None:
        d = torch.where(keep, ref - logps, 0.0)
        kl = d.exp() - d - 1
        loss = loss + kl_coef * kl
    loss = torch.where(keep, loss, 0.0)
    n = keep.sum().clamp(min=1)
    total = {"token_mean": loss.sum() / n, "sequence_mean": (loss.sum(1) / keep.sum(1).clamp(min=1)).mean(),
             "sum": loss.sum()}[reduction]
    return total, logps, torch.where(keep, kl, 0.0).sum() / n, (~use & keep).sum() / n


def balance64(x, top_k, ids=None, mask=None, z_coef=0.0):
    g, n, e = x.shape
    keep = torch.ones(g, n, dtype=torch.bool) if mask is None else mask
    x = torch.where(keep[..., None], x, 0.0)
    if ids is None:  # the rank of each expert: how many are larger, or as large with a lower index
        a, b = x.detach()[..., :, None], x.detach()[..., None, :]
        at = torch.arange(e)
        chosen = ((b > a) | ((b == a) & (at[None, :] < at[:, None]))).sum(-1) < top_k
        counts = (chosen & keep[..., None]).sum(1)
    else:
        counts = torch.stack([(ids[i][keep[i]].reshape(-1, 1) == torch.arange(e)).sum(0) for i in range(g)])
    tokens = keep.sum(1).clamp(min=1).double()[:, None]
    lse = torch.logsumexp(x, -1)
    p = torch.where(keep[..., None], (x - lse[..., None]).exp(), 0.0)
    loss = e * (counts / tokens * p.sum(1) / tokens).sum(1)
    return loss + z_coef * (torch.where(keep, lse, 0.0) ** 2).sum(1) / tokens[:, 0], counts


def _double(x):
    return x.detach().cpu().double().requires_grad_()


# ---------------------------------------------------------------- preference

SIZES = [(1, 1, 1), (1, 3, 2), (1, 1, 7), (2, 5, 33), (3, 17, 1001), (2, 4, 8192), (2, 3, 9001), (1, 2, 40003),
         (1, 2, 131072)]


def _preference(dev, size, dtype, layout="plain", seed=0, **kw):
    p, t, v = size
    labels = _labels(2 * p, t, v, seed + 1)
    x = _logits(2 * p, t, v, dtype, seed, layout, dev)
    ref, _ = _logps64(_double(x), labels)
    ref = (ref.sum(1) + 2 * torch.randn(2 * p, generator=_gen(seed + 2), dtype=torch.float64)).detach().float()
    if kw.get("average_logps"):
        ref = ref / t
    got = ops.preference_loss(x, labels.to(dev), ref.to(dev), **kw)
    x64 = _double(x)
    return got, x, preference64(x64, labels, ref.double(), **kw), x64


def _check_preference(got, x, want, x64, beta=0.1, average=False):
    t = x.shape[1]
    # A sum of T log-probabilities, each within 1e-5 + 2^-22 |logp| (below 64).
    slack = (1 if average else t) * 3e-5
    _close(got.logps, want[1], 0, slack + 2e-7 * float(want[1].detach().abs().max()))
    # |d loss / d m| <= max(beta, 2 |m - 1 / (2 beta)|): the margin's error carries over.
    slope = max(beta, 2 * (float(want[0].detach().abs().max()) ** 0.5 if want[0].numel() else 0))
    _close(got.loss, want[0], 1e-6, 2 * slack * slope + 1e-6)
    return slope, slack


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_preference_loss_and_gradient(dev, dtype, size):
    got, x, want, x64 = _preference(dev, size, dtype)
    _check_preference(got, x, want, x64)
    got.loss.backward()
    want[0].backward()
    assert x.grad.dtype == dtype and x.grad.shape == x.shape
    _close(x.grad, x64.grad, UNIT[dtype], 4e-5 * 0.1 + FLOOR[dtype])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("layout", ["sliced", "shifted", "time_first", "vocab_strided"])
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, (2, 5, 1001)), (torch.float16, (2, 5, 1000)),
                                        (torch.float32, (2, 5, 9003)), (torch.bfloat16, (2, 3, 16384))])
def test_preference_layouts(dev, layout, dtype, size):
    got, x, want, x64 = _preference(dev, size, dtype, layout)
    _check_preference(got, x, want, x64)
    (grad,) = torch.autograd.grad(got.loss, x)
    want[0].backward()
    _close(grad, x64.grad, UNIT[dtype], 4e-5 * 0.1 + FLOOR[dtype])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kw", [
    {"kind": "sigmoid", "label_smoothing": 0.2, "reduction": "sum", "beta": 0.5},
    {"kind": "hinge", "beta": 0.3}, {"kind": "hinge", "beta": 0.05, "reduction": "none"},
    {"kind": "ipo", "beta": 0.2, "average_logps": True}, {"kind": "ipo", "beta": 0.5, "reduction": "sum"},
    {"kind": "sigmoid", "average_logps": True, "reduction": "none", "beta": 2.0}])
def test_preference_kinds_and_reductions(dev, kw):
    got, x, want, x64 = _preference(dev, (5, 11, 517), torch.float32, **kw)
    slope, slack = _check_preference(got, x, want, x64, kw["beta"], kw.get("average_logps", False))
    weight = torch.randn(got.loss.shape, generator=_gen(9))
    (got.loss * weight.to(dev)).sum().backward()
    (want[0] * weight.double()).sum().backward()
    # The ipo coefficient moves by twice the margin's error.
    _close(x.grad, x64.grad, 4e-5, (4e-5 * slope + 2 * slack * (kw["kind"] == "ipo")) * 3 + 4e-5 * kw["beta"])


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_logps_backpropagate_beside_the_loss(dev):
    got, x, want, x64 = _preference(dev, (3, 7, 130), torch.float32, average_logps=True)
    w = torch.randn(6, generator=_gen(4))
    (got.loss * 2 + (got.logps * w.to(dev)).sum()).backward(retain_graph=True)
    (want[0] * 2 + (want[1] * w.double()).sum()).backward(retain_graph=True)
    _close(x.grad, x64.grad, 4e-5, 4e-5 * 3)
    x.grad = x64.grad = None
    (got.logps * w.to(dev)).sum().backward()  # a second time through the same graph, the loss left out
    (want[1] * w.double()).sum().backward()
    _close(x.grad, x64.grad, 4e-5, 4e-5 * 3)


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_empty_sequences_and_poisoned_ignored_rows(dev):
    p, t, v = 2, 6, 300
    labels = _labels(2 * p, t, v, 1)
    labels[0] = labels[3] = -100  # a chosen and a rejected answer without tokens
    x = _logits(2 * p, t, v, torch.float32, 2, device=dev).detach()
    ignored = (labels == -100).to(dev)
    x[ignored] = torch.tensor([math.nan, math.inf, -math.inf, 0.0], device=dev).repeat(v // 4)
    x.requires_grad_()
    ref = torch.tensor([0.5, -20.0, -30.0, -1.0])
    for average in (False, True):
        x.grad = None
        got = ops.preference_loss(x, labels.to(dev), ref.to(dev), average_logps=average)
        x64 = _double(x)
        want = preference64(x64, labels, ref.double(), average_logps=average)
        _check_preference(got, x, want, x64)
        assert float(got.logps[0]) == 0 and float(got.logps[3]) == 0
        got.loss.backward()
        want[0].backward()
        assert not x.grad[ignored].any()
        _close(x.grad[~ignored], x64.grad[~ignored.cpu()], 4e-5, 4e-6)


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_without_any_token_or_position(dev):
    ref = torch.tensor([1.0, 3.0], device=dev)
    for t in (0, 4):
        x = torch.randn(2, t, 9, device=dev, requires_grad=True)
        got = ops.preference_loss(x, torch.full((2, t), -100, device=dev), ref, beta=0.5)
        _close(got.loss, torch.log1p(torch.tensor(-1.0, dtype=torch.float64).exp()), 1e-6, 0)  # m = -1 + 3
        got.loss.backward()
        assert x.grad.shape == x.shape and not x.grad.any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_vocabulary_entries(dev, dtype):
    """Entries at -inf or the type's lowest value have no probability and no gradient; their own label is impossible."""
    x = _logits(2, 3, 77, dtype, 5, device=dev).detach()
    x[:, :, 10:20] = -math.inf
    x[:, :, 30:40] = torch.finfo(dtype).min
    x.requires_grad_()
    labels = torch.tensor([[1, 2, 3], [4, -100, 50]])
    ref = torch.tensor([-9.0, -8.0])
    got = ops.preference_loss(x, labels.to(dev), ref.to(dev))
    x64 = _double(x)
    want = preference64(x64, labels, ref.double())
    _check_preference(got, x, want, x64)
    got.loss.backward()
    want[0].backward()
    _close(x.grad, x64.grad, UNIT[dtype], 4e-6 + FLOOR[dtype])
    assert not x.grad[:, :, 10:20].any() and not x.grad[:, :, 30:40].any()
    labels[0, 0] = 15
    got = ops.preference_loss(x, labels.to(dev), ref.to(dev))
    assert float(got.logps[0]) == -math.inf and float(got.loss) == math.inf


@pytest.mark.parametrize("dev", DEVICES)
def test_a_row_of_nothing_but_minus_infinity_is_nan(dev):
    x = torch.full((2, 1, 40), -math.inf, device=dev)
    x[1] = 0
    got = ops.preference_loss(x, torch.zeros(2, 1, dtype=torch.long, device=dev), torch.zeros(2, device=dev))
    assert math.isnan(float(got.logps[0])) and math.isnan(float(got.loss))
    _close(got.logps[1], -torch.tensor(40.0).log(), 1e-6, 0)


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_gradient_against_differences(dev):
    got, x, _, x64 = _preference(dev, (2, 4, 29), torch.float32, beta=0.7, label_smoothing=0.1)
    (grad,) = torch.autograd.grad(got.loss, x)
    labels = _labels(4, 4, 29, 1)
    ref, _ = _logps64(_double(x), labels)
    ref = (ref.sum(1) + 2 * torch.randn(4, generator=_gen(2), dtype=torch.float64)).detach().float().double()
    h = 1e-5
    for at in [(0, 0, 3), (1, 2, 28), (2, 1, 0), (3, 3, 17), (0, 1, int(labels[0, 1].clamp(min=0)))]:
        ends = []
        for step in (h, -h):
            moved = x64.detach().clone()
            moved[at] += step
            ends.append(float(preference64(moved, labels, ref, beta=0.7, label_smoothing=0.1)[0]))
        # Central differences: h^2 / 6 of a third derivative below 1, and 1e-16 / h of rounding.
        assert abs(float(grad[at]) - (ends[0] - ends[1]) / (2 * h)) < 4e-5 * 0.7 + 1e-9


# ---------------------------------------------------------------- policy


def _policy(dev, size, dtype, layout="plain", seed=0, per_token=True, has_old=True, has_ref=False, **kw):
    b, t, v = size
    labels = _labels(b, t, v, seed + 1)
    x = _logits(b, t, v, dtype, seed, layout, dev)
    now, _ = _logps64(_double(x), labels, kw.get("temperature", 1.0))
    now, g = now.detach(), _gen(seed + 3)
    adv = torch.randn((b, t) if per_token else (b,), generator=g)
    noise = 0.25 * torch.randn(b, t, generator=g)
    lo, hi = kw.get("clip", (0.2, 0.2))
    for edge in (1 - lo, 1 + hi):  # no ratio so near the edge that rounding decides its side
        noise = torch.where((noise.exp() - edge).abs() < 1e-3, noise + 0.01, noise)
    old = (now - noise).float() if has_old else None
    ref = (now + 0.5 * torch.randn(b, t, generator=g)).float() if has_ref else None
    up = lambda z: None if z is None else z.to(dev)  # noqa: E731
    got = ops.policy_loss(x, labels.to(dev), up(adv), up(old), up(ref), **kw)
    x64 = _double(x)
    wide = lambda z: None if z is None else z.double()  # noqa: E731
    return got, x, policy64(x64, labels, wide(adv), wide(old), wide(ref), **kw), x64, labels


def _check_policy(got, want, weight):
    _close(got.logps, want[1], 2**-22, 1e-5)
    # A token's loss is at most |A| r (r below e) with a ratio within 2e-5: sums of `weight` tokens' worth.
    _close(got.loss, want[0], 1e-6, 5 * 3 * 2e-5 * weight)
    _close(got.kl, want[2], 1e-5, 3e-5)
    _close(got.clip_fraction, want[3], 1e-6, 0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_policy_loss_and_gradient(dev, dtype, size):
    got, x, want, x64, _ = _policy(dev, size, dtype, has_ref=True, kl_coef=0.1)
    _check_policy(got, want, 1)
    got.loss.backward()
    want[0].backward()
    bound = 15 if x.shape[1] else 0  # |A| r
    _close(x.grad, x64.grad, UNIT[dtype], 4e-5 * bound + FLOOR[dtype])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("layout", ["sliced", "shifted", "time_first", "vocab_strided"])
@pytest.mark.parametrize("dtype,v", [(torch.bfloat16, 1001), (torch.float16, 1000), (torch.float32, 9003),
                                     (torch.bfloat16, 16384), (torch.bfloat16, 70001)])
def test_policy_layouts(dev, layout, dtype, v):
    got, x, want, x64, _ = _policy(dev, (3, 4, v), dtype, layout, per_token=False)
    _check_policy(got, want, 1)
    (grad,) = torch.autograd.grad(got.loss, x)
    want[0].backward()
    _close(grad, x64.grad, UNIT[dtype], 4e-5 * 15 + FLOOR[dtype])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kw", [
    {"has_old": False, "per_token": False}, {"temperature": 0.7}, {"reduction": "sum"}, {"reduction": "sequence_mean"},
    {"clip": (0.1, 0.4), "has_ref": True, "kl_coef": 0.05}, {"clip": (1.0, 1e9)},
    {"temperature": 3.0, "reduction": "sequence_mean", "has_ref": True, "kl_coef": 0.3, "per_token": False}])
def test_policy_forms(dev, kw):
    got, x, want, x64, labels = _policy(dev, (4, 13, 331), torch.float32, **kw)
    weight = labels.numel() if kw.get("reduction") == "sum" else 1
    _check_policy(got, want, weight)
    scale = 0.37  # a loss that does not end the graph
    w = torch.randn(4, 13, generator=_gen(8))
    (got.loss * scale).backward(retain_graph=True)
    (want[0] * scale).backward(retain_graph=True)
    bound = 4e-5 * 15 * max(1, 1 / kw.get("temperature", 1))
    _close(x.grad, x64.grad, 4e-5, bound)
    first = x.grad.clone()
    x.grad = None
    (got.loss * scale).backward(retain_graph=True)  # the graph again
    _close(x.grad, first, 4e-5, bound)
    x.grad = x64.grad = None
    (got.loss + (got.logps * w.to(dev)).sum()).backward()
    (want[0] + (want[1] * w.double()).sum()).backward()
    _close(x.grad, x64.grad, 4e-5, bound + 4e-5 * 4)
    assert not got.kl.requires_grad and not got.clip_fraction.requires_grad


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("reduction", ["token_mean", "sequence_mean", "sum"])
def test_policy_empty_rollouts_and_poisoned_ignored_rows(dev, reduction):
    b, t, v = 3, 5, 64
    labels = _labels(b, t, v, 1)
    labels[1] = -100
    x = _logits(b, t, v, torch.float32, 2, device=dev).detach()
    ignored = (labels == -100).to(dev)
    x[ignored] = math.nan
    x.requires_grad_()
    old = torch.full((b, t), -4.0)
    adv = torch.randn(b, t, generator=_gen(3))
    poisoned = torch.where(labels == -100, math.nan, old), torch.where(labels == -100, math.inf, adv)
    got = ops.policy_loss(x, labels.to(dev), poisoned[1].to(dev), poisoned[0].to(dev), poisoned[0].to(dev), kl_coef=0.1,
                          clip=(0.9, 3.0), reduction=reduction)
    x64 = _double(x)
    want = policy64(x64, labels, adv.double(), old.double(), old.double(), kl_coef=0.1, clip=(0.9, 3.0), reduction=reduction)
    kl_bound = float(want[2].detach()) * 15 + 5
    _close(got.loss, want[0], 1e-5, 2e-5 * kl_bound)
    got.loss.backward()
    want[0].backward()
    assert not x.grad[ignored].any()
    _close(x.grad[~ignored], x64.grad[~ignored.cpu()], 4e-5, 4e-5 * kl_bound)
    none = ops.policy_loss(x, torch.full_like(labels, -100).to(dev), adv.to(dev), reduction=reduction)
    assert float(none.loss) == 0 and float(none.kl) == 0 and float(none.clip_fraction) == 0
    x.grad = None
    none.loss.backward()
    assert not x.grad.any()


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_small_kl_keeps_its_digits(dev):
    """exp(d) - d - 1 of d near 1e-3 is 5e-7: cancellation in 32 bits would leave nothing of it."""
    x = torch.zeros(1, 64, 16, device=dev)
    logp = -math.log(16.0)
    d = torch.linspace(-2e-3, 2e-3, 64, dtype=torch.float64)
    ref = (d + logp).float()
    got = ops.policy_loss(x, torch.zeros(1, 64, dtype=torch.long, device=dev), torch.zeros(1, device=dev),
                          ref_logps=ref.view(1, -1).to(dev), kl_coef=1.0)
    d = ref.double() - logp
    # d itself is known to 2^-23 |logp|, 3.3e-7 beside 1e-3.
    _close(got.kl, (d.exp() - d - 1).mean(), 2e-3, 0)


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_reports_an_infinite_distance_without_using_it(dev):
    x = torch.randn(2, 3, 11, generator=_gen(0)).to(dev).requires_grad_()
    y, adv = torch.zeros(2, 3, dtype=torch.long, device=dev), torch.ones(2, device=dev)
    ref = torch.full((2, 3), -math.inf, device=dev)
    got, want = ops.policy_loss(x, y, adv, ref_logps=ref), ops.policy_loss(x, y, adv)
    assert float(got.kl) == math.inf and torch.equal(got.loss, want.loss)
    assert torch.equal(torch.autograd.grad(got.loss, x)[0], torch.autograd.grad(want.loss, x)[0])
    empty = ops.policy_loss(x[:, :0], y[:, :0], adv)
    (grad,) = torch.autograd.grad(empty.loss, x)
    assert float(empty.loss) == 0 and empty.logps.shape == (2, 0) and not grad.any()


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_gradient_against_differences(dev):
    kw = dict(kl_coef=0.2, clip=(0.3, 0.3), temperature=0.9)
    got, x, _, x64, labels = _policy(dev, (2, 4, 23), torch.float32, has_ref=True, **kw)
    (grad,) = torch.autograd.grad(got.loss, x)
    now = _logps64(_double(x), labels, 0.9)[0].detach()
    g = _gen(3)
    adv = torch.randn(2, 4, generator=g).double()
    noise = 0.25 * torch.randn(2, 4, generator=g)
    for edge in (0.7, 1.3):
        noise = torch.where((noise.exp() - edge).abs() < 1e-3, noise + 0.01, noise)
    old = (now - noise).float().double()
    ref = (now + 0.5 * torch.randn(2, 4, generator=g)).float().double()
    h = 1e-6
    for at in [(0, 0, 3), (1, 2, 22), (0, 3, 0), (1, 1, int(labels[1, 1].clamp(min=0)))]:
        ends = []
        for step in (h, -h):
            moved = x64.detach().clone()
            moved[at] += step
            ends.append(float(policy64(moved, labels, adv, old, ref, **kw)[0]))
        assert abs(float(grad[at]) - (ends[0] - ends[1]) / (2 * h)) < 4e-5 * 15 + 1e-8


# ---------------------------------------------------------------- router balance

ROUTERS = [(1, 1, 1, 1), (1, 5, 8, 2), (2, 33, 60, 4), (3, 257, 64, 8), (1, 70, 16, 16), (2, 9, 7, 3), (1, 40, 256, 8),
           (1, 13, 1000, 5), (5, 300, 128, 1), (2, 21, 96, 6)]


def _router(size, dtype, seed, dev, ties=False):
    g, n, e, _ = size
    x = 2 * torch.randn(g, n, e, generator=_gen(seed))
    if ties:
        x = x.round()
    return x.to(dtype).to(dev).requires_grad_()


def _check_balance(got, want, x, x64, dtype, z_coef=0.0):
    assert got.counts.dtype == torch.int64 and torch.equal(got.counts.cpu(), want[1])
    # Means of probabilities within 1e-5 of themselves; lse within 1e-5, squared.
    _close(got.loss, want[0], 2e-5, 1e-6)
    w = torch.linspace(0.5, 2.0, x.shape[0])
    got.loss.backward(w.to(x.device))
    want[0].backward(w.double())
    # E p (f - f.p) / N with f up to 1 and p up to 1.
    bound = 2 * x.shape[2] / max(x.shape[1], 1) + z_coef * 40
    _close(x.grad, x64.grad, UNIT[dtype], 2e-5 * bound + FLOOR[dtype])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", ROUTERS)
def test_balance_loss_counts_and_gradient(dev, dtype, size):
    x = _router(size, dtype, 0, dev)
    x64 = _double(x)
    _check_balance(ops.router_balance_loss(x, size[3], z_coef=0.01), balance64(x64, size[3], z_coef=0.01), x, x64, dtype, 0.01)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("size", ROUTERS)
def test_balance_ties_go_to_the_lowest_index(dev, size):
    x = _router(size, torch.float32, 1, dev, ties=True)
    x.data[0, 0] = 0.0
    x.data[0, 0, ::2] = -0.0  # equal to 0
    x64 = _double(x)
    _check_balance(ops.router_balance_loss(x, size[3]), balance64(x64, size[3]), x, x64, torch.float32)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("size", ROUTERS)
@pytest.mark.parametrize("given", [False, True])
def test_balance_masked_tokens_and_given_experts(dev, size, given):
    g, n, e, k = size
    x = _router(size, torch.float32, 2, dev).detach()
    mask = torch.rand(g, n, generator=_gen(5)) < 0.6
    mask[-1] = False  # a group without tokens
    x[~mask.to(dev)] = math.nan
    x.requires_grad_()
    ids = torch.randint(0, e, (g, n, k), generator=_gen(6)) if given else None
    x64 = _double(x)
    got = ops.router_balance_loss(x, k, None if ids is None else ids.to(dev), mask.to(dev), z_coef=0.1)
    _check_balance(got, balance64(x64, k, ids, mask, 0.1), x, x64, torch.float32, 0.1)
    assert float(got.loss[-1]) == 0 and not x.grad[~mask.to(dev)].any()


@pytest.mark.parametrize("dev", DEVICES)
def test_balance_shapes_and_strides(dev):
    base = torch.randn(2, 3, 40, 30, generator=_gen(0)).to(dev)
    x64 = base.cpu().double()
    want = balance64(x64.reshape(6, 40, 30), 4)
    got = ops.router_balance_loss(base, 4)
    assert got.loss.shape == (2, 3) and got.counts.shape == (2, 3, 30)
    _close(got.loss.reshape(6), want[0], 2e-5, 1e-6)
    assert torch.equal(got.counts.cpu().reshape(6, 30), want[1])
    flat = ops.router_balance_loss(base[0, 0], 4)
    assert flat.loss.shape == () and flat.counts.shape == (30,)
    _close(flat.loss, want[0][0], 2e-5, 1e-6)
    for view in (base[0, :, ::2, 3:27], base[0].transpose(1, 2), base[:1, 0].expand(3, 40, 30)):
        leaf = view.detach().requires_grad_()
        leaf64 = _double(view)
        _check_balance(ops.router_balance_loss(leaf, 3), balance64(leaf64, 3), leaf, leaf64, torch.float32)


@pytest.mark.parametrize("dev", DEVICES)
def test_balance_masked_experts_and_no_tokens(dev):
    x = torch.randn(1, 6, 12, generator=_gen(0)).to(dev)
    x[..., 5:] = -math.inf
    x.requires_grad_()
    x64 = _double(x)
    got, want = ops.router_balance_loss(x, 2), balance64(x64, 2)
    assert torch.equal(got.counts.cpu(), want[1])
    _close(got.loss, want[0], 2e-5, 1e-6)
    got.loss.sum().backward()
    assert torch.isfinite(x.grad).all() and not x.grad[..., 5:].any()
    empty = torch.zeros(2, 0, 4, device=dev, requires_grad=True)
    got = ops.router_balance_loss(empty, 1)
    assert not got.loss.any() and not got.counts.any()
    got.loss.sum().backward()
    assert empty.grad.shape == empty.shape


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("e,k", [(8, 8), (60, 60), (64, 1), (300, 3)])
def test_balance_of_experts_used_alike(dev, e, k):
    """The loss is top_k and there is nothing to push: the gradient keeps no rounding of the shares."""
    n = 3 * e
    x = _router((1, n, e, k), torch.float32, 0, dev)
    ids = (torch.arange(n)[:, None] * k + torch.arange(k)).remainder(e).unsqueeze(0)  # each expert n k / e times
    got = ops.router_balance_loss(x, k, ids.to(dev))
    assert got.counts.unique().tolist() == [n * k // e]
    _close(got.loss, torch.full((1,), float(k)), 2e-6, 0)
    got.loss.sum().backward()
    if dev == "cuda":
        assert not x.grad.any()
    else:  # the sums of the shares, each within 2^-22 of k, over the tokens
        assert float(x.grad.abs().max()) <= 2e-6 * k / n


@pytest.mark.parametrize("dev", DEVICES)
def test_balance_gradient_against_differences(dev):
    x = _router((1, 9, 10, 2), torch.float32, 3, dev)
    ids = torch.randint(0, 10, (1, 9, 2), generator=_gen(1))
    (grad,) = torch.autograd.grad(ops.router_balance_loss(x, 2, ids.to(dev), z_coef=0.3).loss.sum(), x)
    h = 1e-5
    for at in [(0, 0, 0), (0, 4, 9), (0, 8, 3)]:
        ends = []
        for step in (h, -h):
            moved = x.detach().cpu().double()
            moved[at] += step
            ends.append(float(balance64(moved, 2, ids, z_coef=0.3)[0]))
        assert abs(float(grad[at]) - (ends[0] - ends[1]) / (2 * h)) < 2e-5 * (2 * 10 / 9 + 12) + 1e-9


# ---------------------------------------------------------------- refusals, errors, streams


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x, y = torch.randn(2, 3, 5, device=dev), torch.zeros(2, 3, dtype=torch.long, device=dev)
    ref, adv = torch.zeros(2, device=dev), torch.zeros(2, device=dev)
    for args, kw in [((x[0], y, ref), {}), ((x, y[:, :2], ref), {}), ((x, y.float(), ref), {}), ((x, y, ref[:1]), {}),
                     ((x[:1], y[:1], ref[:1]), {}), ((x.long(), y, ref), {}), ((x[..., :0], y, ref), {}),
                     ((x, y, ref.clone().requires_grad_()), {}), ((x, y, ref), {"beta": 0.0}),
                     ((x, y, ref), {"beta": math.nan}), ((x, y, ref), {"kind": "other"}),
                     ((x, y, ref), {"reduction": "token_mean"}), ((x, y, ref), {"label_smoothing": 0.5}),
                     ((x, y, ref), {"label_smoothing": 0.1, "kind": "hinge"})]:
        with pytest.raises(ValueError):
            ops.preference_loss(*args, **kw)
    for args, kw in [((x, y, adv[:1]), {}), ((x[:0], y[:0], adv[:0]), {}), ((x, y, adv, ref), {}),
                     ((x, y, adv, None, ref), {}), ((x, y, adv), {"kl_coef": 0.1}), ((x, y, adv), {"temperature": 0.0}),
                     ((x, y, adv), {"clip": (1.5, 0.2)}), ((x, y, adv), {"clip": (0.2, -1.0)}),
                     ((x, y, adv), {"reduction": "mean"}), ((x, y, adv.clone().requires_grad_()), {})]:
        with pytest.raises(ValueError):
            ops.policy_loss(*args, **kw)
    for args, kw in [((x[0, 0], 1), {}), ((x, 0), {}), ((x, 6), {}), ((x, 2, y), {}), ((x, 1, None, y[:1]), {}),
                     ((x.long(), 1), {}), ((x, 1, torch.zeros(2, 3, 1, device=dev)), {})]:
        with pytest.raises(ValueError):
            ops.router_balance_loss(*args, **kw)


@pytest.mark.gpu
def test_unsupported_types_and_devices_are_refused_on_the_gpu():
    x, y = torch.randn(2, 3, 5, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    with pytest.raises(TypeError):
        ops.preference_loss(x.double(), y, torch.zeros(2, device="cuda"))
    with pytest.raises(TypeError):
        ops.router_balance_loss(x.double(), 1)
    with pytest.raises(ValueError):
        ops.preference_loss(x, y.cpu(), torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.preference_loss(x, y, torch.zeros(2))
    with pytest.raises(RuntimeError):
        ops.router_balance_loss(torch.zeros(1, 2, 1025, device="cuda"), 1)


def test_out_of_range_ids_raise_on_the_cpu():
    x = torch.randn(2, 3, 5)
    y = torch.tensor([[0, 5, 1], [1, 1, 1]])
    with pytest.raises(ValueError):
        ops.preference_loss(x, y, torch.zeros(2))
    with pytest.raises(ValueError):
        ops.policy_loss(x, -y, torch.zeros(2))
    with pytest.raises(ValueError):
        ops.router_balance_loss(x, 1, y.unsqueeze(-1))


@pytest.mark.gpu
def test_out_of_range_ids_are_left_out_and_reported_on_the_gpu():
    ops.check_device_errors()
    x = torch.randn(2, 3, 5, device="cuda", requires_grad=True)
    y = torch.tensor([[0, 5, 1], [1, -3, 2]], device="cuda")
    ref = torch.zeros(2, device="cuda")
    fine = torch.where((y < 0) | (y > 4), -100, y)
    for call in (lambda y: ops.preference_loss(x, y, ref), lambda y: ops.policy_loss(x, y, ref)):
        want = call(fine)
        (want_grad,) = torch.autograd.grad(want.loss, x)
        ops.check_device_errors()
        got = call(y)
        (grad,) = torch.autograd.grad(got.loss, x)
        with pytest.raises(RuntimeError, match="error 5"):
            ops.check_device_errors()
        assert torch.equal(got.loss, want.loss) and torch.equal(got.logps, want.logps) and torch.equal(grad, want_grad)
    ids = torch.tensor([[[0], [7], [2]]], device="cuda")
    counts = ops.router_balance_loss(x[:1], 1, ids).counts
    with pytest.raises(RuntimeError, match="error 5"):
        ops.check_device_errors()
    assert counts.tolist() == [[1, 0, 1, 0, 0]]


@pytest.mark.gpu
def test_results_repeat_bit_for_bit_and_follow_the_current_stream():
    torch.cuda.synchronize()
    first = None
    side = torch.cuda.Stream()
    for k in range(4):
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            out = []
            got, x, *_ = _preference("cuda", (4, 65, 5003), torch.bfloat16)
            out += [got.loss, got.logps, *torch.autograd.grad(got.loss, x)]
            got, x, *_ = _policy("cuda", (4, 65, 5003), torch.bfloat16, has_ref=True, kl_coef=0.1)
            out += [*got, *torch.autograd.grad(got.loss, x)]
            r = _router((3, 999, 60, 4), torch.bfloat16, 0, "cuda")
            bal = ops.router_balance_loss(r, 4)
            out += [bal.loss, bal.counts, *torch.autograd.grad(bal.loss.sum(), r)]
        torch.cuda.synchronize()
        if first is None:
            first = out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("b", [33, 100, 1026])
def test_many_short_sequences(dev, b):
    got, x, want, x64, _ = _policy(dev, (b, 2, 19), torch.float32, has_ref=True, kl_coef=0.1)
    _check_policy(got, want, 1)
    got.loss.backward()
    want[0].backward()
    _close(x.grad, x64.grad, 4e-5, 4e-5 * 15)
    got, x, want, x64 = _preference(dev, (b, 2, 19), torch.float32)
    _check_preference(got, x, want, x64)
    got.loss.backward()
    want[0].backward()
    _close(x.grad, x64.grad, 4e-5, 4e-6)


@pytest.mark.gpu
def test_gradients_are_not_differentiated_again():
    """Under create_graph the gradients are there; what differentiates them raises and says why."""
    x = torch.randn(2, 3, 50, device="cuda", requires_grad=True)
    y, zero = torch.zeros(2, 3, dtype=torch.long, device="cuda"), torch.zeros(2, device="cuda")
    for loss in (lambda: ops.preference_loss(x, y, zero).loss, lambda: ops.policy_loss(x, y, zero + 1).loss,
                 lambda: ops.router_balance_loss(x, 2).loss.sum()):
        (want,) = torch.autograd.grad(loss(), x)
        (grad,) = torch.autograd.grad(loss(), x, create_graph=True)
        assert torch.equal(grad, want)
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            grad.sum().backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_balance_of_no_groups(dev):
    for shape in [(0, 5, 4), (2, 0, 3, 4), (2, 3, 0, 4)]:
        x = torch.zeros(shape, device=dev, requires_grad=True)
        got = ops.router_balance_loss(x, 2, torch.zeros(*shape[:-1], 2, dtype=torch.long, device=dev),
                                      torch.ones(shape[:-1], dtype=torch.bool, device=dev))
        assert got.loss.shape == shape[:-2] and got.counts.shape == (*shape[:-2], 4) and not got.loss.any()
        got.loss.sum().backward()
        assert x.grad.shape == x.shape


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets():
    """The last rows of logits with more than 2^31 elements, and of rows far apart."""
    v, t = 131072, 8200  # 2.15e9 elements: 4.3 GB of bf16
    x = torch.zeros(2, t, v, device="cuda", dtype=torch.bfloat16)
    x[1, -1, 77] = 3.0
    labels = torch.full((2, t), -100, device="cuda")
    labels[0, 0], labels[1, -1] = 5, 77
    x.requires_grad_()
    got = ops.preference_loss(x, labels, torch.zeros(2, device="cuda"), beta=1.0)
    want = [-math.log(v), 3 - math.log(v - 1 + math.exp(3.0))]
    _close(got.logps, torch.tensor(want), 0, 3e-5)
    (grad,) = torch.autograd.grad(got.loss, x)
    c = 1 / (1 + math.exp(want[0] - want[1]))  # the chosen answer's push
    assert abs(float(grad[1, -1, 77]) + 0 - (c * (1 - math.exp(want[1])))) < 2**-8 * c
    assert abs(float(grad[0, 0, 5]) + c) < 2**-8 * c
    assert int((grad[:, 1:-1] != 0).sum()) == 0


@pytest.mark.gpu
def test_losses_under_graph_capture():
    labels = _labels(4, 9, 700, 1).cuda()
    x = _logits(4, 9, 700, torch.bfloat16, 0, device="cuda")
    ref, adv = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    r = _router((2, 65, 16, 2), torch.float32, 0, "cuda")

    def step():
        a, b, c = ops.preference_loss(x, labels, ref), ops.policy_loss(x, labels, adv), ops.router_balance_loss(r, 2)
        return [a.loss, b.loss, c.loss, c.counts, *torch.autograd.grad(a.loss + b.loss, x), *torch.autograd.grad(c.loss.sum(), r)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [w.clone() for w in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_native_forms_are_the_ones_that_run():
    assert set(losses.PAIR_LOSSES) == {"sigmoid", "hinge", "ipo"}
    with torch.no_grad():
        got = ops.preference_loss(torch.zeros(2, 1, 4), torch.zeros(2, 1, dtype=torch.long), torch.zeros(2))
    assert not got.loss.requires_grad and abs(float(got.loss) - math.log(2.0)) < 1e-6


# ---------------------------------------------------------------- gradients entry by entry
# Slack that is the same for a whole row hides all of it but the label's entry: most entries are a coefficient times a
# probability of 1e-5 and less.  So each entry has a bound of its own: 4e-5 of (probability + 1 at the label) times the
# row's coefficient bound, which covers the probability's and the coefficient's own error, and one rounding to the type:
# half a unit in the last place (2^-8 bf16, 2^-11 fp16), half the smallest step below fp16's normal range, and what 32
# bits hold no more digits of (1e-36).

HALF_UNIT = {torch.float32: 0.0, torch.bfloat16: 2**-8, torch.float16: 2**-11}
HALF_STEP = {torch.float32: 1e-36, torch.bfloat16: 1e-36, torch.float16: 2**-25}


def _check_entries(grad, want, x64, labels, row_bound, temperature=1.0):
    """*row_bound*: ``(B, T)``, the size of the terms that a row's coefficient adds up, with all factors."""
    keep = labels != -100
    p = torch.softmax(x64.detach() / temperature, -1)
    p.scatter_add_(2, labels.clamp(min=0)[..., None], torch.ones_like(labels, dtype=p.dtype)[..., None])
    size = want.abs()
    slack = 4e-5 * torch.where(keep, row_bound / temperature, 0.0)[..., None] * p
    off = (grad.detach().double().cpu() - want).abs() - slack - HALF_UNIT[grad.dtype] * (size + slack)
    off = torch.where(keep[..., None], off - HALF_STEP[grad.dtype], off)
    assert float(off.max()) <= 0, (float(off.max()), int((off > 0).sum()), off.numel())
    assert float(size[keep].gt(0).double().mean()) > 0.2  # enough of it is there to be compared


def _policy_row_bound(x64, labels, adv, old, ref, kl_coef, temperature, weight):
    logps = _logps64(x64.detach(), labels, temperature)[0]
    adv = adv.double() if adv.dim() == 2 else adv.double()[:, None]
    size = adv.abs() * (1.0 if old is None else (logps - old.double()).exp())
    if kl_coef:
        size = size + kl_coef * ((ref.double() - logps).exp() + 1)
    return size * weight


def _policy_entries(dev, size, dtype, layout, scale=1.0, adv_scale=1.0, reduction="token_mean", temperature=1.0, kl_coef=0.1):
    b, t, v = size
    labels, g = _labels(b, t, v, 1), _gen(3)
    x = _logits(b, t, v, dtype, 0, layout, dev)
    x64 = _double(x)
    now = _logps64(x64.detach(), labels, temperature)[0]
    adv = adv_scale * (0.5 + torch.rand(b, t, generator=g))
    noise = 0.15 * (2 * torch.rand(b, t, generator=g) - 1)  # within the clip: every row that counts has a gradient
    old, ref = (now - noise).float(), (now + 0.5 * torch.randn(b, t, generator=g)).float()
    kw = dict(kl_coef=kl_coef, temperature=temperature, reduction=reduction)
    got = ops.policy_loss(x, labels.to(dev), adv.to(dev), old.to(dev), ref.to(dev), **kw)
    want = policy64(x64, labels, adv.double(), old.double(), ref.double(), **kw)
    keep = labels != -100
    weight = {"token_mean": (1 / keep.sum().clamp(min=1)).expand(b, t), "sum": torch.ones(b, t),
              "sequence_mean": (1 / keep.sum(1, keepdim=True).clamp(min=1) / b).expand(b, t)}[reduction].double()
    bound = _policy_row_bound(x64, labels, adv, old, ref, kl_coef, temperature, weight) * scale
    (want64,) = torch.autograd.grad(want[0] * scale, x64)
    return got, x, want64, x64, labels, bound, temperature


ENTRY_SIZES = [(3, 17, 1001), (2, 4, 8192), (2, 3, 9001), (2, 9, 32003), (1, 3, 40003), (1, 2, 70001), (1, 2, 131072)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("size", ENTRY_SIZES)
@pytest.mark.parametrize("dtype,scale,adv_scale", [
    (torch.float16, 65536.0, 1 / 6144),  # a scaled loss over 6144 tokens: unscaled, most entries are below fp16's range
    (torch.float16, 2.0**-13, 65536.0 * 4),  # unscaled, the labels' entries are above it
    (torch.bfloat16, 1 / 3, 1.0), (torch.float32, 1 / 3, 1.0)])  # accumulation over three micro-batches
def test_policy_gradient_of_a_scaled_loss_is_rounded_once(dev, size, dtype, scale, adv_scale):
    kl_coef = 0.1 * adv_scale
    got, x, *want = _policy_entries(dev, size, dtype, "shifted", scale, adv_scale, "sum", kl_coef=kl_coef)
    for keep in (True, False):  # the gradient kept by the forward, and the one computed again
        (grad,) = torch.autograd.grad(got.loss * scale, x, retain_graph=keep)
        _check_entries(grad, *want)


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_gradient_of_a_loss_times_nothing(dev):
    """A loss gradient of 0 gives zeros, one of NaN reaches the rows that count and no other."""
    got, x, _, _, labels, _, _ = _policy_entries(dev, (3, 17, 1001), torch.bfloat16, "shifted")
    assert not torch.autograd.grad(got.loss * 0.0, x, retain_graph=True)[0].any()
    got, x, *_ = _policy_entries(dev, (3, 17, 1001), torch.bfloat16, "shifted")
    (grad,) = torch.autograd.grad(got.loss, x, torch.tensor(math.nan, device=dev))
    keep = (labels != -100).to(dev)
    assert grad[keep].isnan().all() and not grad[~keep].any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_temperature_is_applied_in_32_bits(dev, dtype):
    """Logits over a temperature that is no power of two: rounded to a half type they would be off by 2^-9 of 20."""
    b, t, v = 2, 7, 301
    labels, x = _labels(b, t, v, 1), _logits(b, t, v, dtype, 0, device=dev, spread=5.0).detach()
    got = ops.policy_loss(x, labels.to(dev), torch.zeros(b, device=dev), temperature=0.7)
    _close(got.logps, _logps64(_double(x).detach(), labels, 0.7)[0], 2**-22, 1e-5)



@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("layout", ["plain", "shifted"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", ENTRY_SIZES)
def test_policy_gradient_entry_by_entry(dev, layout, dtype, size):
    got, x, *want = _policy_entries(dev, size, dtype, layout)
    _check_entries(torch.autograd.grad(got.loss, x)[0], *want)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [{"reduction": "sum"}, {"reduction": "sequence_mean"}, {"temperature": 0.5}, {"kl_coef": 0.0}])
def test_policy_gradient_forms_entry_by_entry(dev, dtype, kw):
    got, x, *want = _policy_entries(dev, (3, 17, 1001), dtype, "plain", **kw)
    _check_entries(torch.autograd.grad(got.loss, x)[0], *want)


@pytest.mark.parametrize("dev", DEVICES)
def test_forward_mode_derivatives_are_right_or_refused(dev):
    """The kernels have none and say so, whether or not the primal needs a gradient; the CPU forms have them."""
    import torch.autograd.forward_ad as fwd

    g = _gen(0)
    x, y, adv = torch.randn(2, 3, 5, generator=g).to(dev), torch.zeros(2, 3, dtype=torch.long, device=dev), torch.ones(2, device=dev)
    w, (cos, sin) = torch.ones(4, device=dev), torch.ones(2, 3, 2, device=dev)
    q, turn = torch.randn(1, 3, 2, 4, generator=g).to(dev), torch.randn(1, 3, 2, 4, generator=g).to(dev)
    calls = [(lambda z: ops.preference_loss(z, y, adv).loss, x), (lambda z: ops.policy_loss(z, y, adv, adv[:, None] - torch.full_like(x[..., 0], 2.6), clip=(1.0, 1e9)).loss, x),
             (lambda z: ops.router_balance_loss(z, 2).loss.sum(), x),
             (lambda z: (ops.qk_norm_rope(z, q, w, w, cos, sin)[0] * turn).sum(), q),
             (lambda z: (ops.qk_norm_rope(q, q, z, w, cos, sin)[0] * turn).sum(), w),
             (lambda z: ops.policy_loss(x, y, z).loss, adv), (lambda z: ops.policy_loss(x, y, adv, None, z, kl_coef=1.0).loss, -x[..., 0].abs()),
             (lambda z: ops.preference_loss(x, y, z).loss, adv)]
    for call, at in calls:
        for wants in (False, True):
            if wants and call in [c for c, _ in calls[5:]]:
                continue  # a constant that needs a gradient is refused anyway
            way = torch.randn(at.shape, generator=g).to(dev)
            with fwd.dual_level():
                z = fwd.make_dual(at.detach().clone().requires_grad_(wants), way)
                if dev == "cuda":
                    with pytest.raises(NotImplementedError):
                        call(z)
                    call(at)  # no tangent, no refusal
                    continue
                got = fwd.unpack_dual(call(z)).tangent
            h = 1e-3
            ends = [float(call(at + s * h * way)) for s in (1, -1)]
            # Central differences in 32 bits: 1e-6 of losses below 5 over 2 h, and h^2 of a third derivative below 20.
            assert abs(float(got.detach()) - (ends[0] - ends[1]) / (2 * h)) < 5e-3


def test_native_entry_points_refuse_tensors_without_memory():
    """Tensors of functional transforms have none; they are turned away before anything is read."""
    try:
        native = ops.native()
    except RuntimeError:
        pytest.skip("the extension is not built")
    x, y, err = torch.randn(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.zeros(1, dtype=torch.int32)
    w = torch.ones(4)
    tables = torch.ones(3, 2), torch.zeros(3, 2)
    calls = [lambda z: native.preference_loss(z, y, torch.zeros(2), "sigmoid", 0.1, 0.0, False, "mean", -100, err)[0],
             lambda z: native.policy_loss(z, y, torch.zeros(2), None, None, 0.2, 0.2, 0.0, 1.0, "sum", -100, err)[0],
             lambda z: native.balance_loss(z, None, None, 2, 0.0, err)[0].sum(),
             lambda z: native.qk_norm_rope(z[:, :, None, :4], z[:, :, None, :4], w, w, *tables, None, 1e-6, err)[0].sum()]
    for call in calls:
        with pytest.raises(NotImplementedError):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(NotImplementedError):
            torch.func.grad(call)(x)
        with pytest.raises(NotImplementedError):
            torch.func.vmap(call)(x[None])


def _four_losses(x, y, bad):
    """One graph of each operator, with labels, ids or positions off the end where *bad*."""
    w, tables = torch.ones(4, device="cuda", requires_grad=True), (torch.ones(3, 2, device="cuda"), torch.zeros(3, 2, device="cuda"))
    ref, off = torch.zeros(2, device="cuda"), 99 if bad else 0
    q = x[:, :, None, :4]
    return [ops.preference_loss(x, y + off, ref).loss, ops.policy_loss(x, y + off, ref + 1).loss,
            ops.policy_loss(x, y + off, ref + 1).logps.sum(),
            ops.router_balance_loss(x, 1, y[..., None] + off, z_coef=0.1).loss.sum(),
            ops.qk_norm_rope(q, q, w, w, *tables, torch.arange(3, device="cuda") + off)[0].sum()]


@pytest.mark.gpu
def test_a_reported_index_leaves_the_graphs_alone():
    """A bad index is left out and reported; the backward of its graph and of the others on the device goes on."""
    ops.check_device_errors()
    x = torch.randn(2, 3, 5, device="cuda", requires_grad=True)
    y = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    good, bad = _four_losses(x, y, False), _four_losses(x, y, True)
    with pytest.raises(RuntimeError, match="error 5"):
        ops.check_device_errors()
    for loss in good:
        (grad,) = torch.autograd.grad(loss, x)
        assert torch.isfinite(grad).all() and grad.any()
    for loss in bad:
        assert torch.isfinite(torch.autograd.grad(loss, x)[0]).all()
    with pytest.raises(RuntimeError, match="error 5"):  # the backward meets the same labels and positions
        ops.check_device_errors()


@pytest.mark.gpu
def test_a_device_first_used_in_inference_mode_trains_and_reports():
    word = ops._err_words.pop(torch.cuda.current_device(), None)
    try:
        x = torch.randn(2, 3, 5, device="cuda", requires_grad=True)
        y = torch.zeros(2, 3, dtype=torch.long, device="cuda")
        with torch.inference_mode():
            ops.policy_loss(x, y, torch.ones(2, device="cuda"))
        for loss in _four_losses(x, y, False):
            assert torch.autograd.grad(loss, x)[0].any()
        ops.check_device_errors()
        ops.policy_loss(x, y + 9, torch.ones(2, device="cuda"))
        with pytest.raises(RuntimeError, match="error 5"):
            ops.check_device_errors()
        ops.check_device_errors()
    finally:
        if word is not None:
            ops._err_words[torch.cuda.current_device()] = word


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_label_of_the_lowest_logit_keeps_a_finite_log_probability(dev, dtype):
    """A mask that put the type's lowest value where a label points: its log-probability is that value, not -inf."""
    low = torch.finfo(dtype).min
    x = _logits(2, 3, 40, dtype, 0, device=dev).detach()
    x[:, 1, 5] = low
    labels = torch.full((2, 3), -100)
    labels[:, 1] = 5
    want = _logps64(_double(x).detach(), labels)[0]
    assert torch.isfinite(want.float()).all()
    got = ops.policy_loss(x, labels.to(dev), torch.ones(2, device=dev))
    _close(got.logps, want, 2**-22, 1e-5)
    got = ops.preference_loss(x.requires_grad_(), labels.to(dev), torch.zeros(2, device=dev))
    want_loss, want = preference64(_double(x).detach(), labels, torch.zeros(2).double())
    _close(got.logps, want, 2**-22, 1e-5)
    assert torch.isfinite(got.loss)
    _close(got.loss, want_loss, 1e-5, 0.1 * 2 * (1e-5 + 2**-22 * abs(low)))


def test_constants_of_64_bit_logits_keep_their_digits():
    x = torch.randn(2, 3, 11, generator=_gen(0), dtype=torch.float64)
    y, g = torch.randint(0, 11, (2, 3), generator=_gen(1)), _gen(2)
    ref = -2000 + torch.randn(2, generator=g, dtype=torch.float64)  # 32 bits hold these to 1e-4
    _close(ops.preference_loss(x, y, ref).loss, preference64(x, y, ref)[0], 1e-12, 0)
    now = _logps64(x, y)[0]
    adv, old, ref = torch.randn(2, generator=g, dtype=torch.float64), now + 1 / 3, now - 1 / 7
    got, want = ops.policy_loss(x, y, adv, old, ref, kl_coef=0.1), policy64(x, y, adv, old, ref, kl_coef=0.1)
    for a, b in zip(got, want):
        _close(a, b, 1e-12, 1e-15)
