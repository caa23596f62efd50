"""Token scores against ``log_softmax`` in 64 bits.

Tolerances: an exponent t = (x - max) log2(e) / temperature is off by |t| 2^-23 (a subtraction and a product in fp32),
and terms with |t| > 64 do not count in fp32 sums, so every exponential is off by less than 64 2^-23 + 2^-22 < 1e-5
relative; so are sums of them, and logarithms of the sums absolutely. An entropy adds t's own error within the same
bound, a log-probability a rounding of its value. Gradients add the rounding to their type.
"""

import math

import pytest
import torch

from dattri_llm_b200 import ops
from dattri_llm_b200.ops.scores import TokenScores

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TOL = 2e-5
IGNORE = -100


def expected(logits, labels, top_k, temperature, g_logps=None, g_entropy=None):
    x = logits.detach().double().cpu().requires_grad_(True)
    labels = labels.cpu()
    valid = labels != IGNORE
    safe = x.masked_fill(~valid.unsqueeze(-1), 0.0)
    logs = torch.log_softmax(safe / temperature, -1)
    p = logs.exp()
    entropy = -(p * logs.masked_fill(p == 0, 0.0)).sum(-1).masked_fill(~valid, 0.0)
    logps = logs.gather(2, labels.clamp(min=0).unsqueeze(-1)).squeeze(-1).masked_fill(~valid, 0.0)
    ids = torch.sort(safe.detach(), dim=-1, descending=True, stable=True).indices[..., :top_k]
    top = logs.detach().gather(2, ids).masked_fill(~valid.unsqueeze(-1), 0.0)
    ids = ids.masked_fill(~valid.unsqueeze(-1), -1)
    grad = None
    if g_logps is not None:
        # the derivative as a formula: a masked entry's -inf has none through the product above
        ge, gl = g_entropy.double().cpu().unsqueeze(-1), g_logps.double().cpu().unsqueeze(-1)
        one = torch.zeros_like(p).scatter_(2, labels.clamp(min=0).unsqueeze(-1), 1.0)
        finite = logs.masked_fill(p == 0, 0.0)
        grad = (gl * (one - p) - ge * p * (finite + entropy.unsqueeze(-1))) / temperature
        grad = grad.masked_fill(~valid.unsqueeze(-1), 0.0).detach()
        size = ((gl.abs() + ge.abs() * (finite.abs() + entropy.unsqueeze(-1))) * p + gl.abs() * one).detach() / temperature
        return TokenScores(logps.detach(), entropy.detach(), top, ids), grad, size
    return TokenScores(logps.detach(), entropy.detach(), top, ids), None, None


def close(got, want, tol=TOL):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) | torch.isnan(want)
    off = torch.where(same, 0.0, (got - want).abs())
    assert (off <= tol * (1 + torch.where(torch.isfinite(want), want.abs(), 0.0))).all(), off.max()


def check(logits, labels, top_k=5, temperature=1.0, grad=True):
    logits = logits.detach().requires_grad_(grad)
    got = ops.token_scores(logits, labels, top_k=top_k, temperature=temperature)
    gl = ge = None
    if grad:
        gen = torch.Generator().manual_seed(5)
        gl = torch.randn(labels.shape, generator=gen).to(logits.device)
        ge = torch.randn(labels.shape, generator=gen).to(logits.device)
    want, dx, size = expected(logits, labels, top_k, temperature, gl, ge)
    close(got.logps, want.logps)
    close(got.entropy, want.entropy)
    close(got.top_logps, want.top_logps)
    assert torch.equal(got.top_ids.cpu(), want.top_ids)
    assert not got.top_logps.requires_grad
    if grad:
        (d,) = torch.autograd.grad((got.logps, got.entropy), logits, (gl, ge))
        assert d.dtype == logits.dtype and d.shape == logits.shape
        half = torch.finfo(d.dtype).eps / 2
        # below its normal range a type's step is fixed: half of the smallest value; and an exponential below fp32's
        # normal range is 0: its probability is under 2^-126, with a coefficient under |a| + |b| (200 + H), H < 12
        floor = torch.finfo(d.dtype).smallest_normal * torch.finfo(d.dtype).eps
        floor = floor + 2.0 ** -126 * (gl.abs() + ge.abs() * 212).double().cpu().unsqueeze(-1) / temperature
        assert ((d.double().cpu() - dx).abs() <= half * dx.abs() + TOL * size + floor).all()
        assert (d[labels == IGNORE] == 0).all()
    return got


def make(b, t, v, dtype, device, *, seed=0, slack=0, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, t + slack, v, generator=gen) * spread).to(dtype).to(device)[:, :t]
    labels = torch.randint(0, v, (b, t), generator=gen)
    labels[torch.rand(b, t, generator=gen) < 0.25] = IGNORE
    return x, labels.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [1, 7, 33, 256, 1000, 6151, 32003])
def test_against_64_bits(device, dtype, v):
    x, labels = make(2, 9, v, dtype, device)
    check(x, labels, top_k=min(5, v))
    check(x, labels, top_k=min(32, v), temperature=0.7)
    check(x, labels, top_k=0, temperature=2.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("v", [515, 8191])
def test_slices_and_other_strides(device, v):
    x, labels = make(3, 5, v + 3, torch.bfloat16, device, slack=1)
    check(x[..., 1:v + 1], labels.clamp(max=v - 1))  # rows that start at odd places
    check(x.transpose(1, 2).contiguous().transpose(1, 2)[..., :v], labels.clamp(max=v - 1))
    check(x.transpose(0, 1), labels.t().clamp(max=v))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("v", [40, 300, 9001])
def test_equal_logits_go_by_the_lowest_index(device, v):
    x = torch.zeros(1, 6, v, device=device, dtype=torch.bfloat16)
    x[0, 1, 0::2] = -0.0  # equal to 0
    x[0, 2, v // 2:] = 1
    x[0, 3] = torch.arange(v, device=device) % 3
    x[0, 4] = -torch.arange(v, device=device) // 16
    x[0, 5, -40:] = torch.arange(40, device=device, dtype=torch.bfloat16) % 20 + 1
    labels = torch.arange(6, device=device).unsqueeze(0)
    check(x, labels, top_k=32)
    check(x, labels, top_k=1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("v", [64, 700, 9001])
def test_masked_vocabularies(device, v):
    for low in (-math.inf, torch.finfo(torch.bfloat16).min):
        x, labels = make(1, 6, v, torch.bfloat16, device, seed=v)
        labels[:] = 3
        x[:, 0, 10:] = low
        x[:, 1, :-1] = low
        x[:, 2, 3] = low  # the label itself
        x[:, 3, 3:] = low
        x[:, 4] = low  # nothing is left, or all are alike
        got = check(x[:, :4], labels[:, :4], top_k=20)
        assert torch.isinf(got.logps[0, 2]) == math.isinf(low)
        last = ops.token_scores(x[:, 4:5], labels[:, 4:5], top_k=20)
        assert torch.equal(last.top_ids[0, 0].cpu(), torch.arange(20))
        if math.isinf(low):
            assert torch.isnan(last.logps).all() and torch.isnan(last.entropy).all()
        else:
            close(last.entropy, torch.full((1, 1), math.log(v), dtype=torch.float64))


@pytest.mark.parametrize("device", DEVICES)
def test_ignored_rows_are_not_read_and_bad_rows_stay_alone(device):
    x, labels = make(2, 8, 4099, torch.float32, device)
    labels[:] = 1
    x[0, 2] = math.nan
    labels[0, 2] = IGNORE
    x[1, 5] = math.inf
    labels[1, 5] = IGNORE
    check(x, labels)
    labels[0, 2] = 7  # a row of NaN that counts
    x[0, 2] = torch.arange(4099, device=device, dtype=torch.float32)
    x[0, 2, 77] = math.nan
    got = ops.token_scores(x, labels, top_k=3)
    assert torch.isnan(got.logps[0, 2]) and torch.isnan(got.entropy[0, 2]) and torch.isnan(got.top_logps[0, 2]).all()
    assert got.top_ids[0, 2].tolist() == [77, 4098, 4097]
    assert torch.isfinite(got.logps[0, 3:]).all() and torch.isfinite(got.logps[1]).all()
    labels[:] = IGNORE
    got = ops.token_scores(x, labels, top_k=3)
    assert not got.logps.any() and not got.entropy.any() and not got.top_logps.any() and (got.top_ids == -1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_no_tokens_and_no_sequences(device):
    for shape in ((0, 4), (4, 0)):
        x = torch.zeros(*shape, 50, device=device, requires_grad=True)
        got = ops.token_scores(x, torch.zeros(shape, dtype=torch.long, device=device), top_k=2)
        assert got.logps.shape == shape and got.top_ids.shape == (*shape, 2)
        (got.logps.sum() + got.entropy.sum()).backward()
        assert x.grad.shape == x.shape


@pytest.mark.parametrize("device", DEVICES)
def test_one_gradient_alone_and_differences(device):
    x, labels = make(1, 4, 130, torch.float32, device)
    x.requires_grad_(True)
    for pick in (0, 1):
        got = ops.token_scores(x, labels, temperature=1.3)[pick]
        (d,) = torch.autograd.grad(got.sum(), x)
        gen = torch.Generator().manual_seed(1)
        way = torch.randn(x.shape, generator=gen).double()
        h = 1e-4
        up, down = (expected((x.detach().double().cpu() + s * h * way), labels, 0, 1.3)[0][pick].sum() for s in (1, -1))
        slope = (d.double().cpu() * way).sum()
        # central differences in 64 bits: off by h^2 times third derivatives of order one
        assert abs(slope - (up - down) / (2 * h)) <= 1e-5 * (1 + d.double().cpu().abs().sum())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, labels = make(2, 3, 40, torch.float32, device)
    for kw in ({"top_k": 33}, {"top_k": -1}, {"temperature": 0.0}, {"temperature": math.inf}):
        with pytest.raises(ValueError):
            ops.token_scores(x, labels, **kw)
    with pytest.raises(ValueError, match="top_k"):
        ops.token_scores(x[..., :8], labels.clamp(max=7), top_k=9)
    with pytest.raises(ValueError):
        ops.token_scores(x[0], labels)
    with pytest.raises(ValueError):
        ops.token_scores(x, labels.float())
    with pytest.raises(ValueError):
        ops.token_scores(x, labels[:, :2])
    labels[1, 1] = 40
    if device == "cpu":
        with pytest.raises(ValueError, match="labels"):
            ops.token_scores(x, labels)
        return
    got = ops.token_scores(x, labels, top_k=2)
    assert got.logps[1, 1] == 0 and (got.top_ids[1, 1] == -1).all()
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_device_errors()
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        y = x.clone().requires_grad_(True)
        (d,) = torch.autograd.grad(ops.token_scores(y, labels.clamp(max=39)).logps.sum(), y, create_graph=True)
        d.sum().backward()


@pytest.mark.gpu
def test_another_stream_and_a_captured_call():
    x, labels = make(2, 7, 5000, torch.bfloat16, "cuda")
    want = ops.token_scores(x, labels, top_k=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.token_scores(x, labels, top_k=4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        held = ops.token_scores(y, labels, top_k=4)
    y.copy_(x)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want, strict=True))


@pytest.mark.gpu
def test_many_rows_and_long_ones_agree_with_themselves():
    """The largest vocabularies, against torch in fp32 on the device: rows of 131,000 entries in every type."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, labels = make(1, 3, 131071, dtype, "cuda", spread=2.0)
        check(x, labels, top_k=32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logits_far_from_zero(device, dtype):
    """Where neighbouring numbers of the type are further apart than any exponential reaches, and at the ends of its range."""
    top = torch.finfo(dtype).max
    x, labels = make(1, 6, 2051, dtype, device)
    labels[:] = 5
    for row, at in enumerate((1e4, -1e4, 6e4, top, -top, 300.0)):
        x[0, row] = at
        steps = torch.randint(0, 4, (2051,), generator=torch.Generator().manual_seed(row)).to(device)
        for _ in range(3):  # one to three representable numbers below it, or above where it is the lowest
            lower = torch.nextafter(x[0, row], torch.full_like(x[0, row], top if row == 4 else -top))
            x[0, row] = torch.where(steps > 0, lower, x[0, row])
            steps -= 1
    check(x, labels, top_k=32, grad=False)
    check(x, labels, top_k=0, temperature=7.0, grad=False)


@pytest.mark.parametrize("device", DEVICES)
def test_alternatives_crowded_into_few_places(device):
    """The best logits next to one another, and more equal ones than a row's short list holds."""
    for v in (600, 9001, 40000):
        x, labels = make(1, 5, v, torch.bfloat16, device)
        labels[:] = 0
        x[0, 0, 8:48] = torch.arange(40, device=device, dtype=torch.bfloat16) + 20
        x[0, 1, v // 2:] = 30.0
        x[0, 2, ::3] = 25.0
        x[0, 3, -33:] = 40.0
        x[0, 4] = -math.inf
        x[0, 4, 7] = 1.0
        check(x[:, :4], labels[:, :4], top_k=32)
        got = ops.token_scores(x[:, 4:], labels[:, 4:], top_k=5)
        assert got.top_ids[0, 0].tolist() == [7, 0, 1, 2, 3] and got.entropy[0, 0] == 0


def test_launch_checks_name_a_bad_label():
    from dattri_llm_b200.ops import checks

    labels = torch.tensor([[0, IGNORE, 9]])
    checks.VALIDATORS["token_scores"]((torch.zeros(1, 3, 10), labels, 0, 1.0, IGNORE, None), {})
    with pytest.raises(ValueError, match="token_scores"):
        checks.VALIDATORS["token_scores"]((torch.zeros(1, 3, 9), labels, 0, 1.0, IGNORE, None), {})


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [148 * 32 - 4, 148 * 32])
def test_middle_rows_by_warps_and_by_blocks(rows):
    """Rows of 9,001 logits, few enough for a block to each and many enough for a warp."""
    gen = torch.Generator().manual_seed(rows)
    logits = (torch.randn(4, rows // 4, 9001, generator=gen) * 3).to(torch.bfloat16)
    labels = torch.randint(0, 9001, (4, rows // 4), generator=gen)
    got = ops.token_scores(logits.cuda(), labels.cuda(), top_k=7)
    cut = (slice(None), slice(0, 40))
    logs = torch.log_softmax(logits[cut].double(), -1)
    want = logs.gather(2, labels[cut].unsqueeze(-1)).squeeze(-1)
    assert ((got.logps[cut].cpu().double() - want).abs() <= TOL * (1 + want.abs())).all()
    entropy = -(logs.exp() * logs).sum(-1)
    assert ((got.entropy[cut].cpu().double() - entropy).abs() <= TOL * (1 + entropy)).all()
    ids = torch.sort(logits[cut].double(), dim=-1, descending=True, stable=True).indices[..., :7]
    assert torch.equal(got.top_ids[cut].cpu(), ids)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [1000, 20000])
def test_rows_further_apart_than_32_bits_count(v):
    """Two rows 2^31 elements apart: their scores and gradients are those of the rows side by side."""
    far = torch.zeros(2**31 + v, dtype=torch.bfloat16, device="cuda").as_strided((1, 2, v), (0, 2**31, 1))
    near, labels = make(1, 2, v, torch.bfloat16, "cuda")
    far.copy_(near)
    got = []
    for x in (far, near):
        x = x.detach().requires_grad_(True)
        r = ops.token_scores(x, labels, top_k=3)
        got.append((r.logps, r.entropy, r.top_logps, r.top_ids, torch.autograd.grad((r.logps.sum() + r.entropy.sum()), x)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*got, strict=True))
