"""RMS norm of q / k heads with rotation against its definition in 64 bits.

Tolerances.  In 32 bits a sum of squares of up to 512 terms and its root are within ``2e-6`` of
themselves; a rotated element is a sum of two products below ``4 |w| |n|`` (``|n| <= sqrt(D)``),
each a few roundings off: ``1e-6`` of ``8 sqrt(D)``.  Half types add a unit of the result
(``2^-8`` bf16, ``2^-10`` fp16 allowed, half of it possible).  A weight gradient sums tokens x
heads terms, each within ``2e-6`` of its size: their absolute sum bounds the error.
"""

import math

import pytest
import torch

from dattri_llm_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
UNIT = {torch.float32: 1e-6, torch.bfloat16: 2**-8, torch.float16: 2**-10}
EPS = 1e-6

# (B, T, Hq, Hk, D, R)
SIZES = [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 77, 8, 1, 128, 128), (3, 5, 6, 3, 96, 48), (2, 9, 7, 7, 80, 40),
         (1, 4, 3, 2, 256, 64), (1, 2, 2, 1, 512, 512), (2, 3, 2, 1, 30, 10), (1, 6, 4, 4, 62, 62), (2, 33, 5, 1, 192, 96),
         (1, 3, 2, 2, 64, 0), (1, 2, 1, 3, 34, 4)]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tables(n, r):
    half = r // 2
    ang = torch.outer(torch.arange(n, dtype=torch.float64), 1.0 / (10000.0 ** (torch.arange(half, dtype=torch.float64) / max(half, 1))))
    return ang.cos().float(), ang.sin().float()


def rotated64(x, w, cos, sin, at):
    """The definition: normalise, scale, turn the pairs (i, i + R / 2) of the first R elements as complex numbers."""
    half = cos.shape[1]
    y = x / ((x ** 2).mean(-1, keepdim=True) + EPS).sqrt() * w
    turn = torch.complex(cos.double(), sin.double())[at][:, :, None]
    z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
    return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)


def _inputs(size, dtype, wdtype, dev, layout="plain", seed=0):
    b, t, hq, hk, d, r = size
    g = _gen(seed)
    if layout == "projection":  # slices of one projection's output, at an odd offset where the width allows it
        x = torch.randn(b, t, (hq + 2 * hk) * d, generator=g).to(dtype).to(dev)
        q, k = x[..., :hq * d].view(b, t, hq, d), x[..., hq * d:(hq + hk) * d].view(b, t, hk, d)
    elif layout == "heads_first":
        q, k = (torch.randn(b, h, t, d, generator=g).to(dtype).to(dev).transpose(1, 2) for h in (hq, hk))
    elif layout == "odd":
        q, k = (torch.randn(b, t, h, d + 3, generator=g).to(dtype).to(dev)[..., 1:d + 1] for h in (hq, hk))
    elif layout == "strided":
        q, k = (torch.randn(b, t, h, d, 2, generator=g).to(dtype).to(dev)[..., 0] for h in (hq, hk))
    else:
        q, k = (torch.randn(b, t, h, d, generator=g).to(dtype).to(dev) for h in (hq, hk))
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(wdtype).to(dev).requires_grad_() for _ in range(2))
    return q.detach().requires_grad_(), k.detach().requires_grad_(), qw, kw


def _run(size, dtype, wdtype, dev, layout="plain", positions=None, table=None, grads="heads_first"):
    b, t, hq, hk, d, r = size
    leaves = _inputs(size, dtype, wdtype, dev, layout)
    cos, sin = _tables(table or t, r)
    q, k = ops.qk_norm_rope(*leaves, cos.to(dev), sin.to(dev), None if positions is None else positions.to(dev), eps=EPS)
    assert q.dtype == dtype and q.is_contiguous() and k.is_contiguous()
    at = (torch.arange(t) if positions is None else positions).expand(b, t)
    wide = [x.detach().cpu().double().requires_grad_() for x in leaves]
    want = [rotated64(x, w, cos, sin, at) for x, w in zip(wide[:2], wide[2:])]
    g = _gen(7)
    outer = [torch.randn(b, h, t, d, generator=g).to(dtype).transpose(1, 2) for h in (hq, hk)]
    if grads == "contiguous":
        outer = [o.contiguous() for o in outer]
    torch.autograd.backward([q, k], [o.to(dev) for o in outer])
    torch.autograd.backward(want, [o.double() for o in outer])
    return (q, k), want, leaves, wide, outer


def _close(got, want, rtol, atol):
    torch.testing.assert_close(got.detach().double().cpu(), want.detach().double(), rtol=rtol, atol=atol)


def _check(size, dtype, got, want, leaves, wide, outer):
    b, t, hq, hk, d, r = size
    for y, y64 in zip(got, want):
        _close(y, y64, UNIT[dtype], 1e-6 * 8 * math.sqrt(d))
    for i in range(2):
        x, x64, w, w64 = leaves[i], wide[i], leaves[i + 2], wide[i + 2]
        assert x.grad.dtype == x.dtype and w.grad.dtype == w.dtype
        # dx = r (dy w - n mean(dy w n)), |dy w| below 12, r = 1 / |x|: bounded by 4e-6 of 12 r (1 + sqrt(D)).
        rms = (x64.detach() ** 2).mean(-1).sqrt().min() + math.sqrt(EPS) if x64.numel() else torch.tensor(1.0)
        _close(x.grad, x64.grad, UNIT[dtype], 4e-6 * 12 * float(1 / rms) * (1 + math.sqrt(d)))
        n = x64.detach() / ((x64.detach() ** 2).mean(-1, keepdim=True) + EPS).sqrt()
        size_of_sum = (n.abs() * outer[i].double().abs().amax(-1, keepdim=True) * 2).sum((0, 1, 2)).max() if n.numel() else 0.0
        _close(w.grad, w64.grad, UNIT[w.dtype], 4e-6 * float(size_of_sum))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(dev, dtype, wdtype, size):
    _check(size, dtype, *_run(size, dtype, wdtype, dev))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("layout", ["projection", "heads_first", "odd", "strided"])
@pytest.mark.parametrize("size", [(2, 9, 6, 2, 64, 64), (1, 5, 3, 1, 96, 48), (2, 3, 2, 1, 30, 10)])
def test_layouts(dev, layout, size):
    for dtype in (torch.bfloat16, torch.float32):
        _check(size, dtype, *_run(size, dtype, dtype, dev, layout, grads="contiguous"))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", [1, 4])
def test_positions(dev, t):
    size = (3, t, 4, 2, 64, 64)
    for positions in (torch.randint(0, 100, (3, t), generator=_gen(1)), torch.arange(t).flip(0) + 50,
                      torch.randint(0, 100, (3, t), generator=_gen(2)).int()):
        _check(size, torch.bfloat16, *_run(size, torch.bfloat16, torch.bfloat16, dev, positions=positions.long(), table=100))
    leaves = _inputs(size, torch.float32, torch.float32, dev)
    cos, sin = (x.to(dev) for x in _tables(100, 64))
    a = ops.qk_norm_rope(*leaves, cos, sin, torch.arange(t, device=dev).int())
    b = ops.qk_norm_rope(*leaves, cos, sin)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dev", DEVICES)
def test_one_output_used_and_broadcast_inputs(dev):
    """Gradients where only k's output is used, and of a key head shared by a broadcast."""
    q, k, qw, kw = _inputs((2, 3, 4, 1, 64, 64), torch.float32, torch.float32, dev)
    cos, sin = (x.to(dev) for x in _tables(3, 64))
    shared = k.expand(2, 3, 4, 64)
    _, ko = ops.qk_norm_rope(q, shared, qw, kw, cos, sin, eps=EPS)
    ko.sum().backward()  # a gradient whose strides are all zero
    k64, kw64 = k.detach().cpu().double().requires_grad_(), kw.detach().cpu().double().requires_grad_()
    want = rotated64(k64.expand(2, 3, 4, 64), kw64, cos.cpu(), sin.cpu(), torch.arange(3).expand(2, 3))
    want.sum().backward()
    _close(k.grad, k64.grad, 1e-6, 4 * 4e-6 * 12 * 9)
    _close(kw.grad, kw64.grad, 1e-6, 4e-6 * 24 * 4)
    assert q.grad is None or not q.grad.any()


@pytest.mark.parametrize("dev", DEVICES)
def test_zero_heads_no_tokens_and_large_values(dev):
    q, k, qw, kw = _inputs((1, 2, 2, 1, 64, 64), torch.float32, torch.float32, dev)
    cos, sin = (x.to(dev) for x in _tables(2, 64))
    zero = torch.zeros_like(q).requires_grad_()
    big = (k.detach() * 1e15).requires_grad_()  # squares of 1e30 stay within 32 bits
    qo, ko = ops.qk_norm_rope(zero, big, qw, kw, cos, sin, eps=EPS)
    assert not qo.any() and torch.isfinite(ko).all()
    (qo.sum() + ko.sum()).backward()
    assert torch.isfinite(zero.grad).all() and torch.isfinite(big.grad).all()
    q, k, qw, kw = _inputs((2, 0, 2, 1, 64, 64), torch.bfloat16, torch.float32, dev)
    qo, ko = ops.qk_norm_rope(q, k, qw, kw, cos, sin)
    assert qo.shape == (2, 0, 2, 64)
    (qo.sum() + ko.sum()).backward()
    assert not qw.grad.any() and not kw.grad.any()


@pytest.mark.parametrize("dev", DEVICES)
def test_gradient_against_differences(dev):
    size = (1, 3, 2, 1, 16, 8)
    _, _, leaves, wide, outer = _run(size, torch.float32, torch.float32, dev)
    cos, sin = _tables(3, 8)
    h, at = 1e-6, torch.arange(3).expand(1, 3)

    def total(x, w, g):
        return float((rotated64(x, w, cos, sin, at) * g.double()).sum())

    for i in range(2):
        for pos in [(0, 0, 0, 0), (0, 1, 0, 5), (0, 2, 0, 15), (0, 2, 0, 9)]:
            ends = []
            for step in (h, -h):
                x = wide[i].detach().clone()
                x[pos] += step
                ends.append(total(x, wide[i + 2].detach(), outer[i]))
            assert abs(float(leaves[i].grad[pos]) - (ends[0] - ends[1]) / (2 * h)) < 4e-6 * 12 * 25 + 1e-6
        for e in (0, 7, 15):
            ends = []
            for step in (h, -h):
                w = wide[i + 2].detach().clone()
                w[e] += step
                ends.append(total(wide[i].detach(), w, outer[i]))
            assert abs(float(leaves[i + 2].grad[e]) - (ends[0] - ends[1]) / (2 * h)) < 4e-6 * 6 * 40 + 1e-6


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    q, k, qw, kw = (x.detach() for x in _inputs((2, 3, 4, 2, 64, 64), torch.float32, torch.float32, dev))
    cos, sin = (x.to(dev) for x in _tables(3, 64))
    for args in [(q[0], k[0], qw, kw, cos, sin), (q, k[:1], qw, kw, cos, sin), (q, k[..., :32], qw, kw, cos, sin),
                 (q, k.bfloat16(), qw, kw, cos, sin), (q, k, qw[:32], kw, cos, sin), (q, k, qw.double(), kw, cos, sin),
                 (q, k, qw, kw, cos[:2], sin[:2]), (q, k, qw, kw, cos, sin[:2]), (q[..., :33], k[..., :33], qw[:33], kw[:33], cos[:, :8], sin[:, :8]),
                 (q[..., :32], k[..., :32], qw[:32], kw[:32], cos, sin), (q, k, qw, kw, cos, sin, torch.zeros(2, device=dev)),
                 (q, k, qw, kw, cos, sin, torch.zeros(2, 3, device=dev)),
                 (q, k, qw, kw, cos.clone().requires_grad_(), sin)]:
        with pytest.raises(ValueError):
            ops.qk_norm_rope(*args)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    q, k, qw, kw = (x.detach() for x in _inputs((1, 2, 2, 1, 64, 64), torch.float32, torch.float32, "cuda"))
    cos, sin = (x.cuda() for x in _tables(2, 64))
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q.double(), k.double(), qw, kw, cos, sin)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q, k, qw.double(), kw.double(), cos, sin)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(q, k, qw.cpu(), kw, cos, sin)
    with pytest.raises(RuntimeError):
        wide = torch.zeros(1, 2, 1, 514, device="cuda")
        ops.qk_norm_rope(wide, wide, wide[0, 0, 0], wide[0, 0, 0], cos, sin)


def test_positions_out_of_range_raise_on_the_cpu():
    q, k, qw, kw = _inputs((1, 2, 2, 1, 64, 64), torch.float32, torch.float32, "cpu")
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, qw, kw, *_tables(4, 64), torch.tensor([3, 4]))


@pytest.mark.gpu
def test_positions_out_of_range_are_held_and_reported_on_the_gpu():
    ops.check_device_errors()
    q, k, qw, kw = (x.detach() for x in _inputs((1, 2, 2, 1, 64, 64), torch.float32, torch.float32, "cuda"))
    cos, sin = (x.cuda() for x in _tables(4, 64))
    got = ops.qk_norm_rope(q, k, qw, kw, cos, sin, torch.tensor([-1, 9], device="cuda"))
    with pytest.raises(RuntimeError, match="error 5"):
        ops.check_device_errors()
    want = ops.qk_norm_rope(q, k, qw, kw, cos, sin, torch.tensor([0, 3], device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_repeats_streams_and_graph_capture():
    size = (2, 130, 8, 2, 128, 128)
    leaves = _inputs(size, torch.bfloat16, torch.bfloat16, "cuda", "projection")
    cos, sin = (x.cuda() for x in _tables(130, 128))
    outer = [torch.randn(2, 130, h, 128, generator=_gen(3)).bfloat16().cuda() for h in (8, 2)]

    def step():
        q, k = ops.qk_norm_rope(*leaves, cos, sin)
        return [q, k, *torch.autograd.grad((q, k), leaves, outer)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [x.clone() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("heads", [(1, 1), (4, 3), (9, 2)])
@pytest.mark.parametrize("d", [30, 64, 96, 256])
def test_weight_gradients_without_eps(dev, heads, d):
    """With eps = 0 only a head of zeros has no norm: heads that fill no whole step of the kernel leave no NaN."""
    q, k, qw, kw = _inputs((1, 3, *heads, d, d - d % 4), torch.float32, torch.float32, dev)
    cos, sin = (x.to(dev) for x in _tables(3, d - d % 4))
    outer = [torch.randn(1, 3, h, d, generator=_gen(7)) for h in heads]
    out = ops.qk_norm_rope(q, k, qw, kw, cos, sin, eps=0.0)
    torch.autograd.backward(out, [o.to(dev) for o in outer])
    for x, w, y, o in zip((q, k), (qw, kw), out, outer):
        x64, w64 = x.detach().cpu().double().requires_grad_(), w.detach().cpu().double().requires_grad_()
        n = x64 / (x64 ** 2).mean(-1, keepdim=True).sqrt()
        turn = torch.complex(cos.cpu().double(), sin.cpu().double())[None, :, None]
        z, half = n * w64, cos.shape[1]
        z2 = torch.complex(z[..., :half], z[..., half:2 * half]) * turn
        want = torch.cat([z2.real, z2.imag, z[..., 2 * half:]], -1)
        want.backward(o.double())
        _close(y, want.detach(), 1e-6, 1e-6 * 8 * math.sqrt(d))
        rms = float((x64.detach() ** 2).mean(-1).sqrt().min())
        _close(x.grad, x64.grad, 1e-6, 4e-6 * 12 / rms * (1 + math.sqrt(d)))
        size_of_sum = (n.detach().abs() * o.double().abs().amax(-1, keepdim=True) * 2).sum((0, 1, 2)).max()
        _close(w.grad, w64.grad, 1e-6, 4e-6 * float(size_of_sum))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("heads", [(0, 0), (0, 2), (3, 0)])
def test_tensors_without_heads(dev, heads):
    """Gradients of no heads at all, and of one tensor's heads beside none of the other's."""
    q, k, qw, kw = _inputs((2, 3, *heads, 64, 64), torch.float32, torch.float32, dev)
    cos, sin = (x.to(dev) for x in _tables(3, 64))
    out = ops.qk_norm_rope(q, k, qw, kw, cos, sin, eps=EPS)
    assert [y.shape[2] for y in out] == list(heads)
    (out[0].sum() + out[1].sum()).backward()
    for x, w, h in zip((q, k), (qw, kw), heads):
        assert x.grad.shape == x.shape and torch.isfinite(w.grad).all()
        assert bool(w.grad.any()) == (h > 0)
