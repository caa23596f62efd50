"""The gated delta rule, chunked and token by token, against the recurrence in 64 bits and autograd through it.

Tolerances. Results are rounded once (``eps / 2`` of each value at most). Before that come products of operands held to
2^-16 with sums in fp32, a handful in a row (state, right-hand side, solve, write, read; as many again in the backward), each
adding errors of 2^-16 of its terms, which are larger than their sum where it cancels: 2^-9 of a tensor's root mean
square covers five such steps with terms up to 25 times the result. The kernel for single tokens and the forms on the CPU
work in fp32 throughout: 2^-18. A final state is fp32 but comes from the same halves: 2^-12.
"""

import functools

import pytest
import torch

from dattri_llm_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NAMES = ("q", "k", "v", "a", "b", "a_log", "dt_bias")


def make(b, t, hk, h, dk, dv, dtype, device, *, seed=0, state=False, layout="sliced", decay=2.0):
    gen = torch.Generator().manual_seed(seed)
    rnd = functools.partial(torch.randn, generator=gen)
    width = 2 * hk * dk + h * dv
    if layout == "sliced":  # q, k and v side by side, gates side by side
        mixed = torch.nn.functional.silu(rnd(b, t, width) * 1.5).to(dtype).to(device)
        gates = rnd(b, t, 2 * h).to(dtype).to(device)
    elif layout == "odd":  # rows that start anywhere
        mixed = torch.nn.functional.silu(rnd(b, t, width + 3) * 1.5).to(dtype).to(device)[..., 1:width + 1]
        gates = rnd(b, t, 2 * h + 1).to(dtype).to(device)[..., 1:]
    else:  # heads before tokens
        mixed = torch.nn.functional.silu(rnd(b, t, width) * 1.5).to(dtype).to(device)
        gates = rnd(b, t, 2 * h).to(dtype).to(device)
    cut = lambda lo, n, d: mixed[..., lo:lo + n * d].unflatten(-1, (n, d))  # noqa: E731
    x = {"q": cut(0, hk, dk), "k": cut(hk * dk, hk, dk), "v": cut(2 * hk * dk, h, dv), "a": gates[..., :h], "b": gates[..., h:2 * h]}
    if layout == "heads first":
        x = {n: y.transpose(1, 2).contiguous().transpose(1, 2) for n, y in x.items()}
    x["a_log"] = (torch.rand(h, generator=gen) * 2 * decay + 0.01).log().to(dtype).to(device)
    x["dt_bias"] = (rnd(h) - 2).to(dtype).to(device)
    x = {n: y.detach() for n, y in x.items()}
    first = (rnd(b, h, dk, dv) * 0.5).to(device) if state else None
    return x, first


def recurrence(x, first, scale=None):
    """Token by token in 64 bits, differentiable."""
    q, k, v, a, b, a_log, dt_bias = (x[n] for n in NAMES)
    group = v.shape[2] // q.shape[2]
    unit = lambda y: y / (y.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    q, k = unit(q).repeat_interleave(group, 2) * (scale or q.shape[3] ** -0.5), unit(k).repeat_interleave(group, 2)
    decay = torch.exp(-a_log.exp() * torch.nn.functional.softplus(a + dt_bias))
    beta = torch.sigmoid(b)
    state = first if first is not None else v.new_zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3])
    outs = []
    for t in range(v.shape[1]):
        state = state * decay[:, t, :, None, None]
        e = beta[:, t, :, None] * (v[:, t] - (state * k[:, t, :, :, None]).sum(2))
        state = state + k[:, t, :, :, None] * e[:, :, None]
        outs.append((state * q[:, t, :, :, None]).sum(2))
    return torch.stack(outs, 1), state


def gate_terms(x, out, g_out, dv):
    """On the CPU the log-decay's gradient at a token is a sum over the rest of its chunk of what tokens give less what they
    take (q . dq - v . dv), whose terms cancel: up to 64 of them with errors of random sign, 8 times one's. Those errors' size
    for each gate's gradient."""
    wide = {n: x[n].detach().double().cpu() for n in ("a", "a_log", "dt_bias", "v")}
    each = (out * g_out.double().cpu()).sum(-1).abs() + (wide["v"] * dv).sum(-1).abs()
    dt = wide["a"] + wide["dt_bias"]
    da = 8 * each.square().mean((0, 1)).sqrt() * wide["a_log"].exp() * torch.sigmoid(dt).square().mean((0, 1)).sqrt()
    n = each[..., 0].numel() ** 0.5
    ratio = (torch.nn.functional.softplus(dt) / torch.sigmoid(dt)).square().mean((0, 1)).sqrt()
    return {"a": da.detach(), "dt_bias": (da * n).detach(), "a_log": (da * n * ratio).detach()}


def gate_sums(x, da):
    """The gradients of a_log and dt_bias are sums of all tokens' shares, of either sign, each with errors of its own size: what such
    a sum comes to where signs are random, whatever they happen to cancel to in one head."""
    dt = (x["a"].detach().double() + x["dt_bias"].detach().double()).cpu()
    ratio = torch.nn.functional.softplus(dt) / torch.sigmoid(dt)  # of a token's share for a_log to that for dt_bias
    return {"dt_bias": da.square().sum((0, 1)).sqrt(), "a_log": (da * ratio).square().sum((0, 1)).sqrt()}


def close(name, got, want, dtype, slack, terms=0.0):
    got, want = got.detach().double().cpu(), want.detach()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    if not want.numel():
        return
    rms = want.square().mean().sqrt()
    off = (got - want).abs()
    # fp16 has a fixed step below its normal range
    floor = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = off > torch.finfo(dtype).eps / 2 * want.abs() + slack * (rms + want.abs() + terms) + floor
    assert not bad.any(), f"{name}: off by {(off / (rms + want.abs())).max():.3g}, {int(bad.sum())} of {bad.numel()}"


def exact(x, first, g_out, g_last, scale=None):
    wide = {n: y.detach().double().cpu().requires_grad_(True) for n, y in x.items()}
    start = first.detach().double().cpu().requires_grad_(True) if first is not None else None
    out, last = recurrence(wide, start, scale)
    loss = (out * g_out.double().cpu()).sum() + ((last * g_last.double().cpu()).sum() if g_last is not None else 0.0)
    inputs = [wide[n] for n in NAMES] + ([start] if first is not None else [])
    grads = torch.autograd.grad(loss, inputs)
    return out, last, dict(zip((*NAMES, "state"), grads, strict=False))


def check(shape, dtype, device, *, state=False, layout="sliced", g_state=False, decay=2.0, seed=0, scale=None, change=None, terms=1):
    x, first = make(*shape, dtype, device, seed=seed, state=state, layout=layout, decay=decay)
    if change is not None:
        change(x)
    for y in x.values():
        y.requires_grad_(True)
    if first is not None:
        first.requires_grad_(True)
    out, last = ops.gated_delta_rule(*(x[n] for n in NAMES), initial_state=first, output_final_state=True, scale=scale)
    assert out.dtype == dtype and last.dtype == torch.float32
    gen = torch.Generator().manual_seed(seed + 1)
    g_out = torch.randn(out.shape, generator=gen).to(dtype).to(device)
    g_last = (torch.randn(last.shape, generator=gen) * 0.3).to(device) if g_state else None
    want, want_last, grads = exact(x, first, g_out, g_last, scale)
    inputs = [x[n] for n in NAMES] + ([first] if first is not None else [])
    outs = (out, last) if g_state else (out,)
    got = torch.autograd.grad(outs, inputs, (g_out, g_last) if g_state else (g_out,))
    cpu = device == "cpu"
    close("out", out, want, dtype, terms * 2.0 ** (-18 if cpu else -9))
    close("state", last, want_last, torch.float32, terms * 2.0 ** (-18 if cpu else -12))
    sums = gate_terms(x, want.detach(), g_out, grads["v"]) if cpu else gate_sums(x, grads["a"])
    for n, g in zip((*NAMES, "state"), got, strict=False):
        close("d" + n, g, grads[n], g.dtype, terms * 2.0 ** (-16 if cpu else -9), sums.get(n, 0.0))


SHAPES = [  # batch, tokens, key heads, value heads, key dim, value dim
    (1, 1, 1, 1, 8, 8), (2, 3, 1, 2, 16, 24), (1, 63, 2, 2, 64, 64), (1, 64, 1, 1, 128, 128), (2, 65, 1, 3, 72, 32),
    (1, 128, 2, 4, 128, 96), (1, 200, 1, 8, 32, 40), (3, 130, 2, 4, 64, 136), (1, 257, 1, 2, 96, 200), (1, 70, 3, 3, 120, 8),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(device, shape):
    check(shape, torch.float32 if device == "cpu" else torch.bfloat16, device)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_gates_that_nearly_close(device):
    """Heads that keep e^-1 to e^-40 of a state in a token, each measured by itself: what passes a gate is summed as such, not as
    a difference of what a token takes and gives, so that a head's gradient has its own size's errors."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    x, _ = make(2, 150, 2, 4, 64, 64, dtype, device)
    x["a_log"] = torch.tensor([1.0, 2.0, 4.0, 16.0], device=device).log()
    x["dt_bias"] = torch.full((4,), 1.0, device=device)
    for y in x.values():
        y.requires_grad_(True)
    out, _ = ops.gated_delta_rule(*(x[n] for n in NAMES))
    g_out = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    _, _, grads = exact(x, None, g_out, None)
    got = torch.autograd.grad(out, [x["a"], x["a_log"], x["dt_bias"]], g_out)
    wide = {n: x[n].detach().double().cpu() for n in ("a", "a_log", "dt_bias")}
    dt = wide["a"] + wide["dt_bias"]
    ratio = torch.nn.functional.softplus(dt) / torch.sigmoid(dt)  # of a token's shares in the gradients of a_log and a
    for h in range(4):
        da = grads["a"][..., h]
        each = {"a": da, "dt_bias": da, "a_log": da * ratio[..., h]}
        for n, g in zip(("a", "a_log", "dt_bias"), got, strict=True):
            size = each[n].square().mean().sqrt() * (1.0 if n == "a" else each[n].numel() ** 0.5)
            off, want = (g[..., h].double().cpu() - grads[n][..., h]).abs(), grads[n][..., h].abs()
            assert (off <= (torch.finfo(g.dtype).eps / 2 + 2.0 ** -9) * want + 2.0 ** -9 * size + 1e-37).all(), (n, h, (off / size).max())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_fp16(shape):
    check(shape, torch.float16, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 70, 1, 5, 72, 64), (2, 66, 1, 6, 64, 128), (1, 130, 2, 14, 128, 64), (1, 70, 1, 8, 128, 128), (1, 65, 2, 10, 128, 200)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_value_heads_of_a_key_head(dtype, shape):
    """Their rows of dq and dk are added up in clusters of 5 to 8, each of which owns a multiple of 16 rows."""
    check(shape, dtype, "cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["odd", "heads first"])
def test_layouts(device, layout):
    for dtype in ((torch.float32,) if device == "cpu" else (torch.bfloat16, torch.float16)):
        check((2, 100, 2, 4, 48, 56), dtype, device, layout=layout, state=True, g_state=True)


@pytest.mark.parametrize("device", DEVICES)
def test_states_in_and_out(device):
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    for shape in SHAPES[::2]:
        check(shape, dtype, device, state=True, g_state=True, seed=3, scale=0.5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("decay", [0.001, 40.0])
def test_slow_and_fast_forgetting(device, decay):
    check((1, 150, 1, 2, 64, 64), torch.float32 if device == "cpu" else torch.bfloat16, device, state=True, decay=decay)


@pytest.mark.parametrize("device", DEVICES)
def test_closed_gates_and_empty_keys(device):
    """Tokens that write nothing, forget all, or have keys of zeros."""

    def change(x):
        x["b"][:, 5] = -200.0
        x["b"][:, 70:75] = -200.0
        x["b"][:, 20] = 200.0
        x["k"][:, 30] = 0
        x["q"][:, 31] = 0
        x["v"][:, 32] = 0
        x["a"][:, 90] = 3e4
        x["a"][:, 33:35] = -200.0  # no forgetting at all

    check((1, 140, 1, 2, 64, 64), torch.float32 if device == "cpu" else torch.bfloat16, device, state=True, change=change)


@pytest.mark.parametrize("device", DEVICES)
def test_repeated_keys(device):
    """One key over a whole chunk: the triangular system is as far from the identity as it gets. Its rows have up to 63 terms
    near one where other keys' terms cancel, each with a rounding of its own: errors of random sign grow by sqrt(64) = 8."""

    def change(x):
        x["k"][:] = x["k"][:, :1]
        x["b"][:] = 4.0

    check((1, 128, 1, 1, 64, 64), torch.float32 if device == "cpu" else torch.bfloat16, device, decay=0.01, change=change, terms=8)


@pytest.mark.parametrize("device", DEVICES)
def test_no_tokens(device):
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    x, first = make(2, 0, 1, 2, 16, 16, dtype, device, state=True)
    for y in x.values():
        y.requires_grad_(True)
    first.requires_grad_(True)
    out, last = ops.gated_delta_rule(*(x[n] for n in NAMES), initial_state=first, output_final_state=True)
    assert out.shape == (2, 0, 2, 16) and torch.equal(last, first)
    (last * 2).sum().backward()
    assert torch.equal(first.grad, torch.full_like(first, 2.0))
    assert x["a_log"].grad is None or not x["a_log"].grad.any()
    with torch.no_grad():
        state = first.detach().clone()
        assert ops.gated_delta_step(*(x[n].detach() for n in NAMES), state).shape == (2, 0, 2, 16)
        assert torch.equal(state, first)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 8, 8), (3, 1, 2, 4, 128, 128), (2, 4, 1, 3, 72, 40), (5, 2, 2, 2, 64, 96), (1, 7, 1, 8, 32, 200)])
def test_token_by_token(device, dtype, shape):
    for layout in ("sliced", "odd"):
        x, state = make(*shape, dtype, device, state=True, layout=layout)
        want, want_last = recurrence({n: y.double().cpu() for n, y in x.items()}, state.double().cpu())
        out = ops.gated_delta_step(*(x[n] for n in NAMES), state)
        close("out", out, want, dtype, 2.0 ** -18)
        close("state", state, want_last, torch.float32, 2.0 ** -18)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(40, 1, 4, 8, 128, 128), (100, 3, 1, 3, 72, 40), (37, 2, 8, 16, 32, 104), (75, 1, 2, 4, 128, 136)])
def test_token_by_token_of_many_sequences(dtype, shape):
    """More heads than two for each SM; the state's heads further apart than they are large."""
    x, state = make(*shape, dtype, "cuda", state=True, layout="odd")
    b, h = state.shape[:2]
    held = torch.full((b, h + 1, *state.shape[2:]), 7.0, device="cuda")
    held[:, :h] = state
    want, want_last = recurrence({n: y.double() for n, y in x.items()}, state.double())
    out = ops.gated_delta_step(*(x[n] for n in NAMES), held[:, :h])
    close("out", out, want.cpu(), dtype, 2.0 ** -18)
    close("state", held[:, :h], want_last.cpu(), torch.float32, 2.0 ** -18)
    assert (held[:, h:] == 7).all()


@pytest.mark.parametrize("device", DEVICES)
def test_prefill_then_decode(device):
    """A prompt in chunks and new tokens one at a time give what the whole sequence gives; the state may be a slice."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    x, _ = make(2, 90, 1, 2, 64, 32, dtype, device)
    want, want_last = recurrence({n: y.double().cpu() for n, y in x.items()}, None)
    part = lambda lo, hi: [y[:, lo:hi] if y.dim() > 1 else y for y in (x[n] for n in NAMES)]  # noqa: E731
    with torch.no_grad():
        out, last = ops.gated_delta_rule(*part(0, 77), output_final_state=True)
        cache = torch.zeros(3, 2, 4, 64, 32, device=device)
        cache[1, :, 1:3] = last
        state = cache[1, :, 1:3]
        rest = [ops.gated_delta_step(*part(t, t + 1), state) for t in range(77, 90)]
    close("out", torch.cat([out, *rest], 1), want, dtype, 2.0 ** -9)
    close("state", state, want_last, torch.float32, 2.0 ** -12)
    assert not cache[0].any() and not cache[2].any() and not cache[1, :, 0].any() and not cache[1, :, 3].any()


def test_gradients_against_differences():
    x, first = make(1, 70, 1, 2, 8, 8, torch.float64, "cpu", state=True)
    wide = [x[n].double().requires_grad_(True) for n in NAMES] + [first.double().requires_grad_(True)]
    fn = lambda *z: ops.gated_delta_rule(*z[:7], initial_state=z[7], output_final_state=True)  # noqa: E731
    assert torch.autograd.gradcheck(fn, wide, fast_mode=True, atol=1e-6)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    x, first = make(2, 5, 1, 2, 16, 16, dtype, device, state=True)
    args = [x[n] for n in NAMES]

    def swapped(name, y):
        return [y if n == name else x[n] for n in NAMES]

    for name, y in (("k", x["k"][:, :4]), ("v", x["v"][:, :, :, 0]), ("a", x["a"][..., :1]), ("a_log", x["a_log"][:1]),
                    ("v", x["v"][:1])):
        with pytest.raises(ValueError):
            ops.gated_delta_rule(*swapped(name, y))
        with pytest.raises(ValueError):
            ops.gated_delta_step(*swapped(name, y), first)
    with pytest.raises(TypeError):
        ops.gated_delta_rule(*swapped("v", x["v"].half()))
    with pytest.raises(ValueError):
        ops.gated_delta_rule(*args, scale=-1.0)
    with pytest.raises(ValueError):
        ops.gated_delta_rule(*args, initial_state=first[:1])
    with pytest.raises(TypeError):
        ops.gated_delta_step(*args, first.half())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gated_delta_step(*swapped("v", x["v"].clone().requires_grad_(True)), first)
    if device == "cpu":
        return
    for shape in ((1, 5, 1, 9, 16, 16), (1, 5, 1, 1, 12, 16), (1, 5, 1, 1, 16, 12), (1, 5, 1, 1, 136, 16)):
        y, _ = make(*shape, dtype, device)
        with pytest.raises(ValueError):
            ops.gated_delta_rule(*(y[n] for n in NAMES))
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        ops.gated_delta_rule(*(x[n].float() for n in NAMES))
    with pytest.raises(ValueError, match="contiguous"):
        ops.gated_delta_step(*args, first.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="overlap"):
        ops.gated_delta_step(*args, first[:1].expand(2, -1, -1, -1))
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        v = x["v"].clone().requires_grad_(True)
        (d,) = torch.autograd.grad(ops.gated_delta_rule(*swapped("v", v))[0].sum(), v, create_graph=True)
        d.sum().backward()


@pytest.mark.gpu
def test_another_stream_and_a_captured_pass():
    x, first = make(1, 150, 1, 2, 64, 64, torch.bfloat16, "cuda", state=True)
    for y in x.values():
        y.requires_grad_(True)
    args = [x[n] for n in NAMES]

    def one():
        out, last = ops.gated_delta_rule(*args, initial_state=first, output_final_state=True)
        return (out, last, *torch.autograd.grad((out, last), args, (torch.ones_like(out), torch.ones_like(last))))

    want = one()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = one()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    graph = torch.cuda.CUDAGraph()
    del got, want
    with torch.cuda.graph(graph):
        held = one()
    with torch.no_grad():
        x["v"].mul_(0.5)
    graph.replay()
    again = [y.clone() for y in held]
    want = one()
    assert all(torch.equal(a, b) for a, b in zip(again, want, strict=True))


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits_and_two_graphs_share_nothing():
    shape = (2, 300, 2, 8, 128, 128)
    x, _ = make(*shape, torch.bfloat16, "cuda")
    y, _ = make(*shape, torch.bfloat16, "cuda", seed=9)
    outs = []
    for z in (x, y):
        for t in z.values():
            t.requires_grad_(True)
        outs.append(ops.gated_delta_rule(*(z[n] for n in NAMES))[0])
    g = torch.ones_like(outs[0])
    late = [torch.autograd.grad(o, [z[n] for n in NAMES], g) for o, z in zip(outs[::-1], (y, x), strict=True)][::-1]
    for z, grads in zip((x, y), late, strict=True):
        alone = torch.autograd.grad(ops.gated_delta_rule(*(z[n] for n in NAMES))[0], [z[n] for n in NAMES], g)
        assert all(torch.equal(a, b) for a, b in zip(alone, grads, strict=True))


@pytest.mark.gpu
def test_the_last_of_many_sequences_is_as_it_is_alone():
    """Workspaces of more than 2^32 bytes (eight sequences of 8,192 tokens): every sequence's results are its own, to the bit."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    b, t, hk, h, d = 8, 8192, 8, 16, 128
    rnd = functools.partial(torch.randn, generator=gen, device="cuda", dtype=torch.bfloat16)
    x = [rnd(b, t, hk, d), rnd(b, t, hk, d), rnd(b, t, h, d), rnd(b, t, h), rnd(b, t, h)]
    shared = [torch.zeros(h, device="cuda"), torch.full((h,), -3.0, device="cuda")]
    g = rnd(b, t, h, d)
    results = []
    for cut in (slice(None), slice(b - 1, b)):
        own = [y[cut].detach().requires_grad_(True) for y in x]
        out, last = ops.gated_delta_rule(*own, *shared, output_final_state=True)
        results.append([y[-1] for y in (out, last, *torch.autograd.grad(out, own, g[cut]))])
    assert all(torch.isfinite(y).all() for y in results[1])
    assert all(torch.equal(p, q) for p, q in zip(*results, strict=True))


@pytest.mark.gpu
def test_states_that_32_bits_do_not_count():
    """2^31 elements of state and more: the last sequences step as they do by themselves."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    b, few, hk, h, d = 2**31 // (16 * 128 * 128) + 20, 20, 8, 16, 128  # few * h: enough for the blocks that stay
    rnd = functools.partial(torch.randn, generator=gen, device="cuda")
    x = [y.to(torch.bfloat16) for y in (rnd(b, 1, hk, d), rnd(b, 1, hk, d), rnd(b, 1, h, d), rnd(b, 1, h), rnd(b, 1, h))]
    shared = [torch.zeros(h, device="cuda"), torch.full((h,), -3.0, device="cuda")]
    state = torch.zeros(b, h, d, d, device="cuda")
    state[-few:] = rnd(few, h, d, d)
    own = state[-few:].clone()
    with torch.no_grad():
        out = ops.gated_delta_step(*x, *shared, state)
        want = ops.gated_delta_step(*(y[-few:] for y in x), *shared, own)
    assert torch.equal(out[-few:], want) and torch.equal(state[-few:], own)


@pytest.mark.parametrize("device", DEVICES)
def test_states_whose_heads_share_memory_are_refused(device):
    """Strides that are large enough each by itself, but not together: head (0, 1) is head (1, 0)."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    x, first = make(3, 1, 1, 2, 16, 16, dtype, device, state=True)
    args = [x[n] for n in NAMES]
    one = 16 * 16
    memory = torch.zeros(8 * one, device=device)
    for outer in ((one, one), (one, 2 * one), (one, one + 16), (2 * one, 2 * one + 16), (0, one), (one, 0)):
        with pytest.raises(ValueError, match="overlap"):
            ops.gated_delta_step(*args, memory.as_strided((3, 2, 16, 16), (*outer, 16, 1)))
    assert not memory.any()
    want = first.clone()
    out = ops.gated_delta_step(*args, want)
    for outer in ((2 * one, one), (one, 3 * one), (2 * one + 64, one + 16), (one + 16, 4 * one), (2 * one, 3 * one)):  # apart
        state = memory.as_strided((3, 2, 16, 16), (*outer, 16, 1))
        state.copy_(first)
        assert torch.equal(ops.gated_delta_step(*args, state), out) and torch.equal(state, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(330, 1, 1, 1, 64, 64), (75, 2, 2, 4, 128, 96), (60, 3, 1, 5, 8, 104), (149, 2, 2, 2, 120, 120)])
def test_many_heads_of_few_and_of_many_columns(dtype, shape):
    """On either side of the width from which on CTAs stay."""
    x, state = make(*shape, dtype, "cuda", state=True)
    want, want_last = recurrence({n: y.double() for n, y in x.items()}, state.double())
    out = ops.gated_delta_step(*(x[n] for n in NAMES), state)
    close("out", out, want.cpu(), dtype, 2.0 ** -18)
    close("state", state, want_last.cpu(), torch.float32, 2.0 ** -18)
