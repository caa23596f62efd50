"""The AdamW step of many tensors and the optimizer over it, against the formula in 64 bits and ``torch.optim.AdamW``.

Tolerances count roundings: a result is rounded once to its type (``eps / 2`` relative); before that come a handful of
fp32 operations on values no larger than the terms of each sum (2^-21 of them covers eight). A code of 4 bits of
significand is off by 2^-4 of its value, or by half a step of the smallest codes (2^-10 of the scale).
"""

import copy

import pytest
import torch

import dattri_llm_b200 as bw
from dattri_llm_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HYPER = {"lr": 3e-3, "betas": (0.9, 0.99), "eps": 1e-7, "weight_decay": 0.1}
SLACK = 2.0 ** -21


def make(shapes, dtype, device, *, bits, grad_dtype=None, seed=0, offset=0):
    gen = torch.Generator().manual_seed(seed)
    params, grads, m, v, scales = [], [], [], [], []
    for i, shape in enumerate(shapes):
        n = int(torch.tensor(shape).prod()) if shape else 1

        def place(x, dt):  # at an odd place of a larger buffer, where the test asks for it
            buf = torch.empty(n + offset, dtype=dt, device=device)
            out = buf[offset:].view(shape)
            out.copy_(x)
            return out

        p = place(torch.randn(shape, generator=gen), dtype)
        g = place(torch.randn(shape, generator=gen) * 10.0 ** (-(i % 5)), grad_dtype or dtype)
        if n > 6:
            g.view(-1)[:3] = 0
        m0 = torch.randn(shape, generator=gen).to(device) * 10.0 ** (-(i % 5))
        v0 = (torch.randn(shape, generator=gen).to(device) * 10.0 ** (-(i % 5))).square()
        if bits == 32:
            m.append(place(m0, torch.float32))
            v.append(place(v0, torch.float32))
        else:
            sc = torch.zeros(2, -(-n // 256), device=device)
            for x, row, to in ((m0, 0, m), (v0.sqrt(), 1, v)):
                flat = torch.nn.functional.pad(x.reshape(-1), (0, -n % 256)).view(-1, 256)
                if n:
                    sc[row] = flat.abs().amax(1) / 448
                codes = (flat / sc[row][:, None].clamp(min=1e-30)).clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)[:n]
                to.append(place(torch.zeros(shape), torch.float8_e4m3fn))
                to[-1].copy_(codes.view(shape))
            scales.append(sc)
        params.append(p)
        grads.append(g)
    return params, grads, m, v, scales or None


def exact(p, g, m, v, step, maximize=False):
    b1, b2 = HYPER["betas"]
    p, g, m, v = (x.double() for x in (p, -g if maximize else g, m, v))
    terms = b1 * m.abs() + (1 - b1) * g.abs()  # of m: where they cancel, their roundings do not
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    by = HYPER["lr"] / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + HYPER["eps"])
    return p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - by * m, m, v, by * terms


def check(shapes, dtype, device, bits, step, **kw):
    maximize = kw.pop("maximize", False)
    params, grads, m, v, scales = make(shapes, dtype, device, bits=bits, **kw)
    start = []
    for i, p in enumerate(params):
        wide = ops.adamw_moments(m[i], v[i], None if scales is None else scales[i])
        start.append((p.clone(), grads[i].clone(), wide[0].clone(), wide[1].clone()))
    ops.adamw_step(params, grads, m, v, scales, step=step, maximize=maximize, **HYPER)
    half = torch.finfo(dtype).eps / 2
    for i, p in enumerate(params):
        old, g, m0, v0 = start[i]
        want, wm, wv, move = exact(old, g, m0, v0, step, maximize)
        off = (p.double() - want).abs()
        assert (off <= half * want.abs() + SLACK * (old.double().abs() + move.abs()) + torch.finfo(dtype).smallest_normal).all()
        gm, gv = ops.adamw_moments(m[i], v[i], None if scales is None else scales[i])
        terms_m = m0.double().abs() + g.double().abs()
        terms_v = v0.double() + g.double().square()
        if bits == 32:
            assert ((gm.double() - wm).abs() <= SLACK * terms_m).all()
            assert ((gv.double() - wv).abs() <= SLACK * terms_v + 1e-44).all()
            continue
        n = p.numel()
        for got, true, row, smallest in ((gm, wm, 0, 2.0 ** -10), (gv.sqrt(), wv.sqrt(), 1, 2.0 ** -9)):
            flat = torch.nn.functional.pad(true.reshape(-1), (0, -n % 256)).view(-1, 256)
            scale = flat.abs().amax(1) / 448 if n else flat.new_zeros(0)
            assert ((scales[i][row].double() - scale).abs() <= SLACK * (scale + terms_m.amax() / 448 if n else scale)).all()
            each = scale.repeat_interleave(256)[:n].view(p.shape)
            assert ((got.double() - true).abs() <= (2.0 ** -4 + SLACK) * true.abs() + (smallest + SLACK) * each).all()
            if row == 1:
                assert (got[true > 0] > 0).all()  # a root that is not zero keeps a code
                assert (got[true == 0] == 0).all()


SHAPES = [(3,), (256,), (257,), (0,), (1,), (17, 31), (8192,), (8200,), (3, 5, 7), (64, 256), ()]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("step", [1, 1000])
def test_step_matches_the_formula(device, bits, dtype, step):
    check(SHAPES, dtype, device, bits, step)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_that_start_anywhere_and_gradients_in_32_bits(device, bits):
    check(SHAPES, torch.bfloat16, device, bits, 3, offset=1)
    check(SHAPES, torch.bfloat16, device, bits, 3, grad_dtype=torch.float32, maximize=True)
    check(SHAPES, torch.float16, device, bits, 3, grad_dtype=torch.float32, offset=3)
    check(SHAPES, torch.float32, device, bits, 3, offset=2)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_one_launch_takes_and_a_large_one(bits):
    check([(1 + i % 700,) for i in range(1111)], torch.float32, "cuda", bits, 2)
    check([(1037, 4099)], torch.bfloat16, "cuda", bits, 2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_axes_in_any_order(device, bits):
    """A transposed parameter and a gradient laid out otherwise: the same numbers as contiguous ones give."""
    torch.manual_seed(0)
    w = torch.randn(40, 33, device=device)
    g = torch.randn(40, 33, device=device)
    results = []
    for p, grad in ((w.t().contiguous().t(), g.clone()), (w.clone(), g.t().contiguous().t())):
        state = ops.adamw_state(p, bits)
        ops.adamw_step([p], [grad], [state[0]], [state[1]], None if bits == 32 else [state[2]], step=1, **HYPER)
        m, _ = ops.adamw_moments(*state)
        assert m.stride() == p.stride()
        results.append(p.clone())
    assert torch.equal(results[0], results[1])  # the step uses the moments before they become codes


@pytest.mark.parametrize("device", DEVICES)
def test_state_of_zeros_and_tiny_and_infinite_gradients(device):
    p = torch.ones(600, device=device)
    m, v, s = ops.adamw_state(p, 8)
    ops.adamw_step([p], [torch.zeros(600, device=device)], [m], [v], [s], step=1, **HYPER)
    assert torch.equal(s, torch.zeros_like(s)) and torch.isfinite(p).all()
    g = torch.full((600,), 1e-30, device=device)
    g[300:] = 0
    ops.adamw_step([p], [g], [m], [v], [s], step=2, **HYPER)
    assert torch.isfinite(p).all() and all(torch.isfinite(x).all() for x in ops.adamw_moments(m, v, s))
    g = torch.zeros(600, device=device)
    g[5] = float("nan")
    g[300] = float("inf")
    ops.adamw_step([p], [g], [m], [v], [s], step=3, **HYPER)
    assert torch.isnan(p[5]) and torch.isnan(p[300])  # as every AdamW has it
    assert torch.isfinite(p[512:]).all()  # their block is theirs alone


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    p = torch.randn(8, 4, device=device)
    m, v, _ = ops.adamw_state(p)
    g = torch.randn_like(p)
    ok = {"step": 1, "lr": 0.1}
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p, p], [g, g], [m, m.clone()], [v, v.clone()], **ok)
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p], [g], [m], [m], **ok)
    with pytest.raises(ValueError, match="needs a gradient"):
        ops.adamw_step([p], [], [m], [v], **ok)
    with pytest.raises(ValueError, match="shape"):
        ops.adamw_step([p], [g[:4]], [m], [v], **ok)
    with pytest.raises(ValueError, match="strides"):
        ops.adamw_step([p], [g], [m.t().contiguous().t()], [v], **ok)
    with pytest.raises(TypeError):
        ops.adamw_step([p], [g], [m.to(torch.bfloat16)], [v], **ok)
    with pytest.raises(TypeError):
        ops.adamw_step([p], [g], [m], [v], [torch.zeros(2, 1, device=device)], **ok)
    with pytest.raises(ValueError, match="scales"):
        m8, v8, s = ops.adamw_state(p, 8)
        ops.adamw_step([p], [g], [m8], [v8], [torch.zeros(2, 3, device=device)], **ok)
    with pytest.raises(NotImplementedError):
        ops.adamw_step([p], [g.to_sparse()], [m], [v], **ok)
    with pytest.raises(ValueError, match="step"):
        ops.adamw_step([p], [g], [m], [v], step=0, lr=0.1)
    with pytest.raises(ValueError):
        ops.adamw_state(p, 4)
    with pytest.raises(ValueError, match="state_bits"):
        bw.AdamW([torch.nn.Parameter(p)], state_bits=16)


def _steps(opt, p, grads):
    for g in grads:
        p.grad = g.clone()
        opt.step()


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_follows_torch(device):
    torch.manual_seed(1)
    start = torch.randn(50, 70, device=device)
    grads = [torch.randn(50, 70, device=device) for _ in range(12)]
    mine, theirs, coded = (torch.nn.Parameter(start.clone()) for _ in range(3))
    kw = {"lr": 1e-2, "betas": (0.9, 0.95), "weight_decay": 0.2}
    a, b, c = bw.AdamW([mine], **kw), torch.optim.AdamW([theirs], **kw), bw.AdamW([coded], state_bits=8, **kw)
    _steps(a, mine, grads)
    _steps(b, theirs, grads)
    _steps(c, coded, grads)
    # 12 steps of at most lr (1 + small) each, every one of them off by some 2^-21 of its parts
    assert (mine - theirs).abs().max() <= 12 * SLACK * (start.abs().max() + 1)
    # a code is off by 2^-4 each step and a moment remembers 10 or 20 steps of it: well below the 0.12 the weights move
    assert (coded - theirs).abs().max() <= 12 * kw["lr"] * 0.5
    assert c.state[coded]["exp_avg"].dtype == torch.float8_e4m3fn
    assert torch.equal(a.moment(mine, "exp_avg"), a.state[mine]["exp_avg"])
    assert ((c.moment(coded, "exp_avg") - b.state[theirs]["exp_avg"]).abs() <= 0.5).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_saved_and_loaded_it_goes_on_as_before(device, bits):
    torch.manual_seed(2)
    start = torch.randn(300, device=device, dtype=torch.bfloat16)
    grads = [torch.randn(300, device=device, dtype=torch.bfloat16) for _ in range(6)]
    p = torch.nn.Parameter(start.clone())
    opt = bw.AdamW([p], state_bits=bits)
    _steps(opt, p, grads[:3])
    saved, weights = copy.deepcopy(opt.state_dict()), p.detach().clone()
    _steps(opt, p, grads[3:])
    q = torch.nn.Parameter(weights)
    other = bw.AdamW([q], state_bits=bits)
    other.load_state_dict(saved)
    assert other.state[q]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)  # not the weights' type
    _steps(other, q, grads[3:])
    assert torch.equal(p, q)


@pytest.mark.parametrize("device", DEVICES)
def test_what_autograd_saved_is_seen_to_have_changed(device):
    w = torch.nn.Parameter(torch.randn(4, 4, device=device))
    x = torch.randn(4, 4, device=device, requires_grad=True)
    y = (x @ w).sum()
    w.grad = torch.ones_like(w)
    bw.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("device", DEVICES)
def test_snapshots_read_coded_states(device):
    """The optimizer-state reader gives 8-bit moments as the numbers they stand for."""
    from dattri_llm_b200.gradient.optimizer_state import OptimizerSnapshot, optimizer_from_state_dict

    torch.manual_seed(3)
    model = torch.nn.Sequential(torch.nn.Linear(9, 5)).to(device)
    opt = bw.AdamW(model.parameters(), state_bits=8)
    for _ in range(3):
        model(torch.randn(4, 9, device=device)).square().sum().backward()
        opt.step()
        opt.zero_grad()
    reader = OptimizerSnapshot(model, opt)
    assert reader.optimizer_type == "AdamW" and reader.step_count("0") == 3
    weight, bias = model[0].weight, model[0].bias
    want = torch.cat([opt.moment(weight, "exp_avg_sq"), opt.moment(bias, "exp_avg_sq").unsqueeze(1)], 1).reshape(-1)
    got = reader.state("0", "exp_avg_sq")
    assert got.dtype == torch.float32 and torch.equal(got.reshape(-1).sort().values, want.sort().values)
    direction = reader.precondition("0", torch.randn(2, got.numel(), device=device))
    assert torch.isfinite(direction).all()
    names = [n for n, _ in model.named_parameters()]
    again = optimizer_from_state_dict(model, copy.deepcopy(opt.state_dict()), names, optimizer_cls=bw.AdamW)
    assert torch.equal(OptimizerSnapshot(model, again).state("0", "exp_avg"), reader.state("0", "exp_avg"))


@pytest.mark.gpu
def test_another_stream_and_a_captured_step():
    torch.manual_seed(4)
    p, g = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")
    m, v, s = ops.adamw_state(p, 8)
    want = p.clone()
    wm, wv, ws = ops.adamw_state(p, 8)
    for _ in range(3):
        ops.adamw_step([want], [g], [wm], [wv], [ws], step=1, lr=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.adamw_step([p], [g], [m], [v], [s], step=1, lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw_step([p], [g], [m], [v], [s], step=1, lr=0.1)
    graph.replay()
    graph.replay()
    assert torch.equal(p, want) and torch.equal(s, ws)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_whose_squares_overflow_move_nothing(device, bits):
    p, g = torch.ones(300, device=device), torch.zeros(300, device=device)
    g[7] = 1e25
    m, v, s = ops.adamw_state(p, bits)
    ops.adamw_step([p], [g], [m], [v], None if s is None else [s], step=1, lr=0.1, weight_decay=0.0)
    assert torch.equal(p, torch.ones_like(p))  # m / inf


@pytest.mark.gpu
def test_elements_that_32_bits_do_not_count():
    """The last elements of a tensor of more than 2^31 move as they do by themselves (whole blocks before them)."""
    n = 2**31 + 700
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v, s = ops.adamw_state(p, 8)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for x in (p, g):
        x[2**31 - 256:] = torch.randn(956, generator=gen, device="cuda")
    few = [x[2**31 - 256:].clone() for x in (p, g)]
    fm, fv, fs = ops.adamw_state(few[0], 8)
    for step in (1, 2):
        ops.adamw_step([p], [g], [m], [v], [s], step=step, lr=0.1)
        ops.adamw_step([few[0]], [few[1]], [fm], [fv], [fs], step=step, lr=0.1)
    assert torch.equal(p[2**31 - 256:], few[0]) and not p[:2**31 - 256].any()
    assert torch.equal(m[2**31 - 256:].view(torch.uint8), fm.view(torch.uint8))
    assert torch.equal(v[2**31 - 256:].view(torch.uint8), fv.view(torch.uint8))
    assert torch.equal(s[:, -fs.shape[1]:], fs)


def check_one_step(p, g, m, v, scales, step, *, lr, betas, eps):
    """A step without weight decay against the formula in 64 bits on the moments that the state stood for before it.  Beside what
    the module's tolerances count, a sum of products below fp32's normal range is rounded to steps of 2^-149, in four
    roundings by 2^-148 together, half of it relative to the root."""
    bits8 = scales is not None
    old = p.double()
    m0, v0 = (x.double() for x in ops.adamw_moments(m, v, scales))
    g = g.double()
    ops.adamw_step([p], [g.to(p.dtype)], [m], [v], [scales] if bits8 else None, step=step, lr=lr, betas=betas, eps=eps, weight_decay=0.0)
    b1, b2 = betas
    wm, wv = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    terms = b1 * m0.abs() + (1 - b1) * g.abs()
    root_off = torch.where(wv > 0, (2.0 ** -149 / wv.clamp(min=1e-300)).clamp(max=1.0), 0.0)
    by = lr / (1 - b1 ** step) / ((wv / (1 - b2 ** step)).sqrt() + eps)
    by = torch.where(terms > 0, by, 0.0)
    want = old - by * wm
    half = torch.finfo(p.dtype).eps / 2
    assert torch.isfinite(p).all()
    assert ((p.double() - want).abs() <= half * want.abs() + (SLACK + 2 * root_off) * (old.abs() + by * terms)).all()
    gm, gv = (x.double() for x in ops.adamw_moments(m, v, scales))
    if not bits8:
        assert ((gm - wm).abs() <= SLACK * terms + 2.0 ** -148).all()
        assert ((gv - wv).abs() <= SLACK * wv + 2.0 ** -148).all()
        return
    n = p.numel()
    roots = v.double() * scales[1].double().repeat_interleave(256)[:n]  # not through the reader, which squares them in 32 bits
    for got, true, off, smallest in ((gm, wm, 0.0, 2.0 ** -10), (roots, wv.sqrt(), root_off, 2.0 ** -9)):
        flat = torch.nn.functional.pad((true.abs() * (1 + off)).reshape(-1), (0, -n % 256)).view(-1, 256)
        each = (flat.amax(1) / 448).repeat_interleave(256)[:n].view(p.shape)
        spread = SLACK * terms if true is wm else 0.0
        assert ((got - true).abs() <= (2.0 ** -4 + SLACK + off) * true.abs() + (smallest + SLACK) * each + spread).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_finite_moments_stay_numbers(device, bits, dtype):
    """Gradients up to 1e17, whose moments' scales pass 256 from 1.2e6 on, in some elements of some blocks, over several steps: none of the
    elements beside them is lost.  One tensor moves by whole vectors, one by single elements."""
    gen = torch.Generator().manual_seed(5)
    for offset in (0, 1):
        n = 256 * 5 + 40
        p = (torch.randn(n + offset, generator=gen)).to(device, dtype)[offset:]
        m, v, s = ops.adamw_state(p, bits)
        for step in range(1, 6):
            g = torch.randn(n, generator=gen)
            if step != 4:
                for block, size in enumerate((1.0, 1.3e6, 2e6, 1e10, 1e15)):
                    g[block * 256 + 7 * step] *= size
                g[-3] = -1e17
            check_one_step(p, g.to(device, dtype), m, v, s, step, lr=3e-3, betas=(0.9, 0.99), eps=1e-8)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_roots_below_the_normal_range(device, bits):
    """Gradients of 1e-21 to 1e-17 with eps = 0: their squares are subnormal numbers of fp32 (from 1e-44 on), their roots are not."""
    gen = torch.Generator().manual_seed(6)
    for offset in (0, 1):
        n = 256 * 3 + 40
        p = torch.randn(n + offset, generator=gen).to(device)[offset:]
        m, v, s = ops.adamw_state(p, bits)
        for step in range(1, 4):
            g = 10.0 ** (-21 + 4 * torch.rand(n, generator=gen)) * (1 - 2 * (torch.rand(n, generator=gen) < 0.5).float())
            check_one_step(p, g.to(device), m, v, s, step, lr=3e-3, betas=(0.9, 0.99), eps=0.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_state_of_torchs_own_adamw_goes_on(device, bits, dtype):
    """Its moments are taken as they are, its groups' settings too; a parameter that it has no state of gets one of `bits`."""
    torch.manual_seed(7)
    kw = {"lr": 1e-2, "betas": (0.9, 0.95), "weight_decay": 0.2}
    first, late = (torch.nn.Parameter(torch.randn(40, 9, device=device).to(dtype)) for _ in range(2))
    theirs = torch.optim.AdamW([first, late], **kw)
    _steps(theirs, first, [torch.randn_like(first) for _ in range(3)])
    mine = bw.AdamW([first, late], lr=5.0, state_bits=bits)
    mine.load_state_dict(copy.deepcopy(theirs.state_dict()))
    group = mine.param_groups[0]
    assert group["lr"] == kw["lr"] and group["state_bits"] == bits and late not in mine.state
    m0, v0 = (theirs.state[first][key].double() for key in ("exp_avg", "exp_avg_sq"))
    for key, was in (("exp_avg", m0), ("exp_avg_sq", v0)):
        assert torch.equal(mine.moment(first, key).double(), was)
    old, g = first.detach().double(), torch.randn_like(first)
    first.grad, late.grad = g, g.clone()
    mine.step()
    (b1, b2), g = kw["betas"], g.double()
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    by = kw["lr"] / (1 - b1 ** 4) / ((v / (1 - b2 ** 4)).sqrt() + 1e-8)
    want, terms = old * (1 - kw["lr"] * kw["weight_decay"]) - by * m, by * (b1 * m0.abs() + (1 - b1) * g.abs())
    off = (first.double() - want).abs()
    assert (off <= torch.finfo(dtype).eps / 2 * want.abs() + SLACK * (old.abs() + terms)).all()
    assert int(mine.state[first]["step"]) == 4 and int(mine.state[late]["step"]) == 1
    assert mine.state[late]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)


@pytest.mark.parametrize("key", ["amsgrad", "differentiable"])
def test_settings_that_would_be_dropped_are_refused(key):
    p = torch.nn.Parameter(torch.randn(5))
    theirs = torch.optim.AdamW([p], **{key: True})
    if key == "amsgrad":  # a differentiable step needs weights that are no leaves
        p.grad = torch.ones_like(p)
        theirs.step()
    p = torch.nn.Parameter(p.detach().clone())
    mine = bw.AdamW([p])
    with pytest.raises(NotImplementedError, match=key):
        mine.load_state_dict(theirs.state_dict())
    assert not mine.state and not mine.param_groups[0][key]  # it is as it was
    with pytest.raises(NotImplementedError, match=key):
        mine.add_param_group({"params": [torch.nn.Parameter(torch.ones(2))], key: True})
    assert len(mine.param_groups) == 1
    with pytest.raises(NotImplementedError, match=key):
        bw.AdamW([{"params": [p], key: True}])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_without_axes_goes_on_after_it_is_loaded(device, bits):
    torch.manual_seed(8)
    p = torch.nn.Parameter(torch.tensor(0.5, device=device, dtype=torch.bfloat16))
    grads = [torch.randn((), device=device, dtype=torch.bfloat16) for _ in range(6)]
    opt = bw.AdamW([p], state_bits=bits)
    _steps(opt, p, grads[:3])
    saved, q = copy.deepcopy(opt.state_dict()), torch.nn.Parameter(p.detach().clone())
    other = bw.AdamW([q], state_bits=bits)
    other.load_state_dict(saved)
    assert torch.equal(other.moment(q, "exp_avg"), opt.moment(p, "exp_avg"))
    _steps(opt, p, grads[3:])
    _steps(other, q, grads[3:])
    assert torch.equal(p, q) and torch.equal(other.moment(q, "exp_avg_sq"), opt.moment(p, "exp_avg_sq"))


@pytest.mark.parametrize("device", DEVICES)
def test_counts_of_a_fused_optimizer_are_kept_on_the_host(device):
    p = torch.nn.Parameter(torch.randn(30, device=device))
    theirs = torch.optim.AdamW([p], fused=True)
    _steps(theirs, p, [torch.randn(30, device=device) for _ in range(2)])
    saved = copy.deepcopy(theirs.state_dict())
    for copied in (saved, {**saved, "state": {0: {**saved["state"][0], "step": 2}}}):  # a number, as old checkpoints have it
        mine = bw.AdamW([p])
        mine.load_state_dict(copied)
        step = mine.state[p]["step"]
        assert step.device.type == "cpu" and float(step) == 2.0
        _steps(mine, p, [torch.randn(30, device=device)])
        assert float(step) == 3.0 and float(theirs.state[p]["step"]) == 2.0


@pytest.mark.parametrize("device", DEVICES)
def test_restored_without_a_class_coded_states_are_read_as_numbers(device):
    from dattri_llm_b200.gradient.optimizer_state import OptimizerSnapshot, optimizer_from_state_dict

    torch.manual_seed(9)
    model = torch.nn.Sequential(torch.nn.Linear(9, 5)).to(device)
    names = [n for n, _ in model.named_parameters()]
    saved = {}
    for bits in (8, 32):
        opt = bw.AdamW(model.parameters(), state_bits=bits)
        model(torch.randn(4, 9, device=device)).square().sum().backward()
        opt.step()
        saved[bits] = copy.deepcopy(opt.state_dict())
        again = optimizer_from_state_dict(model, saved[bits], names)
        assert isinstance(again, bw.AdamW) == (bits == 8)
        for key in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(OptimizerSnapshot(model, again).state("0", key), OptimizerSnapshot(model, opt).state("0", key))
    with pytest.raises(ValueError, match="8-bit codes"):
        optimizer_from_state_dict(model, saved[8], names, optimizer_cls=torch.optim.NAdam)


class _Mine(bw.AdamW):
    pass


def test_a_class_that_reads_codes_is_kept():
    from dattri_llm_b200.gradient.optimizer_state import optimizer_from_state_dict

    model = torch.nn.Linear(3, 2)
    opt = bw.AdamW(model.parameters(), state_bits=8)
    model(torch.ones(1, 3)).sum().backward()
    opt.step()
    again = optimizer_from_state_dict(model, opt.state_dict(), [n for n, _ in model.named_parameters()], optimizer_cls=_Mine)
    assert type(again) is _Mine and again.state[model.weight]["exp_avg"].dtype == torch.float8_e4m3fn


@pytest.mark.parametrize("device", DEVICES)
def test_scales_given_twice_are_refused(device):
    params = [torch.ones(300, device=device) for _ in range(2)]
    m, v, s = zip(*(ops.adamw_state(p, 8) for p in params), strict=True)
    before = [x.clone() for x in (*params, *s)]
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step(params, [p.clone() for p in params], m, v, [s[0], s[0]], step=1, lr=0.1)
    assert all(torch.equal(x, y) for x, y in zip((*params, *s), before, strict=True))
    empty = [torch.ones(0, device=device) for _ in range(2)]  # nothing to write
    m, v, s = zip(*(ops.adamw_state(p, 8) for p in empty), strict=True)
    ops.adamw_step(empty, [p.clone() for p in empty], m, v, [s[0], s[0]], step=1, lr=0.1)


def test_coded_states_are_restored_by_a_function_that_makes_the_class():
    import functools

    from dattri_llm_b200.gradient.optimizer_state import optimizer_from_state_dict

    model = torch.nn.Linear(3, 2)
    names = [n for n, _ in model.named_parameters()]
    opt = bw.AdamW(model.parameters(), state_bits=8)
    model(torch.ones(1, 3)).sum().backward()
    opt.step()
    again = optimizer_from_state_dict(model, opt.state_dict(), names, optimizer_cls=functools.partial(bw.AdamW, state_bits=8))
    assert torch.equal(again.moment(model.weight, "exp_avg"), opt.moment(model.weight, "exp_avg"))
    with pytest.raises(ValueError, match="8-bit codes"):
        optimizer_from_state_dict(model, opt.state_dict(), names, optimizer_cls=functools.partial(torch.optim.AdamW))


@pytest.mark.parametrize("bits", [8, 32])
def test_hooks_on_loading_are_followed(bits):
    """A hook's dictionary is the one that is loaded, and hooks on the loaded optimizer see its states' own types."""
    torch.manual_seed(10)
    first, second = (torch.nn.Parameter(torch.randn(20).to(torch.bfloat16)) for _ in range(2))
    opt = bw.AdamW([first, second], state_bits=bits)
    first.grad, second.grad = torch.randn_like(first), torch.randn_like(second)
    opt.step()
    other = bw.AdamW([first, second], state_bits=bits)

    def swap(_optimizer, given):
        return {**given, "state": {0: given["state"][1], 1: given["state"][0]}}

    seen = []
    other.register_load_state_dict_pre_hook(swap)
    other.register_load_state_dict_post_hook(lambda o: seen.append(o.state[first]["exp_avg"].dtype))
    other.load_state_dict(opt.state_dict())
    assert torch.equal(other.moment(first, "exp_avg"), opt.moment(second, "exp_avg"))
    assert torch.equal(other.moment(second, "exp_avg_sq"), opt.moment(first, "exp_avg_sq"))
    assert seen == [torch.float32 if bits == 32 else torch.float8_e4m3fn]
    other.load_state_dict(opt.state_dict())
    assert len(seen) == 2


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_is_loaded_into_a_parameter_that_lies_otherwise(device, bits):
    """Blocks of 256 elements go by the order of memory, which the loaded parameter need not share.  A moment that is written as
    a code for a second time is off by another 2^-4 of itself or half a step of the smallest codes."""
    torch.manual_seed(11)
    w = torch.randn(40, 33, device=device)
    w[:, 5] *= 100  # blocks of one order and of the other have other scales
    g = w * torch.rand(40, 33, device=device)
    p = torch.nn.Parameter(w.t().contiguous().t())
    opt = bw.AdamW([p], state_bits=bits)
    _steps(opt, p, [g, 2 * g])
    q = torch.nn.Parameter(w.clone())
    other = bw.AdamW([q], state_bits=bits)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert q.stride() != p.stride() and other.state[q]["exp_avg"].stride() == q.stride()
    for key in ("exp_avg", "exp_avg_sq"):
        want, got = opt.moment(p, key).double(), other.moment(q, key).double()
        if bits == 32:
            assert torch.equal(got, want)
            continue
        if key == "exp_avg_sq":
            want, got = want.sqrt(), got.sqrt()
        each = (want.abs().reshape(-1)[:1280].view(5, 256).amax(1) / 448).repeat_interleave(256)
        off, size = (x.reshape(-1)[:1280] for x in ((got - want).abs(), want.abs()))
        assert (off <= (2.0 ** -4 + SLACK) * size + (2.0 ** -9 + SLACK) * each).all()
    _steps(other, q, [g])
    assert torch.isfinite(q).all()


@pytest.mark.parametrize("device", DEVICES)
def test_axes_of_one_element_do_not_change_the_order(device):
    """Their steps say nothing of where an element lies: codes are loaded as they are."""
    torch.manual_seed(12)
    p = torch.nn.Parameter(torch.randn(1, 300, device=device))
    opt = bw.AdamW([p], state_bits=8)
    _steps(opt, p, [torch.randn(1, 300, device=device) for _ in range(3)])
    q = torch.nn.Parameter(torch.empty_strided((1, 300), (7, 1), device=device).copy_(p.detach()))
    other = bw.AdamW([q], state_bits=8)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for key in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(other.state[q][key].view(torch.uint8), opt.state[p][key].view(torch.uint8))
    assert torch.equal(other.state[q]["scales"], opt.state[p]["scales"])
    g = torch.randn(1, 300, device=device)
    _steps(opt, p, [g])
    _steps(other, q, [g])
    assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_of_another_shape_is_not_spread_over_a_parameter(bits):
    p, q = torch.nn.Parameter(torch.randn(1, 300)), torch.nn.Parameter(torch.randn(3, 300))
    opt, other = bw.AdamW([p], state_bits=bits), bw.AdamW([q], state_bits=bits)
    _steps(opt, p, [torch.randn(1, 300)])
    other.load_state_dict(copy.deepcopy(opt.state_dict()))  # as torch.optim loads it
    with pytest.raises(ValueError):
        _steps(other, q, [torch.randn(3, 300)])


@pytest.mark.parametrize("device", DEVICES)
def test_a_refused_step_changes_nothing(device):
    torch.manual_seed(13)
    p, q = torch.nn.Parameter(torch.randn(4, 3, device=device)), torch.nn.Parameter(torch.randn(4, 3, device=device))
    opt, start = bw.AdamW([p, q]), p.detach().clone()
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q).to_sparse()
    with pytest.raises(NotImplementedError):
        opt.step()
    assert all(float(opt.state[x]["step"]) == 0 for x in (p, q)) and torch.equal(p, start)
    old, q.grad = q.detach().clone(), torch.ones_like(q)
    opt.step()
    assert all(float(opt.state[x]["step"]) == 1 for x in (p, q))
    # the first step: by lr whatever the gradient's size, and the weight's decay
    assert ((old * (1 - 1e-5) - 1e-3 - q).abs() <= 4 * torch.finfo(torch.float32).eps * (1 + old.abs())).all()
