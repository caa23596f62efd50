"""Cases of the operators of trajectory training: the gated delta rule, token scores, and the AdamW step of many tensors.

``run`` makes the calls a training or scoring program makes of ``dattri_llm_b200.ops``
where ``own`` is true, and computes the same in elementary torch operations (32 bits,
rounded once at the end) where it is false.
"""

import math

import torch

own = False

IGNORE = -100
BLOCK = 256  # elements that share a scale of an 8-bit moment
F8_MAX = 448.0
F8_TINY = 2.0 ** -9
CHUNK = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_LOGITS = 8 * 1024 * 128256  # logits of the largest listed score
MOST_PARAMS = 8 * 60_821_504  # weights of the largest listed step
MOST_ROWS = 4 * 2048 * 32 * 128  # values of the largest listed delta rule


def listed():
    return [
        # AdamW. A tiny decoder's weights in 32 bits, first step: latency.
        {"name": "adamw_small", "op": "adamw", "hidden": 64, "kv": 32, "inter": 176, "layers": 2, "vocab": 512,
         "dtype": "fp32", "bits": 32, "step": 1, "packed": False},
        # Odd widths in one flat buffer (tensors that start anywhere), 16-bit floats, moments in 8 bits.
        {"name": "adamw_odd", "op": "adamw", "hidden": 333, "kv": 111, "inter": 1001, "layers": 3, "vocab": 5003,
         "dtype": "fp16", "bits": 8, "step": 17, "packed": True},
        # Eight blocks of the headline model, bf16 weights, moments in 32 bits.
        {"name": "adamw_train", "op": "adamw", "hidden": 2048, "kv": 512, "inter": 8192, "layers": 8, "vocab": 0,
         "dtype": "bf16", "bits": 32, "step": 100, "packed": False},
        # The same with moments in 8 bits.
        {"name": "adamw_train_8bit", "op": "adamw", "hidden": 2048, "kv": 512, "inter": 8192, "layers": 8, "vocab": 0,
         "dtype": "bf16", "bits": 8, "step": 100, "packed": False},
        # Token scores. One short answer of a small vocabulary with its 5 best alternatives: latency.
        {"name": "scores_small", "op": "scores", "batch": 2, "tokens": 16, "vocab": 1024, "dtype": "bf16", "masked": 0.25,
         "sliced": False, "top": 5, "temperature": 1.0, "grad": False},
        # An odd vocabulary in 16-bit floats, logits shifted by a slice, a temperature, gradients of both scores.
        {"name": "scores_odd", "op": "scores", "batch": 5, "tokens": 333, "vocab": 32003, "dtype": "fp16", "masked": 0.4,
         "sliced": True, "top": 3, "temperature": 0.8, "grad": True},
        # The headline model's micro-batch scored for selection: 20 alternatives, no gradient.
        {"name": "scores_eval", "op": "scores", "batch": 8, "tokens": 1024, "vocab": 128256, "dtype": "bf16", "masked": 0.0,
         "sliced": False, "top": 20, "temperature": 1.0, "grad": False},
        # The same micro-batch with an entropy term in the loss.
        {"name": "scores_train", "op": "scores", "batch": 8, "tokens": 1024, "vocab": 128256, "dtype": "bf16", "masked": 0.25,
         "sliced": False, "top": 0, "temperature": 1.0, "grad": True},
        # Gated delta rule. One new token of one sequence, the state held in 32 bits: latency.
        {"name": "delta_step", "op": "step", "batch": 1, "tokens": 1, "k_heads": 16, "v_heads": 32, "dk": 128, "dv": 128,
         "dtype": "bf16"},
        # One new token of 64 sequences.
        {"name": "delta_step_batch", "op": "step", "batch": 64, "tokens": 1, "k_heads": 16, "v_heads": 32, "dk": 128, "dv": 128,
         "dtype": "bf16"},
        # Odd lengths and narrow heads that continue from a state, 16-bit floats, both directions.
        {"name": "delta_odd", "op": "delta", "batch": 3, "tokens": 777, "k_heads": 3, "v_heads": 6, "dk": 64, "dv": 96,
         "dtype": "fp16", "state": True, "grad": True},
        # A training micro-batch of 2048 tokens, two value heads for each key head, both directions.
        {"name": "delta_train", "op": "delta", "batch": 4, "tokens": 2048, "k_heads": 16, "v_heads": 32, "dk": 128, "dv": 128,
         "dtype": "bf16", "state": False, "grad": True},
    ]


def _size(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["adamw", "scores", "step", "delta"])
    if op == "adamw":
        hidden = _size(rng, 33, 2048)
        inter = _size(rng, hidden, 4 * hidden)
        kv = max(1, hidden // rng.choice([1, 2, 4]))
        vocab = rng.choice([0, _size(rng, 257, 32768)])
        one = 2 * hidden * hidden + 2 * kv * hidden + 3 * inter * hidden + 2 * hidden
        layers = max(1, min(_size(rng, 1, 12), (MOST_PARAMS // 2 - vocab * hidden) // one))
        return {"op": op, "hidden": hidden, "kv": kv, "inter": inter, "layers": layers, "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "bits": rng.choice([8, 32]),
                "step": _size(rng, 1, 10000), "packed": rng.random() < 0.4}
    if op == "scores":
        vocab = _size(rng, 257, 131072)
        vocab -= vocab % rng.choice([1, 8, 64])
        tokens = _size(rng, 5, 2048)
        most = max(1, MOST_LOGITS // (2 * vocab * tokens))  # half of the largest: 32-bit logits weigh twice
        return {"op": op, "batch": min(most, _size(rng, 1, 32)), "tokens": tokens, "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "masked": rng.choice([0.0, 0.25, 0.5]),
                "sliced": rng.random() < 0.3, "top": rng.choice([0, 1, 5, 20, 32]), "temperature": rng.choice([1.0, 0.8]),
                "grad": rng.random() < 0.5}
    k_heads = rng.choice([1, 2, 4, 8, 16])
    v_heads = k_heads * rng.choice([1, 2, 4])
    dk, dv = rng.choice([32, 64, 96, 128]), rng.choice([32, 64, 96, 128])
    case = {"op": op, "k_heads": k_heads, "v_heads": v_heads, "dk": dk, "dv": dv}
    if op == "step":
        return {**case, "batch": _size(rng, 1, 96), "tokens": rng.choice([1, 1, 1, 2, 5]), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    tokens = _size(rng, 3, 8192)
    batch = max(1, min(_size(rng, 1, 16), MOST_ROWS // (2 * tokens * v_heads * max(dk, dv))))
    return {**case, "batch": batch, "tokens": tokens, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "state": rng.random() < 0.5,
            "grad": rng.random() < 0.6}


def _shapes(case):
    """The tensors of a decoder, as an optimizer holds them."""
    h, kv, inter = case["hidden"], case["kv"], case["inter"]
    block = [(h, h), (kv, h), (kv, h), (h, h), (inter, h), (inter, h), (h, inter), (h,), (h,)]
    return block * case["layers"] + ([(case["vocab"], h), (h,)] if case["vocab"] else [])


# ---------------------------------------------------------------- inputs


def _to_blocks(x):
    """A tensor's elements as (blocks, BLOCK), zeros behind the last one."""
    flat = x.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def _quantized(x, keep_nonzero):
    """8-bit values of each block relative to its largest magnitude, and the scales."""
    blocks = _to_blocks(x)
    scale = blocks.abs().amax(1) / F8_MAX
    values = blocks / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(1)
    if keep_nonzero:  # a root mean square that is not zero never becomes zero
        values = torch.where(blocks > 0, values.clamp(min=F8_TINY), values)
    return values.clamp(-F8_MAX, F8_MAX).to(torch.float8_e4m3fn).view(-1)[:x.numel()].view(x.shape), scale


def _prepare_adamw(case, gen):
    """Weights, gradients and moments as slices of flat buffers, each on an allocation's boundary unless packed."""
    shapes = _shapes(case)
    dtype = DTYPES[case["dtype"]]
    align = 1 if case["packed"] else 256
    sizes = [math.prod(s) for s in shapes]
    starts, end = [], 0
    for n in sizes:
        starts.append(end)
        end += -(-n // align) * align
    p = torch.randn(end, generator=gen, device="cuda", dtype=dtype).mul_(0.02)
    g = torch.randn(end, generator=gen, device="cuda", dtype=dtype).mul_(1e-3)
    g.view(-1)[: end // 2].mul_(torch.rand(end // 2, generator=gen, device="cuda", dtype=dtype))  # magnitudes differ
    first = case["step"] == 1
    m = torch.randn(end, generator=gen, device="cuda").mul_(0.0 if first else 3e-4)
    v = torch.rand(end, generator=gen, device="cuda").add_(0.01).square_().mul_(0.0 if first else 1e-6)
    if case["vocab"]:  # rows of the embedding that no batch has used
        rows = case["vocab"] // 3
        at = starts[-2]
        for t in (g, m, v):
            t[at:at + rows * case["hidden"]] = 0
    views = lambda t: [t[s:s + n].view(shape) for s, n, shape in zip(starts, sizes, shapes)]  # noqa: E731
    state = {"case": dict(case), "p": p, "params": views(p), "grads": views(g)}
    if case["bits"] == 32:
        return {**state, "m": m, "v": v, "exp_avgs": views(m), "exp_avg_sqs": views(v)}
    counts = [-(-n // BLOCK) for n in sizes]
    scales = torch.zeros(2 * sum(counts), device="cuda")
    m8, v8 = (torch.zeros(end, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2))
    ends = [2 * sum(counts[:i]) for i in range(len(counts))]
    state["scales"] = [scales[e:e + 2 * c].view(2, c) for e, c in zip(ends, counts)]
    state.update(m=m8, v=v8, flat_scales=scales, exp_avgs=views(m8), exp_avg_sqs=views(v8))
    for i, (x, y) in enumerate(zip(views(m), views(v))):
        for row, (to, value, root) in enumerate(((state["exp_avgs"][i], x, False), (state["exp_avg_sqs"][i], y.sqrt(), True))):
            codes, scale = _quantized(value, root)
            to.copy_(codes)
            state["scales"][i][row].copy_(scale)
    return state


def _prepare_scores(case, gen):
    """Logits of a trained model (spread 2.5, the answer's token likely) and labels with an ignored prompt and padding."""
    b, t, vocab = case["batch"], case["tokens"], case["vocab"]
    labels = torch.randint(0, vocab, (b, t), generator=gen, device="cuda")
    valid = t - round(case["masked"] * t)
    start = torch.randint(0, t - valid + 1, (b, 1), generator=gen, device="cuda")
    at = torch.arange(t, device="cuda")
    state = {"case": dict(case), "labels": torch.where((at >= start) & (at < start + valid), labels, IGNORE)}
    rows = torch.randn(b, t + int(case["sliced"]), vocab, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]]).mul_(2.5)
    logits = rows[:, :t]
    up = (math.log(vocab) + 2.0) * torch.rand(b, t, 1, generator=gen, device="cuda").add_(0.5)
    logits.scatter_add_(2, labels.unsqueeze(-1), up.to(rows.dtype))
    state["logits"] = logits.detach().requires_grad_(case["grad"])
    if case["grad"]:
        # Gradients of a loss that sums over the tokens: weights of an answer's tokens, and an entropy bonus. 16-bit floats
        # are trained with a scaled loss, or their gradients vanish.
        scale = 2.0 ** 10 if case["dtype"] == "fp16" else 1.0
        state["g_logps"] = torch.randn(b, t, generator=gen, device="cuda").sub_(1.0).mul_(scale)
        state["g_entropy"] = torch.full((b, t), -0.1 * scale, device="cuda")
    return state


def _prepare_delta(case, gen):
    """One convolution's output holds q, k and v of a token side by side, one projection's both gates."""
    b, t, hk, hv, dk, dv = (case[n] for n in ("batch", "tokens", "k_heads", "v_heads", "dk", "dv"))
    dtype = DTYPES[case["dtype"]]
    grad = case.get("grad", False)
    mixed = torch.nn.functional.silu(torch.randn(b, t, 2 * hk * dk + hv * dv, generator=gen, device="cuda", dtype=dtype).mul_(1.5))
    gates = torch.randn(b, t, 2 * hv, generator=gen, device="cuda", dtype=dtype)
    cut = lambda x, lo, heads, d: x[..., lo:lo + heads * d].view(b, t, heads, d)  # noqa: E731
    state = {"case": dict(case), "q": cut(mixed, 0, hk, dk), "k": cut(mixed, hk * dk, hk, dk), "v": cut(mixed, 2 * hk * dk, hv, dv),
             "b": gates[..., :hv], "a": gates[..., hv:]}
    state["a_log"] = torch.rand(hv, generator=gen, device="cuda").mul_(16).clamp_(min=0.01).log().to(dtype)
    state["dt_bias"] = torch.randn(hv, generator=gen, device="cuda").sub_(2.0).to(dtype)
    if case["op"] == "step" or case["state"]:
        state["state"] = torch.randn(b, hv, dk, dv, generator=gen, device="cuda").mul_(0.3)
    if grad:
        for n in ("q", "k", "v", "a", "b", "a_log", "dt_bias"):
            state[n] = state[n].detach().requires_grad_(True)
        state["g_out"] = torch.randn(b, t, hv, dv, generator=gen, device="cuda", dtype=dtype)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)
    if case["op"] == "scores":
        return _prepare_scores(case, gen)
    return _prepare_delta(case, gen)


# ---------------------------------------------------------------- the framework's calls

HYPER = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}


def _adamw_out(s):
    out = {"params": s["p"], "exp_avg": s["m"], "exp_avg_sq": s["v"]}
    if "flat_scales" in s:
        out["scales"] = s["flat_scales"]
    return out


def _own(s):
    from dattri_llm_b200 import ops

    case = s["case"]
    if case["op"] == "adamw":
        ops.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s.get("scales"), step=case["step"], **HYPER)
        return _adamw_out(s)
    if case["op"] == "scores":
        r = ops.token_scores(s["logits"], s["labels"], top_k=case["top"], temperature=case["temperature"])
        out = {"logps": r.logps.detach(), "entropy": r.entropy.detach()}
        if case["top"]:
            out.update(top_logps=r.top_logps, top_ids=r.top_ids)
        if case["grad"]:
            out["dlogits"] = torch.autograd.grad((r.logps, r.entropy), s["logits"], (s["g_logps"], s["g_entropy"]))[0]
        return out
    gates = (s["a"], s["b"], s["a_log"], s["dt_bias"])
    if case["op"] == "step":
        out = ops.gated_delta_step(s["q"], s["k"], s["v"], *gates, s["state"])
        return {"out": out, "state": s["state"]}
    if not case["grad"]:
        with torch.no_grad():
            out, last = ops.gated_delta_rule(s["q"], s["k"], s["v"], *gates, initial_state=s.get("state"),
                                             output_final_state=case["state"])
        return {"out": out, "state": last} if case["state"] else {"out": out}
    out, _ = ops.gated_delta_rule(s["q"], s["k"], s["v"], *gates, initial_state=s.get("state"))
    names = ("q", "k", "v", "a", "b", "a_log", "dt_bias")
    grads = torch.autograd.grad(out, [s[n] for n in names], s["g_out"])
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


# ---------------------------------------------------------------- the plain forms


def _plain_adamw(s):
    case = s["case"]
    lr, (b1, b2), eps, wd = HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    root2 = math.sqrt(1 - b2 ** case["step"])
    size = lr / (1 - b1 ** case["step"])
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        m, v = s["exp_avgs"][i], s["exp_avg_sqs"][i]
        g = g.float()
        if case["bits"] == 8:
            spread = lambda row: s["scales"][i][row].repeat_interleave(BLOCK)[:p.numel()].view(p.shape)  # noqa: B023, E731
            m32, v32 = m.float() * spread(0), (v.float() * spread(1)).square()
        else:
            m32, v32 = m, v
        m32 = b1 * m32 + (1 - b1) * g
        v32 = b2 * v32 + (1 - b2) * g * g
        p.copy_(p.float() * (1 - lr * wd) - size * m32 / (v32.sqrt() / root2 + eps))
        if case["bits"] == 8:
            for row, (to, value, root) in enumerate(((m, m32, False), (v, v32.sqrt(), True))):
                codes, scale = _quantized(value, root)
                to.copy_(codes)
                s["scales"][i][row].copy_(scale)
        else:
            m.copy_(m32)
            v.copy_(v32)
    return _adamw_out(s)


def _order_keys(x):
    """Whole numbers in the order of x (32 bits), the lower index first among equals."""
    bits = x.contiguous().view(torch.int32)
    bits = torch.where(x == 0, torch.zeros_like(bits), bits)  # -0 and 0 are equal
    ordered = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    return (ordered << 32) + (0xFFFFFFFF - torch.arange(x.shape[-1], device=x.device))


def _plain_scores(s):
    case = s["case"]
    b, t, k = case["batch"], case["tokens"], case["top"]
    out = {"logps": torch.zeros(b, t, device="cuda"), "entropy": torch.zeros(b, t, device="cuda")}
    if k:
        out["top_logps"] = torch.zeros(b, t, k, device="cuda")
        out["top_ids"] = torch.full((b, t, k), -1, device="cuda", dtype=torch.int64)
    if case["grad"]:
        out["dlogits"] = torch.zeros(b, t, case["vocab"], device="cuda", dtype=DTYPES[case["dtype"]])
    for i in range(b):  # a sequence at a time: 32-bit copies of all logits would not fit beside three states
        x = s["logits"][i].detach().float()
        label = s["labels"][i]
        valid = label != IGNORE
        at = label.clamp(min=0).unsqueeze(1)
        if k:
            top = 0xFFFFFFFF - (_order_keys(x).topk(k, dim=-1).values & 0xFFFFFFFF)
        x = x / case["temperature"]
        x = x - x.amax(-1, keepdim=True)
        e = x.exp()
        z = e.sum(-1, keepdim=True)
        p, logs = e / z, x - z.log()
        logp = logs.gather(1, at)
        entropy = -(p * logs).sum(-1, keepdim=True)
        out["logps"][i] = torch.where(valid, logp.squeeze(1), 0.0)
        out["entropy"][i] = torch.where(valid, entropy.squeeze(1), 0.0)
        if k:
            out["top_ids"][i] = torch.where(valid.unsqueeze(1), top, -1)
            out["top_logps"][i] = torch.where(valid.unsqueeze(1), logs.gather(1, top), 0.0)
        if case["grad"]:
            gl, ge = s["g_logps"][i].unsqueeze(1), s["g_entropy"][i].unsqueeze(1)
            d = -p * (gl + ge * (logs + entropy))
            d.scatter_add_(1, at, gl)
            out["dlogits"][i] = torch.where(valid.unsqueeze(1), d / case["temperature"], 0.0)
    return out


def _gates(s, dtype):
    """Log-decay and write strength of every token and value head."""
    dt = s["a"].to(dtype) + s["dt_bias"].to(dtype)
    return -s["a_log"].to(dtype).exp() * torch.nn.functional.softplus(dt), torch.sigmoid(s["b"].to(dtype))


def _unit_rows(s, dtype):
    """q (scaled) and k of every value head, rows of length one."""
    group = s["case"]["v_heads"] // s["case"]["k_heads"]
    unit = lambda x: x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    q, k = unit(s["q"].to(dtype)) * s["case"]["dk"] ** -0.5, unit(s["k"].to(dtype))
    return q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)


def _plain_delta(s):
    """Chunks of 64 tokens: a triangular system within, a state between them."""
    case = s["case"]
    b, t, h, dk, dv = (case[n] for n in ("batch", "tokens", "v_heads", "dk", "dv"))
    q, k = _unit_rows(s, torch.float32)
    g, beta = _gates(s, torch.float32)
    pad = -t % CHUNK
    cut = lambda x: torch.nn.functional.pad(  # noqa: E731
        x.transpose(1, 2), (0, 0, 0, pad) if x.dim() == 4 else (0, pad)).unflatten(2, (-1, CHUNK))
    q, k, v, g, beta = (cut(x) for x in (q, k, s["v"].float(), g, beta))
    total = g.double().cumsum(-1)  # differences of long sums
    lower = torch.ones(CHUNK, CHUNK, device="cuda", dtype=torch.bool).tril()
    decay = (total.unsqueeze(-1) - total.unsqueeze(-2)).masked_fill(~lower, -math.inf).float().exp()
    total = total.float()
    mix = ((k @ k.transpose(-1, -2)) * decay * beta.unsqueeze(-2)).tril(-1)
    rows = [torch.zeros_like(mix[..., 0, :])]
    for i in range(1, CHUNK):  # the inverse of I + mix, less I, row by row
        before = torch.stack(rows, -2)
        rows.append(-mix[..., i, :] - (mix[..., i, :i].unsqueeze(-2) @ before).squeeze(-2))
    inverse = torch.stack(rows, -2) + torch.eye(CHUNK, device="cuda")
    scores = (q @ k.transpose(-1, -2)) * decay
    grown, left = total.exp().unsqueeze(-1), (total[..., -1:] - total).exp().unsqueeze(-1)
    state = s["state"] if "state" in s else torch.zeros(b, h, dk, dv, device="cuda")
    outs = []
    for c in range(q.shape[2]):
        new = beta[:, :, c].unsqueeze(-1) * (inverse[:, :, c] @ (v[:, :, c] - grown[:, :, c] * (k[:, :, c] @ state)))
        outs.append(grown[:, :, c] * (q[:, :, c] @ state) + scores[:, :, c] @ new)
        state = grown[:, :, c, -1:] * state + (left[:, :, c] * k[:, :, c]).transpose(-1, -2) @ new
    out = torch.stack(outs, 2).flatten(2, 3)[:, :, :t].transpose(1, 2)
    return out, state


def _plain_step(s):
    q, k = _unit_rows(s, torch.float32)
    g, beta = _gates(s, torch.float32)
    v, state, outs = s["v"].float(), s["state"], []
    for t in range(s["case"]["tokens"]):
        state.mul_(g[:, t, :, None, None].exp())
        key = k[:, t].unsqueeze(-1)
        write = beta[:, t].unsqueeze(-1) * (v[:, t] - (state * key).sum(-2))
        state.add_(key * write.unsqueeze(-2))
        outs.append((state * q[:, t].unsqueeze(-1)).sum(-2))
    return {"out": torch.stack(outs, 1).to(s["v"].dtype), "state": state}


def _plain(s):
    case = s["case"]
    if case["op"] == "adamw":
        return _plain_adamw(s)
    if case["op"] == "scores":
        return _plain_scores(s)
    if case["op"] == "step":
        return _plain_step(s)
    dtype = DTYPES[case["dtype"]]
    if not case["grad"]:
        with torch.no_grad():
            out, last = _plain_delta(s)
        return {"out": out.to(dtype), "state": last} if case["state"] else {"out": out.to(dtype)}
    out, _ = _plain_delta(s)
    names = ("q", "k", "v", "a", "b", "a_log", "dt_bias")
    grads = torch.autograd.grad(out, [s[n] for n in names], s["g_out"].float())
    return {"out": out.detach().to(dtype), **{"d" + n: g for n, g in zip(names, grads)}}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass has to read, write and compute


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * (n // BLOCK)
        return {"bytes": 3 * size * n + moments, "flops": 15 * n}
    if case["op"] == "scores":
        rows = case["batch"] * (case["tokens"] - round(case["masked"] * case["tokens"]))
        read = rows * case["vocab"] * size
        wrote = case["batch"] * case["tokens"] * case["vocab"] * size if case["grad"] else 0
        return {"bytes": read + wrote + case["batch"] * case["tokens"] * (16 + 12 * case["top"]),
                "flops": rows * case["vocab"] * (12 if case["grad"] else 6)}
    b, t, hk, hv, dk, dv = (case[n] for n in ("batch", "tokens", "k_heads", "v_heads", "dk", "dv"))
    io = b * t * size * (2 * hk * dk + 2 * hv * dv + 2 * hv)  # q, k, v, both gates and the output
    held = b * hv * dk * dv * 4
    if case["op"] == "step":
        return {"bytes": io + 2 * held, "flops": 8 * b * t * hv * dk * dv}
    # A token's products with the state (read twice, written once) and with the tokens before it in its chunk.
    flops = b * t * hv * (6 * dk * dv + CHUNK * (2 * dk + 2 * dv))
    reads = held if case["state"] else 0
    if not case["grad"]:
        return {"bytes": io + 2 * reads, "flops": flops}
    # The backward reads q, k, v, the gates and the output's gradient and writes five gradients.
    grads = b * t * size * (4 * hk * dk + 3 * hv * dv + 4 * hv)
    return {"bytes": io + grads + 2 * reads, "flops": 7 * flops // 2}


# ---------------------------------------------------------------- from the definitions, in 64 bits


def _exact_adamw(case, s):
    b1, b2 = HYPER["betas"]
    out = {n: t.to(torch.float64) for n, t in (("params", s["p"]), ("exp_avg", s["m"]), ("exp_avg_sq", s["v"]))}
    if case["bits"] == 8:
        out["scales"] = s["flat_scales"].double()
    origin = {n: t.data_ptr() for n, t in (("params", s["p"]), ("exp_avg", s["m"]), ("exp_avg_sq", s["v"]))}
    for i, p in enumerate(s["params"]):
        n = p.numel()
        at = {name: (t.data_ptr() - origin[name]) // t.element_size()
              for name, t in (("params", p), ("exp_avg", s["exp_avgs"][i]), ("exp_avg_sq", s["exp_avg_sqs"][i]))}
        place = {name: out[name][a:a + n] for name, a in at.items()}
        m, v = place["exp_avg"].clone(), place["exp_avg_sq"].clone()
        if case["bits"] == 8:
            block = torch.arange(n, device="cuda") // BLOCK
            scales = s["scales"][i].double()
            m, v = m * scales[0][block], (v * scales[1][block]) ** 2
        g = s["grads"][i].reshape(-1).double()
        m += (g - m) * (1 - b1)
        v += (g ** 2 - v) * (1 - b2)
        place["params"] -= HYPER["lr"] * HYPER["weight_decay"] * place["params"]
        place["params"] -= HYPER["lr"] * (m / (1 - b1 ** case["step"])) / ((v / (1 - b2 ** case["step"])).sqrt() + HYPER["eps"])
        if case["bits"] == 32:
            place["exp_avg"].copy_(m)
            place["exp_avg_sq"].copy_(v)
            continue
        at_scale = (s["scales"][i].data_ptr() - s["flat_scales"].data_ptr()) // 4
        for row, (name, x) in enumerate((("exp_avg", m), ("exp_avg_sq", v.sqrt()))):
            top = torch.zeros(scales.shape[1], device="cuda", dtype=torch.float64).scatter_reduce(0, block, x.abs(), "amax")
            scale = top / F8_MAX
            ratio = torch.nan_to_num(x / scale[block])
            if name == "exp_avg_sq":
                ratio = torch.where((x > 0) & (ratio < F8_TINY), F8_TINY, ratio)
            place[name].copy_(ratio.float().to(torch.float8_e4m3fn))
            out["scales"][at_scale + row * len(scale):at_scale + (row + 1) * len(scale)] = scale
    return out


def _exact_scores(case, s):
    k = case["top"]
    parts = {n: [] for n in ("logps", "entropy", "top_logps", "top_ids", "dlogits")}
    for i in range(case["batch"]):
        raw, keep = s["logits"][i].detach().double(), (s["labels"][i] != IGNORE)
        x = raw / case["temperature"]
        lse = torch.logsumexp(x, -1)
        at = s["labels"][i].clamp(min=0)
        p = torch.exp(x - lse[:, None])
        entropy = lse - (p * x).sum(-1)
        parts["logps"].append((x[torch.arange(len(x), device="cuda"), at] - lse) * keep)
        parts["entropy"].append(entropy * keep)
        if k:
            rest, ids = raw.clone(), []
            for _ in range(k):
                best = rest.max(-1, keepdim=True).values
                ids.append((rest == best).to(torch.uint8).argmax(-1))  # the first of the equal ones
                rest.scatter_(1, ids[-1][:, None], -math.inf)
            ids = torch.stack(ids, -1)
            parts["top_ids"].append(torch.where(keep[:, None], ids, -1))
            parts["top_logps"].append((x.gather(1, ids) - lse[:, None]) * keep[:, None])
        if case["grad"]:
            one = torch.zeros_like(x).scatter_(1, at[:, None], 1.0)
            gl, ge = s["g_logps"][i].double()[:, None], s["g_entropy"][i].double()[:, None]
            d = gl * (one - p) - ge * p * (x - lse[:, None] + entropy[:, None])
            parts["dlogits"].append((d * keep[:, None] / case["temperature"]).float())  # at 32 bits: the largest would not fit
    out = {n: torch.stack(v) for n, v in parts.items() if v}
    return out


def _exact_delta(case, s):
    """Token by token, and back: the derivative of each line of the recurrence."""
    f = torch.float64
    group = case["v_heads"] // case["k_heads"]
    raw = {n: s[n].detach().to(f) for n in ("q", "k", "v", "a", "b", "a_log", "dt_bias")}
    lengths = {n: torch.sqrt((raw[n] ** 2).sum(-1, keepdim=True) + 1e-6) for n in ("q", "k")}
    q1, k1 = raw["q"] / lengths["q"], raw["k"] / lengths["k"]
    scale = case["dk"] ** -0.5
    wide = lambda x: x.repeat_interleave(group, 2).permute(1, 0, 2, 3).contiguous()  # noqa: E731  time first
    q, k, v = wide(q1) * scale, wide(k1), raw["v"].permute(1, 0, 2, 3)
    dt = raw["a"] + raw["dt_bias"]
    soft = torch.logaddexp(dt, torch.zeros_like(dt))
    g = (-torch.exp(raw["a_log"]) * soft).permute(1, 0, 2)
    decay, beta = torch.exp(g), (1 / (1 + torch.exp(-raw["b"]))).permute(1, 0, 2)
    t = case["tokens"]
    state = s["state"].to(f).clone() if "state" in s else torch.zeros(case["batch"], case["v_heads"], case["dk"], case["dv"], device="cuda", dtype=f)
    grad = case.get("grad", False)
    every = 32
    marks, out = [], torch.empty(v.shape, device="cuda", dtype=f)

    def one(state, i):
        old = state * decay[i][..., None, None]
        gap = v[i] - torch.einsum("bhkv,bhk->bhv", old, k[i])
        return old, gap, old + torch.einsum("bhk,bhv->bhkv", k[i], beta[i][..., None] * gap)

    for i in range(t):
        if i % every == 0:
            marks.append(state)
        _, _, state = one(state, i)
        out[i] = torch.einsum("bhkv,bhk->bhv", state, q[i])
    result = {"out": out.permute(1, 0, 2, 3)}
    if not grad:
        return {**result, "state": state} if case["op"] == "step" or case["state"] else result
    go = s["g_out"].to(f).permute(1, 0, 2, 3)
    dq, dk, dv, dg, dbeta = (torch.empty(x.shape, device="cuda", dtype=f) for x in (q, k, v, g, beta))
    ds = torch.zeros_like(state)
    for start in range((t - 1) // every * every, -1, -every):
        kept, state = [], marks[start // every]
        for i in range(start, min(t, start + every)):
            old, gap, new = one(state, i)
            kept.append((state, old, gap, new))
            state = new
        for i in range(min(t, start + every) - 1, start - 1, -1):
            before, old, gap, new = kept[i - start]
            dq[i] = torch.einsum("bhkv,bhv->bhk", new, go[i])
            ds = ds + torch.einsum("bhk,bhv->bhkv", q[i], go[i])
            dwrite = torch.einsum("bhkv,bhk->bhv", ds, k[i])
            dv[i] = beta[i][..., None] * dwrite
            dbeta[i] = (dwrite * gap).sum(-1)
            dk[i] = torch.einsum("bhkv,bhv->bhk", ds, beta[i][..., None] * gap) - torch.einsum("bhkv,bhv->bhk", old, dv[i])
            ds = ds - torch.einsum("bhk,bhv->bhkv", k[i], dv[i])
            dg[i] = (ds * before).sum((-1, -2)) * decay[i]
            ds = ds * decay[i][..., None, None]
    narrow = lambda x: x.permute(1, 0, 2, 3).unflatten(2, (-1, group)).sum(3)  # noqa: E731
    through = lambda d, y, n: (d - y * (y * d).sum(-1, keepdim=True)) / n  # noqa: E731
    result["dq"] = through(narrow(dq) * scale, q1, lengths["q"])
    result["dk"] = through(narrow(dk), k1, lengths["k"])
    result["dv"] = dv.permute(1, 0, 2, 3)
    dg, beta, dbeta = (x.permute(1, 0, 2) for x in (dg, beta, dbeta))
    da = dg * -torch.exp(raw["a_log"]) / (1 + torch.exp(-dt))
    result["da"] = da
    result["db"] = dbeta * beta * (1 - beta)
    result["da_log"] = (dg * g.permute(1, 0, 2)).sum((0, 1))
    result["ddt_bias"] = da.sum((0, 1))
    return result


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "adamw":
            return _exact_adamw(case, s)
        if case["op"] == "scores":
            return _exact_scores(case, s)
        return _exact_delta(case, s)
