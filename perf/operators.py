"""Cases of the post-training operators: preference and policy losses, router balance loss, head norms with rotation.

``run`` makes the calls a training or serving program makes of ``dattri_llm_b200.ops``
where ``own`` is true, and computes the same in elementary torch operations (32 bits,
rounded once at the end) where it is false.
"""

import math

import torch

own = False

IGNORE = -100
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_LOGITS = 8 * 1024 * 128256  # logits of the largest listed loss
MOST_ROUTED = 16 * 65536 * 64  # router logits of the largest listed balance loss
MOST_HEADS = 8 * 2048 * 40 * 128  # q and k elements of the largest listed rotation


def listed():
    return [
        # Preference loss. The small configuration's vocabulary, two short pairs: latency.
        {"name": "preference_small", "op": "preference", "pairs": 2, "tokens": 24, "vocab": 1024, "dtype": "bf16",
         "masked": 0.25, "empty": False, "sliced": False, "smoothing": 0.0, "grad": True},
        # Long prompts, an odd vocabulary, logits shifted by a slice, one answer without a token, noisy preferences.
        {"name": "preference_odd", "op": "preference", "pairs": 3, "tokens": 333, "vocab": 32003, "dtype": "fp16",
         "masked": 0.4, "empty": True, "sliced": True, "smoothing": 0.1, "grad": True},
        # The headline model's vocabulary and micro-batch (8 x 1024 tokens) as four pairs.
        {"name": "preference_train", "op": "preference", "pairs": 4, "tokens": 1024, "vocab": 128256, "dtype": "bf16",
         "masked": 0.25, "empty": False, "sliced": False, "smoothing": 0.0, "grad": True},
        # Policy loss. A few short rollouts of a tiny model, an advantage for each token: latency.
        {"name": "policy_small", "op": "policy", "batch": 4, "tokens": 16, "vocab": 512, "dtype": "bf16", "masked": 0.25,
         "empty": False, "sliced": False, "per_token": True, "kl": 0.0, "temperature": 1.0, "reduction": "token_mean"},
        # Logits kept in 32 bits, an odd vocabulary, a KL term, sampling temperature, one empty rollout.
        {"name": "policy_odd", "op": "policy", "batch": 5, "tokens": 257, "vocab": 50277, "dtype": "fp32", "masked": 0.3,
         "empty": True, "sliced": False, "per_token": False, "kl": 0.04, "temperature": 0.8, "reduction": "sequence_mean"},
        # The headline model's vocabulary and micro-batch as rollouts with group-normalised advantages and a KL term.
        {"name": "policy_train", "op": "policy", "batch": 8, "tokens": 1024, "vocab": 128256, "dtype": "bf16", "masked": 0.25,
         "empty": False, "sliced": False, "per_token": False, "kl": 0.04, "temperature": 1.0, "reduction": "token_mean"},
        # Balance loss. One layer of a tiny expert model, router logits in 32 bits: latency.
        {"name": "balance_small", "op": "balance", "groups": 1, "tokens": 64, "experts": 8, "top_k": 2, "dtype": "fp32",
         "masked": 0.0, "given": False, "z": 0.0, "grad": True},
        # 60 experts, odd lengths, padded tokens, the model's own choice of experts, the logits' size held down too.
        {"name": "balance_odd", "op": "balance", "groups": 24, "tokens": 2047, "experts": 60, "top_k": 4, "dtype": "bf16",
         "masked": 0.2, "given": True, "z": 0.001, "grad": True},
        # 16 layers with 64 experts, top 8, 32 sequences of 2048 tokens, every layer's loss in one call.
        {"name": "balance_train", "op": "balance", "groups": 16, "tokens": 65536, "experts": 64, "top_k": 8, "dtype": "bf16",
         "masked": 0.0, "given": False, "z": 0.0, "grad": True},
        # Head norms and rotation. One new token of 8 sequences at positions of their own: latency.
        {"name": "qk_decode", "op": "qk", "batch": 8, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 64, "rotary": 64,
         "dtype": "bf16", "weights": "bf16", "positions": True, "table": 8192, "grad": False},
        # Part of each head rotated, 96-wide heads, odd lengths, 16-bit floats with weights in 32 bits.
        {"name": "qk_odd", "op": "qk", "batch": 3, "tokens": 777, "heads": 12, "kv_heads": 4, "dim": 96, "rotary": 48,
         "dtype": "fp16", "weights": "fp32", "positions": False, "table": 777, "grad": True},
        # The 8B configuration's heads (32 / 8 of 128) at its sequence length of 2048, 8 sequences, both directions.
        {"name": "qk_train", "op": "qk", "batch": 8, "tokens": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "dtype": "bf16", "weights": "bf16", "positions": False, "table": 2048, "grad": True},
    ]


def _size(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["preference", "policy", "balance", "qk"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("preference", "policy"):
        vocab = _size(rng, 257, 131072)
        vocab -= vocab % rng.choice([1, 8, 64])
        tokens = _size(rng, 5, 2048)
        most = max(2, MOST_LOGITS // (2 * vocab * tokens)) // 2  # half of the largest: 32-bit logits weigh twice
        case = {"op": op, "tokens": tokens, "vocab": vocab, "dtype": dtype, "masked": rng.choice([0.0, 0.25, 0.5]),
                "empty": rng.random() < 0.3, "sliced": rng.random() < 0.3}
        if op == "preference":
            return {**case, "pairs": min(most, _size(rng, 1, 16)), "smoothing": rng.choice([0.0, 0.1]), "grad": rng.random() < 0.8}
        return {**case, "batch": 2 * min(most, _size(rng, 1, 16)), "per_token": rng.random() < 0.5, "kl": rng.choice([0.0, 0.04]),
                "temperature": rng.choice([1.0, 0.8]), "reduction": rng.choice(["token_mean", "sequence_mean"])}
    if op == "balance":
        experts = rng.choice([8, 16, 60, 64, 96, 128, 256])
        tokens = _size(rng, 33, 65536)
        return {"op": op, "groups": max(1, min(_size(rng, 1, 32), MOST_ROUTED // (2 * experts * tokens))), "tokens": tokens,
                "experts": experts, "top_k": rng.choice([1, 2, 4, 8]), "dtype": dtype, "masked": rng.choice([0.0, 0.3]),
                "given": rng.random() < 0.4, "z": rng.choice([0.0, 0.001]), "grad": rng.random() < 0.8}
    dim = rng.choice([64, 80, 96, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 3, 4, 7])
    grad = rng.random() < 0.7
    tokens = _size(rng, 65, 4096) if grad else rng.choice([1, 1, 3, _size(rng, 65, 4096)])
    batch = max(1, min(_size(rng, 1, 64), MOST_HEADS // (2 * tokens * (heads + kv_heads) * dim)))
    positions = rng.random() < 0.5
    return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": dim if rng.random() < 0.7 else dim // 2, "dtype": dtype, "weights": rng.choice([dtype, "fp32"]),
            "positions": positions, "table": 8192 if positions else tokens, "grad": grad}


# ---------------------------------------------------------------- inputs


def _answers(case, gen, batch):
    """Labels with an ignored prompt before and padding after each answer."""
    tokens, dev = case["tokens"], "cuda"
    valid = tokens - round(case["masked"] * tokens)
    labels = torch.randint(0, case["vocab"], (batch, tokens), generator=gen, device=dev)
    start = torch.randint(0, tokens - valid + 1, (batch, 1), generator=gen, device=dev)
    at = torch.arange(tokens, device=dev)
    keep = (at >= start) & (at < start + valid)
    if case["empty"]:
        keep[-1] = False
    return torch.where(keep, labels, IGNORE)


def _logits(case, gen, labels):
    """Logits of a trained model: spread 2.5, the answer's token likely; a slice of longer rows where the case shifts."""
    batch, tokens = labels.shape
    vocab = case["vocab"]
    rows = torch.randn(batch, tokens + int(case["sliced"]), vocab, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]]).mul_(2.5)
    logits = rows[:, :tokens]
    up = (math.log(vocab) + 2.0) * torch.rand(batch, tokens, 1, generator=gen, device="cuda").add_(0.5)
    logits.scatter_add_(2, labels.clamp(min=0).unsqueeze(-1), up.to(rows.dtype))
    return logits


def _logps_now(logits, labels, temperature):
    """Log-probabilities of the labels, a sequence at a time."""
    out = []
    for x, y in zip(logits, labels):
        x = x.float() / temperature
        out.append(x.gather(1, y.clamp(min=0).unsqueeze(1)).squeeze(1) - x.logsumexp(1))
    return torch.stack(out)


def _off_the_edge(noise):
    """Log-ratios with none so near the clip at 0.8 or 1.2 that rounding decides its side."""
    ratio = noise.exp()
    near = ((ratio - 0.8).abs() < 1e-3) | ((ratio - 1.2).abs() < 1e-3)
    return torch.where(near, noise * 1.02, noise)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": dict(case)}
    if case["op"] in ("preference", "policy"):
        batch = 2 * case["pairs"] if case["op"] == "preference" else case["batch"]
        state["labels"] = labels = _answers(case, gen, batch)
        logits = _logits(case, gen, labels)
        now = _logps_now(logits, labels, case.get("temperature", 1.0))
        noise = torch.randn(2, *labels.shape, generator=gen, device="cuda")
        if case["op"] == "preference":
            # The reference model's log-probability of each sequence, as a data set keeps it.
            state["ref"] = ((now + 0.3 * noise[0]) * (labels != IGNORE)).sum(1)
            state["logits"] = logits.detach().requires_grad_(case["grad"])
            return state
        state["old"] = now - _off_the_edge(0.15 * noise[0])
        state["ref"] = now + 0.3 * noise[1]
        if case["per_token"]:
            state["advantages"] = torch.randn(labels.shape, generator=gen, device="cuda").add_(0.3)
        else:
            reward = torch.rand(batch, generator=gen, device="cuda")
            state["advantages"] = (reward - reward.mean()) / (reward.std() + 1e-4) + 0.05
        state["logits"] = logits.detach().requires_grad_(True)
        return state
    if case["op"] == "balance":
        shape = (case["groups"], case["tokens"], case["experts"])
        lean = torch.randn(case["groups"], 1, case["experts"], generator=gen, device="cuda")  # experts differ in popularity
        logits = (torch.randn(shape, generator=gen, device="cuda") + 0.5 * lean).to(DTYPES[case["dtype"]])
        state["logits"] = logits.requires_grad_(case["grad"])
        state["mask"] = state["ids"] = None
        if case["masked"]:
            state["mask"] = torch.rand(shape[:2], generator=gen, device="cuda") >= case["masked"]
            state["mask"][-1, shape[1] // 2:] = False
        if case["given"]:
            state["ids"] = logits.detach().float().topk(case["top_k"], dim=-1).indices
        # The coefficient in the training loss; 16-bit floats are trained with a scaled loss, or their gradients vanish.
        scale = 2.0 ** 14 if case["dtype"] == "fp16" else 1.0
        state["weight"] = torch.full((case["groups"],), 0.01 * scale, device="cuda")
        return state
    b, t, h, kv, d = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
    dtype, wdtype = DTYPES[case["dtype"]], DTYPES[case["weights"]]
    # One projection's output holds q, k and v of a token side by side; attention returns gradients head by head.
    qkv = torch.randn(b, t, (h + 2 * kv) * d, generator=gen, device="cuda", dtype=dtype)
    state["q"] = qkv[..., :h * d].view(b, t, h, d).detach().requires_grad_(case["grad"])
    state["k"] = qkv[..., h * d:(h + kv) * d].view(b, t, kv, d).detach().requires_grad_(case["grad"])
    for name in ("q_weight", "k_weight"):
        w = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
        state[name] = w.to(wdtype).requires_grad_(case["grad"])
    half = case["rotary"] // 2
    angles = torch.outer(torch.arange(case["table"], device="cuda", dtype=torch.float32),
                         1.0 / (500000.0 ** (torch.arange(half, device="cuda", dtype=torch.float32) / half)))
    state["cos"], state["sin"] = angles.cos(), angles.sin()
    state["positions"] = None
    if case["positions"]:
        state["positions"] = torch.randint(0, case["table"] - t + 1, (b, 1), generator=gen, device="cuda") + torch.arange(t, device="cuda")
    if case["grad"]:
        state["gq"] = torch.randn(b, h, t, d, generator=gen, device="cuda", dtype=dtype).transpose(1, 2)
        state["gk"] = torch.randn(b, kv, t, d, generator=gen, device="cuda", dtype=dtype).transpose(1, 2)
    return state


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    from dattri_llm_b200 import ops

    case = s["case"]
    if case["op"] == "preference":
        if not case["grad"]:
            with torch.no_grad():
                loss, logps = ops.preference_loss(s["logits"], s["labels"], s["ref"], beta=0.1, label_smoothing=case["smoothing"])
            return {"loss": loss, "logps": logps}
        loss, logps = ops.preference_loss(s["logits"], s["labels"], s["ref"], beta=0.1, label_smoothing=case["smoothing"])
        return {"loss": loss.detach(), "logps": logps.detach(), "dlogits": torch.autograd.grad(loss, s["logits"])[0]}
    if case["op"] == "policy":
        loss, logps, kl, clipped = ops.policy_loss(
            s["logits"], s["labels"], s["advantages"], s["old"], s["ref"] if case["kl"] else None, clip=(0.2, 0.2),
            kl_coef=case["kl"], temperature=case["temperature"], reduction=case["reduction"])
        grad = torch.autograd.grad(loss, s["logits"])[0]
        return {"loss": loss.detach(), "logps": logps.detach(), "kl": kl, "clip_fraction": clipped, "dlogits": grad}
    if case["op"] == "balance":
        if not case["grad"]:
            with torch.no_grad():
                loss, counts = ops.router_balance_loss(s["logits"], case["top_k"], s["ids"], s["mask"], z_coef=case["z"])
            return {"loss": loss, "counts": counts}
        loss, counts = ops.router_balance_loss(s["logits"], case["top_k"], s["ids"], s["mask"], z_coef=case["z"])
        grad = torch.autograd.grad(loss, s["logits"], s["weight"])[0]
        return {"loss": loss.detach(), "counts": counts, "dlogits": grad}
    if not case["grad"]:
        with torch.no_grad():
            q, k = ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"], eps=EPS)
        return {"q": q, "k": k}
    q, k = ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"], eps=EPS)
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["gq"], s["gk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": grads[0], "dk": grads[1], "dqw": grads[2], "dkw": grads[3]}


# ---------------------------------------------------------------- the plain forms


def _softmax_parts(x):
    """exp(x - max), its sum and the log of the sum of exp(x), over the last axis."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True)
    return e, z, (top + torch.log(z)).squeeze(-1)


def _token_logps(x, labels):
    e, z, lse = _softmax_parts(x)
    valid = labels != IGNORE
    at = labels.clamp(min=0).unsqueeze(-1)
    logps = torch.where(valid, x.gather(2, at).squeeze(-1) - lse, 0.0)
    return e, z, at, valid, logps


def _dlogits(e, z, at, valid, coef, dtype):
    """coef (onehot - softmax), zero in ignored rows."""
    coef = torch.where(valid, coef, 0.0).unsqueeze(-1)
    g = e.mul_(-coef / z)
    g.scatter_add_(2, at, coef)
    return torch.where(valid.unsqueeze(-1), g, 0.0).to(dtype)


def _log_sigmoid(x):
    return torch.minimum(x, torch.zeros_like(x)) - torch.log1p(torch.exp(-x.abs()))


def _plain_preference(s):
    case, beta, eps = s["case"], 0.1, s["case"]["smoothing"]
    pairs = case["pairs"]
    logits = s["logits"].detach()
    e, z, at, valid, logps = _token_logps(logits.float(), s["labels"])
    total = logps.sum(1)
    ratio = total - s["ref"]
    m = beta * (ratio[:pairs] - ratio[pairs:])
    loss = (-(1 - eps) * _log_sigmoid(m) - eps * _log_sigmoid(-m)).mean()
    if not case["grad"]:
        return {"loss": loss, "logps": total}
    d = beta * (1 / (1 + torch.exp(-m)) - (1 - eps)) / pairs
    coef = torch.cat([d, -d]).unsqueeze(1).expand_as(valid)
    return {"loss": loss, "logps": total, "dlogits": _dlogits(e, z, at, valid, coef, logits.dtype)}


def _plain_policy(s):
    case, dtype = s["case"], s["logits"].dtype
    x = s["logits"].detach().float()
    if case["temperature"] != 1.0:
        x = x / case["temperature"]
    e, z, at, valid, logps = _token_logps(x, s["labels"])
    adv = s["advantages"] if case["per_token"] else s["advantages"].unsqueeze(1)
    ratio = torch.exp(torch.where(valid, logps - s["old"], 0.0))
    free, held = ratio * adv, ratio.clamp(0.8, 1.2) * adv
    token = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, 0.0)
    kl = torch.zeros_like(logps)
    if case["kl"]:
        d = torch.where(valid, s["ref"] - logps, 0.0)
        kl = torch.expm1(d) - d
        token = token + case["kl"] * kl
        slope = slope - case["kl"] * torch.expm1(d)
    count = valid.sum()
    if case["reduction"] == "token_mean":
        weight = (1.0 / count.clamp(min=1)).expand(valid.shape[0], 1)
    else:
        weight = 1.0 / valid.sum(1, keepdim=True).clamp(min=1) / valid.shape[0]
    loss = (torch.where(valid, token, 0.0) * weight).sum()
    mean = 1.0 / count.clamp(min=1)
    clipped = ((held < free) & valid).sum() * mean
    grad = _dlogits(e, z, at, valid, slope * weight / case["temperature"], dtype)
    return {"loss": loss, "logps": logps, "kl": torch.where(valid, kl, 0.0).sum() * mean, "clip_fraction": clipped, "dlogits": grad}


def _plain_balance(s):
    case, logits = s["case"], s["logits"].detach()
    experts = case["experts"]
    e, z, lse = _softmax_parts(logits.float())
    p = e / z
    mask = torch.ones_like(lse, dtype=torch.bool) if s["mask"] is None else s["mask"]
    ids = s["ids"]
    if ids is None:  # the largest, the lowest index where they tie
        ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :case["top_k"]]
    chosen = mask.unsqueeze(-1).expand_as(ids).reshape(case["groups"], -1)
    counts = torch.zeros(case["groups"], experts, dtype=torch.int64, device=logits.device)
    counts.scatter_add_(1, ids.reshape(case["groups"], -1), chosen.to(torch.int64))
    n = mask.sum(1).clamp(min=1).unsqueeze(-1)
    weights = mask.unsqueeze(-1) / n.unsqueeze(-1)
    f = counts / n
    mean_p = torch.where(mask.unsqueeze(-1), p, 0.0).sum(1) / n
    loss = experts * (f * mean_p).sum(1)
    if case["z"]:
        loss = loss + case["z"] * (torch.where(mask, lse, 0.0).square().sum(1) / n.squeeze(-1))
    if not case["grad"]:
        return {"loss": loss, "counts": counts}
    f = f.unsqueeze(1)
    g = experts * p * (f - (f * p).sum(-1, keepdim=True))
    if case["z"]:
        g = g + 2 * case["z"] * lse.unsqueeze(-1) * p
    g = g * weights * s["weight"].view(-1, 1, 1)
    return {"loss": loss, "counts": counts, "dlogits": torch.where(mask.unsqueeze(-1), g, 0.0).to(logits.dtype)}


def _turn(x, cos, sin, half):
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_qk(s):
    case = s["case"]
    half, tokens = case["rotary"] // 2, case["tokens"]
    cos, sin = (t[:tokens] if s["positions"] is None else t[s["positions"]] for t in (s["cos"], s["sin"]))
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)

    def one(x, w, g):
        x, w = x.detach(), w.detach()
        x32, w32 = x.float(), w.float()
        r = torch.rsqrt(x32.square().mean(-1, keepdim=True) + EPS)
        n = x32 * r
        y = _turn(n * w32, cos, sin, half).to(x.dtype)
        if g is None:
            return y, None, None
        dy = _turn(g.float(), cos, -sin, half)
        dw = (dy * n).sum((0, 1, 2)).to(w.dtype)
        dn = dy * w32
        return y, (r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(x.dtype), dw

    q, dq, dqw = one(s["q"], s["q_weight"], s.get("gq"))
    k, dk, dkw = one(s["k"], s["k_weight"], s.get("gk"))
    if not case["grad"]:
        return {"q": q, "k": k}
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"preference": _plain_preference, "policy": _plain_policy, "balance": _plain_balance,
                "qk": _plain_qk}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work and exact values


def work(case):
    width = {"bf16": 2, "fp16": 2, "fp32": 4}
    size = width[case["dtype"]]
    if case["op"] in ("preference", "policy"):
        batch = 2 * case["pairs"] if case["op"] == "preference" else case["batch"]
        answers = batch - int(case["empty"])
        valid = answers * (case["tokens"] - round(case["masked"] * case["tokens"]))  # an ignored row's logits need no reading
        rows = batch * case["tokens"]
        grad = case.get("grad", True)
        return {"bytes": valid * case["vocab"] * size + grad * rows * case["vocab"] * size + rows * 16,
                "flops": valid * case["vocab"] * (4 + 3 * grad)}
    if case["op"] == "balance":
        n = case["groups"] * case["tokens"]
        return {"bytes": n * case["experts"] * size * (1 + case["grad"]) + n * 8 * case["top_k"] * case["given"],
                "flops": n * case["experts"] * (5 + 5 * case["grad"])}
    n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    table = min(case["table"], case["batch"] * case["tokens"]) * case["rotary"] * 4
    # Forward: x read, y written. Backward: the gradient read and dx written; x is read once for both.
    return {"bytes": n * size * (4 if case["grad"] else 2) + table, "flops": n * (18 if case["grad"] else 7)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("preference", "policy"):
        grad = case.get("grad", True)
        x = s["logits"].detach().double().requires_grad_(grad)
        labels, keep = s["labels"], (s["labels"] != IGNORE).double()
        tau = case.get("temperature", 1.0)
        logps = torch.log_softmax(x / tau if tau != 1.0 else x, -1).gather(2, labels.clamp(min=0)[..., None])[..., 0] * keep
        if case["op"] == "preference":
            total = logps.sum(1)
            chosen, rejected = (total - s["ref"].double()).chunk(2)
            m = 0.1 * (chosen - rejected)
            eps = case["smoothing"]
            ls = torch.nn.functional.logsigmoid
            loss = -((1 - eps) * ls(m) + eps * ls(-m)).mean()
            out = {"loss": loss.detach(), "logps": total.detach()}
            if grad:
                out["dlogits"] = torch.autograd.grad(loss, x)[0]
            return out
        adv = s["advantages"].double() if case["per_token"] else s["advantages"].double()[:, None]
        ratio = torch.exp((logps - s["old"].double()) * keep)
        inside = (ratio * adv <= ratio.detach().clamp(0.8, 1.2) * adv)
        gain = torch.where(inside, ratio * adv, ratio.detach().clamp(0.8, 1.2) * adv)
        d = (s["ref"].double() - logps) * keep
        kl = (torch.expm1(d) - d) * (1 if case["kl"] else 0)
        token = (case["kl"] * kl - gain) * keep
        if case["reduction"] == "token_mean":
            loss = token.sum() / keep.sum().clamp(min=1)
        else:
            loss = (token.sum(1) / keep.sum(1).clamp(min=1)).mean()
        count = keep.sum().clamp(min=1)
        return {"loss": loss.detach(), "logps": logps.detach(), "kl": (kl * keep).sum().detach() / count,
                "clip_fraction": ((~inside) * keep).sum() / count, "dlogits": torch.autograd.grad(loss, x)[0]}
    if case["op"] == "balance":
        x = s["logits"].detach().double().requires_grad_(case["grad"])
        keep = torch.ones(x.shape[:2], dtype=torch.float64, device=x.device) if s["mask"] is None else s["mask"].double()
        ids = s["ids"]
        if ids is None:
            ids = torch.argsort(-x.detach(), dim=-1, stable=True)[..., :case["top_k"]]
        hits = torch.zeros_like(x.detach()).scatter_add_(2, ids, torch.ones_like(ids, dtype=torch.float64)) * keep[..., None]
        n = keep.sum(1).clamp(min=1)
        mean_p = (torch.softmax(x, -1) * keep[..., None]).sum(1) / n[:, None]
        loss = case["experts"] * (hits.sum(1) / n[:, None] * mean_p).sum(1)
        loss = loss + case["z"] * (torch.logsumexp(x, -1).square() * keep).sum(1) / n
        out = {"loss": loss.detach(), "counts": hits.sum(1).to(torch.int64)}
        if case["grad"]:
            out["dlogits"] = torch.autograd.grad(loss, x, s["weight"].double())[0]
        return out
    half = case["rotary"] // 2
    at = torch.arange(case["tokens"], device="cuda") if s["positions"] is None else s["positions"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[at].unsqueeze(-2)
    out = {}
    for name in ("q", "k"):
        x = s[name].detach().double().requires_grad_(case["grad"])
        w = s[name + "_weight"].detach().double().requires_grad_(case["grad"])
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
        y = torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)
        out[name] = y.detach()
        if case["grad"]:
            out["d" + name], out["d%sw" % name] = torch.autograd.grad(y, (x, w), s["g" + name].double())
    return out
