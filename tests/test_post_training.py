"""The post-training losses in the models: head norms in the decoder, loss functions over pairs and rollouts,
the router's balance in expert blocks, launch checks of the new entry points, and the example that runs them together."""

import os
import re
import subprocess
import sys

import pytest
import torch

from dattri_llm_b200 import ops
from dattri_llm_b200.models import (
    LlamaConfig,
    LlamaForCausalLM,
    policy_token_loss,
    preference_pair_loss,
    shift_labels,
    stacked_balance_loss,
    token_logps,
)
from dattri_llm_b200.models.llama import apply_rope
from dattri_llm_b200.ops import checks
from dattri_llm_b200.parallel import moe

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(dev, qk_norm=True):
    model = LlamaForCausalLM(LlamaConfig.tiny(qk_norm=qk_norm))
    model.reset_parameters(seed=0)
    model = model.to(dev, torch.bfloat16 if dev == "cuda" else torch.float32)
    if qk_norm:
        gen = torch.Generator().manual_seed(1)
        for layer in model.model.layers:
            for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                norm.weight.data.copy_(1 + 0.2 * torch.randn(norm.weight.shape, generator=gen))
    return model


def _batch(dev, b=4, t=21):
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 512, (b, t), generator=gen)
    labels = ids.masked_fill(torch.rand(b, t, generator=gen) < 0.3, -100)
    return {"input_ids": ids.to(dev), "labels": labels.to(dev)}


def test_head_norms_are_parameters_only_where_asked_for():
    names = {n.split(".")[-2] for n, _ in _model("cpu").named_parameters()}
    plain = {n.split(".")[-2] for n, _ in _model("cpu", qk_norm=False).named_parameters()}
    assert names - plain == {"q_norm", "k_norm"}


def test_head_norms_of_attention():
    """The attention of the first layer, its norms and rotation written out."""
    model = _model("cpu")
    at = model.model.layers[0].self_attn
    x = torch.randn(2, 9, 128, generator=torch.Generator().manual_seed(0))
    cos, sin = model.model.rotary_emb(9, x.device, x.dtype)
    got = at(x, cos, sin)
    q, k = at.q_proj(x).view(2, 9, 4, 32), at.k_proj(x).view(2, 9, 2, 32)
    q, k = (z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + 1e-5) * n.weight for z, n in ((q, at.q_norm), (k, at.k_norm)))
    q, k = apply_rope(q.transpose(1, 2), k.transpose(1, 2), cos, sin)
    v = at.v_proj(x).view(2, 9, 2, 32).transpose(1, 2)
    k, v = (z.repeat_interleave(2, dim=1) for z in (k, v))
    s = (q @ k.transpose(2, 3) / 32**0.5).masked_fill(~torch.ones(9, 9, dtype=torch.bool).tril(), -torch.inf)
    want = at.o_proj((s.softmax(-1) @ v).transpose(1, 2).reshape(2, 9, -1))
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
def test_head_norms_fused_and_by_module_agree():
    """The fused pass against the modules, which run while a hook watches a norm: outputs and weight gradients."""
    model, batch = _model("cuda"), _batch("cuda")
    grads = []
    launches = []
    for watch in (False, True):
        handles = [layer.self_attn.q_norm.register_forward_hook(lambda *a: None) for layer in model.model.layers] if watch else []
        before = ops.native().post_training_launches()
        loss = preference_pair_loss(model, {**batch, "ref_logps": torch.zeros(4, device="cuda")}, beta=0.1)
        loss.backward()
        launches.append(ops.native().post_training_launches() - before)
        for h in handles:
            h.remove()
        grads.append([p.grad.float().clone() for p in model.parameters()])
        model.zero_grad()
    layers = len(model.model.layers)
    assert launches == [3 + 3 * layers, 3]  # per layer: one forward, two backward
    for a, b in zip(*grads):
        assert float((a - b).norm()) <= 0.05 * float(b.norm()) + 1e-3  # bf16 activations, rounded at other places


def test_shift_labels():
    assert shift_labels(torch.tensor([[1, 2, 3], [4, -100, 5]])).tolist() == [[2, 3, -100], [-100, 5, -100]]


@pytest.mark.parametrize("dev", DEVICES)
def test_losses_of_a_model(dev):
    model, batch = _model(dev), _batch(dev)
    with torch.no_grad():
        logits = model(input_ids=batch["input_ids"]).logits
        labels = batch["labels"][:, 1:]
        logp = torch.log_softmax(logits[:, :-1].float(), -1).gather(2, labels.clamp(min=0)[..., None])[..., 0]
        logp = logp * (labels != -100)
    got = token_logps(model, batch)
    torch.testing.assert_close(got[:, :-1], logp, rtol=1e-4, atol=1e-4)
    assert not got[:, -1].any()
    ref = logp.sum(1) + torch.tensor([1.0, -1.0, 0.5, 2.0], device=dev)
    m = -ref + logp.sum(1)
    m = m[:2] - m[2:]
    loss = preference_pair_loss(model, {**batch, "ref_logps": ref}, beta=0.3)
    torch.testing.assert_close(loss.float(), -torch.nn.functional.logsigmoid(0.3 * m).sum(), rtol=1e-3, atol=1e-3)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    adv = torch.tensor([1.0, -1.0, 0.5, 2.0], device=dev)
    pol = policy_token_loss(model, {**batch, "advantages": adv, "old_logps": token_logps(model, batch) + 0.1})
    r = torch.exp(torch.tensor(-0.1))  # the same policy, once e^0.1 likelier
    want = -(torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv)[:, None] * (labels != -100)).sum()
    torch.testing.assert_close(pol.float(), want.float(), rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("dev", DEVICES)
def test_balance_of_stacked_router_logits(dev):
    gen = torch.Generator().manual_seed(0)
    layers = [torch.randn(3 * 7, 6, generator=gen).to(dev) for _ in range(4)]
    mask = (torch.rand(3, 7, generator=gen) < 0.7).to(dev)
    got = stacked_balance_loss(layers, 2, mask.long())
    for i, x in enumerate(layers):
        one = ops.router_balance_loss(x, 2, mask=mask.reshape(-1))
        torch.testing.assert_close(got.loss[i], one.loss, rtol=1e-6, atol=0)
        assert torch.equal(got.counts[i], one.counts)
    assert int(got.counts[0].sum()) == 2 * int(mask.sum())


def test_expert_blocks_track_their_balance():
    block = moe.ExpertParallelMoE(16, 8, 4, 2, max_tokens=32, device=torch.device("cpu"), dtype=torch.float32)
    torch.nn.init.normal_(block.gate.weight, generator=torch.Generator().manual_seed(0))
    x = torch.randn(3, 5, 16, generator=torch.Generator().manual_seed(1))
    with pytest.raises(ValueError, match="track_balance"):
        moe.balance_loss(block)
    topv, topi = block.route(x)
    assert block.balance is None  # off unless asked for
    block.track_balance = True
    again = block.route(x)
    assert torch.equal(again[0], topv) and torch.equal(again[1], topi)
    assert torch.equal(block.balance.counts, torch.bincount(topi.reshape(-1), minlength=4))
    moe.balance_loss(block).backward()
    assert block.gate.weight.grad.abs().sum() > 0


def test_launch_checks_of_labels_ids_and_positions():
    x, y = torch.zeros(2, 3, 5), torch.tensor([[0, 4, -100], [1, 2, 3]])
    v = checks.VALIDATORS
    v["preference_loss"]((x, y, None, 0, 0.1, 0.0, False, 1, -100, None), {})
    v["policy_loss"]((x, y, None, None, None, 0.8, 1.2, 0.0, 1.0, 0, -100, None), {})
    with pytest.raises(checks.LaunchCheckError, match=r"label\[1\] = 5"):
        v["preference_loss"]((x, y + (y == 4), None, 0, 0.1, 0.0, False, 1, -100, None), {})
    with pytest.raises(checks.LaunchCheckError, match="label"):
        v["policy_loss"]((x, y, None, None, None, 0.8, 1.2, 0.0, 1.0, 0, -1, None), {})
    ids, mask = torch.tensor([[[0, 1], [9, 9]]]), torch.tensor([[True, False]])
    v["balance_loss"]((torch.zeros(1, 2, 4), ids, mask, 2, 0.0, None), {})
    v["balance_loss"]((torch.zeros(1, 2, 4), None, mask, 2, 0.0, None), {})
    with pytest.raises(checks.LaunchCheckError, match="expert id"):
        v["balance_loss"]((torch.zeros(1, 2, 4), ids, None, 2, 0.0, None), {})
    v["qk_norm_rope"]((None, None, None, None, torch.zeros(4, 2), None, torch.tensor([[0, 3]]), 1e-6, None), {})
    v["qk_norm_rope"]((None, None, None, None, torch.zeros(4, 2), None, None, 1e-6, None), {})
    with pytest.raises(checks.LaunchCheckError, match="position"):
        v["qk_norm_rope"]((None, None, None, None, torch.zeros(4, 2), None, torch.tensor([[0, 4]]), 1e-6, None), {})


@pytest.mark.gpu
def test_operators_under_launch_checks():
    """With checks on, good arguments pass and the first bad index is named before anything is launched."""
    x = torch.randn(2, 3, 5, device="cuda", requires_grad=True)
    y, zero = torch.tensor([[0, 4, -100], [1, 2, 3]], device="cuda"), torch.zeros(2, device="cuda")
    q, w = torch.randn(2, 3, 1, 8, device="cuda"), torch.ones(8, device="cuda")
    tables = torch.zeros(3, 4, device="cuda"), torch.ones(3, 4, device="cuda")
    checks.set_checks(True)
    try:
        for bad in (False, True):
            off = 5 if bad else 0
            for call in (lambda: ops.preference_loss(x, y + off, zero), lambda: ops.policy_loss(x, y + off, zero),
                         lambda: ops.router_balance_loss(x[0], 2, torch.full((3, 2), 1 + off, device="cuda")),
                         lambda: ops.qk_norm_rope(q, q, w, w, *tables, torch.tensor([0, 1, 2 + off], device="cuda"))):
                if bad:
                    with pytest.raises(checks.LaunchCheckError):
                        call()
                else:
                    call()
        ops.check_device_errors()
    finally:
        checks.set_checks(False)


@pytest.mark.parametrize("dev", DEVICES)
def test_example_runs(dev):
    env = dict(os.environ, MASTER_PORT="29517")
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "post_training.py"), "--device", dev, "--steps", "2"],
                         env=env, capture_output=True, text=True, timeout=300, check=False)
    assert out.returncode == 0, out.stderr[-2000:]
    first = re.search(r"step 0: preference ([\d.]+)", out.stdout)
    # Four pairs at the reference model itself: 4 log 2.
    assert first and abs(float(first.group(1)) - 2.7726) < (0.05 if dev == "cuda" else 1e-3)
    assert "nan" not in out.stdout


def _tracked_block(**kw):
    block = moe.ExpertParallelMoE(16, 8, 4, 2, max_tokens=32, device=torch.device("cpu"), dtype=torch.float32,
                                  track_balance=True, **kw)
    torch.nn.init.normal_(block.gate.weight, generator=torch.Generator().manual_seed(0))
    return block, torch.randn(3, 5, 16, generator=torch.Generator().manual_seed(1))


def test_a_balance_without_a_graph_is_no_training_loss():
    """A forward without gradients after the training one (an evaluation, a checkpointed block in its reentrant form)
    leaves a balance that would add nothing to the gradients: a backward through it says so."""
    block, x = _tracked_block()
    block.route(x)
    want = float(moe.balance_loss(block).detach())
    with torch.no_grad():
        block.route(x)
        assert float(moe.balance_loss(block)) == pytest.approx(want)
    loss = moe.balance_loss(block)
    assert loss.item() == pytest.approx(want)  # a number to log all the same
    with pytest.raises(RuntimeError, match="without gradients"):
        (loss * 0.01 + block.gate.weight.sum()).backward()
    block.route(x)
    moe.balance_loss(block).backward()
    assert block.gate.weight.grad.abs().sum() > 0


def test_the_balance_of_checkpointed_blocks():
    from torch.utils.checkpoint import checkpoint

    grads = []
    for how in (None, False, True):
        block, x = _tracked_block()
        x.requires_grad_()
        route = lambda z: block.route(z)[0].sum()  # noqa: E731
        y = route(x) if how is None else checkpoint(route, x, use_reentrant=how)
        total = y * 0.1 + moe.balance_loss(block)
        if how:
            with pytest.raises(RuntimeError, match="without gradients"):
                total.backward()
            continue
        total.backward()
        grads.append(block.gate.weight.grad)
    assert torch.equal(*grads)


def test_a_block_with_a_balance_is_copied_and_saved(tmp_path):
    """A reference model is a copy of the trained one; the balance of the last batch stays with the original."""
    import copy

    block, x = _tracked_block()
    block.route(x)
    twin = copy.deepcopy(block)
    assert twin.track_balance and twin.balance is None and block.balance is not None
    moe.balance_loss(block).backward()
    assert block.gate.weight.grad.abs().sum() > 0 and twin.gate.weight.grad is None
    twin.route(x)
    assert torch.equal(twin.balance.counts, block.balance.counts)
    torch.save(block, tmp_path / "block.pt")
    assert torch.load(tmp_path / "block.pt", weights_only=False).balance is None


def test_a_forward_that_is_not_tracked_leaves_no_balance():
    block, x = _tracked_block()
    block.route(x)
    block.track_balance = False
    block.route(x)
    assert block.balance is None
    with pytest.raises(ValueError, match="track_balance"):
        moe.balance_loss(block)


@pytest.mark.gpu
def test_head_norms_of_heads_wider_than_the_kernel_takes():
    """Heads of more than 512 elements go through the modules, as on the CPU."""
    model = LlamaForCausalLM(LlamaConfig.tiny(qk_norm=True, head_dim=528, num_attention_heads=2, num_key_value_heads=1))
    model.reset_parameters(seed=0)
    model, batch = model.to("cuda", torch.bfloat16), _batch("cuda", 2, 9)
    got = model(**batch).logits
    want = model.float()(**batch).logits  # the modules, in 32 bits
    assert float((got.float() - want).norm()) <= 0.05 * float(want.norm())


def test_the_balance_of_a_checkpointed_block_stays_after_its_backward():
    """The recomputation stops once it has what the backward needs, which may be within the router."""
    from torch.utils.checkpoint import checkpoint

    block, x = _tracked_block()
    y = checkpoint(lambda z: block.route(z)[0].sum(), x.requires_grad_(), use_reentrant=False)
    counts = block.balance.counts
    (y + moe.balance_loss(block)).backward()
    assert torch.equal(block.balance.counts, counts)
