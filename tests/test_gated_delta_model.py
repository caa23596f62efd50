"""Hugging Face gated delta nets on the library's kernels, and the operators of a trajectory together: a hybrid decoder
trained by the streamer with 8-bit AdamW, its tokens scored, its per-sample gradients captured."""

from __future__ import annotations

import copy
import math
import tempfile
import warnings

import pytest
import torch
from torch.utils.data import DataLoader

transformers = pytest.importorskip("transformers")

import dattri_llm_b200 as bw  # noqa: E402
from dattri_llm_b200 import ops  # noqa: E402
from dattri_llm_b200.models import accelerate_gated_delta, entropy_regularized_loss, token_logps, token_quality  # noqa: E402
from dattri_llm_b200.models import gated_delta as gd  # noqa: E402

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
VOCAB = 64


def _model(device="cpu", dtype=torch.float32):
    if not hasattr(transformers, "Qwen3NextConfig"):
        pytest.skip("not in this Transformers version")
    warnings.filterwarnings("ignore")
    cfg = transformers.Qwen3NextConfig(
        vocab_size=VOCAB, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=2,
        head_dim=16, linear_num_value_heads=4, linear_num_key_heads=2, linear_key_head_dim=16, linear_value_head_dim=8,
        linear_conv_kernel_dim=4, num_experts=2, num_experts_per_tok=1, moe_intermediate_size=16,
        shared_expert_intermediate_size=16, layer_types=["linear_attention", "full_attention"], max_position_embeddings=256)
    from transformers.models.qwen3_next import modeling_qwen3_next as modeling

    # The model's own PyTorch path, whatever packages with kernels of their own are installed.
    others = ("FusedRMSNormGated", "chunk_gated_delta_rule", "fused_recurrent_gated_delta_rule", "causal_conv1d_fn", "causal_conv1d_update")
    with pytest.MonkeyPatch.context() as patch:
        for name in others:
            patch.setattr(modeling, name, None, raising=False)
        torch.manual_seed(0)
        model = transformers.Qwen3NextForCausalLM(cfg)
    if hasattr(model.config, "_experts_implementation"):
        model.config._experts_implementation = "eager"
    return model.to(device, dtype).eval()


def _ids(b, t, device="cpu", seed=1):
    return torch.randint(0, VOCAB, (b, t), generator=torch.Generator().manual_seed(seed)).to(device)


@pytest.mark.parametrize("padded", [False, True])
def test_forward_and_gradients_match_the_library_model(padded):
    theirs = _model()
    mine = copy.deepcopy(theirs)
    assert accelerate_gated_delta(mine, linears=False) == 1
    ids = _ids(3, 75)
    mask = torch.ones_like(ids)
    if padded:
        mask[1, :20] = 0
    want, got = (m(input_ids=ids, attention_mask=mask).logits for m in (theirs, mine))
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)
    keep = mask.unsqueeze(-1).bool()
    want.masked_fill(~keep, 0).pow(2).mean().backward()
    got.masked_fill(~keep, 0).pow(2).mean().backward()
    for (name, p), q in zip(theirs.named_parameters(), mine.parameters(), strict=True):
        if p.grad is not None or q.grad is not None:
            torch.testing.assert_close(q.grad, p.grad, rtol=1e-3, atol=1e-6, msg=name)


@pytest.mark.parametrize("device", DEVICES)
def test_generation_goes_on_from_the_cached_state(device):
    """A prompt and cached tokens give the logits of the whole sequence."""
    model = _model(device, torch.float32 if device == "cpu" else torch.bfloat16)
    accelerate_gated_delta(model)
    ids = _ids(2, 40, device)
    with torch.no_grad():
        want = model(input_ids=ids).logits
        out = model(input_ids=ids[:, :33], use_cache=True)
        got = [out.logits]
        for t in range(33, 40):
            out = model(input_ids=ids[:, t:t + 1], past_key_values=out.past_key_values, use_cache=True)
            got.append(out.logits)
    state = out.past_key_values.layers[0].recurrent_states
    assert state.dtype == torch.float32
    # two orders of the same sums; on the GPU every layer's output is rounded to bf16 (2^-8) some ten times on the way
    tol = 1e-4 if device == "cpu" else 10 * 2.0 ** -8
    assert (torch.cat(got, 1) - want).abs().max() <= tol * want.abs().max()


def test_a_cached_token_does_not_lose_gradients_in_silence():
    """The step in place has none: where they are wanted, the mixer runs its own forward, and a backward does what the
    library's does (it raises: the cached state was updated in place)."""
    logits = []
    for fast in (False, True):
        model = _model()
        if fast:
            accelerate_gated_delta(model, linears=False)
        ids = _ids(2, 9)
        with torch.no_grad():
            cache = model(input_ids=ids[:, :8], use_cache=True).past_key_values
        logits.append(model(input_ids=ids[:, 8:], past_key_values=cache, use_cache=True).logits)
        with pytest.raises(RuntimeError, match="inplace"):
            logits[-1].square().sum().backward()
    torch.testing.assert_close(logits[1], logits[0], rtol=1e-4, atol=1e-4 * float(logits[0].detach().abs().max()))


@pytest.mark.gpu
def test_bf16_model_stays_near_the_library_model_in_fp32():
    theirs = _model("cuda")
    mine = copy.deepcopy(theirs).to(torch.bfloat16)
    calls = ops.launch_count()
    accelerate_gated_delta(mine)
    ids = _ids(2, 130, "cuda")
    want, got = theirs(input_ids=ids).logits, mine(input_ids=ids).logits
    assert ops.launch_count() > calls
    plain = copy.deepcopy(theirs).to(torch.bfloat16)(input_ids=ids).logits
    # the model's own path in bf16 sets the scale: the kernels keep more digits between the layers' roundings, not fewer
    mine_off, plain_off = ((x.double() - want.double()).norm() for x in (got, plain))
    assert mine_off <= 1.5 * plain_off
    got.float().pow(2).mean().backward()
    want.pow(2).mean().backward()
    for (name, p), q in zip(theirs.named_parameters(), mine.named_parameters(), strict=True):
        if p.grad is not None and "linear_attn" in name:
            assert torch.isfinite(q[1].grad).all()
            cos = torch.nn.functional.cosine_similarity(p.grad.flatten().double(), q[1].grad.flatten().double(), dim=0)
            assert cos > 0.95, name  # gradients of bf16 activations: the direction is that of fp32


@pytest.mark.gpu
def test_a_model_in_fp32_runs_the_model_itself():
    theirs = _model("cuda")
    mine = copy.deepcopy(theirs)
    accelerate_gated_delta(mine, linears=False)
    ids = _ids(2, 30, "cuda")
    assert torch.equal(mine(input_ids=ids).logits, theirs(input_ids=ids).logits)


def test_capture_overrides_keep_the_installed_forward():
    model = _model()
    accelerate_gated_delta(model, linears=False)
    mixers = [m for m in model.modules() if gd.is_gated_delta_mixer(m)]
    ids = _ids(2, 16)
    for _ in range(2):
        hm = bw.HookManager(model, bw.HookManagerConfig(linear_io=[r"linear_attn\.(in_proj_qkvz|in_proj_ba|out_proj)$"]),
                            callbacks=[bw.CaptureCallback()])
        with hm.collect():
            model(input_ids=ids).logits.float().pow(2).sum().backward()
        hm.remove()
        assert all(m.forward.__func__ is gd._mixer_forward for m in mixers)


def _rows(n):
    return [{"input_ids": x, "labels": x} for x in _ids(n, 24, seed=7)]


def _loss(model, batch):
    return entropy_regularized_loss(model, batch, coef=0.1)


@pytest.mark.parametrize("device", DEVICES)
def test_a_trajectory_with_all_of_them(device):
    """A hybrid decoder trained on a few batches by the streamer: its mixers on the gated delta rule, the loss on token scores
    with an entropy term, the update by 8-bit AdamW, every sample's gradient captured and the optimizer's moments
    recorded, the tokens scored before and after; the captured gradients against plain autograd at each step."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    model = _model(device, dtype)
    accelerate_gated_delta(model)
    other = copy.deepcopy(model)
    for m in other.modules():  # a copied module's forward is bound to the original
        if gd.is_gated_delta_mixer(m):
            del m.__dict__["forward"]
    accelerate_gated_delta(other)
    rows = _rows(6)
    batch = {k: torch.stack([r[k] for r in rows]).to(device) for k in rows[0]}
    before = token_quality(model, batch, top_k=3)
    near = token_logps(model, batch)
    assert (before.logps - near).abs().max() <= 2e-5 * (1 + near.abs().max())
    assert (before.top_logps[:, :, 0] >= before.logps)[:, :-1].all()
    assert (before.entropy[:, :-1] <= math.log(VOCAB) + 1e-4).all() and (before.top_ids[:, -1] == -1).all()
    args = bw.AttributionArguments(output_dir=tempfile.mkdtemp(), learning_rate=1e-2, weight_decay=0.1, optim="adamw_8bit",
                                   lr_scheduler_type="constant", seed=5, per_device_train_batch_size=2)
    cfg = bw.HookManagerConfig(linear_io=[r"linear_attn\.(in_proj_qkvz|out_proj)$"])
    streamer = bw.GradientStreamer(model, rows, args, batch_size=2, enable_update=True, loss_fn=_loss, config=cfg,
                                   defer_update=True)
    assert isinstance(streamer.optimizer, bw.AdamW) and streamer.optimizer.param_groups[0]["state_bits"] == 8
    loader = DataLoader(rows, batch_size=2, shuffle=True, generator=torch.Generator().manual_seed(5))
    name = "model.layers.0.linear_attn.out_proj"
    steps = 0
    with streamer:
        for (_step, grad, _hashes), part in zip(streamer, loader, strict=True):
            part = {k: v.to(device) for k, v in part.items()}
            got = grad.materialize().data[name].reshape(2, -1)
            other.load_state_dict(model.state_dict())  # the update is due, not done: the weights of this step
            other.zero_grad()
            _loss(other, part).backward()
            whole = other.get_submodule(name).weight.grad.reshape(-1)
            scale = whole.float().abs().max()
            # bf16 gradients of two samples and their sum: three roundings, and those of one backward pass against another's
            assert ((got.sum(0).float() - whole.float()).abs() <= (1e-5 if device == "cpu" else 4 * 2.0 ** -8) * scale).all()
            steps += 1
    assert steps == 3
    states = streamer.optimizer.state
    assert states and all(st["exp_avg"].dtype == torch.float8_e4m3fn for st in states.values())
    after = token_quality(model, batch)
    moved = (after.logps - before.logps).abs().max()
    assert torch.isfinite(after.logps).all() and moved > 0


def test_moments_of_coded_states_are_recorded():
    """The optimizer-state callback of a trajectory reads 8-bit moments as numbers."""
    model = _model()
    accelerate_gated_delta(model)
    opt = bw.AdamW(model.parameters(), lr=1e-2, state_bits=8)
    callback = bw.OptimizerStateCallback(model, opt)
    hm = bw.HookManager(model, bw.HookManagerConfig(linear_io=[r"linear_attn\.out_proj$"]), callbacks=[callback])
    batch = {"input_ids": _ids(2, 12), "labels": _ids(2, 12)}
    with hm.collect():
        for _ in range(2):
            opt.zero_grad()
            _loss(model, batch).backward()
            opt.step()
    hm.remove()
    weight = model.get_submodule("model.layers.0.linear_attn.out_proj").weight
    records = [r["layers"]["model.layers.0.linear_attn.out_proj"] for r in callback.pre.values()]
    assert not records[0][0].any() and records[1][0].dtype == torch.float32
    assert records[1][0].numel() == weight.numel() and records[1][0].abs().max() > 0 and records[1][1].min() >= 0


def _state_gradients(model, ids, loss):
    """Gradients of a mixer's projection, the only one trained, from a prompt whose cache goes on."""
    weight = model.requires_grad_(False).model.layers[0].linear_attn.in_proj_qkvz.weight.requires_grad_(True)
    cache = model(input_ids=ids[:, :12], use_cache=True).past_key_values
    loss(model, cache).backward()
    return weight.grad


def test_a_prompt_gets_the_gradients_of_cached_tokens():
    """A loss on a cached token reaches the prompt's projections through the state too, as in the library's model."""
    ids = _ids(2, 13)
    grads = []
    for fast in (False, True):
        model = _model()
        if fast:
            accelerate_gated_delta(model, linears=False)
        grads.append(_state_gradients(model, ids, lambda m, cache: m(input_ids=ids[:, 12:], past_key_values=cache,
                                                                      use_cache=True).logits.square().sum()))
    torch.testing.assert_close(grads[1], grads[0], rtol=1e-3, atol=1e-5 * float(grads[0].abs().max()))


@pytest.mark.gpu
def test_a_prompts_state_has_its_gradient_on_the_gpu():
    def loss(_model, cache):
        return cache.layers[0].recurrent_states.float().square().sum()

    want = _state_gradients(_model("cuda"), _ids(2, 13, "cuda"), loss)  # fp32: the model itself
    mine = _model("cuda", torch.bfloat16)
    accelerate_gated_delta(mine)
    got = _state_gradients(mine, _ids(2, 13, "cuda"), loss)
    cos = torch.nn.functional.cosine_similarity(want.flatten().double(), got.flatten().double(), dim=0)
    assert cos > 0.95  # gradients of bf16 activations: the direction is that of fp32


@pytest.mark.parametrize("register", ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                                      "register_full_backward_pre_hook"])
def test_a_watched_convolution_is_called_as_a_module(register, monkeypatch):
    """Whatever kind of hook it has, also where the fused kernel would take it."""
    mixer = next(m for m in _model().modules() if gd.is_gated_delta_mixer(m))
    monkeypatch.setattr(gd.fused, "causal_conv_silu_enabled", lambda x, conv: True)
    monkeypatch.setattr(gd.fused, "causal_conv_silu", lambda x, weight, bias: x * 0)
    seen = []
    handle = getattr(mixer.conv1d, register)(lambda *a: seen.append(1))
    x = torch.randn(2, 5, mixer.conv_dim, requires_grad=True)
    gd._convolved(mixer, x).sum().backward()
    assert seen
    handle.remove()
    assert not gd._convolved(mixer, x).any()


def test_cached_tokens_of_a_model_in_64_bits():
    model = _model(dtype=torch.float64)
    accelerate_gated_delta(model, linears=False)
    ids = _ids(2, 12)
    with torch.no_grad():
        want = model(input_ids=ids).logits[:, 9:]
        out = model(input_ids=ids[:, :9], use_cache=True)
        got = []
        for t in range(9, 12):
            out = model(input_ids=ids[:, t:t + 1], past_key_values=out.past_key_values, use_cache=True)
            got.append(out.logits)
    assert out.past_key_values.layers[0].recurrent_states.dtype == torch.float64
    # the mixer and its state stay in 64 bits; the model's own norms and angles round to 32, in another order of sums
    assert (torch.cat(got, 1) - want).abs().max() <= 1e-5 * want.abs().max()
