"""Train a small expert decoder on preference pairs and on its own rollouts, and attribute both.

    python examples/post_training.py [--device cuda|cpu] [--steps N]

The model has norms on its query and key heads (one kernel with the rotation) and a routed
expert block in every layer.  Each preference step scores chosen against rejected answers
relative to the model's own start, each policy step pushes rollouts by their advantages
within a clip, and both add the router's balance loss.  A capture manager collects every
sequence's projected gradient along the way; at the end the pairs' gradients are compared
with a held-out pair's: which preferences taught the model what the held-out one asks.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from dattri_llm_b200 import HookManager, HookManagerConfig  # noqa: E402
from dattri_llm_b200.gradient import ops as gops  # noqa: E402
from dattri_llm_b200.models import LlamaConfig, LlamaForCausalLM, token_logps  # noqa: E402
from dattri_llm_b200.models.post_training import IGNORE, policy_token_terms, preference_pair_terms  # noqa: E402
from dattri_llm_b200.parallel.moe import ExpertParallelMoE, balance_loss  # noqa: E402

PAIRS, TOKENS, PROMPT = 4, 48, 12
BALANCE = 0.01  # of the router's loss in the training loss


def build(device: torch.device, dtype: torch.dtype) -> LlamaForCausalLM:
    """A decoder with head norms and, in place of each MLP, eight experts of which two are used."""
    cfg = LlamaConfig.tiny(qk_norm=True)
    model = LlamaForCausalLM(cfg)
    model.reset_parameters(seed=0)
    model = model.to(device, dtype)
    gen = torch.Generator().manual_seed(1)
    for layer in model.model.layers:
        moe = ExpertParallelMoE(cfg.hidden_size, 64, 8, 2, max_tokens=2 * PAIRS * TOKENS, device=device, dtype=dtype,
                                track_balance=True)
        draw = lambda *shape: 0.05 * torch.randn(*shape, generator=gen)  # noqa: E731
        moe.load_experts(draw(8, 128, cfg.hidden_size).to(dtype), draw(8, cfg.hidden_size, 64).to(dtype),
                         draw(8, cfg.hidden_size).to(dtype))
        layer.mlp = moe
    return model


def pairs(seed: int, device: torch.device) -> dict:
    """``PAIRS`` prompts, each with a chosen and a rejected answer of its own length."""
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 512, (2 * PAIRS, TOKENS), generator=gen)
    ids[PAIRS:, :PROMPT] = ids[:PAIRS, :PROMPT]
    labels = ids.clone()
    labels[:, :PROMPT] = IGNORE
    ends = torch.randint(PROMPT + 1, TOKENS + 1, (2 * PAIRS, 1), generator=gen)
    labels[torch.arange(TOKENS) >= ends] = IGNORE
    return {"input_ids": ids.to(device), "labels": labels.to(device)}


def run(device: str = "cpu", steps: int = 2) -> dict:
    """Train for *steps* of each kind; returns the losses, expert counts and pair scores."""
    dev = torch.device(device)
    dtype = torch.bfloat16 if dev.type == "cuda" else torch.float32
    model = build(dev, dtype)
    batches = [pairs(seed, dev) for seed in range(steps)]
    held_out = pairs(99, dev)
    for batch in (*batches, held_out):
        batch["ref_logps"] = token_logps(model, batch).sum(1)
    optimizer = torch.optim.SGD([p for p in model.parameters() if p.requires_grad], lr=1e-3)
    hm = HookManager(model, config=HookManagerConfig(
        linear_io=[r"\.(q_proj|k_proj|v_proj|o_proj)$"], projection_kwargs={"__default__": {"style": "logra", "proj_dim": 8}}))

    def pair_rows() -> torch.Tensor:  # the sum of both sequences' gradients, all layers side by side
        data = hm.get_gradient().data
        rows = [v if isinstance(v, torch.Tensor) else gops.materialize(v, "nn.Linear") for _, v in sorted(data.items())]
        rows = torch.cat([r.reshape(2 * PAIRS, -1).float() for r in rows], dim=1)
        return rows[:PAIRS] + rows[PAIRS:]

    losses, taught = [], []
    with hm.collect():
        for step, batch in enumerate(batches):
            hm.set_sample_ids([f"pair{step}.{i % PAIRS}.{'chosen' if i < PAIRS else 'rejected'}" for i in range(2 * PAIRS)])
            loss = preference_pair_terms(model, batch, beta=0.5, reduction="sum").loss
            (loss + BALANCE * balance_loss(model)).backward()
            taught.append(pair_rows())
            optimizer.step()
            optimizer.zero_grad()
            # Rollouts: the same sequences, sampled by the model of a step ago, rewarded for being the chosen ones.
            old = token_logps(model, batch) + 0.05
            rollout = {**batch, "old_logps": old, "ref_logps": old,
                       "advantages": torch.tensor([1.0] * PAIRS + [-1.0] * PAIRS, device=dev)}
            hm.set_sample_ids([f"rollout{step}.{i}" for i in range(2 * PAIRS)])
            terms = policy_token_terms(model, rollout, kl_coef=0.04, reduction="sum")
            (terms.loss + BALANCE * balance_loss(model)).backward()
            hm.get_gradient()
            optimizer.step()
            optimizer.zero_grad()
            losses.append((loss.item(), terms.loss.item()))
        hm.set_sample_ids([f"query.{i}" for i in range(2 * PAIRS)])
        preference_pair_terms(model, held_out, beta=0.5, reduction="sum").loss.backward()
        query = pair_rows()
    hm.remove()
    if dev.type == "cuda":
        from dattri_llm_b200 import ops

        ops.check_device_errors(dev)
    counts = torch.stack([layer.mlp.balance.counts for layer in model.model.layers])
    return {"losses": losses, "counts": counts.cpu(), "scores": torch.cat(taught).cpu() @ query.cpu().T}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--steps", type=int, default=4)
    args = ap.parse_args()
    if args.device == "cuda":
        torch.cuda.set_device(0)
    for key, value in (("MASTER_ADDR", "127.0.0.1"), ("MASTER_PORT", "29511"), ("RANK", "0"), ("WORLD_SIZE", "1")):
        os.environ.setdefault(key, value)
    if args.device == "cuda":
        dist.init_process_group("nccl", device_id=torch.device("cuda", 0))
    else:
        dist.init_process_group("gloo")
    try:
        out = run(args.device, args.steps)
    finally:
        dist.destroy_process_group()
    for step, (pref, pol) in enumerate(out["losses"]):
        print(f"step {step}: preference {pref:.4f}  policy {pol:.4f}")
    print("tokens of each expert, by layer:", out["counts"].tolist())
    print("scores of the training pairs on the held-out pairs:")
    print(out["scores"])


if __name__ == "__main__":
    main()
