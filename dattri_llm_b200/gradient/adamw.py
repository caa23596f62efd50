"""AdamW over the multi-tensor kernel of :func:`dattri_llm_b200.ops.adamw_step`, moments in 32 or 8 bits.

A trajectory's optimizer states outweigh its 16-bit weights four to one; in 8 bits they weigh
as much as the weights.  The update rule is ``torch.optim.AdamW``'s, so everything that reads
optimizer state (snapshots, preconditioned capture, the dynamics of AdamW-influence) follows
it; :meth:`AdamW.moment` gives those readers the numbers that 8-bit states stand for.
"""

from __future__ import annotations

import torch

from dattri_llm_b200.ops.optim import adamw_moments, adamw_state, adamw_state_like, adamw_step


def _refuse(group: dict) -> None:
    """Settings of ``torch.optim.AdamW``'s groups that would change the update and are not implemented here."""
    for key in ("amsgrad", "differentiable"):
        if group.get(key):
            raise NotImplementedError(f"AdamW of this library does not implement {key}=True")


class AdamW(torch.optim.AdamW):
    """``torch.optim.AdamW`` whose step is one launch for all tensors of a group and type.

    Args:
        state_bits: 32 (fp32 moments, whatever the parameters' type) or 8 (e4m3 codes with a
            scale for every 256 elements); also a setting of a parameter group.  It says how the
            states of new parameters are held: loaded ones keep the form that they were saved in.

    The update counts are kept on the host: a step is not captured into a CUDA graph, which
    would repeat one count's bias correction.  Parameters sharded as DTensors (FSDP2) are not
    supported, nor are ``amsgrad`` and ``differentiable``, in a group or in a loaded state.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, maximize: bool = False) -> None:
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize)
        self.defaults["state_bits"] = state_bits
        for group in self.param_groups:
            self._settle(group)

    def _settle(self, group: dict) -> None:
        _refuse(group)
        bits = group.setdefault("state_bits", self.defaults["state_bits"])
        if bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {bits}")
        for p in group["params"]:
            if hasattr(p, "to_local") and hasattr(p, "placements"):
                raise NotImplementedError("AdamW of this library steps whole tensors, not DTensors")

    def add_param_group(self, param_group: dict) -> None:
        _refuse(param_group)
        super().add_param_group(param_group)
        if "state_bits" in self.defaults:  # not while the base class is being made
            self._settle(self.param_groups[-1])

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("this optimizer counts its updates on the host: a captured step would repeat one count's "
                               "bias correction")
        for group in self.param_groups:
            bits = group["state_bits"]
            batches: dict[tuple, list[list]] = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["step"] = torch.tensor(0.0)
                    state["exp_avg"], state["exp_avg_sq"], scales = adamw_state(p, bits)
                    if scales is not None:
                        state["scales"] = scales
                lists = batches.setdefault((p.device, int(state["step"]) + 1, "scales" in state), [[], [], [], [], [], []])
                for to, x in zip(lists, (p, p.grad, state["exp_avg"], state["exp_avg_sq"], state.get("scales"), state["step"]),
                                 strict=True):
                    to.append(x)
            for (_device, step, coded), (params, grads, m, v, scales, counts) in batches.items():
                adamw_step(params, grads, m, v, scales if coded else None, step=step, lr=float(group["lr"]),
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                           maximize=group["maximize"])
                for count in counts:  # a refused step is not counted
                    count += 1
        return loss

    def moment(self, param: torch.Tensor, key: str) -> torch.Tensor | None:
        """State *key* of *param* in the numbers it stands for; ``None`` before its first update."""
        state = self.state.get(param, {})
        if "scales" not in state or key not in ("exp_avg", "exp_avg_sq"):
            return state.get(key)
        m, v = adamw_moments(state["exp_avg"], state["exp_avg_sq"], state["scales"])
        return m if key == "exp_avg" else v

    def load_state_dict(self, state_dict: dict) -> None:
        """As ``torch.optim``'s, without its cast of the states to the parameters' type.  A state of
        ``torch.optim.AdamW`` is taken too; ``state_bits``, which it does not have, stay as they are."""
        bits = [group["state_bits"] for group in self.param_groups]
        final: dict = {}  # what the user's hooks make of the dictionary

        def look(_optimizer, given: dict) -> None:
            for group in given["param_groups"]:
                _refuse(group)
            final.update(given)

        def keep(_optimizer) -> None:
            for group, own in zip(self.param_groups, bits, strict=True):
                group.setdefault("state_bits", own)
                self._settle(group)
            self._keep_types(final)

        # Behind the other hooks on the dictionary, before those on the loaded optimizer.
        hooks = [self.register_load_state_dict_pre_hook(look), self.register_load_state_dict_post_hook(keep, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _keep_types(self, state_dict: dict) -> None:
        """The states as they were saved, which ``torch.optim`` has cast to the parameters' types."""
        saved = state_dict["state"]
        ids = (i for group in state_dict["param_groups"] for i in group["params"])
        params = (p for group in self.param_groups for p in group["params"])
        for i, p in zip(ids, params, strict=True):
            if "step" in saved.get(i, {}):  # fused and capturable optimizers count on the GPU, where each step would wait for it
                self.state[p]["step"] = torch.tensor(float(saved[i]["step"]))
            for key, value in saved.get(i, {}).items():
                if isinstance(value, torch.Tensor) and key != "step":
                    self.state[p][key] = value.detach().to(p.device, copy=True)
            state = self.state.get(p, {})
            if any(state[key].shape != p.shape for key in {"exp_avg", "exp_avg_sq"} & state.keys()):
                continue  # of another parameter: the step refuses it
            if "scales" in state:
                keys = ("exp_avg", "exp_avg_sq", "scales")
                state.update(zip(keys, adamw_state_like(p, *(state[key] for key in keys)), strict=True))
                continue
            for key in {"exp_avg", "exp_avg_sq"} & state.keys():  # another AdamW may keep them in the parameters' type
                state[key] = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(state[key])
