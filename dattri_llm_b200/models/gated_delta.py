"""Gated delta nets of Hugging Face models (Qwen3-Next) on the library's kernels.

Without extra packages the Hugging Face mixer solves each chunk's triangular system row by row
and walks the chunks in eager PyTorch, in fp32, with the keys and queries repeated for every
value head.  :func:`accelerate_gated_delta` installs a forward that calls
:func:`~dattri_llm_b200.ops.gated_delta_rule` (and, for a cached token, the in-place
:func:`~dattri_llm_b200.ops.gated_delta_step`) on the projections themselves: the gates, the
rows' lengths and the heads' sharing are the kernels' part.

Parameters, module names and hook points are unchanged: the projections, ``conv1d``, ``norm``
and ``out_proj`` are still called as modules, so capture hooks see them as before.
"""

from __future__ import annotations

import types

import torch
import torch.nn.functional as F
from torch import nn

from dattri_llm_b200.models.layers import tc_linearize
from dattri_llm_b200.ops import fused
from dattri_llm_b200.ops.delta import MAX_GROUP, MAX_KEY_DIM, gated_delta_rule, gated_delta_step


def _supported(mixer: nn.Module, x: torch.Tensor) -> bool:
    """Whether the kernels (or their form on the CPU) take the mixer's heads in the input's type."""
    if not x.is_cuda:
        return True
    return (x.dtype in (torch.bfloat16, torch.float16) and mixer.head_k_dim % 8 == 0 and mixer.head_k_dim <= MAX_KEY_DIM
            and mixer.head_v_dim % 8 == 0 and mixer.num_v_heads <= MAX_GROUP * mixer.num_k_heads)


def _convolved(mixer: nn.Module, mixed: torch.Tensor) -> torch.Tensor:
    """``silu(conv1d(mixed))`` over the tokens of ``(B, T, C)``."""
    conv = mixer.conv1d
    watched = conv._forward_hooks or conv._forward_pre_hooks or conv._backward_hooks or conv._backward_pre_hooks
    if not watched and mixer.activation in ("silu", "swish") and fused.causal_conv_silu_enabled(mixed, conv):
        return fused.causal_conv_silu(mixed, conv.weight, conv.bias)
    return F.silu(conv(mixed.transpose(1, 2))[..., :mixed.shape[1]]).transpose(1, 2)


def _mixer_forward(self, hidden_states: torch.Tensor, cache_params=None, attention_mask=None, **kwargs):
    """The mixer's forward through :mod:`dattri_llm_b200.ops.delta`."""
    layer = cache_params.layers[self.layer_idx] if cache_params is not None else None
    started = layer is not None and layer.has_previous_state
    tracked = torch.is_grad_enabled() and (hidden_states.requires_grad or any(p.requires_grad for p in self.parameters())
                                           or (started and layer.recurrent_states.requires_grad))
    if not _supported(self, hidden_states) or (started and (hidden_states.shape[1] > 1 or tracked)):  # the step has no gradient
        return type(self).forward(self, hidden_states, cache_params=cache_params, attention_mask=attention_mask, **kwargs)
    if attention_mask is not None and attention_mask.shape[0] > 1 and attention_mask.shape[1] > 1:
        hidden_states = (hidden_states * attention_mask[:, :, None]).to(hidden_states.dtype)  # padding writes nothing
    batch, tokens, _ = hidden_states.shape
    query, key, value, z, b, a = self.fix_query_key_value_ordering(self.in_proj_qkvz(hidden_states),
                                                                   self.in_proj_ba(hidden_states))
    mixed = torch.cat([x.reshape(batch, tokens, -1) for x in (query, key, value)], dim=-1)
    if started:
        mixed = self.causal_conv1d_update(mixed.transpose(1, 2), layer.conv_states, self.conv1d.weight.squeeze(1),
                                          self.conv1d.bias, self.activation).transpose(1, 2)
    else:
        if layer is not None:
            taps = F.pad(mixed.transpose(1, 2), (self.conv_kernel_size - tokens, 0))
            cache_params.update_conv_state(taps, self.layer_idx)
        mixed = _convolved(self, mixed)
    query, key, value = torch.split(mixed, [self.key_dim, self.key_dim, self.value_dim], dim=-1)
    heads = (query.unflatten(-1, (self.num_k_heads, self.head_k_dim)), key.unflatten(-1, (self.num_k_heads, self.head_k_dim)),
             value.unflatten(-1, (self.num_v_heads, self.head_v_dim)))
    gates = (a, b, self.A_log, self.dt_bias)
    if started:
        state = layer.recurrent_states
        wide = torch.promote_types(query.dtype, torch.float32)
        held = state if state.dtype == wide and state.is_contiguous() else state.to(wide).contiguous()
        with torch.no_grad():
            out = gated_delta_step(*heads, *gates, held)
        if held is not state:
            cache_params.update_recurrent_state(held, self.layer_idx)
    else:
        out, last = gated_delta_rule(*heads, *gates, output_final_state=layer is not None)
        if layer is not None:  # with its gradient: later tokens may send one back through it
            if layer.is_recurrent_states_initialized:
                cache_params.update_recurrent_state(last, self.layer_idx)
            else:  # held in 32 bits: the cache itself would take the convolution's type
                layer.recurrent_states, layer.is_recurrent_states_initialized = last, True
    shape = z.shape
    out = self.norm(out.reshape(-1, self.head_v_dim), z.reshape(-1, self.head_v_dim))
    return self.out_proj(out.reshape(shape).reshape(batch, tokens, -1))


def is_gated_delta_mixer(module: nn.Module) -> bool:
    """A Hugging Face gated delta net with the projections and gates that the forward reads."""
    names = ("fix_query_key_value_ordering", "in_proj_qkvz", "in_proj_ba", "conv1d", "A_log", "dt_bias", "norm", "out_proj",
             "causal_conv1d_update", "num_k_heads", "num_v_heads")
    return type(module).__name__.endswith("GatedDeltaNet") and all(hasattr(module, n) for n in names)


def accelerate_gated_delta(model: nn.Module, *, linears: bool = True) -> int:
    """Install the library's gated delta rule on every such mixer of *model* (and, with *linears*,
    put its bias-free linears on the tcgen05 kernels).  Returns the number of mixers.

    On the GPU a mixer runs the rule where its hidden states are bf16 or fp16 and its heads are of sizes that
    :func:`~dattri_llm_b200.ops.gated_delta_rule` takes; otherwise its own forward.  Weights in fp32 have hidden states in fp32, under
    autocast too.  Mixers whose projections are cut otherwise than Qwen3-Next's are left alone and not counted."""
    mixers = [m for m in model.modules() if is_gated_delta_mixer(m)]
    for mixer in mixers:
        mixer.forward = types.MethodType(_mixer_forward, mixer)
    if linears:
        tc_linearize(model)
    return len(mixers)
