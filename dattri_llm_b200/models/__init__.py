"""Model families with B200-tuned implementations: a GPT-2-style decoder (``models.gpt2``)
and Llama (``models.llama``), both built from :class:`TcLinear` projections (tcgen05 GEMMs
with an optional fused LoGra projection tail) and ``nn.LayerNorm`` / ``nn.RMSNorm``-shaped
norms, so the capture hooks see them like any user model.  ``models.mamba2`` accelerates
Hugging Face Mamba2 models in place (a memory-bounded SSD forward, linears on the tcgen05
kernels), ``models.gated_delta`` the gated delta nets of Qwen3-Next;
:func:`tc_linearize` puts any model's linears on them.  ``models.post_training`` has
the loss functions of preference pairs, rollouts and expert routers."""

from dattri_llm_b200.models.gated_delta import accelerate_gated_delta
from dattri_llm_b200.models.gpt2 import GPT2Config, GPT2LMHeadModel
from dattri_llm_b200.models.layers import TcLinear, tc_linearize
from dattri_llm_b200.models.llama import LlamaConfig, LlamaForCausalLM, LlamaModel, token_sum_loss
from dattri_llm_b200.models.mamba2 import accelerate_mamba2, ssd_chunked
from dattri_llm_b200.models.post_training import (
    entropy_regularized_loss,
    policy_token_loss,
    preference_pair_loss,
    shift_labels,
    stacked_balance_loss,
    token_logps,
    token_quality,
)

__all__ = ["GPT2Config", "accelerate_gated_delta", "accelerate_mamba2", "ssd_chunked", "GPT2LMHeadModel", "LlamaConfig", "LlamaForCausalLM", "LlamaModel", "TcLinear",
           "policy_token_loss", "preference_pair_loss", "shift_labels", "stacked_balance_loss", "tc_linearize", "token_logps", "token_quality", "entropy_regularized_loss",
           "token_sum_loss"]
