"""Gemma4TextExpertsFP8Block on B200: routed experts with block-scaled FP8
weights, beside ``Gemma4TextExpertsFP8`` (one scale per output row) and
``Gemma4TextExpertsNVFP4``.

Buffers: ``gate_up_proj`` (E, 2I, H) and ``down_proj`` (E, H, I)
float8_e4m3fn Parameters, ``gate_up_proj_scale`` (E, ceil(2I/128),
ceil(H/128)) and ``down_proj_scale`` (E, ceil(H/128), ceil(I/128)) float32,
one scale per 128 x 128 block of the fused matrix (where I is not a multiple
of 128 a block holds gate and up rows). Forward signature and routing as the
other expert modules (HF transformers 5.5.0 ``Gemma4TextExperts``); any
router's ``(top_k_index, top_k_weights)`` will do, ``gpu.routing.route_topk``'s
among them.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from transformers.activations import ACT2FN
from transformers.models.gemma4.modeling_gemma4 import Gemma4TextExperts

from . import moe_ops


class Gemma4TextExpertsFP8Block(Gemma4TextExperts):
    """Block-scaled FP8 expert container + B200 forward."""

    gate_up_proj: torch.Tensor
    gate_up_proj_scale: torch.Tensor
    down_proj: torch.Tensor
    down_proj_scale: torch.Tensor
    num_experts: int

    def __init__(self, config):
        nn.Module.__init__(self)
        self.num_experts = config.num_experts
        self.hidden_dim = config.hidden_size
        self.intermediate_dim = config.moe_intermediate_size
        self.activation = getattr(config, "hidden_activation", "gelu_pytorch_tanh")
        if self.activation not in moe_ops._ACTIVATIONS:
            raise ValueError(f"hidden_activation={self.activation!r} is not supported by the fused kernels "
                             f"(one of {sorted(moe_ops._ACTIVATIONS)})")
        self.act_fn = ACT2FN["gelu_pytorch_tanh" if self.activation == "gelu_tanh" else self.activation]
        ne, im, hd = self.num_experts, self.intermediate_dim, self.hidden_dim
        if hd % 16 or im % 64 or not 1 <= ne <= 1024:
            raise ValueError(f"hidden_size ({hd}) must be a multiple of 16, moe_intermediate_size ({im}) of 64, "
                             f"num_experts ({ne}) at most 1024")
        blocks = lambda n: -(-n // 128)  # noqa: E731
        for name, out_dim, in_dim in (("gate_up_proj", 2 * im, hd), ("down_proj", hd, im)):
            setattr(self, name, nn.Parameter(torch.empty(ne, out_dim, in_dim, dtype=torch.float8_e4m3fn),
                                             requires_grad=False))
            self.register_buffer(f"{name}_scale", torch.empty(ne, blocks(out_dim), blocks(in_dim),
                                                              dtype=torch.float32), persistent=True)

    def forward(self, hidden_states, top_k_index, top_k_weights):
        return moe_ops.fp8_block_experts(hidden_states, top_k_index, top_k_weights, self.gate_up_proj,
                                         self.gate_up_proj_scale, self.down_proj, self.down_proj_scale,
                                         activation=self.activation)
