"""Differentiable gated layer in stock torch, in fp32 (fp64 for fp64 inputs)."""

import torch
import torch.nn.functional as F

from .fused_linear import ACTIVATIONS


def gated_linear_torch(x, gate_weight, up_weight, gate_bias, up_bias, activation):
    wide = torch.promote_types(x.dtype, torch.float32)

    def product(weight, bias):
        return F.linear(x.to(wide), weight.to(wide), None if bias is None else bias.to(wide))

    return (ACTIVATIONS[activation](product(gate_weight, gate_bias)) * product(up_weight, up_bias)).to(x.dtype)
