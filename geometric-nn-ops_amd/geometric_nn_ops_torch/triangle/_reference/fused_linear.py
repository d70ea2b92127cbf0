"""Differentiable linear layer with activation and residual in stock torch, in fp32 (fp64 for fp64 inputs)."""

import torch
import torch.nn.functional as F

ACTIVATIONS = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu, "silu": F.silu, "sigmoid": torch.sigmoid}


def fused_linear_torch(x, weight, bias=None, activation=None, residual=None):
    wide = torch.promote_types(x.dtype, torch.float32)
    z = F.linear(x.to(wide), weight.to(wide), None if bias is None else bias.to(wide))
    y = ACTIVATIONS[activation](z)
    return (y if residual is None else y + residual.to(wide)).to(x.dtype)
