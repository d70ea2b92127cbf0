"""Differentiable LayerNorm in stock torch, with the statistics in fp32 (fp64 for fp64 inputs)."""

import torch
import torch.nn.functional as F


def layer_norm_torch(x, weight=None, bias=None, eps=1e-5):
    wide = torch.promote_types(x.dtype, torch.float32)
    w, b = (None if t is None else t.to(wide) for t in (weight, bias))
    return F.layer_norm(x.to(wide), x.shape[-1:], w, b, eps).to(x.dtype)
