"""Differentiable per-head norms and rotary positions in stock torch, in fp32 (fp64 for fp64 inputs; the angles
always in fp64)."""

import torch


def _turned(x, pos, frequencies, interleaved):
    """``[B, N, H, R]`` turned by ``pos [B or 1, N]`` times each pair's frequency."""
    angle = pos.to(torch.float64)[:, :, None, None] * torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    cos, sin = torch.cos(angle).to(x.dtype), torch.sin(angle).to(x.dtype)
    if interleaved:
        a, c = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - c * sin, c * cos + a * sin], -1).flatten(-2)
    a, c = x.chunk(2, -1)
    return torch.cat([a * cos - c * sin, c * cos + a * sin], -1)


def _one(x, pos, weight, eps, frequencies, interleaved):
    y = x.to(torch.promote_types(x.dtype, torch.float32))
    if eps is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.to(y.dtype)
    if pos is not None:
        r = 2 * len(frequencies)
        y = torch.cat([_turned(y[..., :r], pos, frequencies, interleaved), y[..., r:]], -1)
    y = y.to(x.dtype).contiguous()
    return y.clone() if y is x else y


def qk_norm_rotary_torch(q, k, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved):
    return (_one(q, q_pos, q_weight, eps, frequencies, interleaved),
            _one(k, k_pos, k_weight, eps, frequencies, interleaved))
