"""Differentiable attention over states of another length in stock torch, in fp32 (fp64 for fp64 inputs)."""

import torch


def cross_attention_torch(q, k, v, bias, mask, scale):
    (B, U, H, D), (V, Hk) = q.shape, k.shape[1:3]
    wide = torch.promote_types(q.dtype, torch.float32)
    if not V:
        empty = [t.sum() for t in (k, v, bias) if t is not None]  # zeros, which keep these in the graph
        return (q.masked_fill(torch.ones((), dtype=torch.bool, device=q.device), 0.0) + sum(empty)).contiguous()
    # rows: the queries of all heads that share a key head
    rows = q.to(wide).reshape(B, U, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, H // Hk * U, D)
    k, v = (t.to(wide).transpose(1, 2) for t in (k, v))
    if mask is not None:  # what masked keys hold reaches nothing
        k, v = (t.masked_fill(~mask[:, None, :, None], 0.0) for t in (k, v))
    s = (rows @ k.transpose(-1, -2) * scale).view(B, H, U, V)
    if bias is not None:
        s = s + bias.to(wide)
    if mask is not None:
        s = s.masked_fill(~mask[:, None, None, :], float("-inf"))
    dead = s.detach().amax(-1, keepdim=True) == float("-inf")  # nothing is kept
    p = torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0)
    o = (p.view(B, Hk, H // Hk * U, V) @ v).view(B, Hk, H // Hk, U, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, U, H, D).to(q.dtype).contiguous()
