"""Gradients under saved-tensor hooks and activation checkpoints: the same bits as without them."""

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

from geometric_nn_ops_torch.triangle import fused_linear, layer_norm, relative_position_bias

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _under(kind, block, *leaves):
    """The block's output with what it saves kept as ``kind`` says, and nothing else holding it."""
    if kind == "checkpoint":
        return checkpoint(block, *leaves, use_reentrant=False)
    if kind == "cpu":
        with save_on_cpu():
            return block(*leaves)
    with saved_tensors_hooks(torch.clone, lambda t: t):
        return block(*leaves)


def _same_gradients(block, leaves, dout):
    """The gradients without hooks, and bit for bit the same ones under each kind of them, with the memory that
    the forward left free taken by other values before the backward."""
    plain = torch.autograd.grad(block(*leaves), leaves, dout)
    for kind in ("clone", "cpu", "checkpoint"):
        out = _under(kind, block, *leaves)
        taken = [torch.full((1 << k,), -999, device=DEV, dtype=torch.int64) for k in range(4, 18) for _ in range(4)]
        got = torch.autograd.grad(out, leaves, dout)
        del taken
        for a, e in zip(got, plain):
            assert torch.equal(a, e), kind


@pytest.mark.parametrize("last", [False, True], ids=["heads_first", "heads_last"])
@pytest.mark.parametrize("mixed", [False, True], ids=["one_type", "mixed_types"])
def test_relative_position_bias(last, mixed):
    """Positions made inside the block, those of mixed types converted there once more."""
    u, v, h = 70, 131, 6
    table = torch.randn(32, h, generator=torch.Generator().manual_seed(1)).to(DEV).requires_grad_()
    dout = torch.randn((2, u, v, h) if last else (2, h, u, v), generator=torch.Generator().manual_seed(2)).to(DEV)
    base = torch.arange(2 * v, device=DEV).view(2, v) * 3

    def block(t):
        k = base + 5
        q = k[:, -u:] - 40
        return relative_position_bias(t, q.int() if mixed else q, k, max_distance=128, channels_last=last)

    _same_gradients(block, [table], dout)


def test_layer_norm():
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(301, 96, generator=g).bfloat16().to(DEV) for _ in range(2))
    weight, bias = (torch.randn(96, generator=g).to(DEV) for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    _same_gradients(lambda x, w, b: layer_norm(x * 1.5, w, b), leaves, dy)


@pytest.mark.parametrize("m,i,o", [(45, 40, 24), (300, 61, 13), (32800, 64, 72)])
def test_fused_linear(m, i, o):
    g = torch.Generator().manual_seed(4)
    x, r, dy = (torch.randn(m, k, generator=g).bfloat16().to(DEV) for k in (i, o, o))
    w, b = (torch.randn(*s, generator=g).mul(i ** -0.5).bfloat16().to(DEV) for s in ((o, i), (o,)))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    _same_gradients(lambda x, w, b, r: fused_linear(x * 1.5, w, b, "silu", r), leaves, dy)


def test_fused_linear_from_unaligned_operands():
    """Hooks that keep what they are given in one flat buffer return it at any address."""
    m, i, o = 45, 40, 24
    g = torch.Generator().manual_seed(5)
    x, dy = (torch.randn(m, k, generator=g).bfloat16().to(DEV) for k in (i, o))
    w = torch.randn(o, i, generator=g).mul(i ** -0.5).bfloat16().to(DEV)
    leaves = [t.requires_grad_() for t in (x, w)]
    plain = torch.autograd.grad(fused_linear(x, w, None, "gelu"), leaves, dy)

    def shifted(t):
        return torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].copy_(t.reshape(-1)).view(t.shape)

    with saved_tensors_hooks(shifted, lambda t: t):
        y = fused_linear(x, w, None, "gelu")
    for a, e in zip(torch.autograd.grad(y, leaves, dy), plain):
        assert torch.equal(a, e)
