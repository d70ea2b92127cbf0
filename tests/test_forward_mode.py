"""Forward-mode differentiation of layer_norm, fused_linear and relative_position_bias: a dual tensor's
tangent arrives, on a CPU-only host against differences and on the GPU as the torch path gives it.

Differences: the operators' third derivatives are below 100 at these inputs, (f(x + h v) - f(x - h v)) / 2h is off
by h^2 / 6 of that and by 2^-53 |f| / h; h = 1e-5 leaves 1e-8."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from geometric_nn_ops_torch import _ops
from geometric_nn_ops_torch.triangle import fused_linear, layer_norm, relative_position_bias
from geometric_nn_ops_torch.triangle._reference.fused_linear import fused_linear_torch
from geometric_nn_ops_torch.triangle._reference.layer_norm import layer_norm_torch
from geometric_nn_ops_torch.triangle._reference.relative_position import relative_position_bias_torch

POS = torch.arange(9)[None] * 3


def _leaves(op, dtype):
    g = torch.Generator().manual_seed(1)
    shapes = {"norm": [(5, 24), (24,), (24,)], "linear": [(5, 24), (16, 24), (16,), (5, 16)], "bias": [(32, 3)]}[op]
    return [torch.randn(*s, generator=g).to(dtype) for s in shapes]


def _call(op, t):
    if op == "norm":
        return layer_norm(*t)
    if op == "linear":
        return fused_linear(t[0], t[1], t[2], "silu", t[3])
    return relative_position_bias(t[0], POS.to(t[0].device), max_distance=20)


def _torch_path(op, t):
    if op == "norm":
        return layer_norm_torch(*t)
    if op == "linear":
        return fused_linear_torch(t[0], t[1], t[2], "silu", t[3])
    pos = POS.to(t[0].device)
    return relative_position_bias_torch(t[0], pos, pos, 20, "log", True, False)


def test_what_carries_a_tangent():
    x, y = torch.ones(3), torch.ones(3)
    assert not _ops.carries_tangent(x, None)
    with fwad.dual_level():
        d = fwad.make_dual(x, y)
        assert _ops.carries_tangent(None, y, d) and not _ops.carries_tangent(x, y, None)
        with torch.no_grad():
            assert _ops.carries_tangent(d)
    seen = []
    torch.func.jvp(lambda t: (seen.append(_ops.carries_tangent(t)), t * 2)[1], (x,), (y,))
    assert seen == [True] and not _ops.carries_tangent(x)


@pytest.mark.parametrize("op", ["norm", "linear", "bias"])
def test_tangents_against_differences(op):
    leaves = _leaves(op, torch.float64)
    for k in range(len(leaves)):
        v = torch.randn(leaves[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)
        with fwad.dual_level():
            got = fwad.unpack_dual(_call(op, [fwad.make_dual(t, v) if j == k else t for j, t in enumerate(leaves)])).tangent
        h = 1e-5
        ends = [_call(op, [t + s * v if j == k else t for j, t in enumerate(leaves)]) for s in (h, -h)]
        assert ((ends[0] - ends[1]) / (2 * h) - got).abs().max() < 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("op", ["norm", "linear", "bias"])
def test_tangents_on_the_gpu(op, dtype):
    """In every call: alone, beside leaves that require grad, under no_grad, by torch.func.jvp."""
    leaves = [t.cuda() for t in _leaves(op, dtype)]
    for k in range(len(leaves)):
        v = torch.randn(leaves[k].shape, generator=torch.Generator().manual_seed(k)).to(dtype).cuda()

        def dual(f, grad=False, k=k, v=v):
            with fwad.dual_level():
                t = [u.clone().requires_grad_(grad and u.is_floating_point()) for u in leaves]
                out = fwad.unpack_dual(f(op, [fwad.make_dual(u, v) if j == k else u for j, u in enumerate(t)]))
                return out.primal.detach(), out.tangent.detach()

        def run(f, k=k, v=v):
            got = [*dual(f), *dual(f, grad=True)]
            with torch.no_grad():
                got += dual(f)
            return got + [*torch.func.jvp(lambda t: f(op, leaves[:k] + [t] + leaves[k + 1:]), (leaves[k],), (v,))]

        for got, want in zip(run(_call), run(_torch_path)):
            assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "linear", "bias"])
def test_calls_without_a_tangent_keep_the_kernels(op):
    leaves = [t.cuda() for t in _leaves(op, torch.bfloat16)]
    with torch.no_grad():
        want = _call(op, leaves)
        with fwad.dual_level():
            assert torch.equal(_call(op, leaves), want)
        f = lambda *t: _call(op, list(t))  # noqa: E731
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves), want)
