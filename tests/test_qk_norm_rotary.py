"""qk_norm_rotary on a CPU-only host: the torch path and its gradients, the refusals, and the C entry points'
argument errors."""

import ctypes
import math
import os
import pathlib
import subprocess
import sys

import pytest
import torch

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import qk_norm_rotary
from geometric_nn_ops_torch.triangle._kernels import qk_norm_rotary as _hip


def _rotated(x, pos, freqs, interleaved):
    """Element by element, in Python's own arithmetic."""
    out, r = x.clone().double(), 2 * len(freqs)
    for j, f in enumerate(freqs):
        i0, i1 = (2 * j, 2 * j + 1) if interleaved else (j, j + r // 2)
        for n, p in enumerate(pos):
            c, s = math.cos(p * f), math.sin(p * f)
            a, b = x[:, n, :, i0].double(), x[:, n, :, i1].double()
            out[:, n, :, i0], out[:, n, :, i1] = a * c - b * s, b * c + a * s
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_torch_path(interleaved, dtype):
    g = torch.Generator().manual_seed(1)
    q, k, w = (torch.randn(*s, generator=g).to(dtype) for s in ((2, 3, 4, 10), (2, 5, 2, 10), (10,)))
    qp, kp = [0, 7, 100_003], [3, 2, 1, 0, -9]
    got = qk_norm_rotary(q, k, torch.tensor(qp), torch.tensor(kp, dtype=torch.int32), q_weight=w, rotary_dim=6,
                         interleaved=interleaved, eps=1e-3, base=500.0)
    freqs = [500.0 ** (-2 * j / 6) for j in range(3)]
    tol = {torch.float32: 1e-6, torch.float64: 1e-9, torch.bfloat16: 2.0 ** -8}[dtype]
    for x, weight, pos, y in ((q, w, qp, got[0]), (k, None, kp, got[1])):
        n = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-3).sqrt()
        want = _rotated(n if weight is None else n * weight.double(), pos, freqs, interleaved)
        assert y.dtype == dtype and y.shape == x.shape
        assert ((y.double() - want).abs() <= tol * (1 + want.abs())).all()


def test_defaults_and_frequencies():
    x = torch.randn(1, 4, 2, 8, generator=torch.Generator().manual_seed(2))
    pos = torch.arange(4)
    same = qk_norm_rotary(x, x, pos)
    assert torch.equal(same[0], same[1])
    freqs = [10000.0 ** (-2 * j / 8) for j in range(4)]
    assert torch.equal(qk_norm_rotary(x, x, pos, frequencies=freqs)[0], same[0])
    assert torch.equal(qk_norm_rotary(x, x, pos[None], pos.int())[1], same[0])
    only = qk_norm_rotary(x, x, None, pos, eps=None)
    assert torch.equal(only[0], x) and not torch.equal(only[1], x)
    norm = qk_norm_rotary(x, x)[0]
    assert (norm.square().mean(-1) - 1).abs().max() < 1e-5


@pytest.mark.parametrize("interleaved", [False, True])
def test_torch_path_gradients(interleaved):
    g = torch.Generator().manual_seed(3)
    args = [torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
            for s in ((1, 3, 2, 6), (1, 2, 1, 6), (6,), (6,))]
    assert torch.autograd.gradcheck(
        lambda q, k, a, b: qk_norm_rotary(q, k, torch.tensor([5, 6, 70]), torch.tensor([1, 2]), q_weight=a, k_weight=b,
                                          rotary_dim=4, interleaved=interleaved), args)


@pytest.mark.parametrize("eps", [None, 1e-6])
@pytest.mark.parametrize("pos", [None, torch.arange(3)])
def test_the_results_are_fresh_and_contiguous(pos, eps):
    """Also where nothing is normed or turned, and whatever the layout of the rows."""
    for x in (torch.randn(2, 3, 4, 8), torch.randn(2, 4, 3, 8).transpose(1, 2), torch.randn(2, 3, 4, 8).bfloat16()):
        before = x.clone()
        for y in qk_norm_rotary(x, x, pos, eps=eps):
            assert y.is_contiguous()
            y.zero_()
        assert torch.equal(x, before)


def test_refusals():
    q, k, pos = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 2, 8), torch.arange(3)
    with pytest.raises(ValueError, match=r"\[batch, tokens, heads, head_dim\]"):
        qk_norm_rotary(q[0], k)
    with pytest.raises(ValueError, match="floating-point"):
        qk_norm_rotary(q.long(), k.long())
    with pytest.raises(ValueError, match="k must have q's batch and head dim"):
        qk_norm_rotary(q, k[..., :4])
    with pytest.raises(ValueError, match="k must have q's batch"):
        qk_norm_rotary(q, k[:1])
    with pytest.raises(ValueError, match="k must be torch.float32"):
        qk_norm_rotary(q, k.half())
    with pytest.raises(ValueError, match="k_pos is required"):
        qk_norm_rotary(q, k, pos)
    with pytest.raises(ValueError, match="q_pos must be int32 or int64"):
        qk_norm_rotary(q, k, pos.float(), torch.arange(5))
    with pytest.raises(ValueError, match=r"k_pos must have shape \[5\] or \[2, 5\]"):
        qk_norm_rotary(q, k, pos, pos)
    with pytest.raises(ValueError, match="q_pos must have shape"):
        qk_norm_rotary(q, k, pos.expand(3, 3), torch.arange(5))
    with pytest.raises(ValueError, match="q_pos is on meta"):
        qk_norm_rotary(q, q, pos.to("meta"))
    with pytest.raises(ValueError, match=r"q_weight must have shape \(8,\)"):
        qk_norm_rotary(q, k, q_weight=torch.zeros(4))
    with pytest.raises(ValueError, match="k_weight must be torch.float32"):
        qk_norm_rotary(q, k, k_weight=torch.zeros(8).half())
    with pytest.raises(ValueError, match="one dtype"):
        qk_norm_rotary(q.half(), k.half(), q_weight=torch.zeros(8), k_weight=torch.zeros(8).half())
    with pytest.raises(ValueError, match="goes with a norm"):
        qk_norm_rotary(q, k, q_weight=torch.zeros(8), eps=None)
    for r in (0, 3, 10):
        with pytest.raises(ValueError, match="rotary_dim must be an even number from 2 to 8"):
            qk_norm_rotary(q, q, pos, rotary_dim=r)
    with pytest.raises(ValueError, match="base must be positive"):
        qk_norm_rotary(q, q, pos, base=0.0)
    with pytest.raises(ValueError, match="frequencies must hold"):
        qk_norm_rotary(q, q, pos, frequencies=[1.0] * 5)
    with pytest.raises(ValueError, match="frequencies must hold"):
        qk_norm_rotary(q, q, pos, frequencies=[1.0], rotary_dim=4)


def test_what_the_kernels_take():
    def q(d):
        return torch.empty(1, 2, 3, d, device="meta")

    assert _hip.supports(q(8), q(8), 8) and _hip.supports(q(256), q(256), 0) and _hip.supports(q(72), q(72), 24)
    assert not _hip.supports(q(264), q(264), 8) and not _hip.supports(q(12), q(12), 8) and not _hip.supports(q(16), q(16), 6)


def test_argument_errors():
    lib = _lib.load()
    a = _lib.QkRotaryArgs()

    def refused(text, fn=lib.gnn_qk_rotary_fwd):
        assert fn(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    assert lib.gnn_qk_rotary_fwd(None, None) == _lib.GNN_ERR_ARG
    assert lib.gnn_qk_rotary_bwd(None, None) == _lib.GNN_ERR_ARG
    assert lib.gnn_qk_rotary_parts(None, 0) == 0
    a.dtype = 9
    refused(b"dtype")
    a.dtype, a.param_dtype = _lib.GNN_BF16, _lib.GNN_F16
    refused(b"weights")
    a.param_dtype = _lib.GNN_F32
    refused(b"4 or 8 bytes")
    a.pos_bytes = 8
    for d, r in ((0, 0), (12, 0), (264, 0), (16, 24), (16, 4), (16, -8)):
        a.D, a.R = d, r
        refused(b"multiple of 8")
    a.D = a.R = 16
    a.pos[0] = 4096
    refused(b"frequencies")
    host = (ctypes.c_double * 8)()
    a.frequencies, a.B = ctypes.addressof(host), -1
    refused(b"negative")
    a.B, a.N[0], a.H[0] = 1, 4, 2
    refused(b"required")
    a.x[0], a.out[0], a.weight[0] = 4096, 4096, 4096
    refused(b"go with norms")
    a.norm, a.out[0] = 1, 4097
    refused(b"aligned")
    a.out[0] = None
    refused(b"required", lib.gnn_qk_rotary_bwd)
    a.dy[0] = 4096
    refused(b"parts", lib.gnn_qk_rotary_bwd)
    a.parts[0], a.dweight[0] = 1, 4096
    refused(b"partial", lib.gnn_qk_rotary_bwd)
    assert lib.gnn_qk_rotary_parts(ctypes.byref(a), 0) == 1 and lib.gnn_qk_rotary_parts(ctypes.byref(a), 2) == 0
    a.N[0] = 0  # nothing to do
    assert lib.gnn_qk_rotary_fwd(ctypes.byref(a), None) == 0


HUGE = """
import ctypes
from geometric_nn_ops_torch import _lib
lib = _lib.load()
for b, n, h in ((1, 3, 1 << 32), (8, 3, 1 << 40), (1 << 30, 1 << 16, 1 << 20), (1 << 62, 1 << 62, 1 << 20), (1, 1 << 34, 1)):
    a = _lib.QkRotaryArgs()
    a.D = a.R = 8
    a.B, a.N[0], a.H[0] = b, n, h
    assert lib.gnn_qk_rotary_parts(ctypes.byref(a), 0) == 0
    a.dtype = a.param_dtype = _lib.GNN_BF16
    a.pos_bytes, a.x[0], a.dy[0], a.out[0], a.parts[0] = 8, 4096, 4096, 4096, 1
    for fn in (lib.gnn_qk_rotary_fwd, lib.gnn_qk_rotary_bwd):
        assert fn(ctypes.byref(a), None) < 0, (b, n, h)
a.B, a.N[0], a.H[0] = 1, 1 << 14, (1 << 20) - 1
assert lib.gnn_qk_rotary_parts(ctypes.byref(a), 0) > 0
"""


def test_sizes_beyond_any_grid_are_refused():
    """Heads past 2^31, and products past 64 bits; in a process of its own, which a division by zero would end."""
    root = pathlib.Path(__file__).resolve().parent.parent / "geometric-nn-ops_amd"
    run = subprocess.run([sys.executable, "-c", HUGE], env={**os.environ, "PYTHONPATH": str(root)}, capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stderr[-500:])


def test_args_match_the_c_layout(tmp_path):
    root = pathlib.Path(__file__).resolve().parent.parent
    c = _lib.QkRotaryArgs
    body = 'printf("%zu\\n", sizeof(gnn_qk_rotary_args));' + "".join(
        f'printf("%zu\\n", offsetof(gnn_qk_rotary_args, {f[0]}));' for f in c._fields_)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnn_triangle.h"\nint main(void) {' + body +
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == [ctypes.sizeof(c), *(getattr(c, f[0]).offset for f in c._fields_)]
