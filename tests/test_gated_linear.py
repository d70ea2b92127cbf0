"""gated_linear on a CPU-only host: the torch path and its gradients, the refusals, and the C entry points'
argument errors."""

import ctypes
import pathlib
import subprocess

import pytest
import torch

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import gated_linear
from geometric_nn_ops_torch.triangle._kernels import gated_linear as _hip

ACTS = [None, "relu", "gelu", "silu", "sigmoid"]


def _formula(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "silu":
        return z / (1 + (-z).exp())
    return 1 / (1 + (-z).exp()) if act == "sigmoid" else z


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_torch_path(act, dtype):
    g = torch.Generator().manual_seed(1)
    x, wg, wu, bg, bu = (torch.randn(*s, generator=g).to(dtype) for s in ((2, 3, 7), (5, 7), (5, 7), (5,), (5,)))
    xd = x.double()
    want = _formula(xd @ wg.double().t() + bg.double(), act) * (xd @ wu.double().t() + bu.double())
    got = gated_linear(x, wg, wu, bg, bu, act)
    assert got.dtype == dtype and got.shape == (2, 3, 5)
    tol = {torch.float32: 2e-6, torch.float64: 1e-14, torch.bfloat16: 2.0 ** -8}[dtype]
    assert ((got.double() - want).abs() <= tol * (1 + want.abs())).all()


def test_the_activation_is_the_gates():
    x, w = torch.randn(3, 4), torch.randn(2, 4)
    assert torch.equal(gated_linear(x, w, torch.zeros(2, 4), up_bias=torch.ones(2)), torch.nn.functional.silu(x @ w.t()))


@pytest.mark.parametrize("act", ACTS)
def test_torch_path_gradients(act):
    g = torch.Generator().manual_seed(2)
    args = [torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
            for s in ((4, 6), (3, 6), (3, 6), (3,), (3,))]
    assert torch.autograd.gradcheck(lambda *t: gated_linear(*t, act), args)


def test_refusals():
    x, w = torch.zeros(2, 3, 8), torch.zeros(5, 8)
    with pytest.raises(ValueError, match=r"gate_weight must have shape \[outputs, 8\]"):
        gated_linear(x, w.t(), w)
    with pytest.raises(ValueError, match="gate_weight must have shape"):
        gated_linear(x, torch.zeros(0, 8), torch.zeros(0, 8))
    with pytest.raises(ValueError, match=r"up_weight must have shape \(5, 8\)"):
        gated_linear(x, w, torch.zeros(4, 8))
    with pytest.raises(ValueError, match="activation must be one of"):
        gated_linear(x, w, w, activation="tanh")
    with pytest.raises(ValueError, match="gate_bias must have shape"):
        gated_linear(x, w, w, torch.zeros(8))
    with pytest.raises(ValueError, match="up_bias must have shape"):
        gated_linear(x, w, w, up_bias=torch.zeros(5, 1))
    with pytest.raises(ValueError, match="up_weight must be torch.float32 like x"):
        gated_linear(x, w, w.half())
    with pytest.raises(ValueError, match="up_weight is on meta"):
        gated_linear(x, w, torch.zeros(5, 8, device="meta"))
    with pytest.raises(ValueError, match="floating-point"):
        gated_linear(x.long(), w, w)
    with pytest.raises(ValueError, match="floating-point"):
        gated_linear(torch.tensor(1.0), w, w)


def test_what_the_kernels_take():
    def w(o, i):
        return torch.empty(o, i, device="meta")

    assert _hip.supports(w(1, 1)) and _hip.supports(w(1 << 19, 1 << 20))
    assert not _hip.supports(w((1 << 19) + 1, 8)) and not _hip.supports(w(8, (1 << 20) + 1))


def test_argument_errors():
    lib = _lib.load()
    a = _lib.GatedLinearArgs()

    def refused(text, fn=lib.gnn_gated_linear, args=a):
        assert fn(ctypes.byref(args), None) == _lib.GNN_ERR_ARG
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    for fn in (lib.gnn_gated_linear, lib.gnn_gated_turn, lib.gnn_gated_linear_wgrad):
        assert fn(None, None) == _lib.GNN_ERR_ARG
    assert lib.gnn_gated_linear_wgrad_slices(None) == 0
    refused(b"required")
    a.x = a.wg = a.wu = a.out = 4096
    a.dtype = 9
    refused(b"dtype")
    a.dtype, a.precision = _lib.GNN_BF16, 5
    refused(b"precision")
    a.precision, a.activation = 0, 5
    refused(b"activation")
    a.activation = 0
    refused(b"positive")
    a.M, a.I, a.O, a.out_cols = 4, 12, 5, 5
    refused(b"out_cols")
    a.out_cols = 8
    refused(b"16 bytes")
    a.I = a.x_ld = a.wg_ld = 16
    a.wu_ld = 8
    refused(b"pitches")
    a.wu_ld, a.out_ld = 16, 4
    refused(b"pitches")
    a.dy, a.dy_ld, a.out_ld = 4096, 5, 15
    refused(b"pitches")
    a.out_ld, a.dy = 16, 4097
    refused(b"aligned")
    a.dy, a.wu = 4096, 4104
    refused(b"16-byte")

    t = _lib.GatedTurnArgs()
    refused(b"required", lib.gnn_gated_turn, t)
    t.wg = t.wu = t.dst = 4096
    t.dtype = 9
    refused(b"dtype", lib.gnn_gated_turn, t)
    t.dtype, t.I, t.O, t.wg_ld, t.wu_ld = _lib.GNN_F16, 8, 5, 8, 8
    for cols in (0, 4, 5, 12):
        t.out_cols = cols
        refused(b"multiple of 8", lib.gnn_gated_turn, t)
    t.out_cols, t.wu_ld = 8, 7
    refused(b"pitches", lib.gnn_gated_turn, t)
    t.wu_ld, t.dst = 8, 4104
    refused(b"aligned", lib.gnn_gated_turn, t)


def test_rows_beyond_any_grid_are_refused():
    """Rounding them up to tiles passes 64 bits: no launch of what is left of the product."""
    lib = _lib.load()
    a = _lib.GatedLinearArgs()
    a.x = a.wg = a.wu = a.out = 4096
    a.dtype, a.I, a.O, a.out_cols, a.x_ld, a.wg_ld, a.wu_ld, a.out_ld = _lib.GNN_BF16, 16, 8, 8, 16, 16, 16, 8
    for rows in ((1 << 40) + 1, (1 << 63) - 1):
        a.M = rows
        assert lib.gnn_gated_linear(ctypes.byref(a), None) == _lib.GNN_ERR_ARG and b"2^40" in lib.gnn_last_error()
    a.O, a.out_cols, a.out_ld, a.M = 1 << 29, 1 << 29, 1 << 29, 1 << 40
    assert lib.gnn_gated_linear(ctypes.byref(a), None) == _lib.GNN_ERR_UNSUPPORTED


def test_parameter_gradients_refuse_what_they_cannot_write():
    lib = _lib.load()
    a = _lib.GatedLinearWgradArgs()

    def refused(text):
        assert lib.gnn_gated_linear_wgrad(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    a.dz, a.x, a.partial, a.dwg = 4096, 8192, 4096, 4096
    a.M, a.O, a.I, a.dz_ld, a.x_ld, a.dtype = 64, 32, 16, 64, 16, _lib.GNN_BF16
    refused(b"slices")
    a.slices = 1
    for outputs in (0, 33):
        a.outputs = outputs
        refused(b"outputs")
    a.outputs, a.dwg = 30, None
    refused(b"output is required")
    a.dbu = 4097
    refused(b"aligned")
    a.dbu, a.O = None, 30
    refused(b"multiple of 8")
    a.O, a.dz_ld = 32, 32
    refused(b"pitches")


def test_args_match_the_c_layout(tmp_path):
    root = pathlib.Path(__file__).resolve().parent.parent
    structs = {"gnn_gated_linear_args": _lib.GatedLinearArgs, "gnn_gated_turn_args": _lib.GatedTurnArgs,
               "gnn_gated_linear_wgrad_args": _lib.GatedLinearWgradArgs}
    body = "".join(f'printf("%zu\\n", sizeof({s}));' + "".join(
        f'printf("%zu\\n", offsetof({s}, {f[0]}));' for f in c._fields_) for s, c in structs.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnn_triangle.h"\nint main(void) {' + body +
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    want = [v for c in structs.values() for v in (ctypes.sizeof(c), *(getattr(c, f[0]).offset for f in c._fields_))]
    assert [int(v) for v in out] == want
