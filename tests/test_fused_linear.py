"""fused_linear on a CPU-only host: the torch path and its gradients, the refusals, the rows that the
kernels are given, and the C entry points' argument errors."""

import ctypes
import pathlib
import subprocess

import pytest
import torch

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import fused_linear
from geometric_nn_ops_torch.triangle._kernels import fused_linear as _hip

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
    x, w, b, r = (torch.randn(*s, generator=g).to(dtype) for s in ((2, 3, 7), (5, 7), (5,), (2, 3, 5)))
    want = _formula(x.double() @ w.double().t() + b.double(), act) + r.double()
    got = fused_linear(x, w, b, act, r)
    assert got.dtype == dtype and got.shape == (2, 3, 5)
    tol = {torch.float32: 1e-6, torch.float64: 1e-14, torch.bfloat16: 2.0 ** -8}[dtype]
    assert ((got.double() - want).abs() <= tol * (1 + want.abs())).all()


@pytest.mark.parametrize("act", ACTS)
def test_torch_path_gradients(act):
    g = torch.Generator().manual_seed(2)
    args = [torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
            for s in ((4, 6), (3, 6), (3,), (4, 3))]
    assert torch.autograd.gradcheck(lambda x, w, b, r: fused_linear(x, w, b, act, r), args)


def test_refusals():
    x, w = torch.zeros(2, 3, 8), torch.zeros(5, 8)
    with pytest.raises(ValueError, match=r"weight must have shape \[outputs, 8\]"):
        fused_linear(x, w.t())
    with pytest.raises(ValueError, match="weight must have shape"):
        fused_linear(x, torch.zeros(0, 8))
    with pytest.raises(ValueError, match="weight must have shape"):
        fused_linear(x, torch.zeros(8))
    with pytest.raises(ValueError, match="activation must be one of"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="bias must have shape"):
        fused_linear(x, w, torch.zeros(8))
    with pytest.raises(ValueError, match="residual must have shape"):
        fused_linear(x, w, residual=torch.zeros(5))
    with pytest.raises(ValueError, match="bias must be torch.float32 like x"):
        fused_linear(x, w, torch.zeros(5).half())
    with pytest.raises(ValueError, match="weight must be torch.float32 like x"):
        fused_linear(x, w.bfloat16())
    with pytest.raises(ValueError, match="residual is on meta"):
        fused_linear(x, w, residual=torch.zeros(2, 3, 5, device="meta"))
    with pytest.raises(ValueError, match="floating-point"):
        fused_linear(x.long(), w)
    with pytest.raises(ValueError, match="floating-point"):
        fused_linear(torch.tensor(1.0), w)


def test_argument_errors():
    lib = _lib.load()
    assert lib.gnn_linear(None, None) == _lib.GNN_ERR_ARG
    a = _lib.LinearArgs()

    def refused(text, fn=lib.gnn_linear, args=a):
        assert fn(ctypes.byref(args), None) == _lib.GNN_ERR_ARG
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    refused(b"required")
    a.x = a.w = a.out = 4096
    a.dz = 1
    refused(b"required")
    a.dz, a.dtype = 0, 9
    refused(b"dtype")
    a.dtype, a.precision = _lib.GNN_BF16, 5
    refused(b"precision")
    a.precision, a.activation = 0, 5
    refused(b"activation")
    a.activation = 0
    refused(b"positive")
    a.M, a.I, a.O, a.out_cols = 4, 12, 5, 4
    refused(b"out_cols")
    a.out_cols = 5
    refused(b"16 bytes")
    a.I = a.x_ld = 16
    a.w_ld = 8
    refused(b"pitches")
    a.w_ld, a.out_ld = 16, 4
    refused(b"pitches")
    a.out_ld, a.out = 5, 4097
    refused(b"aligned")
    a.out, a.x = 4096, 4104
    refused(b"16-byte")

    assert lib.gnn_column_sums(None, None) == _lib.GNN_ERR_ARG
    assert lib.gnn_column_sums_parts(0, 5) == 0 and lib.gnn_column_sums_parts(1, 5) == 1
    c = _lib.ColumnSumsArgs()
    refused(b"required", lib.gnn_column_sums, c)
    c.d = c.partial = 4096
    refused(b"positive", lib.gnn_column_sums, c)
    c.M, c.O, c.parts, c.dtype = 4, 5, 1, _lib.GNN_BF16
    c.d = 4097
    refused(b"aligned", lib.gnn_column_sums, c)


def test_args_match_the_c_layout(tmp_path):
    root = pathlib.Path(__file__).resolve().parent.parent
    structs = {"gnn_linear_args": _lib.LinearArgs, "gnn_column_sums_args": _lib.ColumnSumsArgs,
               "gnn_linear_wgrad_args": _lib.LinearWgradArgs, "gnn_pad_rows_args": _lib.PadRowsArgs}
    body = "".join(f'printf("%zu\\n", sizeof({s}));' + "".join(
        f'printf("%zu\\n", offsetof({s}, {f[0]}));' for f in c._fields_) for s, c in structs.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnn_triangle.h"\nint main(void) {' + body +
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    want = [v for c in structs.values() for v in (ctypes.sizeof(c), *(getattr(c, f[0]).offset for f in c._fields_))]
    assert [int(v) for v in out] == want


def test_parameter_gradients_refuse_what_they_cannot_write():
    lib = _lib.load()
    a = _lib.LinearWgradArgs()

    def refused(text):
        assert lib.gnn_linear_wgrad(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    assert lib.gnn_linear_wgrad(None, None) == _lib.GNN_ERR_ARG and lib.gnn_linear_wgrad_slices(None) == 0
    a.dz, a.x, a.partial, a.dw = 4096, 8192, 4096, 4096
    a.M, a.O, a.I, a.dz_ld, a.x_ld, a.dtype = 64, 32, 16, 32, 16, _lib.GNN_BF16
    refused(b"slices")
    a.slices = 1
    for outputs in (0, 33):
        a.outputs = outputs
        refused(b"outputs")
    a.outputs, a.dw = 30, None
    refused(b"dw is required")
    a.dw, a.db = 4096, 4097
    refused(b"aligned")
    a.db, a.partial = None, 4098
    refused(b"")
    a.partial, a.x = 4096, 8196
    refused(b"")
    a.x, a.O = 8192, 30
    refused(b"")


def test_calls_that_take_a_transposed_weight_or_dx():
    lib = _lib.load()
    a = _lib.LinearArgs()
    a.x = a.w = a.out = a.side = 4096
    a.M, a.I, a.O, a.out_cols, a.x_ld, a.w_ld, a.side_ld, a.out_ld = 1 << 16, 128, 512, 512, 128, 128, 512, 512
    a.dtype, a.dz, a.activation, a.dx, a.dx_ld = _lib.GNN_BF16, 1, 1, 4096, 128
    assert lib.gnn_linear_takes_dx(ctypes.byref(a)) == 1 and lib.gnn_linear_takes_transposed(ctypes.byref(a)) == 1
    for name, value in (("M", 64), ("dtype", _lib.GNN_F32), ("I", 512), ("dx", 4098), ("O", 516), ("activation", 0)):
        was = getattr(a, name)
        setattr(a, name, value)
        assert lib.gnn_linear_takes_dx(ctypes.byref(a)) == 0, name
        if name != "O" and name != "I":
            assert lib.gnn_linear(ctypes.byref(a), None) in (_lib.GNN_ERR_ARG, _lib.GNN_ERR_UNSUPPORTED)
        setattr(a, name, was)
    a.M, a.dx, a.w_transposed, a.w_ld = 64, None, 1, 512
    assert lib.gnn_linear(ctypes.byref(a), None) == _lib.GNN_ERR_UNSUPPORTED
    assert b"transposed" in lib.gnn_last_error()


def test_padding_refuses_what_it_cannot_write():
    lib = _lib.load()
    a = _lib.PadRowsArgs()

    def refused(text):
        assert lib.gnn_pad_rows(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
        assert text in lib.gnn_last_error()

    assert lib.gnn_pad_rows(None, None) == _lib.GNN_ERR_ARG
    refused(b"required")
    a.src, a.dst, a.dtype, a.rows, a.cols, a.row_stride, a.col_stride = 4096, 8192, _lib.GNN_BF16, 3, 13, 13, 1
    for ld in (0, 8, 13, 20):  # fewer than the columns, or no multiple of 16 bytes
        a.ld = ld
        refused(b"multiple of 16 bytes")
    a.ld, a.rows = 16, 0
    refused(b"positive")
    a.rows, a.src = 3, 4097
    refused(b"aligned")
    a.src, a.dst = 4098, 8200
    refused(b"aligned")
    a.dst, a.dtype = 8192, 77
    refused(b"dtype")
    lib.gnn_last_error()


def test_the_fitted_normal_distribution():
    """The polynomials of the 16-bit gelu and its slope, read from the source and evaluated in fp32, against the
    normal distribution in 64 bits: within the bounds that the source states, and zero or one far out."""
    text = (pathlib.Path(__file__).resolve().parent.parent / "geometric-nn-ops_amd/csrc/linear_common.hpp").read_text()

    def poly(name, m):
        c = [float(v.rstrip("f")) for v in text.split(f"float {name}[] = {{")[1].split("}")[0].replace("\n", " ").split(", ")]
        out = torch.full_like(m, c[-1])
        for k in reversed(c[:-1]):
            out = out * m + torch.tensor(k, dtype=torch.float32)
        return out.double()

    m = torch.linspace(0, 16, 160001)
    z = m.double()
    tail, pdf = torch.special.ndtr(-z), torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    near = torch.exp2(poly("P", m))
    # 2e-7 of the fit, and a step of the fp32 evaluation's argument (below 2 where the tail counts): 2^-23 of the tail
    assert (z * (near - tail).abs() <= 2e-7 + z * tail * 2.0 ** -22).all()
    inner = z <= 5.5
    assert ((near / tail - 1).abs()[inner] <= 1.6e-4).all()
    slope = poly("S", m) * torch.exp2(-0.7213475204444817 * z * z)
    assert ((slope - (tail - z * pdf)).abs() <= 4e-7).all()
    assert near[-1] < 1e-100 and slope[-1].abs() < 1e-45


def test_dx_comes_with_dz_in_rows_that_hold_it():
    lib = _lib.load()
    a = _lib.LinearArgs()
    a.x = a.w = a.out = a.side = a.dx = 4096
    a.M, a.I, a.O, a.out_cols, a.x_ld, a.w_ld, a.side_ld, a.out_ld = 1 << 16, 128, 512, 512, 128, 128, 512, 512
    a.dtype, a.dz, a.activation, a.dx_ld = _lib.GNN_BF16, 1, 1, 128
    a.out = None
    assert lib.gnn_linear(ctypes.byref(a), None) == _lib.GNN_ERR_ARG and b"required" in lib.gnn_last_error()
    a.out = 4096
    for pitch in (120, 0, -128):
        a.dx_ld = pitch
        assert lib.gnn_linear(ctypes.byref(a), None) == _lib.GNN_ERR_ARG and b"pitches" in lib.gnn_last_error(), pitch
