"""layer_norm on a CPU-only host: the torch path and its gradients against the formulas in float64, the
refusals, the row addressing that the kernels are given, and the C entry points' argument errors."""

import ctypes

import pytest
import torch

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import layer_norm
from geometric_nn_ops_torch.triangle._kernels.rows import as_rows


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_torch_path(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 5, 24, generator=g).to(dtype)
    w, b = torch.randn(24, generator=g).to(dtype), torch.randn(24, generator=g).to(dtype)
    x64 = x.double()
    d = x64 - x64.mean(-1, keepdim=True)
    want = d / (d.pow(2).mean(-1, keepdim=True) + 1e-3).sqrt() * w.double() + b.double()
    got = layer_norm(x, w, b, eps=1e-3)
    assert got.dtype == dtype and got.shape == x.shape
    tol = {torch.float32: 2e-6, torch.float64: 1e-14, torch.bfloat16: 2.0 ** -8}[dtype]
    assert ((got.double() - want).abs() <= tol * (1 + want.abs())).all()


def test_torch_path_gradients():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 7, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(7, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(7, generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(layer_norm, (x, w, b))


def test_refusals():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="weight must have shape"):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="bias must have shape"):
        layer_norm(x, None, torch.ones(2, 8))
    with pytest.raises(ValueError, match="like x, or torch.float32"):
        layer_norm(x, torch.ones(8, dtype=torch.float16))
    with pytest.raises(ValueError, match="one dtype"):
        layer_norm(x.half(), torch.ones(8), torch.ones(8).half())
    with pytest.raises(ValueError, match="floating-point"):
        layer_norm(torch.zeros(2, 8, dtype=torch.int32))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError, match="weight is on meta"):
        layer_norm(x, torch.ones(8, device="meta"))


@pytest.mark.parametrize("make", [
    lambda t: t, lambda t: t.transpose(0, 1), lambda t: t[:, :, 3:11], lambda t: t.transpose(0, 1)[..., 1:9],
    lambda t: t[::2], lambda t: t[0, 0], lambda t: t[:1, 2:3], lambda t: t[:, :1].expand(6, 4, 16),
    lambda t: t.transpose(1, 2), lambda t: t.view(2, 3, 5, 16).transpose(0, 2), lambda t: t[..., ::2],
    lambda t: t[..., :1], lambda t: t[:0],
])
def test_rows_address_every_element(make):
    t = make(torch.arange(6 * 5 * 16, dtype=torch.float32).reshape(6, 5, 16))
    r, rows, inner, outer, stride = as_rows(t)
    k = t.shape[-1]
    assert rows * k == t.numel() and (rows == 0 or 1 <= inner <= rows)
    flat = torch.as_strided(r, (r.untyped_storage().nbytes() // 4,), (1,), 0)
    at = r.storage_offset()
    for i, row in enumerate(t.reshape(-1, k)):
        a = at + i // inner * outer + i % inner * stride
        assert torch.equal(flat[a:a + k], row)


def test_argument_errors():
    lib = _lib.load()
    assert lib.gnn_layer_norm_fwd(None, None) == _lib.GNN_ERR_ARG
    a = _lib.LayerNormFwdArgs()
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
    assert b"required" in lib.gnn_last_error()
    a.x = a.y = 4096
    a.rows, a.K, a.x_inner, a.x_stride, a.dtype = 4, 0, 4, 8, _lib.GNN_BF16
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
    assert b"positive" in lib.gnn_last_error()
    a.K, a.mean = 8, 4096
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
    assert b"together" in lib.gnn_last_error()
    a.mean, a.x_inner = None, 5
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
    assert b"inner" in lib.gnn_last_error()
    a.x_inner, a.x = 4, 4097
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
    assert b"aligned" in lib.gnn_last_error()
    a.x, a.weight, a.param_dtype = 4096, 4096, _lib.GNN_F16
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG
    assert b"parameters" in lib.gnn_last_error()
    a.param_dtype, a.K = _lib.GNN_F32, 16385
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_UNSUPPORTED
    a.dtype = 9
    assert lib.gnn_layer_norm_fwd(ctypes.byref(a), None) == _lib.GNN_ERR_ARG

    assert lib.gnn_layer_norm_bwd(None, None) == _lib.GNN_ERR_ARG
    b = _lib.LayerNormBwdArgs()
    b.x = b.dy = b.mean = b.rstd = 4096
    assert lib.gnn_layer_norm_bwd(ctypes.byref(b), None) == _lib.GNN_ERR_ARG
    assert b"dx and partial" in lib.gnn_last_error()
    b.dx = 4096
    b.rows, b.K, b.x_inner, b.dy_inner, b.dtype = 4, 8, 4, 4, _lib.GNN_BF16
    assert lib.gnn_layer_norm_bwd(ctypes.byref(b), None) == _lib.GNN_ERR_ARG
    assert b"parts" in lib.gnn_last_error()
    b.parts, b.dy_inner = 1, 0
    assert lib.gnn_layer_norm_bwd(ctypes.byref(b), None) == _lib.GNN_ERR_ARG
    b.dy_inner, b.K = 4, 16385
    assert lib.gnn_layer_norm_bwd(ctypes.byref(b), None) == _lib.GNN_ERR_UNSUPPORTED
    assert lib.gnn_layer_norm_bwd_parts(0, 8, _lib.GNN_BF16) == 0
    assert lib.gnn_layer_norm_bwd_parts(3, 8, _lib.GNN_BF16) == 1


def test_args_match_the_c_layout(tmp_path):
    import pathlib
    import subprocess

    root = pathlib.Path(__file__).resolve().parent.parent
    structs = {"gnn_layer_norm_fwd_args": _lib.LayerNormFwdArgs, "gnn_layer_norm_bwd_args": _lib.LayerNormBwdArgs}
    body = "".join(f'printf("{s} %zu\\n", sizeof({s}));' + "".join(
        f'printf("{s}.{f[0]} %zu\\n", offsetof({s}, {f[0]}));' for f in c._fields_) for s, c in structs.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnn_triangle.h"\nint main(void) {' + body +
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        key, value = line.split()
        struct, _, field = key.partition(".")
        cls = structs[struct]
        assert int(value) == (getattr(cls, field).offset if field else ctypes.sizeof(cls)), key
