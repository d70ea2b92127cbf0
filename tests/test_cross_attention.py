"""cross_attention on a CPU-only host: the torch path and its gradients, the refusals, and the C entry points'
argument errors."""

import ctypes
import os
import pathlib
import subprocess
import sys

import pytest
import torch

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import cross_attention
from geometric_nn_ops_torch.triangle._kernels import cross_attention as _hip


def _formula(q, k, v, bias, mask, scale):
    """Head by head and row by row."""
    (B, U, H, D), Hk = q.shape, k.shape[2]
    out = torch.zeros(B, U, H, D, dtype=torch.float64)
    for b in range(B):
        keep = torch.ones(k.shape[1], dtype=torch.bool) if mask is None else mask[b]
        for h in range(H):
            kh, vh = k[b, keep, h * Hk // H].double(), v[b, keep, h * Hk // H].double()
            for u in range(U):
                x = kh @ q[b, u, h].double() * scale
                if bias is not None:
                    x = x + bias[b % bias.shape[0], h, u, keep].double()
                if keep.any():
                    out[b, u, h] = torch.softmax(x, 0) @ vh
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("shared", [False, True])
def test_torch_path(dtype, shared):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(*s, generator=g).to(dtype) for s in ((3, 4, 6, 5), (3, 7, 2, 5), (3, 7, 2, 5)))
    bias = torch.randn(1 if shared else 3, 6, 4, 7, generator=g).to(dtype)
    mask = torch.rand(3, 7, generator=g) < 0.6
    mask[1] = False  # nothing is left there
    tol = {torch.float32: 2e-6, torch.float64: 1e-13, torch.bfloat16: 2.0 ** -8}[dtype]
    for b, m, s in ((None, None, None), (bias, None, 0.3), (None, mask, None), (bias, mask, None)):
        got = cross_attention(q, k, v, b, m, s)
        want = _formula(q, k, v, b, m, 5 ** -0.5 if s is None else s)
        assert got.dtype == dtype and got.shape == q.shape
        assert ((got.double() - want).abs() <= tol * (1 + want.abs())).all()
        if m is not None:
            assert not got[1].any()


def test_torch_path_gradients():
    g = torch.Generator().manual_seed(2)
    q, k, v, bias = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
                     for s in ((2, 3, 4, 3), (2, 5, 2, 3), (2, 5, 2, 3), (1, 4, 3, 5)))
    mask = torch.tensor([[True, False, True, True, False], [False] * 5])
    assert torch.autograd.gradcheck(lambda *t: cross_attention(*t, mask), (q, k, v, bias))


def test_masked_keys_have_no_effect():
    g = torch.Generator().manual_seed(3)
    q, k, v, bias = (torch.randn(*s, generator=g) for s in ((1, 3, 2, 4), (1, 5, 2, 4), (1, 5, 2, 4), (1, 2, 3, 5)))
    mask = torch.tensor([[True, True, False, True, False]])
    want = cross_attention(q, k[:, [0, 1, 3]], v[:, [0, 1, 3]], bias[..., [0, 1, 3]])
    for what in (float("nan"), float("inf"), -3e38):
        k[:, ~mask[0]] = v[:, ~mask[0]] = what
        bias[..., ~mask[0]] = what
        leaves = [t.clone().requires_grad_() for t in (q, k, v, bias)]
        got = cross_attention(*leaves, mask)
        assert (got - want).abs().max() < 1e-6
        for t in torch.autograd.grad(got.sum(), leaves):
            assert torch.isfinite(t).all()


def test_a_bias_that_leaves_nothing():
    q = torch.randn(1, 2, 1, 4)
    bias = torch.zeros(1, 1, 2, 3)
    bias[0, 0, 1] = float("-inf")
    out = cross_attention(q, torch.ones(1, 3, 1, 4), torch.ones(1, 3, 1, 4), bias)
    assert (out[0, 0] - 1).abs().max() < 1e-6 and not out[0, 1].any()


def test_no_keys():
    q, k, b = torch.ones(2, 3, 4, 8, requires_grad=True), torch.ones(2, 0, 2, 8, requires_grad=True), torch.ones(1, 4, 3, 0)
    out = cross_attention(q, k, k, b.requires_grad_())
    assert out.shape == q.shape and not out.any()
    for t, x in zip(torch.autograd.grad(out.sum(), [q, b]), (q, b)):
        assert t.shape == x.shape and not t.any()


def test_no_keys_whatever_the_queries_hold():
    q, k, v = (torch.full((1, 2, 2, 8), float("nan"), requires_grad=True), *(torch.ones(1, 0, 1, 8, requires_grad=True) for _ in "kv"))
    out = cross_attention(q, k, v)
    assert out.shape == q.shape and not out.any()
    for t, x in zip(torch.autograd.grad(out.sum(), [q, k, v]), (q, k, v)):
        assert t.shape == x.shape and not t.any()


@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("keys", [0, 1, 5])
def test_the_result_is_contiguous(keys, heads):
    """Whatever the layout of the queries, as the kernels' is."""
    q, k = torch.randn(2, 4, 3, 8).transpose(1, 2), torch.randn(2, heads, keys, 8).transpose(1, 2)
    for t in (q, q[:, :1], q.double()):
        assert cross_attention(t, k.to(t.dtype), k.to(t.dtype)).is_contiguous()


def test_refusals():
    q, k, bias = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 2, 8), torch.zeros(2, 4, 3, 5)
    with pytest.raises(ValueError, match=r"\[batch, queries, heads, head_dim\]"):
        cross_attention(q[0], k, k)
    with pytest.raises(ValueError, match="floating-point"):
        cross_attention(q.long(), k, k)
    for bad in (k[:1], k[..., :4], torch.zeros(2, 5, 3, 8), torch.zeros(2, 5, 0, 8), k[0]):
        with pytest.raises(ValueError, match=r"k must be \[2, keys, key_heads, 8\]"):
            cross_attention(q, bad, bad)
    with pytest.raises(ValueError, match="v must have k's shape"):
        cross_attention(q, k, k[:, :4])
    for bad in (bias[:, :1], bias[0], bias[..., :1], bias.expand(2, 4, 3, 5)[:, :, :1]):
        with pytest.raises(ValueError, match="bias must have shape"):
            cross_attention(q, k, k, bad)
    with pytest.raises(ValueError, match="k must be torch.float32 like q"):
        cross_attention(q, k.half(), k.half())
    with pytest.raises(ValueError, match="bias must be torch.float32 like q"):
        cross_attention(q, k, k, bias.half())
    with pytest.raises(ValueError, match="mask must be bool"):
        cross_attention(q, k, k, mask=torch.ones(2, 5))
    with pytest.raises(ValueError, match=r"mask must have shape \(2, 5\)"):
        cross_attention(q, k, k, mask=torch.ones(5, dtype=torch.bool))
    with pytest.raises(ValueError, match="mask is on meta"):
        cross_attention(q, k, k, mask=torch.ones(2, 5, dtype=torch.bool, device="meta"))
    with pytest.raises(ValueError, match="k is on meta"):
        cross_attention(q, k.to("meta"), k.to("meta"))
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale must be positive"):
            cross_attention(q, k, k, scale=s)


def test_what_the_kernels_take():
    def t(b, n, h, d):
        return torch.empty(b, n, h, d, device="meta")

    assert _hip.supports(t(1, 1, 1, 8), t(1, 1, 1, 8)) and _hip.supports(t(2, 9, 4, 128), t(2, 1 << 20, 2, 128))
    for d in (4, 12, 136, 256):
        assert not _hip.supports(t(1, 1, 1, d), t(1, 1, 1, d))
    assert not _hip.supports(t(1, 1, 1, 8), t(1, 1 << 30, 1, 8))
    assert not _hip.supports(t(1, 1, 1 << 16, 64), t(1, 1, 1, 64))


def test_tokens_far_apart_are_copied():
    def t(shape, stride, dtype=torch.bfloat16):
        return torch.empty_strided(shape, stride, dtype=dtype, device="meta")

    near = (2, 9, 4, 64), (1 << 40, (1 << 24) - 1, 64, 1)
    far = (2, 9, 4, 64), (1 << 40, 1 << 24, 64, 1)
    assert _hip._heads(t(*near)).stride() == near[1]
    assert _hip._heads(t(*far)).is_contiguous() and _hip._heads(t(*near, torch.float32)).is_contiguous()
    turned = (2, 9, 4, 64), (1 << 40, 64, 1 << 30, 1)  # heads before tokens: apart only where rows count them
    assert _hip._heads(t(*turned)).stride() == turned[1] and _hip._heads(t(*turned), 2).is_contiguous()


@pytest.mark.parametrize("cls,name", [(_lib.CrossAttnArgs, "gnn_cross_attn_fwd"), (_lib.CrossAttnBwdArgs, "gnn_cross_attn_bwd")])
def test_argument_errors(cls, name):
    lib = _lib.load()
    fn, size = getattr(lib, name), getattr(lib, name.replace("_fwd", "") + "_workspace_bytes")
    a = cls()

    def refused(text, code=_lib.GNN_ERR_ARG):
        assert fn(ctypes.byref(a), None) == code
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    assert fn(None, None) == _lib.GNN_ERR_ARG and size(None) == 0
    a.dtype = 9
    refused(b"dtype")
    a.dtype, a.precision = _lib.GNN_BF16, 7
    refused(b"precision")
    a.precision = 0
    for d in (0, 4, 12, 136):
        a.D = d
        refused(b"head dim", _lib.GNN_ERR_UNSUPPORTED)
    a.D = 64
    refused(b"positive")
    a.B, a.U, a.V, a.H, a.Hk = 1, 4, 5, 6, 4
    refused(b"multiple of Hk")
    a.Hk = 2
    for s in (0.0, -1.0, float("nan"), float("inf")):
        a.scale = s
        refused(b"scale")
    a.scale = 1.0
    refused(b"required")
    a.q = a.k = a.v = 4096
    refused(b"required")
    a.k = 4097
    refused(b"aligned")
    a.k = 4096
    for field, at, far in (("q", 1, 1 << 24), ("k", 1, 1 << 24), ("v", 1, -1), ("q", 2, 1 << 29), ("q", 1, 1 << 62)):
        strides = getattr(a, field + "_stride")
        strides[at] = far
        refused(b"2^31", _lib.GNN_ERR_UNSUPPORTED)
        assert size(ctypes.byref(a)) == 0
        strides[at] = 0
    a.o = 4096
    if cls is _lib.CrossAttnArgs:
        a.o = 4104
        refused(b"16-byte")
        a.o, a.o_low = 4096, 4104
        refused(b"16-byte")
        a.o_low, a.U, a.Hk, a.V = None, 1, 1, 1 << 16  # keys split over workgroups
        assert size(ctypes.byref(a)) % 4 == 0 and size(ctypes.byref(a)) > 0
        refused(b"workspace", _lib.GNN_ERR_WORKSPACE)
        return
    a.dout = a.dq = a.stats = 4096
    a.dk = 4096
    refused(b"together")
    a.dv, a.dbias = 4096, 4096
    refused(b"dbias with bias")
    a.bias, a.shared_bias, a.bias_stride[0] = 4096, 1, 5
    refused(b"batch stride 0")
    a.bias_stride[0], a.dv = 0, 4104
    refused(b"16 bytes")
    a.dv = 4096
    for strides in (a.o_stride, a.do_stride):
        strides[1] = 1 << 24
        refused(b"2^31", _lib.GNN_ERR_UNSUPPORTED)
        strides[1] = 0
    assert size(ctypes.byref(a)) >= 4 * 6 * 4
    refused(b"workspace", _lib.GNN_ERR_WORKSPACE)


def test_heads_far_apart_are_taken_or_copied():
    """What the host side leaves in place the library takes: both count 64 tokens and the heads of one of them."""
    lib = _lib.load()
    most = (1 << 31) // 2  # elements of 2 bytes
    for group in (2, 3, 8):
        for head in (most // group - 64, most // group + 64, (most - 64 * 64) // (group - 1) - 64, (most - 64 * 64) // (group - 1) + 64):
            q = torch.empty_strided((1, 3, group, 64), (1 << 40, 64, head, 1), dtype=torch.bfloat16, device="meta")
            in_place = _hip._heads(q, group).stride() == q.stride()
            a = _lib.CrossAttnBwdArgs()
            a.dtype, a.D, a.B, a.U, a.V, a.H, a.Hk, a.scale = _lib.GNN_BF16, 64, 1, 3, 5, group, 1, 1.0
            a.q = a.k = a.v = 4096
            a.q_stride = _lib.I64x3(*q.stride()[:3])
            taken = lib.gnn_cross_attn_bwd_workspace_bytes(ctypes.byref(a)) > 0
            assert taken == in_place, (group, head)
    a.q_stride[2] = (1 << 63) - 1  # no overflow on the way
    assert lib.gnn_cross_attn_bwd_workspace_bytes(ctypes.byref(a)) == 0


HUGE = '''
import ctypes, sys
from geometric_nn_ops_torch import _lib
lib = _lib.load()
for b, u, v, h, hk in ((1 << 30, (1 << 30) - 1, 2, 1 << 30, 1 << 30), (1 << 29, 1 << 20, 127, 1 << 30, 1 << 30),
                       (1 << 24, 1 << 20, 1, 1 << 29, 1 << 24), (1 << 16, 1, 1 << 30, 1 << 14, 1 << 14)):
    for cls, name in ((_lib.CrossAttnArgs, "gnn_cross_attn"), (_lib.CrossAttnBwdArgs, "gnn_cross_attn_bwd")):
        a = cls()
        a.dtype, a.D, a.B, a.U, a.V, a.H, a.Hk, a.scale = _lib.GNN_BF16, 64, b, u, v, h, hk, 1.0
        a.q = a.k = a.v = a.o = 4096
        if "bwd" in name:
            a.dout = a.dq = a.dk = a.dv = a.stats = 4096
        assert getattr(lib, name + "_workspace_bytes")(ctypes.byref(a)) == 0
        fn = getattr(lib, name if "bwd" in name else name + "_fwd")
        assert fn(ctypes.byref(a), None) == _lib.GNN_ERR_UNSUPPORTED and b"grid" in lib.gnn_last_error()
'''


def test_sizes_beyond_any_grid_are_refused():
    """Their products pass 64 bits; in a process of its own, which a division by zero would end."""
    root = pathlib.Path(__file__).resolve().parent.parent / "geometric-nn-ops_amd"
    run = subprocess.run([sys.executable, "-c", HUGE], env={**os.environ, "PYTHONPATH": str(root)}, capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stderr[-500:])


def test_args_match_the_c_layout(tmp_path):
    root = pathlib.Path(__file__).resolve().parent.parent
    structs = {"gnn_cross_attn_args": _lib.CrossAttnArgs, "gnn_cross_attn_bwd_args": _lib.CrossAttnBwdArgs}
    body = "".join(f'printf("%zu\\n", sizeof({s}));' + "".join(
        f'printf("%zu\\n", offsetof({s}, {f[0]}));' for f in c._fields_) for s, c in structs.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnn_triangle.h"\nint main(void) {' + body +
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    want = [v for c in structs.values() for v in (ctypes.sizeof(c), *(getattr(c, f[0]).offset for f in c._fields_))]
    assert [int(v) for v in out] == want
