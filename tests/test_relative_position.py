"""relative_position_bias on a CPU-only host: buckets against their definition distance by distance, the
torch path's values and gradients, the refusals, and the C entry points' argument errors."""

import ctypes
import pathlib
import subprocess
from fractions import Fraction

import pytest
import torch

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import relative_position_bias
from geometric_nn_ops_torch.triangle._reference.relative_position import buckets_torch, log_borders, side_buckets


def bucket(ahead, num_buckets, max_distance, spacing, bidirectional):
    """One bucket, from the definition, in exact rationals."""
    if spacing == "clip":
        if bidirectional:
            return max(-max_distance, min(max_distance, ahead)) + max_distance
        return max(0, min(max_distance, -ahead))
    n, near = side_buckets(num_buckets, bidirectional)
    d = min(abs(ahead) if bidirectional else max(-ahead, 0), max_distance)
    side = d
    if d >= near:
        m = n - near
        ratio, whole = Fraction(d, near), Fraction(max_distance, near)
        side = near + max(k for k in range(m) if ratio**m >= whole**k)
    return side + (n if bidirectional and ahead > 0 else 0)


CASES = [(32, 128, "log", True), (32, 128, "log", False), (8, 20, "log", True), (64, 1000, "log", True),
         (7, 11, "log", False), (2, 2, "log", False), (4, 2, "log", True), (33, 17, "log", False), (12, 7, "log", True),
         (65, 32, "clip", True), (33, 32, "clip", False), (3, 1, "clip", True), (2, 1, "clip", False)]


@pytest.mark.parametrize("case", CASES)
def test_buckets(case):
    far = case[1]
    pos = torch.arange(-far - 3, far + 4)
    got = buckets_torch(torch.zeros(1, 1, dtype=torch.int64), pos[None], *case)[0, 0]
    want = [bucket(int(p), *case) for p in pos]
    assert got.tolist() == want
    assert min(want) >= 0 and max(want) <= case[0] - 1


def test_borders_ascend():
    for n in range(2, 40):
        near = n // 2
        for far in (near + 1, near + 2, 3 * near + 1, 1000, 10**6):
            if far <= near:
                continue
            b = log_borders(n, near, far)
            assert len(b) == n - near - 1 and list(b) == sorted(b) and all(near <= d <= far for d in b)


@pytest.mark.parametrize("channels_last", [False, True])
def test_torch_path(channels_last):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(32, 3, generator=g, dtype=torch.float64, requires_grad=True)
    q, k = torch.randint(0, 300, (2, 5), generator=g), torch.randint(0, 300, (2, 9), generator=g)
    out = relative_position_bias(w, q, k, max_distance=128, channels_last=channels_last)
    assert out.shape == ((2, 5, 9, 3) if channels_last else (2, 3, 5, 9))
    for b in range(2):
        for i in range(5):
            for j in range(9):
                row = w[bucket(int(k[b, j] - q[b, i]), 32, 128, "log", True)]
                assert torch.equal(out[b, i, j] if channels_last else out[b, :, i, j], row)
    assert torch.autograd.gradcheck(
        lambda t: relative_position_bias(t, q, k, max_distance=128, channels_last=channels_last), (w,))


def test_batches_and_defaults():
    w = torch.randn(65, 4)
    pos = torch.arange(7)
    a = relative_position_bias(w, pos, max_distance=32, spacing="clip")
    assert a.shape == (1, 4, 7, 7)
    b = relative_position_bias(w, pos.int(), torch.stack([pos, pos + 5]), max_distance=32, spacing="clip")
    assert b.shape == (2, 4, 7, 7) and torch.equal(b[:1], a) and not torch.equal(b[1:], a)
    assert relative_position_bias(w, pos[:0], pos, max_distance=32, spacing="clip").shape == (1, 4, 0, 7)
    with pytest.raises(ValueError, match="batches 2 and 3"):
        relative_position_bias(w, pos.expand(2, 7), pos.expand(3, 7), max_distance=32, spacing="clip")


def test_refusals():
    w, pos = torch.randn(32, 4), torch.arange(6)
    ok = dict(max_distance=128)
    with pytest.raises(ValueError, match="num_buckets, heads"):
        relative_position_bias(w[0], pos, **ok)
    with pytest.raises(ValueError, match="num_buckets, heads"):
        relative_position_bias(w.long(), pos, **ok)
    with pytest.raises(ValueError, match="int32 or int64"):
        relative_position_bias(w, pos.float(), **ok)
    with pytest.raises(ValueError, match="int32 or int64"):
        relative_position_bias(w, pos, pos.bool(), **ok)
    with pytest.raises(ValueError, match="batch, length"):
        relative_position_bias(w, pos.view(1, 2, 3), **ok)
    with pytest.raises(ValueError, match="key_pos is on meta"):
        relative_position_bias(w, pos, pos.to("meta"), **ok)
    with pytest.raises(ValueError, match="spacing must be"):
        relative_position_bias(w, pos, spacing="linear", **ok)
    with pytest.raises(ValueError, match="at least 1"):
        relative_position_bias(w, pos, max_distance=0)
    with pytest.raises(ValueError, match="257 buckets"):
        relative_position_bias(w, pos, spacing="clip", **ok)
    with pytest.raises(ValueError, match="129 buckets"):
        relative_position_bias(w, pos, spacing="clip", bidirectional=False, **ok)
    with pytest.raises(ValueError, match="even number"):
        relative_position_bias(torch.randn(31, 4), pos, **ok)
    with pytest.raises(ValueError, match="even number"):
        relative_position_bias(torch.randn(2, 4), pos, **ok)
    with pytest.raises(ValueError, match="2 buckets"):
        relative_position_bias(torch.randn(1, 4), pos, bidirectional=False, **ok)
    with pytest.raises(ValueError, match="above the 8"):
        relative_position_bias(w, pos, max_distance=8)


def test_argument_errors():
    lib = _lib.load()
    assert lib.gnn_relpos_fwd(None, None) == _lib.GNN_ERR_ARG
    assert lib.gnn_relpos_bwd(None, None) == _lib.GNN_ERR_ARG
    assert lib.gnn_relpos_parts(None) == 0
    a = _lib.RelposArgs()

    def refused(text, code=_lib.GNN_ERR_ARG, fn=lib.gnn_relpos_fwd):
        assert fn(ctypes.byref(a), None) == code
        assert text in lib.gnn_last_error(), lib.gnn_last_error()

    a.dtype = 9
    refused(b"dtype")
    a.dtype, a.pos_bytes = _lib.GNN_BF16, 2
    refused(b"4 or 8 bytes")
    a.pos_bytes = 8
    refused(b"positive")
    a.B = a.U = a.V = a.H = 4
    a.buckets = 32
    refused(b"max_distance")
    a.max_distance = 128
    refused(b"clip needs")
    a.log_spacing, a.two_sided = 1, 1
    refused(b"borders")
    border = (ctypes.c_int32 * 7)(12, 16, 23, 32, 46, 64, 129)
    a.border = ctypes.addressof(border)
    refused(b"ascend")
    border[6] = 91
    refused(b"are required")
    refused(b"are required", fn=lib.gnn_relpos_bwd)
    assert lib.gnn_relpos_parts(ctypes.byref(a)) >= 1
    a.table = a.query_pos = a.key_pos = 4096
    a.out = 4097
    refused(b"aligned")
    a.V = 1 << 30
    refused(b"below 2^31")
    a.V, a.max_distance = 4, 8
    refused(b"above half")
    a.max_distance, a.buckets = 128, 31
    refused(b"2 buckets a side")
    a.log_spacing, a.max_distance, a.buckets, a.out = 0, 2048, 4097, 4096
    refused(b"4096 buckets", _lib.GNN_ERR_UNSUPPORTED)
    a.log_spacing, a.two_sided, a.buckets, a.max_distance = 1, 0, 600, 2000
    refused(b"256 logarithmic", _lib.GNN_ERR_UNSUPPORTED)


def test_args_match_the_c_layout(tmp_path):
    root = pathlib.Path(__file__).resolve().parent.parent
    cls = _lib.RelposArgs
    body = 'printf("%zu\\n", sizeof(gnn_relpos_args));' + "".join(
        f'printf("%zu\\n", offsetof(gnn_relpos_args, {f[0]}));' for f in cls._fields_)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gnn_triangle.h"\nint main(void) {' + body +
                   "return 0;}")
    subprocess.run(["gcc", "-std=c11", f"-I{root / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in out] == [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
