"""What the backward passes are given when autograd hands back other tensors than the forward saved
(saved-tensor hooks, activation checkpoints), on a CPU-only host: the library is replaced by a recorder."""

import ctypes
import types

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

from geometric_nn_ops_torch import _lib
from geometric_nn_ops_torch.triangle import _fused_linear, _layer_norm, _relative_position


@pytest.fixture
def recorded(monkeypatch):
    """Calls as ``(entry point, copy of its arguments)``; the library's queries answer 1."""
    calls = []

    def call(name, args, device):
        calls.append((name, type(args).from_buffer_copy(args)))

    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(
        gnn_relpos_parts=lambda a: 1, gnn_layer_norm_bwd_parts=lambda *a: 1))
    return calls


HOW = (8, "clip", True, False)


def _read(address, stride, rows, n):
    """int64 ``[rows, n]`` at an address; the memory belongs to a tensor that the test holds."""
    return [[ctypes.c_int64.from_address(address + 8 * (r * stride + j)).value for j in range(n)] for r in range(rows)]


def test_relative_position_reads_the_unpacked_positions(recorded):
    table = torch.randn(17, 2, requires_grad=True)
    q, k = torch.arange(4)[None].repeat(2, 1) + 7, torch.arange(5)[None].repeat(2, 1) - 3
    # what comes back lies elsewhere, in another pitch or order
    for lay_out in (torch.clone, lambda t: torch.nn.functional.pad(t, (0, 3))[:, :t.shape[1]],
                    lambda t: t.t().contiguous().t()):
        recorded.clear()
        held = []

        def unpack(t, held=held):
            held.append(t)
            return t

        with saved_tensors_hooks(lay_out, unpack):
            out = _relative_position._RelativePositionHip.apply(table, q.clone(), k.clone(), HOW)
        out.backward(torch.ones_like(out))
        assert len(held) == 2
        name, a = recorded[-1]
        assert name == "gnn_relpos_bwd"
        for got, stride, at, want in ((held[0], a.query_stride, a.query_pos, q), (held[1], a.key_stride, a.key_pos, k)):
            if got.stride(1) == 1:
                assert at == got.data_ptr() and stride == got.stride(0)
            else:  # laid out anew, dense
                assert at != got.data_ptr() and stride == got.shape[1]
            assert torch.equal(got, want)
            if got.stride(1) == 1:
                assert _read(at, stride, *want.shape) == want.tolist()


def test_relative_position_in_a_checkpoint_reads_the_recomputed_positions(recorded):
    table = torch.randn(17, 2, requires_grad=True)
    start = torch.arange(64)[None]

    def block(t):
        pos = start + 5  # nobody but the graph holds it
        return _relative_position._RelativePositionHip.apply(t, pos, pos, HOW)

    out = checkpoint(block, table, use_reentrant=False)
    taken = [torch.full_like(start, -999) for _ in range(64)]  # what the first forward's positions left free
    out.backward(torch.ones_like(out))
    assert [name for name, _ in recorded] == ["gnn_relpos_fwd", "gnn_relpos_fwd", "gnn_relpos_bwd"]
    first, again, bwd = (a for _, a in recorded)
    assert first.query_pos != again.query_pos and len(taken) == 64
    assert (bwd.query_pos, bwd.key_pos) == (again.query_pos, again.key_pos)


def test_layer_norm_reads_the_unpacked_statistics(monkeypatch):
    """Each row's mean and 1 / standard deviation, whatever pitch they come back in."""
    rows, found = 6, []

    def floats(address):
        return [ctypes.c_float.from_address(address + 4 * r).value for r in range(rows)]

    def call(name, args, device):
        if name == "gnn_layer_norm_fwd":
            for at, base in ((args.mean, 10.0), (args.rstd, 20.0)):
                for r in range(rows):
                    ctypes.c_float.from_address(at + 4 * r).value = base + r
        else:
            found.append(floats(args.mean) + floats(args.rstd))

    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(gnn_layer_norm_bwd_parts=lambda *a: 1))
    x = torch.randn(rows, 16, requires_grad=True)
    for pack in (torch.clone, lambda t: torch.nn.functional.pad(t, (0, 5))[..., :t.shape[-1]],
                 lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        with saved_tensors_hooks(pack, lambda t: t):
            y = _layer_norm._LayerNormHip.apply(x, None, None, 1e-5)
        y.backward(torch.ones_like(y))
        assert found.pop() == [10.0 + r for r in range(rows)] + [20.0 + r for r in range(rows)]


def test_fused_linear_reads_unpacked_operands_in_whole_chunks(monkeypatch):
    """The kernels take x and the weight in aligned 16-byte chunks, wherever the two come back."""
    m, i, o = 6, 16, 8
    x, w = torch.randn(m, i, requires_grad=True), torch.randn(o, i, requires_grad=True)
    found = []

    def rows(address, ld, n, k):
        assert address % 16 == 0 and ld % 4 == 0 and ld >= k
        return torch.tensor([[ctypes.c_float.from_address(address + 4 * (r * ld + j)).value for j in range(k)]
                             for r in range(n)])

    def call(name, args, device):
        if name == "gnn_linear" and args.dz:
            found.append((rows(args.x, args.x_ld, m, i), rows(args.w, args.w_ld, o, i)))
        elif name == "gnn_linear_wgrad":
            found.append(rows(args.x, args.x_ld, m, i))
        elif name == "gnn_pad_rows":  # copies element by element
            for r in range(args.rows):
                for c in range(args.ld):
                    at = args.src + 4 * (r * args.row_stride + c * args.col_stride)
                    ctypes.c_float.from_address(args.dst + 4 * (r * args.ld + c)).value = (
                        ctypes.c_float.from_address(at).value if c < args.cols else 0.0)

    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(
        gnn_linear_takes_transposed=lambda a: 0, gnn_linear_takes_dx=lambda a: 0, gnn_linear_wgrad_slices=lambda a: 1))

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype)[1:]
        return flat.copy_(t.reshape(-1)).view(t.shape)

    def spread(t):
        return torch.stack([t, -t], -1)[..., 0]

    for pack in (torch.clone, shifted, spread, lambda t: t.t().contiguous().t()):
        with saved_tensors_hooks(pack, lambda t: t):
            y = _fused_linear._FusedLinearHip.apply(x, w, None, "silu", None)
        torch.autograd.grad(y, (x, w), torch.ones_like(y))
        (in_dz, weight), in_dw = found
        found.clear()
        assert torch.equal(in_dz, x) and torch.equal(weight, w) and torch.equal(in_dw, x)
