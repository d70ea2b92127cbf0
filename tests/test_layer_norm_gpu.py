"""layer_norm on the GPU against the formulas in float64.

Bounds. fp32 sums go through at most 32 elements of a lane and 10 steps of the team: the mean is off by at
most 42 U mean|x|, 1 / sigma by a relative 64 U, so the normalised value by E = 64 U (rstd mean|x| + |xhat|).
A gradient's sums add the same counts; the parameters' sums run over at most 128 rows in a lane and are
then added pairwise: 256 U of the sum of absolute values."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import layer_norm
from op_helpers import DTYPES, IDS, U, assert_within, directional, replays_match

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-5

SHAPES = [(1, 1), (1, 7), (3, 8), (5, 9), (2, 16), (33, 64), (130, 100), (257, 128), (7, 200), (65, 384), (9, 511),
          (19, 520), (12, 768), (5, 1025), (6, 1537), (5, 2048), (4, 3001), (9, 4104), (3, 5003), (2, 7000), (2, 8192),
          (3, 12289), (2, 16384), (70001, 16)]


def _inputs(rows, k, dtype, wdtype, seed=0, shift=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, k, generator=g) * (0.5 + torch.rand(k, generator=g)) + shift).to(dtype)
    w = (1 + 0.2 * torch.randn(k, generator=g)).to(wdtype)
    b = (0.2 * torch.randn(k, generator=g)).to(wdtype)
    dy = torch.randn(rows, k, generator=g).to(dtype)
    return x, w, b, dy


def _exact(x, w, b, dy=None, eps=EPS):
    """y and its fp32 slack, and with dy: dx, dw, db with theirs (all float64)."""
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double()
    d = x - x.mean(-1, keepdim=True)
    r = 1 / (d.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    xh = d * r
    e = 64 * U * (r * x.abs().mean(-1, keepdim=True) + xh.abs())
    # the deviations' squares carry the mean's error too: a relative error of 1 / sigma of E's size
    spread = (e * xh.abs()).mean(-1, keepdim=True)
    e = e + xh.abs() * spread
    out = [(xh * w + b, e * w.abs() + 4 * U * (xh * w).abs() + 4 * U * b.abs())]
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    dx = r * (g - m1 - xh * m2)
    slack = r * (64 * U * (g.abs() + a1 + xh.abs() * a2) + e * a2 + xh.abs() * (g.abs() * e).mean(-1, keepdim=True))
    slack = slack + (64 * U + spread) * r * (g.abs() + a1 + xh.abs() * a2)
    out.append((dx, slack))
    out.append(((dy * xh).sum(0), 256 * U * (dy * xh).abs().sum(0) + (dy.abs() * e).sum(0)))
    out.append((dy.sum(0), 256 * U * dy.abs().sum(0)))
    return out


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_forward_and_gradients(rows, k, dtype):
    # the parameters in the rows' type at even widths, in fp32 at odd ones
    x, w, b, dy = _inputs(rows, k, dtype, dtype if k % 2 == 0 else torch.float32, seed=rows + k)
    exact = _exact(x, w, b, dy)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, EPS)
    assert y.dtype == dtype and y.is_contiguous()
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    with torch.no_grad():
        assert torch.equal(layer_norm(*leaves, EPS), y)
    for name, got, (want, slack) in zip(("y", "dx", "dw", "db"), (y, *grads), exact):
        assert_within(f"{name} {rows}x{k}", got, want, slack)


@pytest.mark.parametrize("params", ["none", "weight", "bias"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_parameters_left_out(dtype, params):
    x, w, b, dy = _inputs(37, 96, dtype, dtype, seed=3)
    w, b = (w if params == "weight" else None), (b if params == "bias" else None)
    exact = _exact(x, w, b, dy)
    named = [("x", x), ("w", w), ("b", b)]
    leaves = {n: t.to(DEV).requires_grad_() for n, t in named if t is not None}
    y = layer_norm(leaves["x"], leaves.get("w"), leaves.get("b"), EPS)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to(DEV))))
    assert_within("y", y, *exact[0])
    for n, (want, slack) in zip(("x", "w", "b"), exact[1:]):
        if n in grads:
            assert_within(n, grads[n], want, slack)


def test_only_the_gradients_asked_for():
    x, w, b, dy = _inputs(50, 128, torch.bfloat16, torch.bfloat16, seed=4)
    exact = _exact(x, w, b, dy)
    for i, name in enumerate(("x", "w", "b")):
        args = [t.to(DEV) for t in (x, w, b)]
        args[i].requires_grad_()
        (got,) = torch.autograd.grad(layer_norm(*args, EPS), [args[i]], dy.to(DEV))
        assert_within(name, got, *exact[1 + i])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views_are_read_in_place(dtype):
    """Column slices at odd offsets, transposed pair tensors (one and two batches, the latter by a copy),
    a row step, expanded rows, a strided last dimension; the output gradient in the same variety."""
    g = torch.Generator().manual_seed(5)
    base = torch.randn(2, 6, 6, 100, generator=g).to(dtype).to(DEV)
    views = [base[..., 3:67], base[:1].transpose(1, 2), base.transpose(1, 2), base[:, ::2, :, 1:50],
             base[:1, :1, :1].expand(2, 3, 4, 100), base[..., ::2], base[0, 0], base[0, 0, 0, 5:38]]
    for i, x in enumerate(views):
        k = x.shape[-1]
        w = (1 + 0.1 * torch.randn(k, generator=g)).to(DEV)
        grads_out = torch.randn(2, *x.shape, generator=g).to(dtype).to(DEV)
        for dy in (grads_out[0], grads_out.transpose(0, 1)[:, 1] if x.dim() > 1 else grads_out[1],
                   grads_out[0].sum().expand(x.shape)):
            if dy.shape != x.shape:
                continue
            xl, wl = x.detach().requires_grad_(), w.clone().requires_grad_()
            y = layer_norm(xl, wl, None, EPS)
            dx, dw = torch.autograd.grad(y, [xl, wl], dy)
            exact = _exact(x.cpu().reshape(-1, k), w.cpu(), None, dy.cpu().reshape(-1, k))
            for name, got, (want, slack) in zip(("y", "dx", "dw"), (y, dx, dw), exact):
                assert_within(f"view {i} {name}", got.reshape(want.shape), want, slack)


def test_large_means_keep_the_variance():
    """Rows whose mean is 1000 deviations away: the variance comes from the deviations, not from a
    difference of squares (which would leave nothing of it in fp32)."""
    x, w, b, _ = _inputs(64, 640, torch.float32, torch.float32, seed=6, shift=1000.0)
    assert_within("y", layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), EPS), *_exact(x, w, b)[0])


def test_constant_rows_and_rows_that_are_not_finite():
    x = torch.randn(9, 130, generator=torch.Generator().manual_seed(7))
    x[2] = 0.0
    x[3] = 2.5
    x[5, 17] = float("inf")
    x[6, 129] = float("nan")
    b = torch.linspace(-1, 1, 130)
    y = layer_norm(x.to(DEV), None, b.to(DEV), EPS).cpu()
    assert torch.equal(y[2], b) and torch.equal(y[3], b)
    assert y[5].isnan().any() and y[6].isnan().all()
    keep = [0, 1, 4, 7, 8]
    want, slack = _exact(x[keep], None, b)[0]
    assert_within("other rows", y[keep], want, slack)


def test_no_rows():
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.empty(*shape, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        w = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        b = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        y = layer_norm(x, w, b)
        assert y.shape == x.shape
        dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_wide_rows_and_float64_take_the_torch_path():
    x = torch.randn(2, 16385, device=DEV, requires_grad=True)
    y = layer_norm(x)
    want, slack = _exact(x.detach().cpu(), None, None)[0]
    assert ((y.detach().cpu().double() - want).abs() <= 1e-5 * (1 + want.abs())).all()
    torch.autograd.grad(y.sum(), x)
    x = torch.randn(3, 40, device=DEV, dtype=torch.float64)
    want = _exact(x.cpu(), None, None)[0][0]
    assert ((layer_norm(x).cpu() - want).abs() < 1e-12).all()


def test_gradient_against_differences():
    x, w, b, dy = _inputs(12, 72, torch.float32, torch.float32, seed=8)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves, EPS), leaves, dy.to(DEV))
    point = [t.double() for t in (x, w, b)]
    for i in range(3):
        v = torch.randn(point[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)

        def f(t, i=i):
            args = point[:i] + [t] + point[i + 1:]
            return (_exact(*args)[0][0] * dy.double()).sum()

        want = directional(f, point[i], v)
        got = (grads[i].double().cpu() * v).sum()
        # the difference is off by h^2 / 6 third derivatives, the gradient by some U of its terms
        assert abs(got - want) <= 1e-5 * (grads[i].double().cpu() * v).abs().sum()


def test_second_derivative_raises():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_offsets_beyond_32_bits():
    rows, k = (1 << 24) + 5, 131
    x = torch.empty(rows, k, device=DEV, dtype=torch.bfloat16)
    tail = torch.randn(64, k, generator=torch.Generator().manual_seed(9)).bfloat16()
    x[:-64].fill_(1.0)
    x[-64:] = tail.to(DEV)
    dy = torch.zeros_like(x)
    dy[-64:] = tail.flip(0).to(DEV)
    w = torch.ones(k, device=DEV, requires_grad=True)
    x.requires_grad_()
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    exact = _exact(tail, None, None, tail.flip(0))
    assert not y[:-64].any() and not dx[:-64].any()
    assert_within("y", y[-64:], *exact[0])
    assert_within("dx", dx[-64:], *exact[1])
    assert_within("dw", dw, *exact[2])


def test_calls_repeat_bit_for_bit_and_replay_in_a_graph():
    x, w, b, dy = (t.to(DEV) for t in _inputs(3000, 384, torch.bfloat16, torch.float32, seed=10))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def block():
        y = layer_norm(*leaves, EPS)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    def equal(got, want, replay):
        assert torch.equal(got, want), replay

    replays_match(block, equal)


def test_another_stream():
    x, w, b, dy = (t.to(DEV) for t in _inputs(500, 256, torch.float16, torch.float16, seed=11))
    want = layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm(x * 1, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_operator_registration():
    import geometric_nn_ops_torch._ops  # noqa: F401

    x, w, b, _ = (t.to(DEV) for t in _inputs(6, 40, torch.bfloat16, torch.bfloat16, seed=12))
    torch.library.opcheck(torch.ops.gnn_amd.layer_norm_fwd.default, (x, w, b, 1e-5),
                          test_utils=("test_schema", "test_faketensor"))
    with torch.no_grad():
        compiled = torch.compile(lambda t: layer_norm(t, w, b), fullgraph=True, backend="aot_eager")(x)
        assert torch.equal(compiled, layer_norm(x, w, b))
