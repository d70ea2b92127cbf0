"""fused_linear on the GPU against the formulas in float64.

Bounds. A product over K terms whose absolute values sum to S is off by at most min(K, 16 + 4 sqrt(K)) U S in
fp32 (rounding errors of random sign; K U S at the very worst), plus 3 * 2^-18 S where fp32 operands are split
into two bf16 parts (each operand's rest is 2^-18, the product of the two small parts 2^-18 again). The
activations add their own error (ACT below; the slopes are at most 1.2 and change by at most 1 per unit). dz
is rounded to the operands' type before the products: independent errors of at most half a step each, so
that a sum over terms t is off by less than six deviations, 2 sqrt(3) half sqrt(sum t^2)."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import (attention_pair_bias, fused_linear, layer_norm, relative_position_bias,
                                             triangle_attention)
from op_helpers import DTYPES, IDS, U, assert_within, directional, half_step, replays_match

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = [None, "relu", "gelu", "silu", "sigmoid"]
SHAPES = [(1, 1, 1), (1, 8, 8), (1, 384, 1536), (3, 7, 5), (17, 33, 65), (64, 128, 512), (129, 200, 131), (300, 64, 1),
          (5, 1, 300), (257, 512, 128), (2049, 131, 257), (40, 4100, 72), (700, 1024, 1000), (130, 72, 4100)]


class precision:
    def __init__(self, mode):
        self.mode = mode

    def __enter__(self):
        self.was = torch.backends.cuda.matmul.fp32_precision
        torch.backends.cuda.matmul.fp32_precision = self.mode

    def __exit__(self, *exc):
        torch.backends.cuda.matmul.fp32_precision = self.was


def _inputs(m, i, o, dtype, bias=True, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, i, generator=g).to(dtype)
    w = (torch.randn(o, i, generator=g) * i ** -0.5).to(dtype)
    b = (0.3 * torch.randn(o, generator=g)).to(dtype) if bias else None
    r = torch.randn(m, o, generator=g).to(dtype) if residual else None
    dy = torch.randn(m, o, generator=g).to(dtype)
    return x, w, b, r, dy


def _sum_error(k):
    return min(k, 16 + 4 * k ** 0.5) * U


def _act(z, act):
    """y, its slope, and what computing either may lose beside the error of z."""
    s = torch.sigmoid(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0 * z, 0 * z
    if act == "gelu":
        cdf, pdf = torch.special.ndtr(z), torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
        lost = (z * z + 8) * 4 * U
        return z * cdf, cdf + z * pdf, z.abs() * (2e-7 + lost * cdf), 2e-7 + lost * (cdf + z.abs() * pdf)
    if act == "silu":
        lost = (z.abs() + 8) * 4 * U
        return z * s, s * (1 + z * (1 - s)), lost * (z * s).abs(), lost * s * (1 + 2 * z.abs() * (1 - s))
    if act == "sigmoid":
        lost = (z.abs() + 8) * 4 * U
        return s, s * (1 - s), lost * s, lost * s
    return z, torch.ones_like(z), 0 * z, 0 * z


def _exact(x, w, b, r, act, dy=None, split=False):
    """(value, slack) of y and, with dy, of dx, dw, db."""
    dtype = x.dtype
    x, w = x.double(), w.double()
    per = 3 * 2.0 ** -18 if split else 0.0
    size = x.abs() @ w.abs().t()
    z = x @ w.t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    ez = (_sum_error(x.shape[1]) + per) * size + 2 * U * z.abs()
    y, slope, ey, es = _act(z, act)
    slack = 1.2 * ez + ey + 4 * U * y.abs()
    if r is not None:
        y = y + r.double()
        slack = slack + 2 * U * y.abs()
    out = [(y, slack)]
    if dy is None:
        return out
    dy = dy.double()
    dz = dy * slope
    if act is None:
        edz, half = 0 * dz, 0.0
    else:
        edz, half = dy.abs() * (ez + es) + 4 * U * dz.abs(), half_step(dtype) if dtype != torch.float32 else U
        if act == "relu":
            edz = edz * 0 + dy.abs() * (z.abs() <= ez)
        edz = edz + torch.finfo(dtype).tiny * torch.finfo(dtype).eps

    def product(a, c, k, extra=0.0):
        """a @ c with a = dz (or its transpose)."""
        ea = edz if a.shape == dz.shape and a.data_ptr() == dz.data_ptr() else edz.t()
        lost = (_sum_error(k) + extra) * (a.abs() @ c.abs()) + ea @ c.abs()
        return a @ c, lost + 2 * 3 ** 0.5 * half * (a.square() @ c.square()).sqrt()

    out.append(product(dz, w, w.shape[0], per))
    out.append(product(dz.t(), x, x.shape[0]))
    db = dz.sum(0)
    out.append((db, _sum_error(x.shape[0]) * dz.abs().sum(0) + edz.sum(0) + 2 * 3 ** 0.5 * half * dz.square().sum(0).sqrt()))
    return out


def _run(m, i, o, dtype, act, bias, residual, seed, split=False):
    x, w, b, r, dy = _inputs(m, i, o, dtype, bias, residual, seed)
    exact = _exact(x, w, b, r, act, dy, split)
    leaves = {n: t.to(DEV).requires_grad_() for n, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    y = fused_linear(leaves["x"], leaves["w"], leaves.get("b"), act, leaves.get("r"))
    assert y.dtype == dtype and y.is_contiguous()
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to(DEV))))
    with torch.no_grad():
        assert torch.equal(fused_linear(leaves["x"], leaves["w"], leaves.get("b"), act, leaves.get("r")), y)
    name = f"{m}x{i}->{o} {act}"
    assert_within(f"y {name}", y, *exact[0])
    for n, (want, slack) in zip("xwb", exact[1:]):
        if n in grads:
            assert_within(f"d{n} {name}", grads[n], want, slack)
    if residual:
        assert torch.equal(grads["r"].cpu(), dy)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,i,o", SHAPES)
def test_forward_and_gradients(m, i, o, dtype):
    act = ACTS[(m + i + o) % 5]
    with precision("ieee"):
        _run(m, i, o, dtype, act, (m + o) % 3 != 0, (m + i) % 2 == 0, seed=m + i + o)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("m,i,o", [(32768, 128, 512), (32791, 40, 72), (40001, 256, 200), (33000, 512, 128), (33333, 400, 24),
                                   (36865, 64, 1024), (33001, 136, 264), (35000, 576, 96), (33000, 16, 8),
                                   (131072, 128, 128)])
def test_many_rows(m, i, o, dtype):
    """The pixels of a pair tensor, where the weight stays in LDS, in every direction of the layer."""
    act = ACTS[(m + i + o) % 5]
    for bias, residual in ((True, False), (False, True)):
        x, w, b, r, dy = (None if t is None else t.to(DEV) for t in _inputs(m, i, o, dtype, bias, residual, seed=o))
        exact = _exact(x, w, b, r, act, dy)
        leaves = {n: t.clone().requires_grad_() for n, t in (("x", x), ("w", w), ("b", b)) if t is not None}
        y = fused_linear(leaves["x"], leaves["w"], leaves.get("b"), act, r)
        grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
        assert_within(f"y {act}", y.detach(), *exact[0])
        for n, (want, slack) in zip("xwb", exact[1:]):
            if n in grads:
                assert_within(f"d{n} {act}", grads[n], want, slack)


def test_many_rows_leave_what_lies_behind():
    """Rows behind the last one of a result inside a larger buffer stay as they were, and so do columns."""
    from geometric_nn_ops_torch import _lib

    m, i, o = 32768 + 5, 64, 40
    x, w, _, _, _ = (None if t is None else t.to(DEV) for t in _inputs(m, i, o, torch.bfloat16, False, False))
    out = torch.full((m + 40, o + 8), 7.0, device=DEV, dtype=torch.bfloat16)
    a = _lib.LinearArgs()
    a.x, a.w, a.out = x.data_ptr(), w.data_ptr(), out.data_ptr()
    a.M, a.I, a.O, a.out_cols, a.x_ld, a.w_ld, a.out_ld, a.dtype = m, i, o, o, i, i, o + 8, _lib.GNN_BF16
    _lib.call("gnn_linear", a, x.device)
    want, slack = _exact(x, w, None, None, None)[0]
    assert_within("y", out[:m, :o], want, slack)
    assert (out[m:] == 7).all() and (out[:, o:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
def test_every_activation(act, dtype):
    with precision("ieee"):
        for bias in (False, True):
            for residual in (False, True):
                _run(193, 96, 160, dtype, act, bias, residual, seed=3)


@pytest.mark.parametrize("act", ACTS)
def test_split_precision(act):
    """fp32 at 'tf32': the products of two bf16 parts, in the backward too."""
    with precision("tf32"):
        _run(150, 264, 136, torch.float32, act, True, True, seed=4, split=True)


def test_the_backward_keeps_the_forwards_precision():
    x, w, b, _, dy = (t if t is None else t.to(DEV) for t in _inputs(64, 128, 96, torch.float32, residual=False))
    x.requires_grad_()
    with precision("ieee"):
        y = fused_linear(x, w, b, "silu")
        (want,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    with precision("tf32"):
        (got,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
def test_extreme_inputs(act, dtype):
    """Activations far out on both sides stay exact zeros, ones or the input itself; a row or an output
    that is not finite stays in its row or column."""
    top = 200.0
    w = torch.eye(8).to(dtype)
    x = torch.tensor([[-top, -30.0, -8.0, -0.0, 0.0, 8.0, 30.0, top], [1.0] * 8]).to(dtype)
    y = fused_linear(x.to(DEV), w.to(DEV), None, act).double().cpu()
    want, slack = _exact(x, w, None, None, act)[0]
    assert_within(str(act), y.to(dtype), want, slack + 1e-12)
    x = torch.randn(6, 8, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[2, 3] = float("nan")
    w = torch.randn(10, 8, generator=torch.Generator().manual_seed(2)).to(dtype)
    b = torch.zeros(10).to(dtype)
    b[7] = float("inf")
    y = fused_linear(x.to(DEV), w.to(DEV), b.to(DEV), act).cpu()
    assert y[2].isnan().all()
    keep = [0, 1, 3, 4, 5]
    cols = [0, 1, 2, 3, 4, 5, 6, 8, 9]
    assert y[keep][:, cols].isfinite().all()
    assert (y[keep][:, 7] == (1.0 if act == "sigmoid" else float("inf"))).all()


def test_views():
    """Rows at odd offsets and pitches, transposed weights, expanded rows and gradients."""
    g = torch.Generator().manual_seed(5)
    big = torch.randn(40, 300, generator=g).bfloat16().to(DEV)
    with precision("ieee"):
        for x, w in ((big[:, 3:67], big[:20, 64:128]), (big[:, 8:72], big[:30, 9:73]),
                     (big[:1, 8:72].expand(7, 64), big[:10, :64]), (big[:36, :16].t(), big[:12, 4:40]),
                     (big[:, ::4], big[:9, 100:175]), (big[3:4, 1:41], big[5:6, 1:41]),
                     (big[:, :40].unflatten(0, (4, 10)).transpose(0, 1), big[:40, :17].t())):
            m = x.numel() // x.shape[-1]
            o = w.shape[0]
            x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
            dyw = torch.randn(m, 2 * o, generator=g).bfloat16().to(DEV)
            r = torch.randn(*x.shape[:-1], o + 3, generator=g).bfloat16().to(DEV)[..., 3:]
            y = fused_linear(x, w, None, "gelu", r)
            for dy in (dyw[:, 1:1 + o].reshape(y.shape), dyw[0, 0].expand(y.shape),
                       dyw[:1, :o].expand(m, o).reshape(y.shape)):
                dx, dw = torch.autograd.grad(y, [x, w], dy, retain_graph=True)
                exact = _exact(x.detach().cpu().reshape(m, -1), w.detach().cpu(), None, r.cpu().reshape(m, o), "gelu",
                               dy.cpu().reshape(m, o))
                for name, got, (want, slack) in zip(("y", "dx", "dw"), (y, dx, dw), exact):
                    assert_within(name, got.detach().reshape(want.shape), want, slack)


def test_only_the_gradients_asked_for():
    x, w, b, r, dy = _inputs(70, 40, 24, torch.float16, seed=6)
    exact = _exact(x, w, b, r, "silu", dy)
    for k, name in enumerate("xwb"):
        args = [t.to(DEV) for t in (x, w, b, r)]
        args[k].requires_grad_()
        (got,) = torch.autograd.grad(fused_linear(args[0], args[1], args[2], "silu", args[3]), [args[k]], dy.to(DEV))
        assert_within(name, got, *exact[1 + k])
    args = [t.to(DEV) for t in (x, w, b, r)]
    args[3].requires_grad_()
    (got,) = torch.autograd.grad(fused_linear(args[0], args[1], args[2], "silu", args[3]), [args[3]], dy.to(DEV))
    assert torch.equal(got.cpu(), dy)


def test_no_rows():
    x = torch.empty(3, 0, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(5, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    b = torch.ones(5, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = fused_linear(x, w, b, "relu")
    assert y.shape == (3, 0, 5)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and not dw.any() and not db.any()


def test_float64_takes_the_torch_path():
    x, w = torch.randn(4, 9, device=DEV, dtype=torch.float64), torch.randn(3, 9, device=DEV, dtype=torch.float64)
    assert (fused_linear(x, w, activation="relu") - (x @ w.t()).clamp(min=0)).abs().max() < 1e-12


@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid"])
def test_gradient_against_differences(act):
    x, w, b, r, dy = _inputs(30, 24, 17, torch.float32, seed=7)
    with precision("ieee"):
        leaves = [t.to(DEV).requires_grad_() for t in (x, w, b, r)]
        grads = torch.autograd.grad(fused_linear(leaves[0], leaves[1], leaves[2], act, leaves[3]), leaves, dy.to(DEV))
    point = [t.double() for t in (x, w, b, r)]
    for k in range(4):
        v = torch.randn(point[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)

        def f(t, k=k):
            a = point[:k] + [t] + point[k + 1:]
            return ((_act(a[0] @ a[1].t() + a[2], act)[0] + a[3]) * dy.double()).sum()

        want = directional(f, point[k], v)
        got = grads[k].double().cpu() * v
        # the difference is off by h^2 / 6 third derivatives, the gradient by some U of its terms
        assert abs(got.sum() - want) <= 1e-5 * got.abs().sum()


def test_second_derivative_raises():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    w = torch.randn(8, 32, device=DEV)
    (dx,) = torch.autograd.grad(fused_linear(x, w, None, "silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_offsets_beyond_32_bits():
    m, i, o = (1 << 23) + 77, 16, 520
    w = (torch.randn(o, i, generator=torch.Generator().manual_seed(8)) / 4).bfloat16()
    tail = torch.randn(200, i, generator=torch.Generator().manual_seed(9)).bfloat16()
    x = torch.zeros(m, i, device=DEV, dtype=torch.bfloat16)
    x[-200:] = tail.to(DEV)
    x.requires_grad_()
    y = fused_linear(x, w.to(DEV), None, "relu")
    assert y.numel() > 1 << 32
    dy = torch.zeros_like(y)
    dyt = torch.randn(200, o, generator=torch.Generator().manual_seed(10)).bfloat16()
    dy[-200:] = dyt.to(DEV)
    (dx,) = torch.autograd.grad(y, x, dy)
    exact = _exact(tail, w, None, None, "relu", dyt)
    assert not y[:-200].any() and not dx[:-200].any()
    assert_within("y", y[-200:].detach(), *exact[0])
    assert_within("dx", dx[-200:], *exact[1])


@pytest.mark.parametrize("m,i,o", [(1, 384, 1536), (700, 130, 200), (3000, 128, 512)])
def test_calls_repeat_bit_for_bit_and_replay_in_a_graph(m, i, o):
    x, w, b, r, dy = (t.to(DEV) for t in _inputs(m, i, o, torch.bfloat16, seed=11))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]

    def block():
        y = fused_linear(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
        return (y.detach(), *torch.autograd.grad(y, leaves[:3], dy))

    def equal(got, want, replay):
        assert torch.equal(got, want), replay

    replays_match(block, equal)


def test_operator_registration():
    import geometric_nn_ops_torch._ops  # noqa: F401

    x, w, b, r, _ = (t.to(DEV) for t in _inputs(6, 40, 24, torch.bfloat16, seed=12))
    torch.library.opcheck(torch.ops.gnn_amd.fused_linear_fwd.default, (x, w, b, "gelu", r),
                          test_utils=("test_schema", "test_faketensor"))
    with torch.no_grad():
        f = lambda t: fused_linear(t, w, b, "gelu", r)  # noqa: E731
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(x), f(x))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 24), (5, 7), (65, 63), (64, 130), (1000, 131)])
def test_rows_of_whole_chunks(rows, cols, dtype):
    from geometric_nn_ops_torch.triangle._kernels.fused_linear import _chunked

    base = torch.randn(2 * rows + 1, 2 * cols + 3, generator=torch.Generator().manual_seed(7)).to(DEV, dtype)
    turned = torch.randn(cols, rows, generator=torch.Generator().manual_seed(8)).to(DEV, dtype)
    views = [base[:rows, :cols].contiguous(), base[1:rows + 1, 1:cols + 1], base[:2 * rows:2, 0:2 * cols:2], turned.t(),
             base[:1, :cols].expand(rows, cols)]
    for t in views:
        got = _chunked(t)
        pitch = got.stride(0) if rows > 1 else got.shape[1]
        assert got.shape == (rows, -(-cols // 8) * 8) and got.data_ptr() % 16 == 0 and pitch * got.element_size() % 16 == 0
        assert torch.equal(got[:, :cols], t) and not got[:, cols:].any()


def test_chunked_rows_are_copied_only_where_they_must():
    base = torch.arange(4 * 64, dtype=torch.bfloat16, device=DEV).reshape(4, 64)
    from geometric_nn_ops_torch.triangle._kernels.fused_linear import _chunked

    for t, same in ((base, True), (base[:, 8:24], True), (base[:, 4:20], False), (base[:, :13], False),
                    (base.t()[:8, :2].t(), True), (base[:, ::4], False), (base[:1].expand(3, 64), False), (base[1:2, 16:24], True),
                    (torch.arange(66, dtype=torch.bfloat16, device=DEV)[2:].view(1, 64), False)):
        c = _chunked(t)
        assert torch.equal(c[:, :t.shape[1]], t) and not c[:, t.shape[1]:].any()
        assert c.shape[1] % 8 == 0 and c.stride(1) == 1 and c.stride(0) % 8 == 0 and c.data_ptr() % 16 == 0
        assert c.stride(0) >= c.shape[1]
        assert (c.data_ptr() == t.data_ptr()) == same


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("m,i,o", [(32770, 64, 4), (32768, 72, 13), (300, 64, 4), (40, 200, 13)])
def test_nothing_around_the_operands_is_read(m, i, o, act, dtype):
    """Weight, rows, bias and output gradient as parts of tensors that hold NaN everywhere else."""
    def within(t, columns):
        buf = torch.full((t.shape[0] + 40, t.shape[1] + (16 if columns else 0)), float("nan"), device=DEV, dtype=dtype)
        part = buf[16:16 + t.shape[0], 8:8 + t.shape[1]] if columns else buf[16:16 + t.shape[0]]
        part.copy_(t)
        return part

    x, w, b, _, dy = _inputs(m, i, o, dtype, residual=False, seed=11)
    plain = [x.to(DEV), w.to(DEV), b.to(DEV)]
    parts = [within(x, False), within(w, False), within(b[:, None], False)[:, 0]]
    results = []
    for leaves, d in ((plain, dy.to(DEV)), (parts, within(dy, True))):
        leaves = [t.requires_grad_() for t in leaves]
        y = fused_linear(*leaves, act)
        results.append((y, *torch.autograd.grad(y, leaves, d)))
    for name, a, e in zip(("y", "dx", "dw", "db"), results[1], results[0]):
        assert torch.equal(a, e), name


def test_operands_changed_in_place_before_the_backward():
    """Refused where the graph keeps the operand itself; a padded copy keeps the forward's values."""
    for i in (64, 61):
        x, w, b, _, dy = (None if t is None else t.to(DEV) for t in _inputs(50, i, 40, torch.bfloat16, residual=False))
        w.requires_grad_()
        want = torch.autograd.grad(fused_linear(x, w, b, "silu"), w, dy)[0]
        y = fused_linear(x, w, b, "silu")
        x.zero_()
        if i % 8 == 0:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, w, dy)
        else:
            assert torch.equal(torch.autograd.grad(y, w, dy)[0], want)


@pytest.mark.parametrize("i", [4, 8, 12, 16, 20, 28, 132, 260, 500])
@pytest.mark.parametrize("m,o", [(1, 1), (5, 40), (33, 24), (700, 200)])
@pytest.mark.parametrize("mode", ["ieee", "bf16x3"])
def test_full_precision_rows_of_whole_chunks(m, o, i, mode):
    """The C entry takes fp32 rows of any number of 16-byte chunks; NaN follows each row, and the last one."""
    from geometric_nn_ops_torch import _lib

    x, w, b, r, _ = _inputs(m, i, o, torch.float32, seed=i)
    bufs = []
    for t in (x, w):
        buf = torch.full((t.shape[0] + 2, i + 4), float("nan"), device=DEV)
        buf[:t.shape[0], :i] = t.to(DEV)
        bufs.append(buf)
    out, bd, rd = torch.empty(m, o, device=DEV), b.to(DEV), r.to(DEV)
    a = _lib.LinearArgs()
    a.x, a.w, a.bias, a.side, a.out = bufs[0].data_ptr(), bufs[1].data_ptr(), bd.data_ptr(), rd.data_ptr(), out.data_ptr()
    a.M, a.I, a.O, a.out_cols, a.x_ld, a.w_ld, a.side_ld, a.out_ld = m, i, o, o, i + 4, i + 4, o, o
    a.dtype, a.precision, a.activation = _lib.GNN_F32, _lib.PRECISION_CODE[mode], _lib_act("silu")
    _lib.call("gnn_linear", a, out.device)
    want, slack = _exact(x, w, b, r, "silu")[0]
    if mode == "bf16x3":
        # x in [2^e, 2^(e+1)) is hi + lo + rest: |x - hi| <= 2^(e-8), half a bf16 step, so that lo has an exponent of
        # e - 9 at most (or is exact) and |rest| <= 2^(e-17). A product loses both rests and lo lo:
        # (2^-17 + 2^-17 + 2^-16) |x w| = 2^-15 |x w|. One short sum can be off by all of that (the slope is below 1.2).
        slack = slack + 1.2 * 2.0 ** -15 * (x.double().abs() @ w.double().abs().t())
    assert_within(f"{m}x{i}->{o}", out, want, slack)


def _lib_act(name):
    from geometric_nn_ops_torch.triangle._kernels.fused_linear import ACTIVATION_CODE

    return ACTIVATION_CODE[name]


def _slopes(act, dtype, m, top):
    """``(got, exact)`` slopes at m x 8 points within ``top``: dx of a layer whose weight is the identity and whose output
    gradient is 1, where z is x and dx is dz, to the last bit."""
    x = torch.linspace(-top, top, 8 * m, dtype=torch.float64).to(dtype).view(m, 8).to(DEV).requires_grad_()
    w = torch.eye(8, dtype=dtype, device=DEV)
    (dx,) = torch.autograd.grad(fused_linear(x, w, None, act), x, torch.ones(m, 8, dtype=dtype, device=DEV))
    return x.detach().double(), dx


@pytest.mark.parametrize("m", [700, 33000])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_sigmoid_slope_far_out(dtype, m):
    """e / (1 + e)^2, e = exp(-|z|), keeps its digits where the sigmoid rounds to 1. The exponential's argument is off
    by 2 U |z| where it is scaled to base 2 first (its result by 2 U), the sum, the reciprocal and three products by
    2 U each at most; both roundings of the result (dz, dx) are of the same value."""
    with precision("ieee"):
        z, got = _slopes("sigmoid", dtype, m, 60.0)
    e = torch.exp(-z.abs())
    want = e / (1 + e) ** 2
    assert_within("slope", got, want, (2 * z.abs() + 16) * U * want)


@pytest.mark.parametrize("m", [700, 33000])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gelu_slope_far_out(dtype, m):
    """Phi(z) + z phi(z) to where it leaves bf16's range. 16-bit types: the fit is off by 4e-7 (it passes zero near
    z = -0.75), and from |z| = 2 on by less than 3.2e-4 of the value; fp32 and the exponential's argument, z^2 / 2,
    add (z^2 + 16) 4 U of both terms."""
    with precision("ieee"):
        z, got = _slopes("gelu", dtype, m, 13.0)
    # not torch.special.ndtr, which is (1 + erf) / 2 and has no digits left beyond z = -8
    cdf, pdf = torch.special.erfc(-z * 0.5 ** 0.5) / 2, torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    want = cdf + z * pdf
    slack = (z * z + 16) * 4 * U * (cdf + z.abs() * pdf)
    if dtype != torch.float32:
        slack = slack + 4e-7 * (z.abs() < 2) + 3.2e-4 * want.abs() * (z < -2) + 4e-7 * (z >= 2)
    assert_within("slope", got, want, slack)
