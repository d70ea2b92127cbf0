"""gated_linear on the GPU against the formulas in float64.

Bounds. Each product's sum is off as fused_linear's is (``_sum_error`` of the terms' absolute values, 3 * 2^-18 of them
where fp32 operands are split) and the activation as its own; a product a b of two values that are off by ea and eb is
off by |a| eb + |b| ea + ea eb and a few U. dzg and dzu are rounded to the operands' type before the products behind
them: independent errors of at most half a step each, so that a sum over terms t is off by less than six deviations,
2 sqrt(3) half sqrt(sum t^2)."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import gated_linear
from op_helpers import DTYPES, IDS, U, assert_within, directional, half_step, replays_match
from test_fused_linear_gpu import ACTS, _act, _sum_error, precision

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(1, 1, 1), (1, 8, 8), (1, 384, 1536), (3, 7, 5), (17, 33, 65), (64, 128, 512), (129, 200, 131), (300, 64, 1),
          (5, 1, 300), (257, 512, 128), (2049, 131, 257), (40, 4100, 72), (700, 1024, 1000), (130, 72, 4100),
          (4000, 72, 520), (6000, 136, 1030)]


def _inputs(m, i, o, dtype, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, i, generator=g).to(dtype)
    wg, wu = ((torch.randn(o, i, generator=g) * i ** -0.5).to(dtype) for _ in range(2))
    bg, bu = ((0.3 * torch.randn(o, generator=g)).to(dtype) if bias else None for _ in range(2))
    return [x, wg, wu, bg, bu], torch.randn(m, o, generator=g).to(dtype)


def _exact(args, act, dy=None, split=False):
    """(value, slack) of y and, with dy, of dx, dwg, dwu, dbg, dbu."""
    dtype = args[0].dtype
    x, wg, wu, bg, bu = (None if t is None else t.double() for t in args)
    per = 3 * 2.0 ** -18 if split else 0.0

    def product(w, b):
        z, size = x @ w.t(), x.abs() @ w.abs().t()
        if b is not None:
            z, size = z + b, size + b.abs()
        return z, (_sum_error(x.shape[1]) + per) * size + 2 * U * z.abs()

    (zg, eg), (zu, eu) = product(wg, bg), product(wu, bu)
    a, slope, ea, es = _act(zg, act)
    ea = 1.2 * eg + ea + 2 * U * a.abs()
    y = a * zu
    out = [(y, a.abs() * eu + zu.abs() * ea + ea * eu + 4 * U * y.abs())]
    if dy is None:
        return out
    dy = dy.double()
    es = eg * (0 if act is None else 1) + es
    if act == "relu":
        es = (zg.abs() <= eg).double()
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    dg, du = dy * zu * slope, dy * a
    eg2 = dy.abs() * (zu.abs() * es + slope.abs() * eu + es * eu) + 6 * U * dg.abs() + tiny
    eu2 = dy.abs() * ea + 4 * U * du.abs() + tiny
    half = half_step(dtype) if dtype != torch.float32 else U
    six = 2 * 3 ** 0.5 * half

    def back(d, e, c, k, extra=0.0):
        return d @ c, (_sum_error(k) + extra) * (d.abs() @ c.abs()) + e @ c.abs(), d.square() @ c.square()

    o, m = wg.shape[0], x.shape[0]
    vg, lg, sg = back(dg, eg2, wg, 2 * o, per)
    vu, lu, su = back(du, eu2, wu, 2 * o, per)
    out.append((vg + vu, lg + lu + six * (sg + su).sqrt()))
    for d, e in ((dg, eg2), (du, eu2)):
        v, lost, sq = back(d.t(), e.t(), x, m)
        out.append((v, lost + six * sq.sqrt()))
    for d, e in ((dg, eg2), (du, eu2)):
        out.append((d.sum(0), _sum_error(m) * d.abs().sum(0) + e.sum(0) + six * d.square().sum(0).sqrt()))
    return out


NAMES = ("y", "dx", "dgate_weight", "dup_weight", "dgate_bias", "dup_bias")


def _run(m, i, o, dtype, act, bias, seed, split=False, device="cpu"):
    args, dy = _inputs(m, i, o, dtype, bias, seed)
    exact = _exact([None if t is None else t.to(device) for t in args], act, dy.to(device), split)
    leaves = [None if t is None else t.to(DEV).requires_grad_() for t in args]
    y = gated_linear(*leaves, act)
    assert y.dtype == dtype and y.is_contiguous() and y.shape == (m, o)
    used = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, used, dy.to(DEV))
    with torch.no_grad():
        assert torch.equal(gated_linear(*leaves, act), y)
    for name, got, (want, slack) in zip(NAMES, (y.detach(), *grads), exact):
        assert_within(f"{name} {m}x{i}->{o} {act}", got, want, slack)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,i,o", SHAPES)
def test_forward_and_gradients(m, i, o, dtype):
    with precision("ieee"):
        _run(m, i, o, dtype, ACTS[(m + i + o) % 5], (m + o) % 3 != 0, seed=m + i + o)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("m,i,o", [(32768, 128, 512), (32791, 40, 72), (40001, 256, 200), (33000, 512, 128),
                                   (36865, 64, 1024), (33001, 136, 264), (33000, 16, 8), (50001, 120, 300)])
def test_many_rows(m, i, o, dtype):
    """The pixels of a pair tensor."""
    _run(m, i, o, dtype, ACTS[(m + i + o) % 5], o % 3 == 0, seed=o, device=DEV)


@pytest.mark.parametrize("m,i,o", [(5000, 1000, 1032), (9000, 264, 2056)])
def test_large_tiles(m, i, o):
    _run(m, i, o, torch.bfloat16, "silu", True, seed=o, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
def test_every_activation(act, dtype):
    with precision("ieee"):
        for bias in (False, True):
            _run(193, 96, 160, dtype, act, bias, seed=3)


@pytest.mark.parametrize("act", ACTS)
def test_split_precision(act):
    """fp32 at 'tf32': the products of two bf16 parts, in the backward too."""
    with precision("tf32"):
        _run(150, 264, 136, torch.float32, act, True, seed=4, split=True)


def test_the_backward_keeps_the_forwards_precision():
    args, dy = _inputs(64, 128, 96, torch.float32)
    args = [t.to(DEV) for t in args]
    args[0].requires_grad_()
    with precision("ieee"):
        y = gated_linear(*args)
        (want,) = torch.autograd.grad(y, args[0], dy.to(DEV), retain_graph=True)
    with precision("tf32"):
        (got,) = torch.autograd.grad(y, args[0], dy.to(DEV))
    assert torch.equal(got, want)


def test_one_bias():
    args, dy = _inputs(40, 24, 30, torch.bfloat16)
    for k in (3, 4):
        used = [t if j != k else None for j, t in enumerate(args)]
        leaves = [None if t is None else t.to(DEV).requires_grad_() for t in used]
        y = gated_linear(*leaves)
        grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(DEV))
        exact = _exact(used, "silu", dy)
        del exact[1 + k]
        for got, (want, slack) in zip((y.detach(), *grads), exact):
            assert_within(str(k), got, want, slack)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
def test_what_is_not_finite_stays_in_its_place(act, dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 8, generator=g).to(dtype)
    x[2, 3] = float("nan")
    wg, wu = (torch.randn(10, 8, generator=g).to(dtype) for _ in range(2))
    b = torch.zeros(10).to(dtype)
    b[7] = float("inf")
    y = gated_linear(*(t.to(DEV) for t in (x, wg, wu)), None, b.to(DEV), act).cpu()
    assert y[2].isnan().all()
    keep, cols = [0, 1, 3, 4, 5], [0, 1, 2, 3, 4, 5, 6, 8, 9]
    assert y[keep][:, cols].isfinite().all() and not y[keep][:, 7].isfinite().all()


def test_far_gates():
    """Gates far out on both sides: zeros, ones or the input itself, and no overflow on the way."""
    for dtype in DTYPES:
        for act in ACTS:
            top = 200.0
            w = torch.eye(8).to(dtype)
            x = torch.tensor([[-top, -30.0, -8.0, -0.0, 0.0, 8.0, 30.0, top]]).to(dtype)
            y = gated_linear(x.to(DEV), w.to(DEV), torch.zeros_like(w).to(DEV), None, torch.ones(8, device=DEV, dtype=dtype), act)
            want, slack = _exact([x, w, 0 * w, None, torch.ones(8)], act)[0]
            assert_within(str(act), y.cpu(), want, slack + 1e-12)


def test_views():
    """Rows at odd offsets and pitches, halves of a stacked weight, transposed weights, expanded gradients."""
    g = torch.Generator().manual_seed(5)
    big = torch.randn(80, 300, generator=g).bfloat16().to(DEV)
    for x, wg, wu in ((big[:, 3:67], big[:20, 64:128], big[20:40, 64:128]), (big[:, 8:72], big[:30, 9:73], big[:30, 80:144]),
                      (big[:1, 8:72].expand(7, 64), big[:10, :64], big[10:20, :64]),
                      (big[:36, :16].t(), big[:12, 4:40], big[:36, :12].t()),
                      (big[:, :40].unflatten(0, (4, 20)).transpose(0, 1), big[:40, :17].t(), big[:40, 20:37].t())):
        m, o = x.numel() // x.shape[-1], wg.shape[0]
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        y = gated_linear(*leaves, activation="gelu")
        dyw = torch.randn(m, 2 * o, generator=g).bfloat16().to(DEV)
        for dy in (dyw[:, 1:1 + o].reshape(y.shape), dyw[0, 0].expand(y.shape)):
            got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            exact = _exact([x.detach().cpu().reshape(m, -1), wg.cpu(), wu.cpu(), None, None], "gelu", dy.cpu().reshape(m, o))
            for name, t, (want, slack) in zip(NAMES, (y.detach(), *got), exact):
                assert_within(name, t.reshape(want.shape), want, slack)


def test_only_the_gradients_asked_for():
    args, dy = _inputs(70, 41, 24, torch.float16, seed=6)
    leaves = [t.to(DEV).requires_grad_() for t in args]
    every = torch.autograd.grad(gated_linear(*leaves), leaves, dy.to(DEV))
    for k in range(5):
        some = [t.to(DEV) for t in args]
        some[k].requires_grad_()
        (got,) = torch.autograd.grad(gated_linear(*some), [some[k]], dy.to(DEV))
        assert torch.equal(got, every[k]), NAMES[1 + k]


def test_the_same_weight_twice():
    args, dy = _inputs(33, 40, 24, torch.float32, seed=6)
    x, w = args[0].to(DEV).requires_grad_(), args[1].to(DEV).requires_grad_()
    with precision("ieee"):
        dx, dw = torch.autograd.grad(gated_linear(x, w, w), [x, w], dy.to(DEV))
    exact = _exact([args[0], args[1], args[1], None, None], "silu", dy)
    assert_within("dx", dx, *exact[1])
    (a, ea), (b, eb) = exact[2:4]
    assert_within("dw", dw, a + b, ea + eb + U * (a.abs() + b.abs()))


def test_no_rows():
    x = torch.empty(3, 0, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w, b = (torch.ones(*s, device=DEV, dtype=torch.bfloat16, requires_grad=True) for s in ((5, 16), (5,)))
    y = gated_linear(x, w, w, b)
    assert y.shape == (3, 0, 5)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_float64_takes_the_torch_path():
    x, w = torch.randn(4, 9, device=DEV, dtype=torch.float64), torch.randn(3, 9, device=DEV, dtype=torch.float64)
    assert (gated_linear(x, w, w, activation="relu") - (x @ w.t()).clamp(min=0) * (x @ w.t())).abs().max() < 1e-12


@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid"])
def test_gradient_against_differences(act):
    args, dy = _inputs(30, 24, 17, torch.float32, seed=7)
    with precision("ieee"):
        leaves = [t.to(DEV).requires_grad_() for t in args]
        grads = torch.autograd.grad(gated_linear(*leaves, act), leaves, dy.to(DEV))
    point = [t.double() for t in args]
    for k in range(5):
        v = torch.randn(point[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)

        def f(t, k=k):
            a = point[:k] + [t] + point[k + 1:]
            return (_act(a[0] @ a[1].t() + a[3], act)[0] * (a[0] @ a[2].t() + a[4]) * dy.double()).sum()

        want = directional(f, point[k], v)
        got = grads[k].double().cpu() * v
        # the difference is off by h^2 / 6 third derivatives, the gradient by some U of its terms
        assert abs(got.sum() - want) <= 1e-5 * got.abs().sum()


def test_second_derivative_raises():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    w = torch.randn(8, 32, device=DEV)
    (dx,) = torch.autograd.grad(gated_linear(x, w, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_offsets_beyond_32_bits():
    m, i, o = (1 << 23) + 77, 16, 264
    g = torch.Generator().manual_seed(8)
    wg, wu = ((torch.randn(o, i, generator=g) / 4).bfloat16() for _ in range(2))
    tail, dyt = torch.randn(200, i, generator=g).bfloat16(), torch.randn(200, o, generator=g).bfloat16()
    x = torch.zeros(m, i, device=DEV, dtype=torch.bfloat16)
    x[-200:] = tail.to(DEV)
    x.requires_grad_()
    y = gated_linear(x, wg.to(DEV), wu.to(DEV))
    assert 2 * y.numel() > 1 << 32  # the gradients' rows
    dy = torch.zeros_like(y)
    dy[-200:] = dyt.to(DEV)
    (dx,) = torch.autograd.grad(y, x, dy)
    exact = _exact([tail, wg, wu, None, None], "silu", dyt)
    assert not y[:-200].any() and not dx[:-200].any()
    assert_within("y", y[-200:].detach(), *exact[0])
    assert_within("dx", dx[-200:], *exact[1])


def test_rows_and_columns_behind_stay_as_they_were():
    from geometric_nn_ops_torch import _lib

    for m, i, o in ((5, 64, 40), (700, 64, 200), (32773, 64, 40)):
        (x, wg, wu, _, _), _ = _inputs(m, i, o, torch.bfloat16, False)
        x, wg, wu = (t.to(DEV) for t in (x, wg, wu))
        out = torch.full((m + 300, o + 8), 7.0, device=DEV, dtype=torch.bfloat16)
        a = _lib.GatedLinearArgs()
        a.x, a.wg, a.wu, a.out = x.data_ptr(), wg.data_ptr(), wu.data_ptr(), out.data_ptr()
        a.M, a.I, a.O, a.out_cols, a.x_ld, a.wg_ld, a.wu_ld, a.out_ld = m, i, o, o, i, i, i, o + 8
        a.activation, a.dtype = 3, _lib.GNN_BF16
        _lib.call("gnn_gated_linear", a, x.device)
        assert_within("y", out[:m, :o], *_exact([x, wg, wu, None, None], "silu")[0])
        assert (out[m:] == 7).all() and (out[:, o:] == 7).all()


@pytest.mark.parametrize("m,i,o", [(1, 384, 1536), (700, 130, 200), (3000, 128, 512), (40000, 128, 264)])
def test_calls_repeat_bit_for_bit_and_replay_in_a_graph(m, i, o):
    args, dy = _inputs(m, i, o, torch.bfloat16, seed=11)
    args, dy = [t.to(DEV) for t in args], dy.to(DEV)

    def block():
        leaves = [t.detach().requires_grad_() for t in args]
        y = gated_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    def equal(got, want, replay):
        assert torch.equal(got, want), f"replay {replay}"

    replays_match(block, equal)


def test_another_stream_and_saved_tensor_hooks():
    from torch.autograd.graph import saved_tensors_hooks

    args, dy = _inputs(333, 72, 200, torch.float16, seed=12)
    leaves, dy = [t.to(DEV).requires_grad_() for t in args], dy.to(DEV)

    def train():
        y = gated_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    def shifted(t):
        return torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].copy_(t.reshape(-1)).view(t.shape)

    want = train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = train()
    torch.cuda.current_stream().wait_stream(side)
    with saved_tensors_hooks(shifted, lambda t: t):
        hooked = train()
    for a, b, e in zip(other, hooked, want):
        assert torch.equal(a, e) and torch.equal(b, e)


def test_traced_and_dual():
    import torch.autograd.forward_ad as fwad

    args, _ = _inputs(9, 16, 24, torch.bfloat16)
    args = [t.to(DEV) for t in args]
    with torch.no_grad():
        f = lambda *t: gated_linear(*t, activation="gelu")  # noqa: E731
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(*args), f(*args))
    x, wg, wu = (t.float() for t in args[:3])
    with fwad.dual_level():
        got = fwad.unpack_dual(gated_linear(fwad.make_dual(x, torch.ones_like(x)), wg, wu)).tangent
    xs = [x.cpu().double() + h for h in (1e-5, -1e-5)]
    ends = [gated_linear(t, wg.cpu().double(), wu.cpu().double()) for t in xs]
    assert ((ends[0] - ends[1]) / 2e-5 - got.cpu().double()).abs().max() < 1e-3
