"""qk_norm_rotary on the GPU against the formulas in float64.

Bounds. A lane adds 16 squares at most and a team 32 lanes in 5 steps, so the mean is off by 24 U of itself and
1 / rms by 12 U and the 3 roundings behind it; with the products by 1 / rms and the weight a normed element is off by
20 U. A fraction of a turn rounds to fp32 by 2^-26 (half a step below 1/2), an angle of 1.6 U, and sine and cosine add
2 U: 4 U. An element of the result is then off by 32 U of |a| + |c| of its pair, and so is an output gradient turned
back (with 8 U); 1 / rms, xhat and the mean of g w xhat enter dx with 64 U of their absolute values together."""

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

from geometric_nn_ops_torch.triangle import qk_norm_rotary
from op_helpers import DTYPES, IDS, U, assert_within, directional, replays_match

pytestmark = pytest.mark.gpu
DEV = "cuda"
# batch, query and key tokens, query and key heads, head dim, rotary dim, neighbours paired
SHAPES = [(1, 1, 1, 1, 1, 8, 8, False), (2, 7, 7, 4, 2, 32, 32, False), (1, 5, 9, 3, 1, 80, 48, True),
          (3, 33, 33, 6, 2, 128, 128, False), (2, 3, 3, 16, 16, 256, 248, True), (1, 300, 300, 2, 2, 64, 0, False),
          (2, 17, 17, 5, 5, 72, 24, False), (8, 1, 1, 32, 8, 128, 128, False), (1, 2500, 3, 9, 1, 96, 96, True),
          (2, 700, 1, 24, 3, 16, 16, False), (1, 1300, 1300, 64, 8, 64, 32, False)]


def _sum_error(k):
    return min(k, 16 + 4 * k ** 0.5) * U


def _pairs(x, r, interleaved):
    return (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])


def _whole(a, c, x, r, interleaved):
    y = x.clone()
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = a, c
    else:
        y[..., :r // 2], y[..., r // 2:r] = a, c
    return y


def _exact(x, w, pos, freqs, interleaved, eps, dy=None):
    """(value, slack) of y and, with dy, of dx and dw."""
    r = 2 * len(freqs)
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    size = 1.0 if eps is None else (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * size
    n = xh * w
    if r:
        angle = pos.double()[:, :, None, None] * torch.tensor(freqs, dtype=torch.float64)
        c, s = angle.cos(), angle.sin()

    def turn(t, back):
        if not r:
            return t, t.abs()
        a, b = _pairs(t, r, interleaved)
        sb = -s if back else s
        both = a.abs() + b.abs()
        return (_whole(a * c - b * sb, b * c + a * sb, t, r, interleaved), _whole(both, both, t.abs(), r, interleaved))

    y, span = turn(n, False)
    out = [(y, 32 * U * span)]
    if dy is None:
        return out
    g, gspan = turn(dy.double(), True)
    if eps is None:
        return out + [(g, 8 * U * gspan), None]
    v, vspan = g * w, gspan * w.abs()
    m, mspan = (v * xh).mean(-1, keepdim=True), (vspan * xh.abs()).mean(-1, keepdim=True)
    out.append((size * (v - xh * m), 64 * U * size * (vspan + xh.abs() * mspan)))
    terms = gspan * xh.abs()
    out.append(((g * xh).sum((0, 1, 2)), (_sum_error(x.numel() // x.shape[-1]) + 40 * U) * terms.sum((0, 1, 2))))
    return out


def _inputs(b, u, v, h, hk, d, dtype, wdtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, dq, dk = (scale * torch.randn(b, n, m, d, generator=g) for n, m in ((u, h), (v, hk), (u, h), (v, hk)))
    q, k, dq, dk = (t.to(dtype) for t in (q, k, dq, dk))
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(wdtype) for _ in range(2))
    pos = [torch.randint(0, 5000, (b, n), generator=g) for n in (u, v)]
    return q, k, dq, dk, qw, kw, pos


def _run(shape, dtype, wdtype, seed=0, eps=1e-6, weights=True, scale=1.0, freqs=None):
    b, u, v, h, hk, d, r, interleaved = shape
    q, k, dq, dk, qw, kw, pos = _inputs(b, u, v, h, hk, d, dtype, wdtype, seed, scale)
    if not weights:
        qw = kw = None
    freqs = [10000.0 ** (-2 * j / r) for j in range(r // 2)] if freqs is None else freqs
    exact = [_exact(x, w, p, freqs, interleaved, eps, dy) for x, w, p, dy in ((q, qw, pos[0], dq), (k, kw, pos[1], dk))]
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, qw, kw) if t is not None]
    kw_args = dict(eps=eps, interleaved=interleaved)
    if weights:
        kw_args.update(q_weight=leaves[2], k_weight=leaves[3])
    if r:
        kw_args.update(q_pos=pos[0].to(DEV), k_pos=pos[1].int().to(DEV) if seed % 2 else pos[1].to(DEV), frequencies=freqs)
    got = qk_norm_rotary(leaves[0], leaves[1], **kw_args)
    grads = torch.autograd.grad(got, leaves, [dq.to(DEV), dk.to(DEV)])
    with torch.no_grad():
        for a, e in zip(qk_norm_rotary(leaves[0], leaves[1], **kw_args), got):
            assert torch.equal(a, e) and a.is_contiguous() and a.dtype == dtype
    for i, name in enumerate("qk"):
        assert_within(f"{name}' {shape}", got[i], *exact[i][0])
        assert_within(f"d{name} {shape}", grads[i], *exact[i][1])
        if weights:
            assert_within(f"d{name}_weight {shape}", grads[2 + i], *exact[i][2])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, dtype):
    _run(shape, dtype, dtype, seed=shape[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("eps,weights", [(1e-6, False), (None, False), (0.5, True)])
def test_norms(eps, weights, dtype):
    _run((2, 19, 19, 4, 2, 64, 64, False), dtype, torch.float32, eps=eps, weights=weights)
    _run((1, 50, 3, 4, 2, 40, 16, True), dtype, torch.float32, eps=eps, weights=weights)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_small_and_large_rows(dtype):
    _run((1, 9, 9, 3, 3, 128, 128, False), dtype, dtype, scale=2.0 ** -9)
    _run((1, 9, 9, 3, 3, 128, 128, False), dtype, dtype, scale=2.0 ** 9)


def test_far_positions_keep_their_angles():
    """Angles of 10^9 rad and more: in fp32 not a digit would be right."""
    d, far = 64, torch.tensor([[0, -5, 10 ** 6 + 1, 2 ** 31 - 1, 10 ** 9 + 7, 2 ** 40 + 1]])
    x = torch.randn(1, 6, 2, d, generator=torch.Generator().manual_seed(4))
    freqs = [10000.0 ** (-2 * j / d) for j in range(d // 2)]
    got = qk_norm_rotary(x.to(DEV), x.to(DEV), far.to(DEV), eps=None)[0]
    value, slack = _exact(x, None, far, freqs, False, None)[0]
    # the exact side's own angle, and the kernel's fraction of a turn, are off by 2^-52 of the angle
    span = slack / (32 * U)
    assert_within("far", got, value, slack + span * far.abs().double()[:, :, None, None] * 2.0 ** -51)


def test_views_are_read_in_place():
    g = torch.Generator().manual_seed(5)
    heads = torch.randn(2, 11, 12, 72, generator=g).bfloat16().to(DEV)
    pos = torch.arange(11, device=DEV)
    w = torch.randn(64, generator=g).to(DEV)
    q, k = heads[:, :, :8, 3:67], heads[:, :, 8:10, 8:]  # an odd address and an aligned one
    want = qk_norm_rotary(q.contiguous(), k.contiguous(), pos, q_weight=w, k_weight=w)
    for a, e in zip(qk_norm_rotary(q, k, pos, q_weight=w, k_weight=w), want):
        assert torch.equal(a, e)
    qt, kt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k))
    for a, e in zip(qk_norm_rotary(qt, kt, pos.expand(2, 11), q_weight=w, k_weight=w), want):
        assert torch.equal(a, e)
    turned = torch.empty(2, 11, 64, 8, device=DEV, dtype=torch.bfloat16).transpose(2, 3).copy_(q)  # no unit stride
    assert torch.equal(qk_norm_rotary(turned, k, pos, q_weight=w, k_weight=w)[0], want[0])

    def grads(q, k, dq, dk):
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        return torch.autograd.grad(qk_norm_rotary(*leaves, pos, q_weight=w), leaves, [dq, dk])

    dq, dk = torch.randn_like(want[0]), torch.randn_like(want[1])
    plain = grads(q.contiguous(), k.contiguous(), dq, dk)
    wide = torch.zeros(2, 11, 8, 130, device=DEV, dtype=torch.bfloat16)
    wide[..., 1:65] = dq
    for a, e in zip(grads(q, kt, wide[..., 1:65], dk), plain):
        assert torch.equal(a, e)
    for a, e in zip(grads(q, k, dq[:1, :1, :1, :1].expand_as(dq), dk),
                    grads(q, k, dq[:1, :1, :1, :1].expand_as(dq).contiguous(), dk)):
        assert torch.equal(a, e)


def test_unaligned_weights():
    q, k, _, _, qw, kw, pos = _inputs(1, 5, 5, 2, 2, 64, torch.float16, torch.float16)
    at = torch.zeros(65, device=DEV, dtype=torch.float16)
    at[1:] = qw.to(DEV)
    args = (q.to(DEV), k.to(DEV), pos[0].to(DEV))
    assert torch.equal(qk_norm_rotary(*args, q_weight=at[1:])[0], qk_norm_rotary(*args, q_weight=qw.to(DEV))[0])


def test_only_what_is_needed():
    shape = (2, 40, 40, 4, 2, 64)
    q, k, dq, dk, qw, kw, pos = (t.to(DEV) if torch.is_tensor(t) else t[0].to(DEV)
                                 for t in _inputs(*shape, torch.bfloat16, torch.bfloat16))

    def grads(names, use=(True, True)):
        leaves = {n: t.detach().clone().requires_grad_(n in names) for n, t in
                  (("q", q), ("k", k), ("qw", qw), ("kw", kw))}
        got = qk_norm_rotary(leaves["q"], leaves["k"], pos, q_weight=leaves["qw"], k_weight=leaves["kw"])
        outs = [(t, d) for t, d, n in zip(got, (dq, dk), use) if n]
        return dict(zip(names, torch.autograd.grad([t for t, _ in outs], [leaves[n] for n in names], [d for _, d in outs],
                                                   allow_unused=True)))

    every = grads(["q", "k", "qw", "kw"])
    for names in (["q"], ["k"], ["qw"], ["kw"], ["q", "kw"], ["qw", "kw"]):
        for n, t in grads(names).items():
            assert torch.equal(t, every[n]), (names, n)
    one = grads(["q", "k", "qw", "kw"], (True, False))  # the keys' output goes nowhere
    assert torch.equal(one["q"], every["q"]) and torch.equal(one["qw"], every["qw"])
    assert not one["k"].any() and not one["kw"].any()


def test_empty_sides():
    w = torch.ones(32, device=DEV, dtype=torch.float16, requires_grad=True)
    for b, u, v, h, hk in ((0, 3, 3, 2, 2), (2, 0, 4, 2, 2), (2, 4, 0, 2, 2), (2, 0, 0, 1, 1), (2, 3, 4, 0, 1)):
        q, k = (torch.randn(b, n, m, 32, device=DEV).half().requires_grad_() for n, m in ((u, h), (v, hk)))
        got = qk_norm_rotary(q, k, torch.arange(u, device=DEV), torch.arange(v, device=DEV), q_weight=w)
        assert got[0].shape == q.shape and got[1].shape == k.shape
        grads = torch.autograd.grad(got, [q, k, w], [torch.ones_like(t) for t in got])
        assert all(torch.isfinite(t).all() for t in grads)
        if not q.numel():
            assert not grads[2].any()


def test_other_dims_take_the_torch_path():
    for d, r in ((12, 12), (320, 64), (16, 12)):
        x = torch.randn(1, 3, 2, d, device=DEV)
        got = qk_norm_rotary(x, x, torch.arange(3, device=DEV), rotary_dim=r)
        want = qk_norm_rotary(x.cpu().double(), x.cpu().double(), torch.arange(3), rotary_dim=r)
        for a, e in zip(got, want):
            assert (a.cpu().double() - e).abs().max() < 1e-5


def test_gradient_against_differences():
    shape = (1, 6, 4, 3, 1, 40, 16, True)
    q, k, dq, dk, qw, kw, pos = _inputs(*shape[:6], torch.float32, torch.float32, seed=7)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, qw, kw)]
    kw_args = dict(rotary_dim=16, interleaved=True)
    got = qk_norm_rotary(leaves[0], leaves[1], pos[0].to(DEV), pos[1].to(DEV), q_weight=leaves[2], k_weight=leaves[3], **kw_args)
    grads = torch.autograd.grad(got, leaves, [dq.to(DEV), dk.to(DEV)])
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i)).double()

        def f(x, i=i):
            a = [x if j == i else t.detach().cpu().double() for j, t in enumerate(leaves)]
            out = qk_norm_rotary(a[0], a[1], *pos, q_weight=a[2], k_weight=a[3], **kw_args)
            return (out[0] * dq.double()).sum() + (out[1] * dk.double()).sum()

        want = directional(f, leaves[i].detach().cpu().double(), d)
        have = (grads[i].cpu().double() * d).sum()
        assert abs(have - want) <= 1e-4 * (grads[i].cpu().double().abs() * d.abs()).sum()


def test_captured_streams_and_hooks():
    q, k, dq, dk, qw, kw, pos = (t.to(DEV) if torch.is_tensor(t) else t[0].to(DEV)
                                 for t in _inputs(2, 130, 130, 8, 2, 64, torch.bfloat16, torch.bfloat16))
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]

    def train():
        got = qk_norm_rotary(leaves[0] * 1, leaves[1] * 1, pos, q_weight=leaves[2], k_weight=leaves[3])
        return [t.detach() for t in got] + list(torch.autograd.grad(got, leaves, [dq, dk]))

    want = train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = train()
    torch.cuda.current_stream().wait_stream(side)
    with saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t):
        hooked = train()
    for a, b, e in zip(other, hooked, want):
        assert torch.equal(a, e) and torch.equal(b, e)

    def block():
        with torch.no_grad():
            return qk_norm_rotary(q, k, pos, q_weight=qw, k_weight=kw)

    def same(a, e, replay):
        assert torch.equal(a, e), f"replay {replay}"

    replays_match(block, same)


def test_captured_backward():
    """Forward and backward in one graph, whose replays give the eager gradients."""
    q, k, dq, dk, qw, kw, pos = (t.to(DEV) if torch.is_tensor(t) else t[0].to(DEV)
                                 for t in _inputs(1, 77, 77, 4, 4, 128, torch.float16, torch.float16))

    def block():
        leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
        got = qk_norm_rotary(leaves[0], leaves[1], pos, q_weight=leaves[2], k_weight=leaves[3])
        return list(torch.autograd.grad(got, leaves, [dq, dk]))

    def same(a, e, replay):
        assert torch.equal(a, e), f"replay {replay}"

    replays_match(block, same)


def test_traced():
    q, k, _, _, qw, kw, pos = (t.to(DEV) if torch.is_tensor(t) else t[0].to(DEV)
                               for t in _inputs(1, 9, 9, 4, 2, 64, torch.bfloat16, torch.bfloat16))

    def f(q, k, pos, w):
        return qk_norm_rotary(q, k, pos, q_weight=w, rotary_dim=32)

    with torch.no_grad():
        for a, e in zip(torch.compile(f, fullgraph=True, backend="aot_eager")(q, k, pos, qw), f(q, k, pos, qw)):
            assert torch.equal(a, e)


def test_second_derivatives_raise():
    q, k, _, _, _, _, pos = _inputs(1, 3, 3, 2, 2, 32, torch.float32, torch.float32)
    q = q.to(DEV).requires_grad_()
    (g,) = torch.autograd.grad(qk_norm_rotary(q, k.to(DEV), pos[0].to(DEV))[0].square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_dual_tensors_take_the_torch_path():
    import torch.autograd.forward_ad as fwad

    q, k, dq, _, _, _, pos = _inputs(1, 3, 3, 2, 2, 32, torch.float32, torch.float32)
    q, k, dq, pos = q.to(DEV), k.to(DEV), dq.to(DEV), pos[0].to(DEV)
    with fwad.dual_level():
        out = fwad.unpack_dual(qk_norm_rotary(fwad.make_dual(q, dq), k, pos)[0]).tangent
    h = 1e-5
    ends = [qk_norm_rotary(q.cpu().double() + s * dq.cpu().double(), k.cpu().double(), pos.cpu())[0] for s in (h, -h)]
    assert ((ends[0] - ends[1]) / (2 * h) - out.cpu().double()).abs().max() < 1e-4
