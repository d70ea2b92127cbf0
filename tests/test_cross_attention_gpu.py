"""cross_attention on the GPU against the formulas in float64.

Bounds, with E(n) = ``_sum_error(n)``. A logit x is off by ex = E(D) sum |scale q k| and 4 U of |x|; a probability, whose
row's sum carries the same errors, by ep = ex + sum_k P ex + 8 U (1 + |x| + |lse|) of itself (the exponent's argument and
the base-2 exponential round once each). Then, linearly:
  o = sum P v:            sum P ep |v| + E(V) sum P |v|
  Delta = dO . o:         that of o times |dO|, E(D) sum |dO o|, and the output's own rounding
  dP = dO . v:            E(D) sum |dO v|
  dS = P (dP - Delta):    |dS| ep + P (errors of dP and Delta) + 4 U P (|dP| + |Delta|)
  dQ, dK, dV:             their terms' errors and E(n) of the sum of their absolute values
16-bit inputs round P and dS once as operands: independent errors of at most half a step each, so that a sum over terms
t is off by less than six deviations, 2 sqrt(3) half sqrt(sum t^2), and of 2^-25 each where fp16 values fall below its
normal range (P is held at 2^10 P there in dV, and in o against a row sum of at least 1). fp32 operands that are split
into two bf16 parts add 3 * 2^-18 of the products' absolute values."""

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

from geometric_nn_ops_torch.triangle import cross_attention, relative_position_bias
from op_helpers import DTYPES, IDS, U, assert_within, directional, half_step, replays_match
from test_fused_linear_gpu import precision

pytestmark = pytest.mark.gpu
DEV = "cuda"
# batch, queries, keys, heads, key heads, head dim, bias (0 none, 1 shared, 2 one a sequence), masked
SHAPES = [(1, 1, 1, 1, 1, 8, 0, False), (2, 1, 300, 8, 2, 64, 2, True), (1, 3, 7, 2, 1, 16, 1, False),
          (2, 5, 129, 4, 4, 32, 1, True), (1, 33, 64, 6, 3, 40, 0, True), (3, 70, 65, 2, 2, 96, 1, True),
          (2, 130, 131, 4, 1, 128, 2, True), (1, 200, 1000, 3, 3, 72, 0, True), (2, 257, 63, 8, 2, 48, 0, False),
          (4, 16, 2100, 8, 1, 128, 0, True), (1, 1, 5000, 4, 4, 128, 1, True), (1, 700, 333, 2, 2, 64, 2, False),
          (2, 9, 4500, 16, 4, 24, 0, True), (1, 2300, 40, 2, 1, 32, 1, False), (5, 129, 193, 2, 2, 32, 1, True)]


def _sum_error(k):
    return min(k, 16 + 4 * k ** 0.5) * U


def _inputs(shape, dtype, seed=0, scale=1.0):
    b, u, v, h, hk, d, bias, masked = shape
    g = torch.Generator().manual_seed(seed)
    q, k, val, dout = ((scale * torch.randn(*s, generator=g)).to(dtype).to(DEV)
                       for s in ((b, u, h, d), (b, v, hk, d), (b, v, hk, d), (b, u, h, d)))
    add = torch.randn(1 if bias == 1 else b, h, u, v, generator=g).to(dtype).to(DEV) if bias else None
    mask = None
    if masked:
        mask = torch.rand(b, v, generator=g) < 0.7
        mask[:, v - v // 5:] = False
        mask[:, 0] = True
        if b > 2:
            mask[1] = False
        mask = mask.to(DEV)
    return [q, k, val, add], mask, dout


def _exact(tensors, mask, dout=None, scale=None, split=False):
    """(value, slack) of the output and, with dout, of the gradients of q, k, v and the bias."""
    dtype, (B, Uq, H, D) = tensors[0].dtype, tensors[0].shape
    V, Hk = tensors[1].shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    half = half_step(dtype) if dtype != torch.float32 else 0.0
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    per = 3 * 2.0 ** -18 if split else 0.0
    six = 2 * 3 ** 0.5 * half

    def heads(t):  # [B, n, h, D] -> [B, H, n, D]
        t = t.double().transpose(1, 2)
        return t if t.shape[1] == H else t.repeat_interleave(G, 1)

    def own(t):  # [B, H, n, D] -> [B, n, Hk, D], summed over the heads that share a key head
        return t.reshape(B, Hk, G, -1, D).sum(2).transpose(1, 2)

    q, k, v = (heads(t) for t in tensors[:3])
    keep = torch.ones(B, V, dtype=torch.bool, device=DEV) if mask is None else mask
    k, v = (t.masked_fill(~keep[:, None, :, None], 0.0) for t in (k, v))
    kt, vt = k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous()
    x = q @ kt * scale
    ex = (_sum_error(D) + per) * scale * (q.abs() @ kt.abs())
    if tensors[3] is not None:
        x = x + tensors[3].double()
    x = x.masked_fill(~keep[:, None, None, :], float("-inf"))
    lse = torch.logsumexp(x, -1, keepdim=True)
    dead = lse == float("-inf")
    P = torch.exp(x - lse.masked_fill(dead, 0.0)).masked_fill(dead, 0.0)
    live = P > 0
    size = torch.where(live, x.abs(), 0.0)
    lsize = lse.abs().masked_fill(dead, 0.0)
    ex = torch.where(live, ex + 4 * U * size, 0.0)
    ep = ex + (P * ex).sum(-1, keepdim=True) + 8 * U * (1 + size + lsize)
    o = P @ v
    eo = (P * ep) @ v.abs() + (_sum_error(V) + per) * (P @ v.abs())
    half_o = six * (P.square() @ v.square()).sqrt() + tiny * v.abs().sum(2, keepdim=True)
    out = [(o.transpose(1, 2), (eo + half_o).transpose(1, 2))]
    if dout is None:
        return out
    do = heads(dout)
    dP = do @ vt
    delta = (do * o).sum(-1, keepdim=True)
    edp = (_sum_error(D) + per) * (do.abs() @ vt.abs())
    size_o = do.abs() * o.abs()
    edelta = (do.abs() * (eo + half_o)).sum(-1, keepdim=True) + _sum_error(D) * size_o.sum(-1, keepdim=True)
    edelta = edelta + 2 * 3 ** 0.5 * half_step(dtype) * size_o.square().sum(-1, keepdim=True).sqrt()
    dS = P * (dP - delta)
    eds = dS.abs() * ep + P * (edp + edelta) + 4 * U * P * (dP.abs() + delta.abs())
    dSt, Pt, edst, ept = (t.transpose(2, 3).contiguous() for t in (dS, P, eds, P * ep))

    def product(a, ea, c, n):
        return (a @ c, ea @ c.abs() + (_sum_error(n) + per) * (a.abs() @ c.abs()) + tiny * c.abs().sum(2, keepdim=True),
                six ** 2 * (a.square() @ c.square()))

    qv, qe, q2 = product(dS, eds, k, V)
    out.append(((scale * qv).transpose(1, 2), (scale * (qe + q2.sqrt())).transpose(1, 2)))
    kv, ke, k2 = product(dSt, edst, q, Uq * G)
    out.append((scale * own(kv), scale * (own(ke) + own(k2).sqrt())))
    vv, ve, v2 = product(Pt, ept, do, Uq * G)
    out.append((own(vv), own(ve) + own(v2).sqrt()))
    out = out[:2] + [(t.masked_fill(~keep[:, :, None, None], 0.0), s) for t, s in out[2:]]
    if tensors[3] is not None:
        if tensors[3].shape[0] == 1:
            dS, eds = dS.sum(0, keepdim=True), eds.sum(0, keepdim=True) + _sum_error(B) * dS.abs().sum(0, keepdim=True)
        out.append((dS, eds))
    return out


NAMES = ("o", "dq", "dk", "dv", "dbias")


def _run(shape, dtype, seed=0, scale=1.0, split=False, attn_scale=None):
    tensors, mask, dout = _inputs(shape, dtype, seed, scale)
    exact = _exact(tensors, mask, dout, attn_scale, split)
    leaves = [t.clone().requires_grad_() for t in tensors if t is not None]
    o = cross_attention(*leaves, *([] if len(leaves) == 4 else [None]), mask, attn_scale)
    assert o.dtype == dtype and o.is_contiguous()
    grads = torch.autograd.grad(o, leaves, dout)
    with torch.no_grad():
        assert torch.equal(cross_attention(*leaves, *([] if len(leaves) == 4 else [None]), mask, attn_scale), o)
    for name, got, (want, slack) in zip(NAMES, (o.detach(), *grads), exact):
        assert_within(f"{name} {shape}", got, want, slack)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, dtype):
    with precision("ieee"):
        _run(shape, dtype, seed=shape[2])


@pytest.mark.parametrize("shape", [(2, 5, 129, 4, 2, 64, 1, True), (1, 140, 200, 2, 2, 128, 0, False)], ids=str)
def test_split_precision(shape):
    with precision("tf32"):
        _run(shape, torch.float32, seed=1, split=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_peaked_and_flat_rows(dtype):
    """Logits of up to some hundred, whose maximum moves from tile to tile, and a scale that flattens them."""
    with precision("ieee"):
        _run((1, 70, 700, 2, 2, 64, 0, False), dtype, seed=2, scale=4.0)
        _run((1, 70, 700, 2, 1, 32, 1, True), dtype, seed=3, attn_scale=1e-3)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_that_rise(dtype):
    """Every tile's logits are above those of the tiles before, by more than the running maximum lets pass."""
    b, u, v, h, d = 1, 40, 600, 2, 32
    tensors, _, dout = _inputs((b, u, v, h, h, d, 2, False), dtype, seed=4)
    tensors[3] += (torch.arange(v, device=DEV) // 7 * 0.25).to(dtype)
    exact = _exact(tensors, None, dout)
    leaves = [t.requires_grad_() for t in tensors]
    with precision("ieee"):
        o = cross_attention(*leaves)
        grads = torch.autograd.grad(o, leaves, dout)
    for name, got, (want, slack) in zip(NAMES, (o.detach(), *grads), exact):
        assert_within(name, got, want, slack)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("u", [1, 40])
def test_masked_keys_have_no_effect(u, dtype):
    """NaN, infinities and the type's lowest value in masked keys, values and biases, and their zero gradients."""
    shape = (3, u, 333, 4, 2, 64, 2, True)
    tensors, mask, dout = _inputs(shape, dtype, seed=5)

    def run():
        leaves = [t.clone().requires_grad_() for t in tensors]
        o = cross_attention(*leaves, mask)
        return [o.detach(), *torch.autograd.grad(o, leaves, dout)]

    want = run()
    assert not want[0][1].any() and all(not t[1].any() for t in want[1:])
    for what in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
        tensors[1][~mask] = tensors[2][~mask] = what
        tensors[3].masked_fill_(~mask[:, None, None, :], what)
        for name, a, e in zip(NAMES, run(), want):
            assert torch.equal(a, e), (name, what)
    for t in want[2:4]:
        assert not t[~mask].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_biases_that_leave_nothing(dtype):
    """Rows whose bias is -inf everywhere give zeros; the lowest value is a logit like any other."""
    shape = (2, 37, 150, 2, 2, 32, 2, False)
    tensors, _, dout = _inputs(shape, dtype, seed=6)
    tensors[3][0, 1, 3] = float("-inf")
    tensors[3][1, 0, 5, :149] = float("-inf")
    leaves = [t.requires_grad_() for t in tensors]
    o = cross_attention(*leaves)
    grads = torch.autograd.grad(o, leaves, dout)
    assert not o[0, 3, 1].any() and not grads[0][0, 3, 1].any() and not grads[3][0, 1, 3].any()
    assert torch.equal(o[1, 5, 0], tensors[2][1, 149, 0])
    exact = _exact([t.detach() for t in tensors], None, dout)
    for name, got, (want, slack) in zip(NAMES, (o.detach(), *grads), exact):
        assert torch.isfinite(got).all()
        assert_within(name, got, want, slack)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("u", [5, 70])
def test_the_lowest_value_is_a_logit_like_any_other(u, dtype):
    """Beside the lowest value of a wide type the products vanish: all keys weigh the same, 1 / V, in both directions."""
    shape = (2, u, 150, 2, 2, 32, 1, False)
    tensors, _, dout = _inputs(shape, dtype, seed=17)
    tensors[3].fill_(torch.finfo(dtype).min)
    leaves = [t.requires_grad_() for t in tensors]
    o = cross_attention(*leaves)
    grads = torch.autograd.grad(o, leaves, dout)
    val, do = tensors[2].detach().double(), dout.double()
    mean = val.mean(1, keepdim=True)
    assert_within("o", o.detach(), mean.expand_as(o), _sum_error(150) * val.abs().mean(1, keepdim=True).expand_as(o))
    dv = do.sum(1, keepdim=True) / 150
    # 1 / 150 is rounded to the operands' type, the same way for all
    slack = (half_step(dtype) + 8 * U + _sum_error(u)) * do.abs().sum(1, keepdim=True) / 150
    assert_within("dv", grads[2], dv.expand_as(val), slack.expand_as(val))
    # dP - Delta, by keys and rows: Delta holds the output's rounding
    dp = torch.einsum("buhd,bvhd->bhuv", do, val - mean) / 150
    lost = torch.einsum("buhd,bvhd->bhuv", do.abs(), val.abs() + mean.abs()) / 150
    dbias = dp.sum(0, keepdim=True)
    assert_within("dbias", grads[3], dbias, (2 * half_step(dtype) + 64 * U) * lost.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("u", [1, 52])
@pytest.mark.parametrize("bias", [0, 1, 2])
def test_one_key(bias, u, dtype):
    """Its probability is 1 whatever its logit: the output is the value and the logits' gradients are zeros, exactly."""
    tensors, _, dout = _inputs((3, u, 1, 4, 2, 128, bias, False), dtype, seed=18, scale=3.0)
    mask = torch.tensor([[True], [False], [True]], device=DEV)
    for m in (None, mask):
        leaves = [t.clone().requires_grad_() for t in tensors if t is not None]
        o = cross_attention(*leaves, *([] if bias else [None]), m)
        grads = torch.autograd.grad(o, leaves, dout)
        keep = torch.ones(3, 1, 1, 1, device=DEV, dtype=dtype) if m is None else m[:, :, None, None].to(dtype)
        assert torch.equal(o, (tensors[2] * keep).repeat_interleave(2, 2).expand(3, u, 4, 128))
        assert not grads[0].any() and not grads[1].any() and (not bias or not grads[3].any())
        want = (dout.double() * keep.double()).view(3, u, 2, 2, 128)
        assert_within("dv", grads[2], want.sum((1, 3))[:, None], _sum_error(2 * u) * want.abs().sum((1, 3))[:, None])


def test_no_keys_no_queries():
    for b, u, v, h, hk in ((0, 3, 4, 2, 2), (2, 0, 4, 2, 1), (2, 3, 0, 2, 2), (1, 3, 4, 0, 1)):
        q, k, val = (torch.randn(b, n, m, 32, device=DEV).half().requires_grad_() for n, m in ((u, h), (v, hk), (v, hk)))
        bias = torch.randn(1, h, u, v, device=DEV).half().requires_grad_()
        o = cross_attention(q, k, val, bias)
        assert o.shape == q.shape and not o.any()
        for t, x in zip(torch.autograd.grad(o, [q, k, val, bias], torch.ones_like(o)), (q, k, val, bias)):
            assert t.shape == x.shape and not t.any()


def test_an_all_masked_batch():
    q, k, val = (torch.randn(2, n, 4, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True) for n in (70, 200, 200))
    mask = torch.zeros(2, 200, dtype=torch.bool, device=DEV)
    for u in (1, 70):
        o = cross_attention(q[:, :u], k, val, mask=mask)
        assert not o.any()
        for t in torch.autograd.grad(o, [q, k, val], torch.ones_like(o)):
            assert not t.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views_are_read_in_place(dtype):
    """Parts of a stacked projection, transposed heads, odd addresses, an expanded batch, a sliced mask and bias."""
    g = torch.Generator().manual_seed(7)
    b, u, v, h, hk, d = 2, 45, 77, 4, 2, 40
    kv = torch.randn(b, v, 2 * hk, d + 3, generator=g).to(dtype).to(DEV)
    k, val = kv[:, :, :hk, 1:1 + d], kv[:, :, hk:, 3:]
    q = torch.randn(b, h, u, d, generator=g).to(dtype).to(DEV).transpose(1, 2)
    bias = torch.randn(b, h, u, v + 9, generator=g).to(dtype).to(DEV)[..., 5:5 + v]
    mask = (torch.rand(b, 3 * v, generator=g) < 0.6).to(DEV)[:, ::3]

    def run(q, k, val, bias, mask, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, val, bias)]
        o = cross_attention(*leaves, mask)
        return [o.detach(), *torch.autograd.grad(o, leaves, dout)]

    dout = torch.randn(b, u, h, d + 1, generator=g).to(dtype).to(DEV)[..., 1:]
    plain = run(*(t.contiguous() for t in (q, k, val, bias, mask, dout)))
    for name, a, e in zip(NAMES, run(q, k, val, bias, mask, dout), plain):
        assert torch.equal(a, e), name
    turned = val.transpose(2, 3).contiguous().transpose(2, 3)  # no unit stride
    for a, e in zip(run(q, k, turned, bias.transpose(2, 3).contiguous().transpose(2, 3), mask, dout), plain):
        assert torch.equal(a, e)
    one = [t[:1].expand(2, *t.shape[1:]) for t in (q, k, val)]
    for a, e in zip(run(*one, bias, mask[:1].expand(2, v), dout[:1, :1].expand_as(dout)),
                    run(*(t.contiguous() for t in one), bias, mask[:1].expand(2, v).contiguous(),
                        dout[:1, :1].expand_as(dout).contiguous())):
        assert torch.equal(a, e)
    # an expanded bias has a gradient for every sequence, a shared one their sum
    every = run(q, k, val, bias[:1].expand(b, h, u, v), mask, dout)
    shared = run(q, k, val, bias[:1], mask, dout)
    assert every[4].shape == (b, h, u, v) and shared[4].shape == (1, h, u, v)
    off = (shared[4].double() - every[4].double().sum(0, keepdim=True)).abs()
    assert (off <= 3 * half_step(dtype) * every[4].double().abs().sum(0, keepdim=True) + 1e-6).all()


def test_only_what_is_needed():
    tensors, mask, dout = _inputs((2, 50, 90, 4, 2, 64, 1, True), torch.bfloat16, seed=8)
    leaves = [t.clone().requires_grad_() for t in tensors]
    every = torch.autograd.grad(cross_attention(*leaves, mask), leaves, dout)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate(tensors)]
        (got,) = torch.autograd.grad(cross_attention(*some, mask), [some[i]], dout)
        assert torch.equal(got, every[i]), NAMES[1 + i]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_small_gradients(dtype):
    """A row spread over many keys, and a small output gradient: fp16 operands keep their digits."""
    tensors, mask, dout = _inputs((1, 64, 6000, 1, 1, 32, 0, False), dtype, seed=9)
    dout = (dout * 2.0 ** -6).to(dtype)
    exact = _exact(tensors, mask, dout, 0.01)
    leaves = [t.clone().requires_grad_() for t in tensors[:3]]
    with precision("ieee"):
        o = cross_attention(*leaves, scale=0.01)
        grads = torch.autograd.grad(o, leaves, dout)
    for name, got, (want, slack) in zip(NAMES, (o.detach(), *grads), exact):
        assert_within(name, got, want, slack)
    dv, want = grads[2].double(), exact[3][0]
    # dv's elements lie around 1e-5, below fp16's normal range (2^-14), where storing one is off by up to half of its
    # smallest step whatever its size: 2^-25, and 2^-25 sqrt(n) in norm
    stored = 2.0 ** -25 * dv.numel() ** 0.5 if dtype == torch.float16 else 0.0
    assert (dv - want).norm() <= 2 * half_step(dtype) * want.norm() + 64 * U * want.norm() + stored


def test_relative_position_bias_of_decoded_queries():
    """The learned bias of a few new queries against the keys so far, read without a copy."""
    b, u, v, h, d = 2, 3, 517, 4, 64
    tensors, mask, dout = _inputs((b, u, v, h, 2, d, 0, True), torch.bfloat16, seed=10)
    table = torch.randn(32, h, device=DEV).bfloat16().requires_grad_()
    key_pos = torch.arange(v, device=DEV).expand(b, v)
    bias = relative_position_bias(table, key_pos[:, -u:], key_pos, max_distance=128, bidirectional=False)
    assert bias.stride(2) != v
    got = cross_attention(*tensors[:3], bias, mask)
    want = cross_attention(*tensors[:3], bias.contiguous(), mask)
    assert torch.equal(got, want)
    (dtable,) = torch.autograd.grad(got, table, dout)
    assert torch.isfinite(dtable).all() and dtable.any()
    exact = _exact([*tensors[:3], bias.detach()], mask)
    assert_within("o", got.detach(), *exact[0])


def test_float64_and_other_head_dims_take_the_torch_path():
    for dtype, d in ((torch.float64, 16), (torch.float32, 12), (torch.bfloat16, 136)):
        q, k = torch.randn(1, 3, 2, d, device=DEV).to(dtype), torch.randn(1, 5, 2, d, device=DEV).to(dtype)
        want = cross_attention(q.cpu().double(), k.cpu().double(), k.cpu().double())
        assert (cross_attention(q, k, k).cpu().double() - want).abs().max() < 0.02


def test_gradient_against_differences():
    tensors, mask, dout = _inputs((2, 6, 9, 4, 2, 16, 1, True), torch.float32, seed=11)
    leaves = [t.requires_grad_() for t in tensors]
    with precision("ieee"):
        grads = torch.autograd.grad(cross_attention(*leaves, mask), leaves, dout)
    point = [t.detach().cpu().double() for t in tensors]
    for k in range(4):
        v = torch.randn(point[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)

        def f(t, k=k):
            a = point[:k] + [t] + point[k + 1:]
            return (cross_attention(*a, mask.cpu()) * dout.cpu().double()).sum()

        want = directional(f, point[k], v)
        got = grads[k].double().cpu() * v
        # the difference is off by h^2 / 6 third derivatives, the gradient by some U of its terms
        assert abs(got.sum() - want) <= 1e-5 * got.abs().sum()


def test_second_derivative_raises():
    q = torch.randn(1, 4, 2, 32, device=DEV, requires_grad=True)
    k = torch.randn(1, 5, 2, 32, device=DEV)
    (dq,) = torch.autograd.grad(cross_attention(q, k, k).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), q)


@pytest.mark.parametrize("u,v,bias", [(1, 3000, 0), (90, 200, 1), (300, 65, 2)])
def test_calls_repeat_and_replay_in_a_graph(u, v, bias):
    tensors, mask, dout = _inputs((2, u, v, 4, 2, 64, bias, True), torch.bfloat16, seed=12)

    def block():
        leaves = [t.detach().requires_grad_() for t in tensors if t is not None]
        o = cross_attention(*leaves, *([] if len(leaves) == 4 else [None]), mask)
        return (o.detach(), *torch.autograd.grad(o, leaves, dout))

    def equal(got, want, replay):
        assert torch.equal(got, want), f"replay {replay}"

    replays_match(block, equal)


def test_another_stream_hooks_and_checkpoints():
    tensors, mask, dout = _inputs((2, 77, 150, 4, 2, 64, 1, True), torch.float16, seed=13)
    leaves = [t.requires_grad_() for t in tensors]

    def train(f=lambda *t: cross_attention(*t, mask)):
        o = f(*leaves)
        return (o.detach(), *torch.autograd.grad(o, leaves, dout))

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
    again = train(lambda *t: checkpoint(lambda *s: cross_attention(*s, mask), *t, use_reentrant=False))
    for a, b, c, e in zip(other, hooked, again, want):
        assert torch.equal(a, e) and torch.equal(b, e) and torch.equal(c, e)


def test_traced_and_dual():
    import torch.autograd.forward_ad as fwad

    tensors, mask, dout = _inputs((2, 7, 30, 4, 2, 32, 1, True), torch.bfloat16, seed=14)
    with torch.no_grad():
        f = lambda *t: cross_attention(*t, mask)  # noqa: E731
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(*tensors), f(*tensors))
    q, k, v = (t.float() for t in tensors[:3])
    with fwad.dual_level():
        got = fwad.unpack_dual(cross_attention(fwad.make_dual(q, dout.float()), k, v)).tangent
    ends = [cross_attention(q.cpu().double() + h * dout.cpu().double(), k.cpu().double(), v.cpu().double())
            for h in (1e-5, -1e-5)]
    assert ((ends[0] - ends[1]) / 2e-5 - got.cpu().double()).abs().max() < 1e-3


def test_offsets_beyond_32_bits():
    """Keys and values of more than 2^32 elements between their first and last row: the last ones count."""
    b, v, hk, d = 1, (1 << 21) + 70, 16, 128
    k = torch.zeros(b, v, hk, d, device=DEV, dtype=torch.bfloat16)
    assert k.numel() > 1 << 32
    g = torch.Generator().manual_seed(15)
    tail = torch.randn(b, 100, hk, d, generator=g).bfloat16().to(DEV)
    k[:, -100:] = tail
    mask = torch.zeros(b, v, dtype=torch.bool, device=DEV)
    mask[:, -100:] = True
    q = torch.randn(b, 3, hk, d, generator=g).bfloat16().to(DEV)
    want = cross_attention(q, tail, tail)
    got = cross_attention(q, k, k, mask=mask)
    assert (got.double() - want.double()).norm() <= 2 * half_step(torch.bfloat16) * want.double().norm()


def test_rows_behind_the_output_stay_as_they_were():
    from geometric_nn_ops_torch import _lib

    for u, v in ((1, 40), (37, 100), (130, 70)):
        (q, k, val, _), _, _ = _inputs((2, u, v, 4, 2, 64, 0, False), torch.bfloat16, seed=16)
        buf = torch.full((q.numel() + 4096,), 7.0, device=DEV, dtype=torch.bfloat16)
        a = _lib.CrossAttnArgs()
        a.q, a.k, a.v, a.o = q.data_ptr(), k.data_ptr(), val.data_ptr(), buf.data_ptr()
        a.B, a.U, a.V, a.H, a.Hk, a.D, a.scale, a.dtype = 2, u, v, 4, 2, 64, 0.125, _lib.GNN_BF16
        for name, t in (("q", q), ("k", k), ("v", val)):
            setattr(a, name + "_stride", _lib.I64x3(*t.stride()[:3]))
        _lib.call("gnn_cross_attn_fwd", a, q.device)
        assert torch.equal(buf[:q.numel()].view_as(q), cross_attention(q, k, val, scale=0.125))
        assert (buf[q.numel():] == 7).all()


@pytest.mark.parametrize("v", [2, 5, 33, 64])
@pytest.mark.parametrize("masked", [False, True])
def test_few_keys_lose_no_bits(v, masked):
    """With up to 64 keys P (dP - Delta) is a small difference, whose terms are held to 2^-16 (two parts of 8 bits):
    P and dS as operands, and o in Delta, which P's two parts enter as well. fp32 arithmetic, E(D) U at most, is below
    another 2^-16. Three roundings of operands to one part would be off by 2^-8 each."""
    B, Uq, H, D = 2, 37, 4, 64
    (q, k, val, _), _, dout = _inputs((B, Uq, v, H, 2, D, 0, False), torch.bfloat16, seed=v)
    mask = None
    if masked:
        mask = torch.ones(B, v, dtype=torch.bool, device=DEV)
        mask[0, 1:] = False  # one key: no gradient
        mask[1, v // 2] = False
    leaves = [t.clone().requires_grad_() for t in (q, k, val)]
    got = torch.autograd.grad(cross_attention(*leaves, mask=mask), leaves, dout)

    q, k, val, dout = (t.double().transpose(1, 2) for t in (q, k, val, dout))
    k, val = (t.repeat_interleave(H // 2, 1) for t in (k, val))
    x = q @ k.transpose(2, 3).contiguous() * D ** -0.5
    keep = torch.ones(B, v, dtype=torch.bool, device=DEV) if mask is None else mask
    p = torch.softmax(x.masked_fill(~keep[:, None, None], float("-inf")), -1)
    dp = dout @ val.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    most = (dout.abs() * (p @ val.abs())).sum(-1, keepdim=True)
    slack = 2.0 ** -15 * (ds.abs() + p * (dp.abs() + 2 * most)) * D ** -0.5
    assert_within("dq", got[0].transpose(1, 2), ds @ k * D ** -0.5, slack @ k.abs())
    if masked:
        assert (got[0][0].double().abs() <= (slack @ k.abs())[0].transpose(0, 1)).all()
