"""cross_attention where little is left of a row: one key under a bias, infinities and NaN, gradients far from one.

Bounds of gradients' digits, in the norm of a row's D elements. Storing one is off by half a step of it, or of fp16's
smallest. The operands dS are off by half a step each, independently: by half / sqrt(3) sqrt(sum dS^2 k^2) in the
mean over the row, of which sqrt(3) times is 6 deviations away for 32 elements on. Delta is off by what p's rounding leaves
in o: one number a row, six deviations are 2 sqrt(3) half sqrt(sum_d dO^2 sum_j p^2 v^2). fp32 arithmetic is off by some U of
the terms, below 2^-16 of them."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import cross_attention
from op_helpers import DTYPES, IDS, U, assert_within, half_step
from test_cross_attention_gpu import NAMES, _exact, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def _train(tensors, mask, dout, scale=None):
    """The output and the gradients of q, k, v and, where there is one, the bias."""
    leaves = [t.detach().clone().requires_grad_() for t in tensors if t is not None]
    o = cross_attention(*leaves, *([] if len(leaves) == 4 else [None]), mask, scale)
    return [o.detach(), *torch.autograd.grad(o, leaves, dout)]


def _torch_path(tensors, mask, dout):
    wide = [None if t is None else t.cpu().double() for t in tensors]
    return _train(wide, None if mask is None else mask.cpu(), dout.cpu().double())


# ---- one key
def _one_key(u, bias, dtype, masked):
    """Three sequences of one key, and the gradients that stock torch has in float64."""
    tensors, _, dout = _inputs((3, u, 1, 4, 2, 128, bias, False), dtype, seed=40)
    mask = torch.tensor([[True], [False], [True]], device=DEV) if masked else None
    return tensors, mask, dout


def _same(got, want, dtype, sums):
    """NaN where stock torch has it. o holds one value or none and dq, dk, dbias are zeros: equal; dv adds ``sums``
    output gradients, each below 6, in fp32."""
    for name, a, e in zip(NAMES, got, want):
        a = a.cpu()
        assert torch.equal(a.isnan(), e.isnan()), name
        a, e = a.double().nan_to_num(nan=0.0), e.nan_to_num(nan=0.0)
        if name != "dv":
            assert torch.equal(a, e), name
        else:
            assert_within(name, a.to(dtype), e, min(sums, 16 + 4 * sums ** 0.5) * U * 6 * sums * torch.ones_like(e))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("u", [1, 52])
@pytest.mark.parametrize("bias", [1, 2])
def test_one_key_that_a_bias_takes_away(bias, u, masked, dtype):
    """A bias of -inf leaves its query nothing: zeros, and nothing of its output gradient in dv."""
    tensors, mask, dout = _one_key(u, bias, dtype, masked)
    tensors[3][:, 1, ::3] = -INF
    got = _train(tensors, mask, dout)
    assert not got[0][:, ::3, 1].any() and got[0][0, :, 0].any()
    _same(got, _torch_path(tensors, mask, dout), dtype, 2 * u)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("u", [1, 52])
@pytest.mark.parametrize("bias", [1, 2])
@pytest.mark.parametrize("what", [INF, NAN])
def test_one_key_whose_bias_is_no_number(what, bias, u, dtype):
    tensors, mask, dout = _one_key(u, bias, dtype, True)
    tensors[3][0, 2, u // 2, 0] = what
    got = _train(tensors, mask, dout)
    assert got[0][0, u // 2, 2].isnan().all() and not got[0][0, u // 2, 0].isnan().any()
    _same(got, _torch_path(tensors, mask, dout), dtype, 2 * u)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("bias", [0, 1, 2])
def test_one_key_and_a_query_that_is_no_number(bias, dtype):
    tensors, mask, dout = _one_key(52, bias, dtype, True)
    tensors[0][2, 7, 3, 5] = NAN
    got = _train(tensors, mask, dout)
    assert got[0][2, 7, 3].isnan().all() and not got[0][2, 7, 2].isnan().any()
    _same(got, _torch_path(tensors, mask, dout), dtype, 104)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("bias", [0, 2])
def test_one_key_of_a_large_logit(bias, dtype):
    """The weight is an exact 1 beside logits of some thousand."""
    tensors, _, dout = _inputs((3, 52, 1, 4, 2, 128, bias, False), dtype, seed=41, scale=30.0)
    o = cross_attention(*tensors)
    assert torch.equal(o, tensors[2].repeat_interleave(2, 2).expand_as(o))
    _same(_train(tensors, None, dout / 30), _torch_path(tensors, None, dout / 30), dtype, 104)


# ---- output gradients that are no numbers
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("what", [INF, NAN])
@pytest.mark.parametrize("shape", [(3, 70, 333, 4, 2, 64, 1, True), (2, 5, 200, 4, 2, 128, 2, True),
                                   (1, 2300, 40, 4, 2, 32, 0, True), (2, 300, 90, 4, 2, 96, 0, True)], ids=str)
def test_an_infinite_output_gradient_stays_with_the_kept_keys(shape, what, dtype):
    """It reaches every kept key of its key head, and no masked one."""
    tensors, mask, dout = _inputs(shape, dtype, seed=42)
    plain = _train(tensors, mask, dout)
    dout[0, 3, 2, 7] = what
    got = _train(tensors, mask, dout)
    for t in got[2:4]:
        assert not t[~mask].any() and not t[0, mask[0], 1].isfinite().all(-1).any()
    if shape[6]:
        kept = mask.any(0, keepdim=True) if shape[6] == 1 else mask  # of a shared bias: by some sequence
        assert not got[4].masked_fill(kept[:, None, None].expand_as(got[4]), 0.0).any()
    for a, e in zip(got[2:4], plain[2:4]):
        assert torch.equal(a[0, :, 0], e[0, :, 0]) and torch.equal(a[1:], e[1:])
    got[1][0, 3, 2] = plain[1][0, 3, 2]
    assert torch.equal(got[1], plain[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("what", [INF, NAN])
@pytest.mark.parametrize("shape", [(2, 70, 333, 4, 2, 64, 1, False), (2, 5, 200, 4, 2, 128, 2, True),
                                   (1, 40, 5000, 2, 1, 32, 2, False), (2, 33, 1, 4, 2, 64, 1, False)], ids=str)
def test_rows_without_keys_have_no_gradient(shape, what, dtype):
    """Whatever their output gradient holds: zeros in dq and dbias, as stock torch has them."""
    tensors, mask, dout = _inputs(shape, dtype, seed=43)
    tensors[3][:, 1, 2:5] = -INF
    plain = _train(tensors, mask, dout)
    dout[:, 2:5, 1] = what
    got = _train(tensors, mask, dout)
    for i in (0, 1, 4):
        assert torch.equal(got[i], plain[i]), NAMES[i]
    assert not got[1][:, 2:5, 1].any() and not got[4][:, 1, 2:5].any()


# ---- gradients far from one
def _digits(tensors, mask, dout, dtype):
    """((value, bound of a row's error), ...) of dq and dk in float64."""
    (B, Uq, H, D), Hk = tensors[0].shape, tensors[1].shape[2]
    half, scale = half_step(dtype), D ** -0.5
    q, k, v, do = (t.double().transpose(1, 2) for t in (*tensors[:3], dout))
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    x = q @ k.transpose(2, 3).contiguous() * scale
    if tensors[3] is not None:
        x = x + tensors[3].double()
    if mask is not None:
        x = x.masked_fill(~mask[:, None, None], -INF)
    P = torch.softmax(x, -1)
    dP = do @ v.transpose(2, 3).contiguous()
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    delta = 2 * 3 ** 0.5 * half * (do.square() * (P.square() @ v.square())).sum(-1, keepdim=True).sqrt()
    dSt, Pt = (t.transpose(2, 3).contiguous() for t in (dS, P))

    def own(t):  # summed over the heads that share a key head
        return t.reshape(B, Hk, H // Hk, -1, D).sum(2)

    def bound(value, spread, by_delta):
        stored = half * value.norm(dim=-1) + (2.0 ** -25 * D ** 0.5 if dtype == torch.float16 else 0.0)
        return stored + scale * ((half + 2.0 ** -16) * spread.sum(-1).sqrt() + by_delta)

    dq, dk = scale * dS @ k, scale * own(dSt @ q)
    return ((dq.transpose(1, 2), bound(dq, dS.square() @ k.square(), (delta * (P @ k)).norm(dim=-1)).transpose(1, 2)),
            (dk.transpose(1, 2), bound(dk, own(dSt.square() @ q.square()),
                                       own((Pt.square() @ (delta * q).square())).sum(-1).sqrt()).transpose(1, 2)))


def _hold_digits(tensors, mask, dout, dtype):
    got = _train(tensors, mask, dout)
    for name, a, (want, bound) in zip(("dq", "dk"), got[1:3], _digits(tensors, mask, dout, dtype)):
        off = (a.double() - want).norm(dim=-1)
        assert (off <= bound).all(), (name, (off / bound).max().item())
    return got


LONG = [(1, 256, 16384, 2, 1, 64, 0, False), (1, 200, 8000, 2, 2, 128, 0, True), (2, 130, 6000, 2, 2, 64, 2, False),
        (2, 130, 6000, 2, 1, 32, 1, False), (1, 64, 5000, 4, 2, 96, 0, True), (1, 150, 4000, 2, 2, 128, 2, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", [8, 10])
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_rows_of_small_gradients_keep_their_digits(shape, size, dtype):
    tensors, mask, dout = _inputs(shape, dtype, seed=44)
    dout = dout * 2.0 ** -size
    got = _hold_digits(tensors, mask, dout, dtype)
    if shape[6]:
        assert_within("dbias", got[4], *_exact(tensors, mask, dout)[4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_each_row_keeps_its_digits(dtype):
    """Output gradients of sizes from row to row apart, an all-masked sequence and a row of zeros among them."""
    tensors, mask, dout = _inputs((3, 140, 3000, 4, 2, 64, 0, True), dtype, seed=45)
    dout *= (2.0 ** -(torch.arange(140, device=DEV) % 11 - 2.0)).to(dtype)[None, :, None, None]
    dout[0, 17] = 0.0
    mask[1] = mask[0]
    _hold_digits(tensors, mask, dout, dtype)
    mask[1] = False
    got = _train(tensors, mask, dout)
    assert all(torch.isfinite(t).all() for t in got) and not got[1][0, 17].any()
    assert not any(t[1].any() for t in got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
def test_large_gradients_stay_finite(d, dtype):
    """dS beyond fp16's 65504, with queries and keys so small that dq and dk are not."""
    tensors, mask, dout = _inputs((2, 200, 70, 4, 2, d, 0, True), dtype, seed=46)
    tensors[0] *= 2.0 ** -6
    tensors[1] *= 2.0 ** -8
    tensors[2] *= 2.0 ** 7
    dout = dout * 2.0 ** 10
    got = _hold_digits(tensors, mask, dout, dtype)
    assert all(torch.isfinite(t).all() for t in got)


def test_heads_far_apart():
    """Two query heads a key head, more than 1 GiB between them: read in place."""
    tensors, mask, dout = _inputs((1, 130, 200, 2, 1, 64, 0, True), torch.bfloat16, seed=47)
    want = _train(tensors, mask, dout)
    apart = (1 << 29) + 4096  # elements
    q = torch.empty(apart + 130 * 64, device=DEV, dtype=torch.bfloat16).as_strided((1, 130, 2, 64), (apart, 64, apart, 1))
    q.copy_(tensors[0])
    q.requires_grad_()
    o = cross_attention(q, *tensors[1:3], None, mask)
    assert torch.equal(o, want[0])
    (dq,) = torch.autograd.grad(o, q, dout)
    assert torch.equal(dq, want[1])


# ---- single queries
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(2, 1, 100, 8, 2, 64, 0, False), (1, 3, 700, 4, 4, 128, 1, True), (3, 8, 200, 4, 1, 32, 2, True),
                                   (1, 1, 9000, 2, 2, 96, 0, True)], ids=str)
def test_single_queries_round_once(shape, dtype):
    """Up to 32 rows a key head p is multiplied in two parts, 2^-16 exact, or in fp16 by half of its smallest step
    against a row sum of at least 1. A logit is off by E(D) = 48 U at most of its terms' absolute values, some 10 here, and
    its probability by twice that: below 2^-13 of itself."""
    tensors, mask, _ = _inputs(shape, dtype, seed=48)
    (B, _, H, D), Hk = tensors[0].shape, tensors[1].shape[2]
    q, k, v = (t.double().transpose(1, 2) for t in tensors[:3])
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    x = q @ k.transpose(2, 3).contiguous() * D ** -0.5
    if tensors[3] is not None:
        x = x + tensors[3].double()
    if mask is not None:
        if B > 2:
            mask[1] = mask[0]
        x = x.masked_fill(~mask[:, None, None], -INF)
    P = torch.softmax(x, -1)
    slack = (2.0 ** -16 + 2.0 ** -13) * (P @ v.abs())
    if dtype == torch.float16:
        slack = slack + 2.0 ** -25 * v.abs().sum(2, keepdim=True) * (P.amax(-1, keepdim=True))
    assert_within("o", cross_attention(*tensors, mask), (P @ v).transpose(1, 2), slack.transpose(1, 2))


@pytest.mark.parametrize("u,v,bias", [(1, 3000, 0), (90, 700, 1), (300, 65, 2)])
def test_powers_of_two_follow_the_data_of_each_replay(u, v, bias):
    """A captured fp16 training call with output gradients of other sizes in its buffer: every replay as the eager call."""
    tensors, mask, dout = _inputs((2, u, v, 4, 2, 64, bias, True), torch.float16, seed=49)
    first = dout.clone()

    def block():
        leaves = [t.detach().requires_grad_() for t in tensors if t is not None]
        o = cross_attention(*leaves, *([] if len(leaves) == 4 else [None]), mask)
        return (o.detach(), *torch.autograd.grad(o, leaves, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    for size in (1.0, 2.0 ** -10, 2.0 ** 9, 0.0):
        dout.copy_(first * size)
        want = [t.clone() for t in block()]
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for name, a, e in zip(NAMES, captured, want):
            assert torch.equal(a, e), (name, size)
        torch.cuda.synchronize()


def test_only_what_is_needed_in_fp16():
    tensors, mask, dout = _inputs((2, 50, 300, 4, 2, 128, 1, True), torch.float16, seed=50)
    every = _train(tensors, mask, dout)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate(tensors)]
        (got,) = torch.autograd.grad(cross_attention(*some, mask), [some[i]], dout)
        assert torch.equal(got, every[1 + i]), NAMES[1 + i]
