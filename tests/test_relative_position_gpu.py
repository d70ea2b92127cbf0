"""relative_position_bias on the GPU: values equal to the table's (a lookup rounds nothing), the table's
gradient against float64 sums.

Bound of the gradient: a lane adds a run of values in fp32 one by one, at most 4096 here, and the partial
sums of lanes and workgroups are added in another 200 steps at most: 4300 U of the sum of absolute values
at the very worst, of which rounding errors of random sign leave the square root; 100 U is taken (its
square is above the 4300 steps)."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import relative_position_bias, triangle_attention
from geometric_nn_ops_torch.triangle._reference.relative_position import buckets_torch
from op_helpers import DTYPES, IDS, U, assert_within, directional, replays_match

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _positions(b, n, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "run":
        return torch.arange(n).expand(b, n).contiguous()
    if kind == "gaps":
        return torch.cumsum(1 + 40 * (torch.rand(b, n, generator=g) < 0.05).long(), 1)
    return torch.randint(-400, 400, (b, n), generator=g)


def _check(b, u, v, h, case, dtype, kind="gaps", last=False, seed=0, pos_dtype=torch.int64):
    buckets, far, spacing, two = case
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(buckets, h, generator=g).to(dtype)
    q, k = _positions(b, u, kind, seed + 1), _positions(b, v, kind, seed + 2)
    dout = torch.randn((b, u, v, h) if last else (b, h, u, v), generator=g).to(dtype)
    rows = buckets_torch(q, k, *case)
    leaf = w.to(DEV).requires_grad_()
    how = dict(max_distance=far, spacing=spacing, bidirectional=two, channels_last=last)
    qd, kd = q.to(DEV, pos_dtype), k.to(DEV, pos_dtype)
    out = relative_position_bias(leaf, qd, kd, **how)
    want = w[rows] if last else w[rows].permute(0, 3, 1, 2)
    assert out.dtype == dtype and out.shape == want.shape
    assert torch.equal(out.detach().cpu(), want)
    with torch.no_grad():
        assert torch.equal(relative_position_bias(leaf, qd, kd, **how), out)
    (grad,) = torch.autograd.grad(out, leaf, dout.to(DEV))
    flat = (dout if last else dout.permute(0, 2, 3, 1)).reshape(-1, h).double()
    exact, size = (torch.zeros(buckets, h, dtype=torch.float64).index_add_(0, rows.reshape(-1), t)
                   for t in (flat, flat.abs()))
    assert_within("dweight", grad, exact, 100 * U * size)


CASES = [(32, 128, "log", True), (32, 128, "log", False), (65, 32, "clip", True), (33, 32, "clip", False)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", CASES, ids=["log2", "log1", "clip2", "clip1"])
@pytest.mark.parametrize("last", [False, True], ids=["heads_first", "heads_last"])
def test_values_and_gradient(case, dtype, last):
    for i, (b, u, v, h) in enumerate([(1, 1, 1, 1), (1, 1, 700, 4), (2, 5, 9, 3), (1, 64, 64, 16), (2, 33, 130, 8),
                                      (1, 70, 531, 5), (1, 3, 2100, 12), (2, 40, 63, 130)]):
        kind = ("run", "gaps", "any")[i % 3]
        _check(b, u, v, h, case, dtype, kind, last, seed=10 * i, pos_dtype=(torch.int64, torch.int32)[i % 2])


@pytest.mark.parametrize("last", [False, True], ids=["heads_first", "heads_last"])
def test_other_tables(last):
    """Few and many buckets: the smallest tables, ones whose bins take several passes, one that does not
    fit LDS in the forward, a head count of several channel tiles."""
    for i, case in enumerate([(2, 2, "log", False), (4, 2, "log", True), (3, 1, "clip", True), (7, 11, "log", False),
                              (64, 1000, "log", True), (512, 3000, "log", False), (801, 400, "clip", True)]):
        _check(1, 20, 300, 9, case, torch.bfloat16, "any", last, seed=100 + i)
    _check(1, 30, 100, 300, (401, 200, "clip", True), torch.float32, "gaps", last, seed=120)
    _check(1, 9, 50, 257, (32, 128, "log", True), torch.float16, "gaps", last, seed=121)


def test_long_rows():
    _check(1, 600, 4100, 2, CASES[0], torch.bfloat16, "run", False, seed=7)
    _check(1, 300, 1000, 64, CASES[2], torch.bfloat16, "run", True, seed=8)


def test_far_positions():
    """Differences beyond 32 bits, and beyond 63, count as far away on their side."""
    w = torch.randn(32, 4, generator=torch.Generator().manual_seed(1)).to(DEV)
    big = 1 << 62
    q = torch.tensor([0, 5, -big - 7, big + 9], device=DEV)
    k = torch.tensor([0, 4, 1 << 33, -(1 << 33), big + 9, -big - 9], device=DEV)
    out = relative_position_bias(w, q, k, max_distance=128)[0].permute(1, 2, 0).cpu()
    for i, a in enumerate(q.tolist()):
        for j, b in enumerate(k.tolist()):
            d = max(-128, min(128, b - a))
            row = buckets_torch(torch.zeros(1, 1, dtype=torch.int64), torch.tensor([[d]]), 32, 128, "log", True)
            assert torch.equal(out[i, j], w.cpu()[row.item()])


def test_output_gradients_in_any_strides():
    w = torch.randn(65, 6, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    pos = torch.arange(40, device=DEV)
    rows = buckets_torch(pos.cpu()[None], pos.cpu()[None], 65, 32, "clip", True).reshape(-1)
    base = torch.randn(2, 40, 6, 40, 2, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    for last in (False, True):
        leaf = w.clone().requires_grad_()
        out = relative_position_bias(leaf, pos, max_distance=32, spacing="clip", channels_last=last)
        views = [base[:1, ..., 0], base[:1, ..., 0].contiguous(), base[0, 0, 0, 0, 0].expand(1, 40, 6, 40)]
        for d in views:  # [1, u, h, v]
            dout = d.permute(0, 1, 3, 2) if last else d.permute(0, 2, 1, 3)
            (grad,) = torch.autograd.grad(out, leaf, dout, retain_graph=True)
            flat = d.permute(0, 1, 3, 2).reshape(-1, 6).double().cpu()
            exact, size = (torch.zeros(65, 6, dtype=torch.float64).index_add_(0, rows, t) for t in (flat, flat.abs()))
            assert_within("dweight", grad, exact, 100 * U * size)


def test_values_that_are_not_finite_stay_in_their_bucket():
    w = torch.zeros(65, 2, device=DEV, requires_grad=True)
    pos = torch.arange(100, device=DEV)
    out = relative_position_bias(w, pos, max_distance=32, spacing="clip")
    dout = torch.ones_like(out)
    dout[0, 0, 10, 13] = float("nan")  # bucket 35 of head 0
    dout[0, 1, 10, 99] = float("inf")  # bucket 64 of head 1
    (grad,) = torch.autograd.grad(out, w, dout)
    bad = torch.zeros(65, 2, dtype=torch.bool)
    bad[35, 0] = bad[64, 1] = True
    assert torch.equal(~grad.isfinite().cpu(), bad)


def test_empty():
    w = torch.randn(32, 4, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.arange(5, device=DEV)
    for q, k in ((pos[:0], pos), (pos, pos[:0]), (pos[None][:0], pos[None][:0])):
        out = relative_position_bias(w, q, k, max_distance=128)
        assert out.numel() == 0
        (grad,) = torch.autograd.grad(out, w, torch.empty_like(out))
        assert grad.shape == w.shape and not grad.any()
    assert relative_position_bias(w[:, :0].detach(), pos, max_distance=128).shape == (1, 0, 5, 5)


def test_expanded_positions_and_table_views():
    g = torch.Generator().manual_seed(4)
    w = torch.randn(32, 8, generator=g).to(DEV)
    pos = torch.arange(60, device=DEV)
    want = relative_position_bias(w[:, 1:4].contiguous(), pos, max_distance=128)
    got = relative_position_bias(w[:, 1:4], torch.arange(120, device=DEV)[::2] // 2, pos.expand(3, 60), max_distance=128)
    assert got.shape == (3, 3, 60, 60) and torch.equal(got, want.expand(3, 3, 60, 60))


def test_attention_reads_the_bias_without_a_copy():
    from geometric_nn_ops_torch.triangle._kernels.triangle_attention import _bias_readable

    w = torch.randn(65, 4, device=DEV, dtype=torch.bfloat16)
    for n in (40, 43):
        bias = relative_position_bias(w, torch.arange(n, device=DEV), max_distance=32, spacing="clip")
        assert _bias_readable(bias.unsqueeze(1))
        q, k, v = torch.randn(3, 1, 5, n, 4, 32, device=DEV, dtype=torch.bfloat16)
        with torch.no_grad():
            assert torch.equal(triangle_attention(q, k, v, bias), triangle_attention(q, k, v, bias.contiguous()))


def test_gradient_against_differences():
    w = torch.randn(32, 3, generator=torch.Generator().manual_seed(5))
    pos = torch.arange(50)
    dout = torch.randn(1, 3, 50, 50, generator=torch.Generator().manual_seed(6))
    leaf = w.to(DEV).requires_grad_()
    (grad,) = torch.autograd.grad(relative_position_bias(leaf, pos.to(DEV), max_distance=40), leaf, dout.to(DEV))
    v = torch.randn(32, 3, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
    rows = buckets_torch(pos[None], pos[None], 32, 40, "log", True)
    want = directional(lambda t: (t[rows].permute(0, 3, 1, 2) * dout.double()).sum(), w.double(), v)
    # linear in the table: the difference is exact but for the cancellation of its two sums
    assert abs((grad.double().cpu() * v).sum() - want) <= 1e-5 * (grad.double().cpu() * v).abs().sum()


def test_second_derivative_raises():
    w = torch.randn(65, 2, device=DEV, requires_grad=True)
    out = relative_position_bias(w, torch.arange(9, device=DEV), max_distance=32, spacing="clip")
    (grad,) = torch.autograd.grad(out.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), w)


def test_offsets_beyond_32_bits():
    """An output of more than 2^32 elements: its first and last queries, and the gradient of a dout that is
    zero but for them."""
    n, h = 23200, 8
    w = torch.randn(32, h, generator=torch.Generator().manual_seed(8)).bfloat16()
    leaf = w.to(DEV).requires_grad_()
    pos = torch.arange(n)
    out = relative_position_bias(leaf, pos.to(DEV), max_distance=128)
    assert out.numel() > 1 << 32
    ends = [0, 1, n - 2, n - 1]
    rows = buckets_torch(pos[None, ends], pos[None], 32, 128, "log", True)
    assert torch.equal(out[:, :, ends].detach().cpu(), w[rows].permute(0, 3, 1, 2))
    dout = torch.zeros_like(out)
    some = torch.randn(1, h, 4, n, generator=torch.Generator().manual_seed(9)).bfloat16()
    dout[:, :, ends] = some.to(DEV)
    (grad,) = torch.autograd.grad(out, leaf, dout)
    flat = some.permute(0, 2, 3, 1).reshape(-1, h).double()
    exact, size = (torch.zeros(32, h, dtype=torch.float64).index_add_(0, rows.reshape(-1), t) for t in (flat, flat.abs()))
    assert_within("dweight", grad, exact, 100 * U * size)


@pytest.mark.parametrize("last", [False, True], ids=["heads_first", "heads_last"])
def test_calls_repeat_bit_for_bit_and_replay_in_a_graph(last):
    w = torch.randn(65, 24, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.arange(211, device=DEV)
    dout = torch.randn((1, 211, 211, 24) if last else (1, 24, 211, 211), device=DEV, dtype=torch.bfloat16)

    def block():
        out = relative_position_bias(w, pos, max_distance=32, spacing="clip", channels_last=last)
        return out.detach(), *torch.autograd.grad(out, w, dout)

    def equal(got, want, replay):
        assert torch.equal(got, want), replay

    replays_match(block, equal)


def test_operator_registration():
    import geometric_nn_ops_torch._ops  # noqa: F401

    w = torch.randn(65, 4, device=DEV)
    q, k = torch.arange(9, device=DEV)[None], torch.arange(13, device=DEV)[None]
    for last in (False, True):
        torch.library.opcheck(torch.ops.gnn_amd.relative_position_bias_fwd.default, (w, q, k, 32, "clip", True, last),
                              test_utils=("test_schema", "test_faketensor"))
    with torch.no_grad():
        f = lambda t: relative_position_bias(t, q, k, max_distance=32, spacing="clip")  # noqa: E731
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(w), f(w))


def test_the_borders_live_as_long_as_the_graph():
    import gc

    from geometric_nn_ops_torch.triangle._kernels import relative_position as kernels

    pos = torch.arange(200, device=DEV)
    grads = []
    for drop in (False, True):
        table = torch.randn(32, 4, generator=torch.Generator().manual_seed(2)).to(DEV).requires_grad_()
        y = relative_position_bias(table, pos, max_distance=100)
        if drop:
            kernels._borders.cache_clear()
            gc.collect()
            others = [(type(kernels._borders(16, 8, 99)))(*range(1, 8)) for _ in range(2000)]  # noqa: F841
        grads.append(torch.autograd.grad(y, table, torch.ones_like(y))[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("h", [1, 2, 3, 5, 8, 16, 31, 33, 64, 65, 129, 200])
def test_channels_last_of_every_width(h, dtype):
    """The gradient of narrow tables, whose channels leave room for several pixels in a wave, and of odd ones;
    the output gradient lies between NaN."""
    u, v, far = 7, 301, 5
    g = torch.Generator().manual_seed(h)
    w = torch.randn(2 * far + 1, h, generator=g).to(dtype)
    q = torch.randint(-9, 300, (2, u), generator=g)
    k = torch.randint(-9, 300, (2, v), generator=g)
    dout = torch.randn(2, u, v, h, generator=g).to(dtype)
    at = (k[:, None, :] - q[:, :, None]).clamp(-far, far) + far
    want = torch.zeros(2 * far + 1, h, dtype=torch.float64).index_add_(0, at.reshape(-1), dout.double().reshape(-1, h))
    size = torch.zeros(2 * far + 1, h, dtype=torch.float64).index_add_(0, at.reshape(-1), dout.double().abs().reshape(-1, h))
    table = w.to(DEV).requires_grad_()
    y = relative_position_bias(table, q.to(DEV), k.to(DEV), max_distance=far, spacing="clip", channels_last=True)
    assert torch.equal(y.detach().cpu(), w[at])
    buf = torch.full((dout.numel() + 512,), float("nan"), device=DEV, dtype=dtype)
    inner = buf[256:256 + dout.numel()].view(dout.shape)
    inner.copy_(dout)
    grad = torch.autograd.grad(y, table, inner)[0]
    assert_within(f"gradient of {h} channels", grad, want, 100 * U * size)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("buckets,h,v", [(64, 500, 3), (256, 100, 61), (256, 101, 7), (255, 257, 5), (128, 193, 1)])
def test_channels_last_tables_outside_lds(buckets, h, v, dtype):
    """Tables above 48 KB whose heads fill no whole chunks, in rows that end inside one: the last pixel lies in the
    last bucket, so that nothing of the table follows it, and NaN lies around the table."""
    far = buckets - 1
    g = torch.Generator().manual_seed(h)
    w = torch.randn(buckets, h, generator=g).to(dtype)
    q = torch.arange(5)[None] + far + 400
    k = torch.randint(0, far, (1, v), generator=g) + 400
    k[0, -1] = 0
    rows = buckets_torch(q, k, buckets, far, "clip", False)
    assert (rows[..., -1] == buckets - 1).all() and w.numel() * w.element_size() > 48 << 10
    buf = torch.full((w.numel() + 128,), float("nan"), device=DEV, dtype=dtype)
    table = buf[64:64 + w.numel()].view(w.shape)
    table.copy_(w)
    how = dict(max_distance=far, spacing="clip", bidirectional=False, channels_last=True)
    with torch.no_grad():
        out = relative_position_bias(table, q.to(DEV), k.to(DEV), **how)
    assert torch.equal(out.cpu(), w[rows])


@pytest.mark.parametrize("case", [(255, 127, "clip", True), (256, 255, "clip", False), (511, 255, "clip", True),
                                  (256, 1000, "log", True), (255, 900, "log", False), (512, 1023, "log", False)],
                         ids=["255", "256", "511", "log256", "log255", "log512"])
def test_tables_whose_bins_and_differences_pass_64_kb(case):
    """Heads first: the bins of 255 or 256 buckets a pass and the table of differences beside them."""
    for i, dtype in enumerate(DTYPES):
        _check(1, 70, 300, 3, case, dtype, ("run", "gaps", "any")[i], seed=200 + i, pos_dtype=(torch.int32, torch.int64)[i % 2])
