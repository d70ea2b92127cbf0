"""cross_attention where little is left of a row: one key under a bias, infinities and NaN."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import cross_attention
from op_helpers import DTYPES, IDS, U, assert_within
from test_cross_attention_gpu import NAMES, _inputs

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
