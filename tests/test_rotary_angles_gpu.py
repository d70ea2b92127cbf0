"""qk_norm_rotary's sine and cosine in fp32, read off pairs (1, 0), against float64.

The angle, reduced to half a turn to both sides in fp64, is rounded once as a fraction of a turn: by U of itself, and the
fp64 product by 2^-52 of the angle. Sine and cosine are off by two units in the last place at most, 4 U of themselves."""

import math

import pytest
import torch

from geometric_nn_ops_torch.triangle import qk_norm_rotary
from op_helpers import U, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _hold(pos, freqs, interleaved):
    d = 2 * len(freqs)
    x = torch.zeros(1, pos.numel(), 1, d)
    first, second = ((slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, d // 2), slice(d // 2, None)))
    x[..., first] = 1.0
    angle = (pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64))[None, :, None]
    near = (angle - 2 * math.pi * torch.round(angle / (2 * math.pi))).abs()
    sin, cos, lost = angle.sin(), angle.cos(), angle.abs() * 2.0 ** -51
    y = qk_norm_rotary(x.to(DEV), x.to(DEV), pos.to(DEV), eps=None, frequencies=freqs, interleaved=interleaved)[0].cpu()
    assert_within("sine", y[..., second], sin, U * near * cos.abs() + 4 * U * sin.abs() + lost)
    assert_within("cosine", y[..., first], cos, U * near * sin.abs() + 4 * U * cos.abs() + lost)


@pytest.mark.parametrize("interleaved", [False, True])
def test_small_angles_keep_their_digits(interleaved):
    """Of 10^-7 to 10^-1: a sine that is off by 2^-23 would have none left."""
    _hold(torch.tensor([0, 1, 2, 3, 17, 100, 999]), [10.0 ** (-7 + j / 12) for j in range(48)], interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_over_many_turns(interleaved):
    g = torch.Generator().manual_seed(1)
    pos = torch.cat([torch.arange(-40, 400), torch.randint(0, 1 << 20, (3000,), generator=g)])
    _hold(pos, [10000.0 ** (-2 * j / 128) for j in range(64)], interleaved)


def test_whole_quarters_of_a_turn():
    """Beside zeros of sine and cosine."""
    _hold(torch.arange(-64, 65), [math.pi / 2 * k / 8 for k in range(1, 9)], False)


def test_gradients_of_small_angles():
    freqs = [10.0 ** (-6 + j / 8) for j in range(32)]
    x, dy = torch.zeros(1, 7, 1, 64, device=DEV, requires_grad=True), torch.zeros(1, 7, 1, 64, device=DEV)
    dy[..., :32] = 1.0
    pos = torch.tensor([1, 2, 3, 5, 17, 100, 999])
    q, _ = qk_norm_rotary(x, x.detach(), pos.to(DEV), eps=None, frequencies=freqs)
    (dx,) = torch.autograd.grad(q, x, dy)
    angle = (pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64))[None, :, None]
    near = (angle - 2 * math.pi * torch.round(angle / (2 * math.pi))).abs()
    assert_within("dx", dx.cpu()[..., 32:], -angle.sin(), U * near * angle.cos().abs() + 4 * U * angle.sin().abs() + angle.abs() * 2.0 ** -51)
