"""Checks shared by the tests of layer_norm, fused_linear and relative_position_bias.

Bounds are elementwise: half a step of the result's type (``torch.finfo(t).eps / 2`` relative to the exact
value) for the one rounding at the end, plus what fp32 arithmetic may lose, counted in units U = 2^-24 of
the sums of absolute values that the operator's formula goes through."""

import torch

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def assert_within(name, got, want, slack):
    """``|got - want| <= half a step of got's type * |want| + slack``, elementwise; ``want`` and ``slack``
    float64. The smallest step of the type counts where values fall below its normal range."""
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} != {tuple(want.shape)}"
    got, slack = got.to(want.device), slack.to(want.device)
    d = (got.double() - want).abs()
    info = torch.finfo(got.dtype)
    bound = half_step(got.dtype) * want.abs() * (1 + 4 * U) + slack * (1 + half_step(got.dtype))
    bound = bound + info.tiny * info.eps
    bad = ~(d <= bound)
    if bad.any():
        i = int((d / bound).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off, worst at {i}: got "
                             f"{got.reshape(-1)[i].item()}, want {want.reshape(-1)[i].item()}, bound "
                             f"{bound.reshape(-1)[i].item():.3g}")


def directional(f, x, v, h=1e-4):
    """Central difference of the float64 scalar function ``f`` at ``x`` along ``v``."""
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


def replays_match(block, check_equal, replays=3):
    """Captures ``block`` into a HIP graph and replays it with eager work between the replays; every
    replay's outputs must equal the eager ones bit for bit."""
    eager = [t.clone() for t in block()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    for replay in range(replays):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, eager):
            check_equal(got, want, replay)
        for got, want in zip(block(), eager):  # eager work between the replays
            check_equal(got, want, replay)
        torch.cuda.synchronize()
