"""gated_linear, qk_norm_rotary and cross_attention as a decoder block over an encoder's states uses them, between
layer_norm, fused_linear and relative_position_bias: outputs and every gradient against the same block written in plain
64-bit torch, its decoding token by token, and the block captured into a graph.

Bounds are relative to a result's norm. A 16-bit stage rounds once, by at most half a step; an fp32 stage sums up to 256
terms, (16 + 4 * 256^0.5) U at most. Up to the gated product lie nine stages at most: a norm, a projection, the
per-head norm with its rotation, logits, probabilities, their sum, the projection with its residual, a norm, and a
projection inside the gated product. None enlarges an error of norm, but each factor of the gated product carries it, so
that it counts twice there; the product's own rounding and the last projection follow: ``STAGES`` = 2 * 9 + 2. A gradient
passes as many again on its way back. Where a gradient vanishes (of the logits, with one key) it is a sum of terms that
cancel, each a product of an output gradient and two rows of norm C^0.5 at most, off by (16 + 4 * 256^0.5) U of them:
``C ||dout||`` times that is the least that counts."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import (cross_attention, fused_linear, gated_linear, layer_norm, qk_norm_rotary,
                                             relative_position_bias)
from op_helpers import DTYPES, IDS, U, half_step, replays_match

pytestmark = pytest.mark.gpu

DEV = "cuda"
C, H, HK, D, FAR = 64, 4, 2, 16, 8
STAGES = 20
FP32 = (16 + 4 * 256 ** 0.5) * U


def _leaves(b, u, v, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def w(*shape, scale=None, shift=0.0):
        scale = shape[-1] ** -0.5 if scale is None else scale
        return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)

    return {
        "x": w(b, u, C, scale=1.0), "states": w(b, v, C, scale=1.0), "table": w(2 * FAR + 1, H, scale=0.5),
        "n1": w(C, scale=0.1, shift=1.0), "n1b": w(C, scale=0.1), "n2": w(C, scale=0.1, shift=1.0),
        "ns": w(C, scale=0.1, shift=1.0), "q": w(H * D, C), "kv": w(2 * HK * D, C),
        "qn": w(D, scale=0.1, shift=1.0), "kn": w(D, scale=0.1, shift=1.0), "out": w(C, H * D), "out_b": w(C, scale=0.1),
        "gate_up": w(8 * C, C), "gate_b": w(4 * C, scale=0.1), "down": w(C, 4 * C),
    }


def _case(b, u, v):
    keep = torch.arange(v) < torch.tensor([v, 0, max(1, v // 3)])[:b, None]  # whole, all padding, a third
    return torch.arange(u) + 5, torch.arange(v), keep


def _block(p, q_pos, k_pos, keep):
    (b, u), v = p["x"].shape[:2], p["states"].shape[1]
    q = fused_linear(layer_norm(p["x"], p["n1"], p["n1b"]), p["q"]).view(b, u, H, D)
    k, val = fused_linear(layer_norm(p["states"], p["ns"]), p["kv"]).view(b, v, 2, HK, D).unbind(2)
    q, k = qk_norm_rotary(q, k, q_pos, k_pos, q_weight=p["qn"], k_weight=p["kn"])
    bias = relative_position_bias(p["table"], q_pos[None], k_pos[None], spacing="clip", max_distance=FAR)
    o = cross_attention(q, k, val, bias, keep)
    x = fused_linear(o.reshape(b, u, H * D), p["out"], p["out_b"], residual=p["x"])
    gate, up = p["gate_up"].chunk(2)
    return fused_linear(gated_linear(layer_norm(x, p["n2"]), gate, up, p["gate_b"]), p["down"], residual=x)


def _plain(p, q_pos, k_pos, keep):
    (b, u), v = p["x"].shape[:2], p["states"].shape[1]

    def norm(x, w, bias=None):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, bias)

    def turned(x, w, pos):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        angle = pos.double()[:, None, None] * 10000.0 ** (-torch.arange(0, D, 2).double() / D)
        a, c = x.chunk(2, -1)
        return torch.cat([a * angle.cos() - c * angle.sin(), c * angle.cos() + a * angle.sin()], -1)

    q = (norm(p["x"], p["n1"], p["n1b"]) @ p["q"].t()).view(b, u, H, D)
    k, val = (norm(p["states"], p["ns"]) @ p["kv"].t()).view(b, v, 2, HK, D).unbind(2)
    q, k = turned(q, p["qn"], q_pos).transpose(1, 2), turned(k, p["kn"], k_pos).transpose(1, 2)
    k, val = (t.repeat_interleave(H // HK, 1) for t in (k, val.transpose(1, 2)))
    bias = p["table"][(k_pos - q_pos[:, None]).clamp(-FAR, FAR) + FAR].permute(2, 0, 1)
    logits = (q @ k.transpose(2, 3) * D ** -0.5 + bias).masked_fill(~keep[:, None, None, :], -1e30)
    probs = torch.softmax(logits, -1) * keep[:, None, None, :]
    x = p["x"] + (probs @ val).transpose(1, 2).reshape(b, u, H * D) @ p["out"].t() + p["out_b"]
    gate, up = p["gate_up"].chunk(2)
    h = norm(x, p["n2"])
    return x + (torch.nn.functional.silu(h @ gate.t() + p["gate_b"]) * (h @ up.t())) @ p["down"].t()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,u,v", [(1, 1, 1), (2, 1, 40), (3, 37, 90), (1, 130, 257), (3, 200, 19)])
def test_block_and_gradients(b, u, v, dtype):
    p, where = _leaves(b, u, v, dtype), _case(b, u, v)
    exact = {k: t.double().requires_grad_() for k, t in p.items()}
    want = _plain(exact, *where)
    dout = torch.randn(want.shape, generator=torch.Generator().manual_seed(5)).to(dtype)
    want_grads = torch.autograd.grad(want, list(exact.values()), dout.double())
    leaves = {k: t.to(DEV).requires_grad_() for k, t in p.items()}
    got = _block(leaves, *(t.to(DEV) for t in where))
    grads = torch.autograd.grad(got, list(leaves.values()), dout.to(DEV))
    step = half_step(dtype) if dtype != torch.float32 else FP32
    least = FP32 * C * float(dout.double().norm())

    def near(name, a, e, stages):
        assert a.dtype == dtype and a.shape == e.shape, name
        off, norm = float((a.detach().double().cpu() - e).norm()), float(e.norm())
        assert off <= max(stages * step * norm, least), f"{name}: off by {off:.3g}, its norm {norm:.3g}"

    near("output", got, want.detach(), STAGES)
    for name, a, e in zip(leaves, grads, want_grads):
        near("gradient of " + name, a, e, 2 * STAGES)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_token_by_token(dtype):
    p, (q_pos, k_pos, keep) = _leaves(2, 21, 70, dtype), _case(2, 21, 70)
    want = _plain({k: t.double() for k, t in p.items()}, q_pos, k_pos, keep)
    p = {k: t.to(DEV) for k, t in p.items()}
    q_pos, k_pos, keep = q_pos.to(DEV), k_pos.to(DEV), keep.to(DEV)
    step = half_step(dtype) if dtype != torch.float32 else FP32
    with torch.no_grad():
        for i in range(21):
            got = _block({**p, "x": p["x"][:, i:i + 1]}, q_pos[i:i + 1], k_pos, keep)
            off = float((got.double().cpu() - want[:, i:i + 1]).norm())
            assert off <= STAGES * step * float(want[:, i:i + 1].norm()), f"token {i}: off by {off:.3g}"


@pytest.mark.parametrize("u", [1, 50])
def test_block_repeats_and_replays_in_a_graph(u):
    p = {k: t.to(DEV) for k, t in _leaves(2, u, 600, torch.bfloat16).items()}
    where = [t.to(DEV) for t in _case(2, u, 600)]

    def block():
        with torch.no_grad():
            return [_block(p, *where)]

    def same(a, e, replay):
        assert torch.equal(a, e), f"replay {replay}"

    replays_match(block, same)


def test_block_on_another_stream():
    p = {k: t.to(DEV).requires_grad_() for k, t in _leaves(2, 33, 90, torch.bfloat16).items()}
    where = [t.to(DEV) for t in _case(2, 33, 90)]

    def run():
        out = _block(p, *where)
        return [out.detach(), *torch.autograd.grad(out, list(p.values()), torch.ones_like(out))]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(2048, 2048, device=DEV)
    for _ in range(20):  # the default stream is at work meanwhile
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    for name, a, e in zip(("output", *p), got, want):
        assert torch.equal(a, e), name
