"""layer_norm, fused_linear and relative_position_bias as a pairformer block uses them, around
triangle_attention and attention_pair_bias: outputs and every gradient against the same block written in
plain 64-bit torch, and the block captured into a graph.

Bounds are relative to a result's norm. A 16-bit stage rounds once, by at most half a step; an fp32 stage
sums up to 256 terms, (16 + 4 * 256^0.5) U at most. The longest path from an input to an output goes through
``STAGES`` of them, none of which enlarges an error of norm (LayerNorms rescale to 1, the products' weights
have norm about 1, residuals add); a gradient passes as many again on its way back. Where a gradient vanishes
(of the logits, with one key) it is a sum of terms that cancel, each a product of an output gradient, a row of
norm C^0.5 and a value of norm C^0.5 at most, off by (16 + 4 * 256^0.5) U of them: ``C ||dout||`` times that is
the least that counts."""

import pytest
import torch

from geometric_nn_ops_torch.triangle import (attention_pair_bias, fused_linear, layer_norm, relative_position_bias,
                                             triangle_attention)
from op_helpers import DTYPES, IDS, U, half_step, replays_match

pytestmark = pytest.mark.gpu

DEV = "cuda"
C, H, D, S = 64, 4, 16, 64
FAR, BUCKETS, LOG_FAR = 8, 16, 40
STAGES = 14


def _leaves(n, b, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def w(*shape, scale=None, shift=0.0):
        scale = shape[-1] ** -0.5 if scale is None else scale
        return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)

    return {
        "z": w(b, n, n, C, scale=1.0), "s": w(b, n, S, scale=1.0),
        "table_z": w(2 * FAR + 1, C, scale=0.5), "table_b": w(BUCKETS, H, scale=0.5),
        "n1w": w(C, scale=0.1, shift=1.0), "n1b": w(C, scale=0.1), "n2w": w(C, scale=0.1, shift=1.0), "n2b": w(C, scale=0.1),
        "nsw": w(S, scale=0.1, shift=1.0),
        "qkv": w(3 * H * D, C), "tri": w(H, C), "gate": w(H * D, C), "gate_b": w(H * D, scale=0.1),
        "out": w(C, H * D), "out_b": w(C, scale=0.1), "up": w(4 * C, C), "up_b": w(4 * C, scale=0.1), "down": w(C, 4 * C),
        "sqkv": w(3 * S, S), "sg": w(S, S), "so": w(S, S), "sup": w(2 * S, S), "sdown": w(S, 2 * S),
    }


def _positions(n, b):
    g = torch.Generator().manual_seed(n)
    return torch.cumsum(1 + 60 * (torch.rand(b, n, generator=g) < 0.1).long(), 1)


def _heads(t, n, b):
    return [x.transpose(1, 2) for x in t.view(b, n, 3, H, S // H).unbind(2)]


def _block(p, pos, mask, smask):
    b, n = pos.shape
    z = p["z"] + relative_position_bias(p["table_z"], pos, spacing="clip", max_distance=FAR, channels_last=True)
    rel = relative_position_bias(p["table_b"], pos, spacing="log", max_distance=LOG_FAR)
    h = layer_norm(z, p["n1w"], p["n1b"])
    q, k, v = fused_linear(h, p["qkv"]).view(b, n, n, 3, H, D).unbind(3)
    bias = fused_linear(h, p["tri"]).permute(0, 3, 1, 2) + rel
    o = triangle_attention(q, k, v, bias=bias, mask=mask)
    o = o.reshape(b, n, n, H * D) * fused_linear(h, p["gate"], p["gate_b"], "sigmoid")
    z = fused_linear(o, p["out"], p["out_b"], residual=z)
    t = fused_linear(layer_norm(z, p["n2w"], p["n2b"]), p["up"], p["up_b"], "gelu")
    z = fused_linear(t, p["down"], residual=z)
    a = layer_norm(p["s"], p["nsw"])
    q, k, v = _heads(fused_linear(a, p["sqkv"]), n, b)
    o, _ = attention_pair_bias(a, q, k, v, rel, proj_g_weight=p["sg"], proj_o_weight=p["so"], mask=smask,
                               z_is_projected=True)
    s = p["s"] + o
    s = fused_linear(fused_linear(s, p["sup"], None, "silu"), p["sdown"], residual=s)
    return z, s


def _plain_bias(table, pos, log):
    d = pos[:, None, :] - pos[:, :, None]
    if not log:
        return table[d.clamp(-FAR, FAR) + FAR]
    n, near = BUCKETS // 2, BUCKETS // 4
    at = d.abs().clamp(max=LOG_FAR)
    far = near + (torch.log(at.double().clamp(min=near) / near) / torch.log(torch.tensor(LOG_FAR / near).double())
                  * (n - near) + 1e-9).long()
    side = torch.where(at < near, at, far.clamp(max=n - 1))
    return table[side + n * (d > 0)].permute(0, 3, 1, 2)


def _plain(p, pos, mask, smask):
    b, n = pos.shape

    def norm(x, w, bias=None):
        y = torch.nn.functional.layer_norm(x, x.shape[-1:], w, bias)
        return y

    def attend(q, k, v, bias, keep):  # [..., H, N, D]
        logits = q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5 + bias
        return torch.softmax(logits.masked_fill(~keep, float("-inf")), -1) @ v

    z = p["z"] + _plain_bias(p["table_z"], pos, False)
    rel = _plain_bias(p["table_b"], pos, True)
    h = norm(z, p["n1w"], p["n1b"])
    q, k, v = (t.transpose(2, 3) for t in (h @ p["qkv"].t()).view(b, n, n, 3, H, D).unbind(3))
    bias = ((h @ p["tri"].t()).permute(0, 3, 1, 2) + rel)[:, None]
    o = attend(q, k, v, bias, mask).transpose(2, 3).reshape(b, n, n, H * D)
    o = o * torch.sigmoid(h @ p["gate"].t() + p["gate_b"])
    z = z + o @ p["out"].t() + p["out_b"]
    t = torch.nn.functional.gelu(norm(z, p["n2w"], p["n2b"]) @ p["up"].t() + p["up_b"])
    z = z + t @ p["down"].t()
    a = norm(p["s"], p["nsw"])
    q, k, v = _heads(a @ p["sqkv"].t(), n, b)
    o = attend(q, k, v, rel, smask[:, None, None, :] > 0).transpose(1, 2).reshape(b, n, S)
    s = p["s"] + (torch.sigmoid(a @ p["sg"].t()) * o) @ p["so"].t()
    s = s + torch.nn.functional.silu(s @ p["sup"].t()) @ p["sdown"].t()
    return z, s


def _case(n, b, dtype):
    p, pos = _leaves(n, b, dtype), _positions(n, b)
    keep = torch.rand(b, n, generator=torch.Generator().manual_seed(3)) < 0.8
    keep[:, 0] = True
    return p, pos, keep


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,b", [(1, 2), (21, 2), (64, 1), (185, 1)])
def test_block_and_gradients(n, b, dtype):
    p, pos, keep = _case(n, b, dtype)
    exact = {k: t.double().requires_grad_() for k, t in p.items()}
    want = _plain(exact, pos, keep[:, None, None, None, :], keep)
    g = torch.Generator().manual_seed(5)
    douts = [torch.randn(t.shape, generator=g).to(dtype) for t in want]
    want_grads = torch.autograd.grad(want, list(exact.values()), [d.double() for d in douts])
    leaves = {k: t.to(DEV).requires_grad_() for k, t in p.items()}
    got = _block(leaves, pos.to(DEV), keep[:, None, None, None, :].to(DEV), keep.to(DEV, dtype))
    grads = torch.autograd.grad(got, list(leaves.values()), [d.to(DEV) for d in douts])
    step = half_step(dtype) if dtype != torch.float32 else (16 + 4 * 256 ** 0.5) * U

    least = (16 + 4 * 256 ** 0.5) * U * C * float(sum(d.double().norm() for d in douts))

    def near(name, a, e, stages):
        assert a.dtype == dtype and a.shape == e.shape, name
        a = a.detach()
        off, scale = float((a.double().cpu() - e).norm()), float(e.norm())
        assert off <= max(stages * step * scale, least), f"{name}: off by {off:.3g}, its norm {scale:.3g}"

    for name, a, e in zip("zs", got, want):
        near(name, a, e.detach(), STAGES)
    for name, a, e in zip(leaves, grads, want_grads):
        near("gradient of " + name, a, e, 2 * STAGES)


def test_block_repeats_and_replays_in_a_graph():
    p, pos, keep = _case(48, 1, torch.bfloat16)
    p = {k: t.to(DEV) for k, t in p.items()}
    pos, mask, smask = pos.to(DEV), keep[:, None, None, None, :].to(DEV), keep.to(DEV, torch.bfloat16)

    def block():
        with torch.no_grad():
            return _block(p, pos, mask, smask)

    def same(a, e, replay):
        assert torch.equal(a, e), f"replay {replay}"

    replays_match(block, same)


def test_block_on_another_stream():
    p, pos, keep = _case(33, 2, torch.bfloat16)
    p = {k: t.to(DEV).requires_grad_() for k, t in p.items()}
    pos, mask, smask = pos.to(DEV), keep[:, None, None, None, :].to(DEV), keep.to(DEV, torch.bfloat16)

    def run():
        outs = _block(p, pos, mask, smask)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, list(p.values()), [torch.ones_like(t) for t in outs]))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(2048, 2048, device=DEV)
    for _ in range(20):  # the default stream is at work meanwhile
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    for name, a, e in zip(("z", "s", *p), got, want):
        assert torch.equal(a, e), name
