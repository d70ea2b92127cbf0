"""The operators of a transformer block beside the pair stream: gated_linear, qk_norm_rotary and cross_attention.

A case is a dict of plain values; "op" names the operator. "train" asks for the forward with everything
requiring grad and for the gradients of a given output gradient; otherwise the forward runs under
inference_mode. "dtype" is the type of every floating tensor.

  gated_linear     m x i -> o: act of one projection times another; "act" is "none", "relu", "gelu", "silu" or
                   "sigmoid"; "stacked": both weights are halves of one tensor
  qk_norm_rotary   b sequences of n tokens, h query and hk key heads of d, the first "rotary" elements of each
                   turned; "start" is the first token's position; "fused": q and k are views of one projection's
                   output, as a layer leaves them; "norm" false leaves the norms out
  cross_attention  b x u queries of h heads against v keys and values of hk heads, all of d; "pad": sequences are
                   padded to v and the mask says where they end ("empty": one of them holds nothing);
                   "bias" is 0 (none), 1 (one for all sequences) or 2 (one each)
"""

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "geometric-nn-ops_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
BASE = 10000.0


def _gated(name, m, i, o, dtype="bf16", *, act="silu", bias=False, stacked=False, train=False):
    c = {"op": "gated_linear", "m": m, "i": i, "o": o, "dtype": dtype, "act": act, "bias": bias, "stacked": stacked,
         "train": train}
    return dict(c, name=name) if name else c


def _rotary(name, b, n, h, hk, d, dtype="bf16", *, rotary=None, interleaved=False, norm=True, start=0, fused=True,
            train=False):
    c = {"op": "qk_norm_rotary", "b": b, "n": n, "h": h, "hk": hk, "d": d, "dtype": dtype,
         "rotary": d if rotary is None else rotary, "interleaved": interleaved, "norm": norm, "start": start,
         "fused": fused, "train": train}
    return dict(c, name=name) if name else c


def _cross(name, b, u, v, h, hk, d, dtype="bf16", *, pad=False, empty=False, bias=0, train=False):
    c = {"op": "cross_attention", "b": b, "u": u, "v": v, "h": h, "hk": hk, "d": d, "dtype": dtype, "pad": pad,
         "empty": empty, "bias": bias, "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through the gated layer of a single-track transition: the call costs more than the kernel
        _gated("gated_token_c384_bf16", 1, 384, 1536),
        # the gated layer of the pair transition in training at the usual crop
        _gated("gated_train_pair_n384_bf16", 384 * 384, 128, 512, train=True),
        # a wide layer, where the matrix units bound the call
        _gated("gated_wide_4096_bf16", 8192, 4096, 8192, stacked=True),
        # full precision at odd widths, in training
        _gated("gated_train_odd_fp32", 4099, 331, 883, "fp32", act="gelu", bias=True, train=True),
        # one new token of each of 8 sequences, far from their start
        _rotary("rotary_token_b8_bf16", 8, 1, 32, 8, 128, start=100_000),
        # queries and keys as the projection leaves them, in training
        _rotary("rotary_train_n4096_bf16", 2, 4096, 16, 16, 128, train=True),
        # an odd length, a head dim that is no power of two, part of it turned, neighbours paired
        _rotary("rotary_train_odd_fp16", 3, 1021, 20, 5, 80, "fp16", rotary=48, interleaved=True, train=True),
        # one new query of each of 8 sequences against a long padded memory, shared heads
        _cross("cross_token_v8191_bf16", 8, 1, 8191, 32, 8, 128, pad=True),
        # a decoder's tokens against an encoder's padded states, in training
        _cross("cross_train_u2048_bf16", 4, 2048, 1400, 16, 16, 64, pad=True, train=True),
        # many queries against a long memory, inference: the matrix units bound the call
        _cross("cross_long_v8192_bf16", 1, 4096, 8192, 32, 8, 128),
        # odd lengths with a learned bias for all sequences, one of them empty, in training
        _cross("cross_train_bias_fp16", 3, 509, 1021, 8, 8, 32, "fp16", pad=True, empty=True, bias=1, train=True),
        # full precision with shared heads, in training
        _cross("cross_train_fp32", 2, 333, 777, 8, 2, 64, "fp32", train=True),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(("gated_linear", "qk_norm_rotary", "cross_attention", "cross_attention"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    train = rng.random() < 0.5
    if op == "gated_linear":
        i, o = (rng.choice((128, 256, 384, 512, 1024, size(16, 4096), size(16, 4096))) for _ in range(2))
        # the work of the wide case, a quarter of it in full precision, a third where there are gradients
        most = 8192 * 4096 * 8192 // (i * o) // (4 if dtype == "fp32" else 1) // (3 if train else 1)
        m = size(1, max(1, min(262144, most, 300_000_000 // ((3 if train else 1) * SIZE[dtype] * (i + 3 * o)))))
        return _gated(None, m, i, o, dtype, act=rng.choice(("silu", "silu", "gelu", "relu", "sigmoid", "none")),
                      bias=rng.random() < 0.4, stacked=rng.random() < 0.4, train=train)
    if op == "qk_norm_rotary":
        d = rng.choice((32, 64, 128, 128, 256, 8 * size(1, 32)))
        hk = size(1, 32)
        h = hk * rng.choice((1, 1, 2, 4, 8))
        rotary = d if rng.random() < 0.6 else 8 * rng.randint(1, d // 8)
        n = size(1, max(1, min(32768, 200_000_000 // ((3 if train else 1) * SIZE[dtype] * (h + hk) * d))))
        b = rng.choice((1, 2, 3)) if n * (h + hk) * d < 30_000_000 else 1
        return _rotary(None, b, n, h, hk, d, dtype, rotary=rotary, interleaved=rng.random() < 0.4,
                       norm=rng.random() < 0.8, start=rng.choice((0, size(1, 1_000_000))), fused=rng.random() < 0.6,
                       train=train)
    d = rng.choice((32, 64, 64, 128, 128, 8 * size(1, 16)))
    hk = size(1, 16)
    h = hk * rng.choice((1, 1, 2, 4, 8))
    v = size(1, 16384)
    bias = rng.choice((0, 0, 1, 2))
    # the work of the long case, a quarter of it in full precision, a fourth where there are gradients
    most = 4096 * 8192 * 32 * 128 // (h * d * v) // (4 if dtype == "fp32" else 1) // (4 if train else 1)
    cells = 4096 * 8192 * 32 // (2 if train or bias else 1) // (h * v)
    u = 1 if rng.random() < 0.25 else size(1, max(1, min(8192, most, cells)))
    b = max(1, min(rng.choice((1, 2, 4, 8)), most // u, cells // u, 400_000_000 // (v * hk * d * SIZE[dtype])))
    pad = rng.random() < 0.6
    return _cross(None, b, u, v, h, hk, d, dtype, pad=pad, empty=pad and rng.random() < 0.3, bias=bias, train=train)


# ------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Valid keys of each sequence: padded batches hold sequences of a half to the whole length."""
    b, v = case["b"], case["v"]
    if not case["pad"]:
        return [v] * b
    found = [v - i * v // (2 * b) for i in range(b)]
    if case["empty"]:
        found[b // 2] = 0
    return found


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)

    state = {"case": case}
    if case["op"] == "gated_linear":
        m, i, o = case["m"], case["i"], case["o"]
        both = normal(2 * o, i, scale=i ** -0.5)
        gate, up = (both[:o], both[o:]) if case["stacked"] else (both[:o].clone(), both[o:].clone())
        leaves = {"x": normal(m, i), "gate_weight": gate, "up_weight": up}
        if case["bias"]:
            leaves.update(gate_bias=normal(o, scale=0.1), up_bias=normal(o, scale=0.1))
        outs = [(m, o)]
    elif case["op"] == "qk_norm_rotary":
        b, n, h, hk, d = (case[k] for k in ("b", "n", "h", "hk", "d"))
        if case["fused"]:  # queries, keys and values of a token side by side
            heads = normal(b, n, h + 2 * hk, d)
            leaves = {"q": heads[:, :, :h], "k": heads[:, :, h:h + hk]}
        else:
            leaves = {"q": normal(b, n, h, d), "k": normal(b, n, hk, d)}
        if case["norm"]:
            leaves.update(q_weight=normal(d, scale=0.1, shift=1.0), k_weight=normal(d, scale=0.1, shift=1.0))
        # sequences begin at places of their own
        first = torch.randint(0, 1000, (b, 1), generator=g, device="cuda") + case["start"]
        state["pos"] = first + torch.arange(n, device="cuda")
        outs = [(b, n, h, d), (b, n, hk, d)]
    else:
        b, u, v, h, hk, d = (case[k] for k in ("b", "u", "v", "h", "hk", "d"))
        leaves = {"q": normal(b, u, h, d), "k": normal(b, v, hk, d), "v": normal(b, v, hk, d)}
        if case["bias"]:
            leaves["bias"] = normal(1 if case["bias"] == 1 else b, h, u, v)
        if case["pad"]:
            ends = torch.tensor(_lengths(case), device="cuda")
            state["mask"] = torch.arange(v, device="cuda") < ends[:, None]
        outs = [(b, u, h, d)]
    if case["train"]:
        state["douts"] = [normal(*s) for s in outs]
        for t in leaves.values():
            t.requires_grad_()
    return dict(state, leaves=leaves)


# --------------------------------------------------------------------------- the plain forms
def _activation(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return z


def _plain_gated(state, x, gate_weight, up_weight, gate_bias=None, up_bias=None):
    gate, up = x @ gate_weight.t(), x @ up_weight.t()
    if gate_bias is not None:
        gate, up = gate + gate_bias, up + up_bias
    return (_activation(gate, state["case"]["act"]) * up,)


def _plain_rotary(state, q, k, q_weight=None, k_weight=None):
    case = state["case"]
    r = case["rotary"]
    # angles of far positions need more than 32 bits
    j = torch.arange(r // 2, device=q.device, dtype=torch.float64)
    angle = state["pos"].double()[:, :, None, None] * BASE ** (-2.0 * j / r)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def one(x, weight):
        if case["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        turned, rest = x[..., :r], x[..., r:]
        if case["interleaved"]:
            a, c = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - c * sin, c * cos + a * sin], -1).flatten(-2)
        else:
            a, c = turned[..., :r // 2], turned[..., r // 2:]
            turned = torch.cat([a * cos - c * sin, c * cos + a * sin], -1)
        return torch.cat([turned, rest], -1)

    return one(q, q_weight), one(k, k_weight)


def _plain_cross(state, q, k, v, bias=None):
    case = state["case"]
    b, u, n, h, hk, d = (case[name] for name in ("b", "u", "v", "h", "hk", "d"))
    # [b, hk, h / hk * u, d] queries of a key head
    rows = q.view(b, u, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * u, d)
    keys, values = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    s = (rows @ keys.transpose(-1, -2).contiguous() * d ** -0.5).view(b, h, u, n)
    if bias is not None:
        s = s + bias
    if "mask" in state:
        s = s.masked_fill(~state["mask"][:, None, None, :], -math.inf)
    # a row whose mask leaves nothing has no maximum, and sums to zero
    top = s.detach().amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min)
    p = torch.exp(s - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).tiny)
    o = p.view(b, hk, h // hk * u, n) @ values
    return (o.view(b, hk, h // hk, u, d).permute(0, 3, 1, 2, 4).reshape(b, u, h, d),)


def _plain(state):
    case, leaves = state["case"], state["leaves"]
    form = {"gated_linear": _plain_gated, "qk_norm_rotary": _plain_rotary, "cross_attention": _plain_cross}[case["op"]]
    wide = {n: t.detach().float().requires_grad_(case["train"]) for n, t in leaves.items()}
    outs = form(state, **wide)
    dtype = DTYPES[case["dtype"]]
    found = [t.detach().to(dtype) for t in outs]
    if case["train"]:
        grads = torch.autograd.grad(outs, list(wide.values()), [t.float() for t in state["douts"]])
        found += [t.to(dtype) for t in grads]
    return found


# --------------------------------------------------------------------------------------- run
def _call(state):
    from geometric_nn_ops_torch.triangle import cross_attention, gated_linear, qk_norm_rotary

    case, leaves = state["case"], state["leaves"]
    if case["op"] == "gated_linear":
        act = None if case["act"] == "none" else case["act"]
        return (gated_linear(leaves["x"], leaves["gate_weight"], leaves["up_weight"], leaves.get("gate_bias"),
                             leaves.get("up_bias"), activation=act),)
    if case["op"] == "qk_norm_rotary":
        return qk_norm_rotary(leaves["q"], leaves["k"], state["pos"], q_weight=leaves.get("q_weight"),
                              k_weight=leaves.get("k_weight"), eps=EPS if case["norm"] else None, base=BASE,
                              rotary_dim=case["rotary"], interleaved=case["interleaved"])
    return (cross_attention(leaves["q"], leaves["k"], leaves["v"], leaves.get("bias"), state.get("mask")),)


def run(state):
    if not own:
        return _plain(state)
    if state["case"]["train"]:
        outs = _call(state)
        return [*outs, *torch.autograd.grad(outs, list(state["leaves"].values()), state["douts"])]
    with torch.inference_mode():
        return list(_call(state))


# -------------------------------------------------------------------------------------- work
def work(case):
    e, train = SIZE[case["dtype"]], case["train"]
    both = 2 if train else 1  # gradients of what is read go out
    if case["op"] == "gated_linear":
        m, i, o = case["m"], case["i"], case["o"]
        read = m * i + 2 * o * i + 2 * o * case["bias"]
        return {"bytes": (both * read + both * m * o) * e, "flops": (12 if train else 4) * m * i * o}
    if case["op"] == "qk_norm_rotary":
        cells = case["b"] * case["n"] * (case["h"] + case["hk"]) * case["d"]
        # x in, y out; dy in, dx out
        return {"bytes": 2 * both * cells * e + 8 * case["b"] * case["n"], "flops": (20 if train else 8) * cells}
    b, u, h, hk, d = (case[n] for n in ("b", "u", "h", "hk", "d"))
    held = sum(_lengths(case))
    q, kv, out = b * u * h * d, 2 * held * hk * d, b * u * h * d
    shared = case["bias"] == 1
    bias = (max(_lengths(case)) if shared else held) * h * u if case["bias"] else 0
    return {"bytes": (both * (q + kv + bias) + both * out) * e + (b * case["v"] if case["pad"] else 0),
            "flops": (14 if train else 4) * held * u * h * d}


# ------------------------------------------------------------------------------------- exact
def _exact_gated(case, douts, x, gate_weight, up_weight, gate_bias=None, up_bias=None):
    zg, zu = (torch.mm(x, w.t().contiguous()) for w in (gate_weight, up_weight))
    if gate_bias is not None:
        zg, zu = zg + gate_bias, zu + up_bias
    s = torch.sigmoid(zg)
    if case["act"] == "relu":
        a, slope = zg.clamp(min=0), (zg > 0).double()
    elif case["act"] == "gelu":
        phi = torch.special.ndtr(zg)
        a, slope = zg * phi, phi + zg * torch.exp(-0.5 * zg * zg) / math.sqrt(2 * math.pi)
    elif case["act"] == "silu":
        a, slope = zg * s, s * (1 + zg * (1 - s))
    elif case["act"] == "sigmoid":
        a, slope = s, s * (1 - s)
    else:
        a, slope = zg, torch.ones_like(zg)
    out = [a * zu]
    if not douts:
        return out
    dg, du = douts[0] * zu * slope, douts[0] * a
    out += [torch.mm(dg, gate_weight) + torch.mm(du, up_weight), torch.mm(dg.t().contiguous(), x),
            torch.mm(du.t().contiguous(), x)]
    return out + ([dg.sum(0), du.sum(0)] if gate_bias is not None else [])


def _exact_rotary(case, pos, douts, q, k, q_weight=None, k_weight=None):
    """Pairs as complex numbers, turned by exp(i angle); back by its conjugate."""
    r = case["rotary"]
    j = torch.arange(0, r, 2, device=pos.device, dtype=torch.float64)
    turn = torch.polar(torch.ones_like(j), pos.double()[..., None] * torch.exp(-j / r * math.log(BASE)))[:, :, None]

    def pairs(x):
        at = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        return torch.complex(*(t.contiguous() for t in at))

    def whole(z, x):
        y = x.clone()
        if case["interleaved"]:
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        else:
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        return y

    outs, grads, weights = [], [], []
    for n, (x, w) in enumerate(((q, q_weight), (k, k_weight))):
        size = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).rsqrt() if case["norm"] else 1.0
        xh = x * size
        y = xh * w if case["norm"] else xh
        outs.append(whole(pairs(y) * turn, y))
        if douts:
            dy = whole(pairs(douts[n]) * turn.conj(), douts[n])
            if case["norm"]:
                weights.append((dy * xh).sum((0, 1, 2)))
                dy = dy * w
                dy = size * (dy - xh * (dy * xh).mean(-1, keepdim=True))
            grads.append(dy)
    return outs + grads + weights


def _exact_cross(case, douts, q, k, v, bias=None):
    """Head by head, over the keys that a sequence holds; gradients by their formulas."""
    b, u, h, hk, d = (case[n] for n in ("b", "u", "h", "hk", "d"))
    o, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dbias = torch.zeros_like(bias) if bias is not None and douts else None
    for i, held in enumerate(_lengths(case)):
        for n in range(h if held else 0):
            m, at = n * hk // h, (0 if case["bias"] == 1 else i, n)
            qs, ks, vs = q[i, :, n].contiguous(), k[i, :held, m].contiguous(), v[i, :held, m].contiguous()
            s = torch.mm(qs, ks.t().contiguous()) / math.sqrt(d)
            if bias is not None:
                s = s + bias[at][:, :held]
            p = torch.softmax(s, -1)
            o[i, :, n] = torch.mm(p, vs)
            if douts:
                do = douts[0][i, :, n].contiguous()
                dv[i, :held, m] += torch.mm(p.t().contiguous(), do)
                dp = torch.mm(do, vs.t().contiguous())
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dq[i, :, n] = torch.mm(ds, ks) / math.sqrt(d)
                dk[i, :held, m] += torch.mm(ds.t().contiguous(), qs) / math.sqrt(d)
                if dbias is not None:
                    dbias[at][:, :held] += ds
    if not douts:
        return [o]
    return [o, dq, dk, dv] + ([dbias] if dbias is not None else [])


def exact(case, seed):
    state = prepare(case, seed)
    wide = {n: t.detach().double() for n, t in state["leaves"].items()}
    douts = [t.double() for t in state.get("douts", ())]
    if case["op"] == "qk_norm_rotary":
        return _exact_rotary(case, state["pos"], douts, **wide)
    return (_exact_gated if case["op"] == "gated_linear" else _exact_cross)(case, douts, **wide)
