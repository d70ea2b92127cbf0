"""The operators around a pairformer's triangle updates: layer_norm, fused_linear and relative_position_bias.

A case is a dict of plain values; "op" names the operator. "train" asks for the forward with everything
requiring grad and for the gradients of a given output gradient; otherwise the forward runs under
inference_mode. "dtype" is the type of every floating tensor, but "wdtype" that of a LayerNorm's parameters.

  layer_norm              rows x k; "params" is "both", "weight" or "none"; "view": x is a column slice of
                          wider rows, as one part of a stacked projection is
  fused_linear            m x i -> o; "act" is "none", "relu", "gelu", "silu" or "sigmoid"
  relative_position_bias  b x u queries against v keys, h heads, "buckets" rows in the table; positions
                          ascend with gaps (chain breaks); "last" has the heads last, as the pair stream does
"""

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "geometric-nn-ops_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(name, rows, k, dtype="bf16", *, train=False, wdtype=None, params="both", view=False):
    c = {"op": "layer_norm", "rows": rows, "k": k, "dtype": dtype, "wdtype": wdtype or dtype, "params": params,
         "train": train, "view": view}
    return dict(c, name=name) if name else c


def _linear(name, m, i, o, dtype="bf16", *, act="none", bias=True, residual=False, train=False):
    c = {"op": "fused_linear", "m": m, "i": i, "o": o, "dtype": dtype, "act": act, "bias": bias, "residual": residual,
         "train": train}
    return dict(c, name=name) if name else c


def _relpos(name, u, v, h, buckets, dtype="bf16", *, b=1, spacing="log", distance=128, two_sided=True, last=False,
            train=False):
    c = {"op": "relative_position_bias", "b": b, "u": u, "v": v, "h": h, "buckets": buckets, "dtype": dtype,
         "spacing": spacing, "distance": distance, "two_sided": two_sided, "last": last, "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the single track of an ordinary crop before its attention: the call costs more than the kernel
        _norm("norm_single_n384_bf16", 384, 384),
        # the pair stream before an update, in training at the usual crop, parameters kept in 32 bits
        _norm("norm_train_pair_n384_bf16", 384 * 384, 128, train=True, wdtype="fp32"),
        # wide rows of an odd width, in training
        _norm("norm_train_wide_k5003_fp16", 8191, 5003, "fp16", train=True),
        # one token through the first layer of a single-track transition
        _linear("linear_token_c384_bf16", 1, 384, 1536, act="gelu"),
        # first layer of the pair transition, inference on an ordinary protein
        _linear("linear_pair_up_n512_bf16", 512 * 512, 128, 512, act="relu"),
        # the same layer in training at the usual crop
        _linear("linear_train_up_n384_bf16", 384 * 384, 128, 512, act="silu", train=True),
        # the transition's second layer, which adds to the stream, in training
        _linear("linear_train_down_n384_bf16", 384 * 384, 512, 128, residual=True, train=True),
        # full precision at odd widths, in training
        _linear("linear_train_odd_fp32", 201 * 201, 131, 257, "fp32", act="silu", residual=True, train=True),
        # a wide layer, where the matrix units bound the call
        _linear("linear_wide_4096_bf16", 8192, 4096, 4096, act="gelu", residual=True),
        # one new query per sequence against the keys so far, which all lie before it
        _relpos("relpos_decode_v8191_bf16", 1, 8191, 16, 32, b=4, two_sided=False),
        # the bias of self attention over a long sequence, in training
        _relpos("relpos_train_n2048_bf16", 2048, 2048, 16, 32, train=True),
        # the clipped residue offsets that seed the pair stream, in training at a large odd crop
        _relpos("relpos_train_pair_n509_bf16", 509, 509, 128, 65, spacing="clip", distance=32, last=True, train=True),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(("layer_norm", "fused_linear", "fused_linear", "relative_position_bias"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    train = rng.random() < 0.5
    if op == "layer_norm":
        k = rng.choice((64, 128, 256, 384, 768, size(8, 8192), size(8, 8192)))
        rows = size(1, min(400000, 320_000_000 // ((4 if train else 2) * SIZE[dtype] * k)))
        return _norm(None, rows, k, dtype, train=train, wdtype=rng.choice((dtype, "fp32")),
                     params=rng.choice(("both", "both", "weight", "none")), view=rng.random() < 0.3)
    if op == "fused_linear":
        i, o = (rng.choice((128, 256, 384, 512, 1024, size(16, 4096), size(16, 4096))) for _ in range(2))
        # the work of the wide case, a quarter of it in full precision, a third where there are gradients
        most = 8192 * 4096 * 4096 // (i * o) // (4 if dtype == "fp32" else 1) // (3 if train else 1)
        m = size(1, max(1, min(262144, most, 400_000_000 // ((3 if train else 1) * SIZE[dtype] * (i + 2 * o)))))
        return _linear(None, m, i, o, dtype, act=rng.choice(("none", "relu", "gelu", "silu", "sigmoid")),
                       bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=train)
    b = rng.choice((1, 1, 2))
    last = rng.random() < 0.4
    h = size(8, 192) if last else size(1, 32)
    most = 260_000_000 // ((2 if train else 1) * SIZE[dtype] * b * h)
    v = size(1, min(8192, most))
    u = min(v, size(1, min(8192, max(1, most // v))))
    two_sided = rng.random() < 0.6
    if rng.random() < 0.5:
        distance = size(1, 64)
        return _relpos(None, u, v, h, (2 if two_sided else 1) * distance + 1, dtype, b=b, spacing="clip",
                       distance=distance, two_sided=two_sided, last=last, train=train)
    buckets = rng.choice((8, 16, 32, 32, 64))
    return _relpos(None, u, v, h, buckets, dtype, b=b, distance=size(buckets, 2000), two_sided=two_sided, last=last,
                   train=train)


# ------------------------------------------------------------------------------------ inputs
def _borders(case):
    """The distances at which the logarithmic part of the table goes on to its next bucket: with n buckets on
    a side and e = n // 2 of them for exact distances, the least d with d >= e * (distance / e) ** (k / (n - e))
    for k = 1 .. n - e - 1, in whole numbers."""
    n = case["buckets"] // (2 if case["two_sided"] else 1)
    e, far = n // 2, case["distance"]
    m = n - e
    found = []
    for k in range(1, m):
        d = int(e * (far / e) ** (k / m))
        while d ** m >= e ** (m - k) * far ** k:
            d -= 1
        while d ** m < e ** (m - k) * far ** k:
            d += 1
        found.append(d)
    return found


def _positions(g, b, n):
    """Residue numbers of b sequences: ascending by one, now and then with a gap."""
    step = 1 + 40 * (torch.rand(b, n, generator=g, device="cuda") < 0.004).long()
    return torch.cumsum(step, 1) - 1


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=case["dtype"], scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(DTYPES[dtype])

    state = {"case": case}
    if case["op"] == "layer_norm":
        rows, k = case["rows"], case["k"]
        # channels of the stream differ in scale and offset
        wide = torch.randn(rows, 2 * k + 8 if case["view"] else k, generator=g, device="cuda")
        wide.mul_(0.5 + torch.rand(wide.shape[1], generator=g, device="cuda")).add_(0.3)
        x = wide.to(DTYPES[case["dtype"]])
        leaves = {"x": x[:, k:2 * k] if case["view"] else x}
        if case["params"] != "none":
            leaves["weight"] = normal(k, dtype=case["wdtype"], scale=0.1, shift=1.0)
        if case["params"] == "both":
            leaves["bias"] = normal(k, dtype=case["wdtype"], scale=0.1)
        out = (rows, k)
    elif case["op"] == "fused_linear":
        m, i, o = case["m"], case["i"], case["o"]
        leaves = {"x": normal(m, i), "weight": normal(o, i, scale=i ** -0.5)}
        if case["bias"]:
            leaves["bias"] = normal(o, scale=0.1)
        if case["residual"]:
            leaves["residual"] = normal(m, o)
        out = (m, o)
    else:
        b, u, v, h = (case[n] for n in ("b", "u", "v", "h"))
        leaves = {"weight": normal(case["buckets"], h)}
        key = _positions(g, b, v)
        state.update(key_pos=key, query_pos=key[:, v - u:].contiguous())
        # a program that looks the table up by hand keeps the borders on the device
        state["borders"] = torch.tensor(_borders(case) if case["spacing"] == "log" else [0], device="cuda")
        out = (b, u, v, h) if case["last"] else (b, h, u, v)
    if case["train"]:
        state["dout"] = normal(*out)
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


def _plain_norm(case, x, weight=None, bias=None):
    d = x - x.mean(-1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5)
    y = y if weight is None else y * weight
    return y if bias is None else y + bias


def _plain_linear(case, x, weight, bias=None, residual=None):
    z = x @ weight.t()
    y = _activation(z if bias is None else z + bias, case["act"])
    return y if residual is None else y + residual


def _plain_buckets(state):
    """[b, u, v] rows of the table."""
    case = state["case"]
    far = case["distance"]
    ahead = state["key_pos"][:, None, :] - state["query_pos"][:, :, None]
    if case["spacing"] == "clip":
        return ahead.clamp(-far, far) + far if case["two_sided"] else (-ahead).clamp(0, far)
    n = case["buckets"] // (2 if case["two_sided"] else 1)
    d = ahead.abs() if case["two_sided"] else (-ahead).clamp(min=0)
    near = n // 2
    side = torch.where(d < near, d, near + torch.bucketize(d, state["borders"], right=True))
    return side + n * (ahead > 0) if case["two_sided"] else side


def _plain_relpos(state):
    case, weight = state["case"], state["leaves"]["weight"]
    rows = _plain_buckets(state)
    out = weight.detach()[rows]
    out = out if case["last"] else out.permute(0, 3, 1, 2).contiguous()
    if not case["train"]:
        return out
    # a bucket's gradient sums up to millions of values: a query's keys in 32 bits, the queries in 64
    dout = state["dout"] if case["last"] else state["dout"].permute(0, 2, 3, 1)
    hit = (rows[:, :, None, :] == torch.arange(case["buckets"], device=rows.device)[:, None]).float()
    return out, torch.matmul(hit, dout.float().contiguous()).double().sum((0, 1)).to(weight.dtype)


def _plain(state):
    case, leaves = state["case"], state["leaves"]
    if case["op"] == "relative_position_bias":
        return _plain_relpos(state)
    form = _plain_norm if case["op"] == "layer_norm" else _plain_linear
    wide = {n: t.detach().float().requires_grad_(case["train"]) for n, t in leaves.items()}
    y = form(case, **wide)
    out = y.detach().to(leaves["x"].dtype)
    if not case["train"]:
        return out
    grads = torch.autograd.grad(y, list(wide.values()), state["dout"].float())
    return (out, *(d.to(t.dtype) for d, t in zip(grads, leaves.values())))


# --------------------------------------------------------------------------------------- run
def _call(state):
    from geometric_nn_ops_torch.triangle import fused_linear, layer_norm, relative_position_bias

    case, leaves = state["case"], state["leaves"]
    if case["op"] == "layer_norm":
        return layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"))
    if case["op"] == "fused_linear":
        return fused_linear(leaves["x"], leaves["weight"], leaves.get("bias"), residual=leaves.get("residual"),
                            activation=None if case["act"] == "none" else case["act"])
    return relative_position_bias(leaves["weight"], state["query_pos"], state["key_pos"], max_distance=case["distance"],
                                  spacing=case["spacing"], bidirectional=case["two_sided"], channels_last=case["last"])


def run(state):
    if not own:
        return _plain(state)
    if state["case"]["train"]:
        out = _call(state)
        return (out, *torch.autograd.grad(out, list(state["leaves"].values()), state["dout"]))
    with torch.inference_mode():
        return _call(state)


# -------------------------------------------------------------------------------------- work
def work(case):
    e, train = SIZE[case["dtype"]], case["train"]
    if case["op"] == "layer_norm":
        rows, k = case["rows"], case["k"]
        count = {"both": 2, "weight": 1, "none": 0}[case["params"]] * k * SIZE[case["wdtype"]]
        # x in, y out; dy in, dx out
        return {"bytes": (4 if train else 2) * rows * k * e + (2 if train else 1) * count,
                "flops": (19 if train else 8) * rows * k}
    if case["op"] == "fused_linear":
        m, i, o = case["m"], case["i"], case["o"]
        weights = i * o + case["bias"] * o
        moved = m * i + weights + m * o * (1 + case["residual"])
        if train:  # dout in; dx and the weights' gradients out; the residual's gradient is dout
            moved += m * o + m * i + weights
        return {"bytes": moved * e, "flops": (6 if train else 2) * m * i * o}
    cells = case["b"] * case["u"] * case["v"]
    table = case["buckets"] * case["h"] * e
    return {"bytes": (2 if train else 1) * (cells * case["h"] * e + table) + 8 * case["b"] * (case["u"] + case["v"]),
            "flops": cells * case["h"] if train else 0}


# ------------------------------------------------------------------------------------- exact
def _exact_norm(case, dy, x, weight=None, bias=None):
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    r = torch.rsqrt(var + 1e-5)
    xh = (x - mean) * r
    w = 1.0 if weight is None else weight
    y = xh * w + (0.0 if bias is None else bias)
    if dy is None:
        return y
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    grads = [dx]
    if weight is not None:
        grads.append((dy * xh).sum(0))
    if bias is not None:
        grads.append(dy.sum(0))
    return (y, *grads)


def _exact_linear(case, dy, x, weight, bias=None, residual=None):
    z = torch.mm(x, weight.t().contiguous())
    if bias is not None:
        z = z + bias
    s = torch.sigmoid(z)
    if case["act"] == "relu":
        y, slope = z.clamp(min=0), (z > 0).double()
    elif case["act"] == "gelu":
        phi = torch.special.ndtr(z)
        y, slope = z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    elif case["act"] == "silu":
        y, slope = z * s, s * (1 + z * (1 - s))
    elif case["act"] == "sigmoid":
        y, slope = s, s * (1 - s)
    else:
        y, slope = z, torch.ones_like(z)
    if residual is not None:
        y = y + residual
    if dy is None:
        return y
    dz = dy * slope
    grads = [torch.mm(dz, weight), torch.mm(dz.t().contiguous(), x)]
    if bias is not None:
        grads.append(dz.sum(0))
    if residual is not None:
        grads.append(dy)
    return (y, *grads)


def _exact_relpos(case, weight, query, key, dout):
    """Bucket by bucket of the distance, looked up in a list that whole-number arithmetic fills."""
    far, two = case["distance"], case["two_sided"]
    n = case["buckets"] // (2 if two else 1)
    near = n // 2
    if case["spacing"] == "clip":
        side = list(range(far + 1))
    else:
        m = n - near
        power = [near ** (m - k) * far ** k for k in range(m)]
        side = [d if d < near else near + sum(d ** m >= p for p in power[1:]) for d in range(far + 1)]
    side = torch.tensor(side, device=weight.device)
    ahead = (key[:, None, :] - query[:, :, None]).clamp(-far, far)
    behind = side[(-ahead).clamp(min=0)]
    if not two:
        rows = behind
    elif case["spacing"] == "clip":
        rows = far + ahead
    else:
        rows = torch.where(ahead > 0, n + side[ahead.clamp(min=0)], behind)
    heads = [weight[:, h][rows] for h in range(case["h"])]
    out = torch.stack(heads, -1 if case["last"] else 1)
    if dout is None:
        return out
    # the pixels in the order of their buckets: a bucket's sum is a difference of running sums
    at, order = torch.sort(rows.reshape(-1))
    ends = torch.searchsorted(at, torch.arange(case["buckets"], device=at.device), right=True)
    grads = []
    for h in range(case["h"]):
        running = torch.cumsum((dout[..., h] if case["last"] else dout[:, h]).reshape(-1).double()[order], 0)
        upto = torch.cat([running.new_zeros(1), running])[ends]
        grads.append(torch.diff(upto, prepend=upto.new_zeros(1)))
    return out, torch.stack(grads, 1)


def exact(case, seed):
    state = prepare(case, seed)
    wide = {n: t.detach().double() for n, t in state["leaves"].items()}
    dout = state.get("dout")
    if case["op"] == "relative_position_bias":
        return _exact_relpos(case, wide["weight"], state["query_pos"], state["key_pos"], dout)
    form = _exact_norm if case["op"] == "layer_norm" else _exact_linear
    return form(case, None if dout is None else dout.double(), **wide)
