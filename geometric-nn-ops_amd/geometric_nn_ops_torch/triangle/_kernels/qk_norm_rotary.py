"""Host side of the HIP per-head norms with rotary positions: ``qk_norm_rotary_hip`` and the gradients,
``qk_norm_rotary_bwd_hip``. Positions come as ``[B or 1, N]`` of one integer dtype, or None."""

import ctypes
import functools

import torch

from ... import _lib

MAX_HEAD_DIM = 256


def supports(q, k, rotary_dim: int) -> bool:
    """Whether the HIP kernels cover these shapes (dtype handled by the caller)."""
    d = q.shape[-1]
    if d % 8 or not 8 <= d <= MAX_HEAD_DIM or rotary_dim % 8:
        return False
    # heads of a side, and workgroups, are numbered in 31 bits
    return max(q.shape[2], k.shape[2]) <= 1 << 20 and max(q.numel(), k.numel()) // d < 1 << 34


@functools.lru_cache(maxsize=256)
def _host(frequencies):
    return (ctypes.c_double * max(1, len(frequencies)))(*frequencies)


def _rows(t):
    """Unit stride over the head dim, the other strides as they are."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _pos(t):
    """Address and batch stride of positions with unit stride along the tokens."""
    if t is None:
        return None, 0
    if t.stride(1) != 1 and t.shape[1] != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else 0


def _call(fn, q, k, dys, pos, weights, outs, dweights, parts, partial, eps, frequencies, interleaved):
    B, U, H, D = q.shape
    V, Hk = k.shape[1:3]
    (q_pos, q_ps), (k_pos, k_ps) = _pos(pos[0]), _pos(pos[1])
    weights = [None if w is None else w.contiguous() for w in weights]
    w = next((t for t in weights if t is not None), q)
    p = q_pos if q_pos is not None else k_pos
    host = _host(frequencies)
    none = (0, 0, 0)
    a = _lib.QkRotaryArgs()
    _lib.pack_qk_rotary(
        a, 0, q.data_ptr(), k.data_ptr(), *(0 if t is None else t.data_ptr() for t in (*dys, *weights, q_pos, k_pos,
                                                                                       *outs, *dweights)),
        ctypes.addressof(host), 0 if partial is None else partial.data_ptr(), B, U, V, H, Hk, D, 2 * len(frequencies),
        *q.stride()[:3], *k.stride()[:3], *(none if dys[0] is None else dys[0].stride()[:3]),
        *(none if dys[1] is None else dys[1].stride()[:3]), q_ps, k_ps, *parts, 0.0 if eps is None else eps,
        eps is not None, interleaved, 4 if p is None else p.element_size(), _lib.DTYPE_CODE[q.dtype],
        _lib.DTYPE_CODE[w.dtype])
    if fn is None:
        lib = _lib.load()
        return [lib.gnn_qk_rotary_parts(ctypes.byref(a), side) for side in (0, 1)]
    _lib.call(fn, a, q.device)
    return None


def qk_norm_rotary_hip(q, k, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved):
    """``(q', k')``, fresh and contiguous."""
    outs = [torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k)]
    if q.numel() or k.numel():
        _call("gnn_qk_rotary_fwd", _rows(q), _rows(k), (None, None), (q_pos, k_pos), (q_weight, k_weight), outs,
              (None, None), (0, 0), None, eps, frequencies, interleaved)
    return tuple(outs)


def qk_norm_rotary_bwd_hip(q, k, dq, dk, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved, need):
    """``(dq, dk, dq_weight, dk_weight)``, None where ``need`` says so, from the output gradients (None: zeros)."""
    xs, dys = [q, k], [dq, dk]
    found = [torch.empty(t.shape, device=t.device, dtype=t.dtype) if n else None for t, n in zip(xs, need[:2])]
    dws = [torch.empty(w.shape, device=w.device, dtype=w.dtype) if n else None
           for w, n in zip((q_weight, k_weight), need[2:])]
    for i in range(2):
        if dys[i] is None or not xs[i].numel():
            for t in (found[i], dws[i]):
                if t is not None:
                    t.zero_()
            xs[i], dys[i] = xs[i][:, :0], None  # nothing of this side in the call
    runs = [xs[i].numel() > 0 and (found[i] is not None or dws[i] is not None) for i in range(2)]
    if any(runs):
        xs, dys = [_rows(t) for t in xs], [None if t is None else _rows(t) for t in dys]
        args = (*xs, dys, (q_pos, k_pos), (q_weight, k_weight), [t if r else None for t, r in zip(found, runs)],
                [t if r else None for t, r in zip(dws, runs)])
        parts = _call(None, *args, (1, 1), None, eps, frequencies, interleaved)
        rows = sum(n for n, t, r in zip(parts, dws, runs) if r and t is not None)
        partial = torch.empty((rows, q.shape[-1]), device=q.device, dtype=torch.float32) if rows else None
        _call("gnn_qk_rotary_bwd", *args, [max(1, n) for n in parts], partial, eps, frequencies, interleaved)
    return (*found, *dws)
