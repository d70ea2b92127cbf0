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
    """Positions with unit stride along the tokens, and their batch stride."""
    if t.stride(1) != 1 and t.shape[1] != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else 0


def _args(q, k, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved, outs, dys=(None, None)):
    """The call's arguments and what they point to, from rows of unit stride."""
    B, U, H, D = q.shape
    V, Hk = k.shape[1:3]
    qp = kp = qs = ks = 0
    pos_bytes = 4
    if q_pos is not None:
        shared = k_pos is q_pos
        q_pos, qs = _pos(q_pos)
        qp, pos_bytes = q_pos.data_ptr(), q_pos.element_size()
        if shared:
            k_pos, kp, ks = q_pos, qp, qs
    if k_pos is not None and not kp:
        k_pos, ks = _pos(k_pos)
        kp, pos_bytes = k_pos.data_ptr(), k_pos.element_size()
    qw = kw = 0
    dtype = param = _lib.DTYPE_CODE[q.dtype]
    if q_weight is not None:
        q_weight = q_weight.contiguous()
        qw, param = q_weight.data_ptr(), _lib.DTYPE_CODE[q_weight.dtype]
    if k_weight is not None:
        k_weight = k_weight.contiguous()
        kw, param = k_weight.data_ptr(), _lib.DTYPE_CODE[k_weight.dtype]
    host = _host(frequencies)
    (dq, dk), (oq, ok) = dys, outs
    a = _lib.QkRotaryArgs()
    _lib.pack_qk_rotary(
        a, 0, q.data_ptr(), k.data_ptr(), 0 if dq is None else dq.data_ptr(), 0 if dk is None else dk.data_ptr(), qw, kw, qp,
        kp, 0 if oq is None else oq.data_ptr(), 0 if ok is None else ok.data_ptr(), 0, 0, ctypes.addressof(host), 0, B, U, V,
        H, Hk, D, 2 * len(frequencies), *q.stride()[:3], *k.stride()[:3], *((0, 0, 0) if dq is None else dq.stride()[:3]),
        *((0, 0, 0) if dk is None else dk.stride()[:3]), qs, ks, 1, 1, 0.0 if eps is None else eps, eps is not None, interleaved, pos_bytes, dtype, param)
    return a, (q_pos, k_pos, q_weight, k_weight, host)


def qk_norm_rotary_hip(q, k, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved):
    """``(q', k')``, fresh and contiguous."""
    outs = (torch.empty(q.shape, device=q.device, dtype=q.dtype), torch.empty(k.shape, device=k.device, dtype=k.dtype))
    if q.numel() or k.numel():
        q, k = _rows(q), _rows(k)
        a, kept = _args(q, k, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved, outs)
        _lib.call("gnn_qk_rotary_fwd", a, q.device)
    return outs


def qk_norm_rotary_bwd_hip(q, k, dq, dk, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved, need):
    """``(dq, dk, dq_weight, dk_weight)``, None where ``need`` says so, from the output gradients (None: zeros)."""
    device, D = q.device, q.shape[3]
    gq = torch.empty(q.shape, device=device, dtype=q.dtype) if need[0] else None
    gk = torch.empty(k.shape, device=device, dtype=k.dtype) if need[1] else None
    gqw = torch.empty((D,), device=device, dtype=q_weight.dtype) if need[2] else None
    gkw = torch.empty((D,), device=device, dtype=k_weight.dtype) if need[3] else None
    if dq is None or not q.numel():  # nothing of this side in the call
        for t in (gq, gqw):
            if t is not None:
                t.zero_()
        q, dq = q[:, :0], None
    if dk is None or not k.numel():
        for t in (gk, gkw):
            if t is not None:
                t.zero_()
        k, dk = k[:, :0], None
    if not ((dq is not None and (need[0] or need[2])) or (dk is not None and (need[1] or need[3]))):
        return gq, gk, gqw, gkw
    q, k = _rows(q), _rows(k)
    dq, dk = None if dq is None else _rows(dq), None if dk is None else _rows(dk)
    a, kept = _args(q, k, q_pos, k_pos, q_weight, k_weight, eps, frequencies, interleaved, (gq, gk), (dq, dk))
    lib, ref, rows = _lib.load(), ctypes.byref(a), 0
    for side, (t, dy) in enumerate(((gqw, dq), (gkw, dk))):
        if dy is None:
            continue
        a.parts[side] = parts = lib.gnn_qk_rotary_parts(ref, side)
        if t is not None:
            a.dweight[side] = t.data_ptr()
            rows += parts
    if rows:
        partial = torch.empty((rows, D), device=device, dtype=torch.float32)
        a.partial = partial.data_ptr()
    _lib.call("gnn_qk_rotary_bwd", a, device)
    return gq, gk, gqw, gkw
