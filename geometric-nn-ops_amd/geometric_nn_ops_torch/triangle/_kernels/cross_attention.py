"""Host side of the HIP attention over states of another length: ``cross_attention_hip`` and the gradients,
``cross_attention_bwd_hip``."""

import ctypes

import torch

from ... import _lib

MAX_HEAD_DIM = 128
_FAR = 1 << 31  # bytes


def supports(q, k) -> bool:
    """Whether the HIP kernels cover these shapes (dtype handled by the caller)."""
    B, U, H, D = q.shape
    if D % 8 or not 8 <= D <= MAX_HEAD_DIM:
        return False
    # rows, keys and workgroups are numbered in 31 bits
    (V, Hk) = k.shape[1:3]
    row_blocks, key_blocks = Hk * ((U * H // Hk + 127) // 128), Hk * ((V + 127) // 128)
    return (H * D < 1 << 22 and B * U * H < 1 << 30 and V <= 1 << 29 and B * max(row_blocks, key_blocks) < 1 << 30
            and row_blocks * ((V + 63) // 64) < 1 << 31)


def _heads(t, group=1):
    """Unit stride over the head dim, the other strides as they are; a copy too where 64 rows of one product, tokens of
    ``group`` heads each, lie 2 GiB apart: the kernels count them in 32 bits."""
    s = t.stride()
    if s[3] == 1 and 64 * s[1] + (group - 1) * s[2] < _FAR // t.element_size():
        return t
    return t.contiguous()


def _bias(t, batch):
    """A bias with unit stride over the keys, and its strides (0 over the batch where one goes with all)."""
    if t is None:
        return None, (0, 0, 0)
    if t.stride(3) != 1 and t.shape[3] != 1:
        t = t.contiguous()
    s = t.stride()
    return t, (0 if t.shape[0] == 1 else s[0], s[1], s[2])


def cross_attention_hip(q, k, v, bias, mask, scale, *, precision, keep=False):
    """``[B, U, H, D]``, fresh and contiguous; with ``keep`` ``(out, low, stats)``: what the rounding of a
    16-bit output left (``None`` in fp32) and what the backward needs of the rows' sums, fp32 ``[B, H, U, 2]``."""
    (B, U, H, D), (V, Hk) = q.shape, k.shape[1:3]
    out = torch.empty((B, U, H, D), device=q.device, dtype=q.dtype)
    low = torch.empty_like(out) if keep and q.dtype is not torch.float32 else None
    stats = torch.empty((B, H, U, 2), device=q.device, dtype=torch.float32) if keep else None
    if not out.numel() or not V:
        out.zero_()
        return (out, low, stats) if keep else out
    q, k, v = _heads(q, H // Hk), _heads(k), _heads(v)
    bias, bs = _bias(bias, B)
    a = _lib.CrossAttnArgs()
    _lib.pack_cross_attn(
        a, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if mask is None else mask.data_ptr(), out.data_ptr(), 0 if low is None else low.data_ptr(),
        0 if stats is None else stats.data_ptr(), 0, 0, B, U, V, H, Hk, D,
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *bs, *((0, 0) if mask is None else mask.stride()), scale,
        _lib.DTYPE_CODE[q.dtype], _lib.PRECISION_CODE[precision], 0)
    size = (_lib._lib or _lib.load()).gnn_cross_attn_workspace_bytes(ctypes.byref(a))
    if size:
        ws = torch.empty(size, device=q.device, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
    _lib.call("gnn_cross_attn_fwd", a, q.device)
    return (out, low, stats) if keep else out


def cross_attention_bwd_hip(q, k, v, bias, mask, out, low, stats, dout, scale, *, precision, need_kv=True, need_bias=True):
    """``(dq, dk, dv, dbias)``; dk and dv None unless ``need_kv``, dbias unless ``need_bias``."""
    (B, U, H, D), (V, Hk) = q.shape, k.shape[1:3]
    dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) if need_kv else None for t in (k, v))
    dbias = torch.empty(bias.shape, device=q.device, dtype=q.dtype) if need_bias else None
    if not q.numel() or not k.numel():
        for t in (dq, dk, dv, dbias):
            if t is not None:
                t.zero_()
        return dq, dk, dv, dbias
    k, v = _heads(k), _heads(v)
    q, out, dout = (_heads(t, H // Hk) for t in (q, out, dout))
    stats, low = stats.contiguous(), None if low is None else low.contiguous()  # in whatever layout saved-tensor hooks return them
    bias, bs = _bias(bias, B)
    a = _lib.CrossAttnBwdArgs()
    _lib.pack_cross_attn_bwd(
        a, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if low is None else low.data_ptr(), dout.data_ptr(),
        0 if bias is None else bias.data_ptr(), 0 if mask is None else mask.data_ptr(), stats.data_ptr(), dq.data_ptr(),
        0 if dk is None else dk.data_ptr(), 0 if dv is None else dv.data_ptr(), 0 if dbias is None else dbias.data_ptr(), 0,
        0, B, U, V, H, Hk, D, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *dout.stride()[:3], *bs,
        *((0, 0) if mask is None else mask.stride()), scale, _lib.DTYPE_CODE[q.dtype], _lib.PRECISION_CODE[precision],
        bias is not None and bias.shape[0] == 1)
    size = _lib.load().gnn_cross_attn_bwd_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(size, device=q.device, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    _lib.call("gnn_cross_attn_bwd", a, q.device)
    return dq, dk, dv, dbias
