"""Host side of the HIP relative position bias: ``relative_position_bias_hip`` and the table's gradient,
``relative_position_bias_bwd_hip``. Positions come as ``[B, U]`` / ``[B, V]`` of one integer dtype."""

import ctypes
import functools

import torch

from ... import _lib
from .._reference.relative_position import log_borders, side_buckets

MAX_BUCKETS = 4096
MAX_BORDERS = 256  # logarithmic buckets of a side


def supports(weight, query_pos, key_pos, max_distance, spacing, bidirectional) -> bool:
    """Whether the HIP kernels cover the call (dtype handled by the caller)."""
    buckets, heads = weight.shape
    if buckets > MAX_BUCKETS or max_distance > 1 << 28:
        return False
    # rows, and 64-element pieces of rows, are numbered in 32 bits
    row, rows = key_pos.shape[1] * heads, query_pos.shape[0] * query_pos.shape[1]
    if row >= (1 << 31) - 4096 or rows * ((row + 63) // 64 + 1) >= 1 << 31:
        return False
    if spacing == "clip":
        return True
    n, near = side_buckets(buckets, bidirectional)
    return n - near <= MAX_BORDERS


@functools.lru_cache(maxsize=256)
def _borders(n: int, near: int, max_distance: int):
    found = log_borders(n, near, max_distance)
    return (ctypes.c_int32 * max(1, len(found)))(*found)


def _pos(t):
    """Unit stride along the positions; the batch may be expanded."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _args(table_ptr, out_ptr, dout_ptr, strides, weight, query_pos, key_pos, max_distance, spacing, bidirectional,
          channels_last):
    buckets, heads = weight.shape
    borders = 0
    if spacing == "log":
        n, near = side_buckets(buckets, bidirectional)
        borders = ctypes.addressof(_borders(n, near, max_distance))
    a = _lib.RelposArgs()
    _lib.pack_relpos(
        a, 0, table_ptr, query_pos.data_ptr(), key_pos.data_ptr(), out_ptr, dout_ptr, 0, borders, 0,
        query_pos.stride(0), key_pos.stride(0), *strides, query_pos.shape[0], query_pos.shape[1], key_pos.shape[1],
        heads, buckets, max_distance, spacing == "log", bidirectional, channels_last, query_pos.element_size(),
        _lib.DTYPE_CODE[weight.dtype], 0, 0)
    return a


def relative_position_bias_hip(weight, query_pos, key_pos, max_distance, spacing, bidirectional, channels_last):
    """``[B, H, U, V]``, a view with a row pitch rounded up to 8 elements (what the attention kernels read
    without a copy), or the contiguous ``[B, U, V, H]``."""
    B, U = query_pos.shape
    V, H = key_pos.shape[1], weight.shape[1]
    query_pos, key_pos, weight = _pos(query_pos), _pos(key_pos), weight.contiguous()
    if channels_last:
        buf = out = torch.empty((B, U, V, H), device=weight.device, dtype=weight.dtype)
        strides = (buf.stride(0), 0, buf.stride(1))
    else:
        buf = torch.empty((B, H, U, (V + 7) // 8 * 8), device=weight.device, dtype=weight.dtype)
        out = buf[..., :V]
        strides = buf.stride()[:3]
    if out.numel():
        a = _args(weight.data_ptr(), buf.data_ptr(), 0, strides, weight, query_pos, key_pos, max_distance, spacing,
                  bidirectional, channels_last)
        _lib.call("gnn_relpos_fwd", a, weight.device)
    return out


def relative_position_bias_bwd_hip(weight, query_pos, key_pos, dout, max_distance, spacing, bidirectional,
                                   channels_last):
    """The table's gradient, like ``weight``."""
    grad = torch.empty(weight.shape, device=weight.device, dtype=weight.dtype)
    if not dout.numel():
        return grad.zero_()
    query_pos, key_pos = _pos(query_pos), _pos(key_pos)
    if channels_last:
        H, V = weight.shape[1], key_pos.shape[1]
        if (H > 1 and dout.stride(3) != 1) or (V > 1 and dout.stride(2) != H):
            dout = dout.contiguous()
        strides = (dout.stride(0), 0, dout.stride(1))
    else:
        if key_pos.shape[1] > 1 and dout.stride(3) != 1:
            dout = dout.contiguous()
        strides = dout.stride()[:3]
    a = _args(0, 0, dout.data_ptr(), strides, weight, query_pos, key_pos, max_distance, spacing, bidirectional,
              channels_last)
    a.parts = _lib.load().gnn_relpos_parts(ctypes.byref(a))
    part = torch.empty((a.parts, *weight.shape), device=weight.device, dtype=torch.float32)
    a.partial, a.dtable = part.data_ptr(), grad.data_ptr()
    _lib.call("gnn_relpos_bwd", a, weight.device)
    return grad
